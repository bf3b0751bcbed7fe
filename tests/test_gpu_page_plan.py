"""GPU: a step's page plan against the plan made request by request."""

import numpy as np
import pytest
import torch

import attention_ref as ref

pytestmark = pytest.mark.gpu


def _state(rng, lengths, width, page_size, free, extra=0):
    """(table, ring, head): each request's held pages in its row, `free` pages in the ring from a head somewhere, in no order."""
    held = [ref.pages_of(min(max(n, 0), width * page_size), page_size) for n in lengths]
    pages = sum(held) + free + extra
    ids = rng.permutation(pages)
    table = np.full((len(lengths), width), -7, np.int64)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = ids[at:at + h]
        at += h
    ring = np.full(max(pages, 1), -9, np.int64)
    head = int(rng.integers(0, 1 << 40))
    ring[(head + np.arange(free)) % len(ring)] = ids[at:at + free]
    return table, ring, head


def _check(hm, device, lengths, added, table, ring, head, tail, rows, page_size, in_place=False, pad=0):
    want = ref.plan(lengths, added, table, ring, head, tail, rows, page_size)
    i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device=device)
    wide = torch.full((len(lengths), table.shape[1] + pad), -5, dtype=torch.int32, device=device)
    wide[:, :table.shape[1]] = i32(table)
    t, r, n, a = wide[:, :table.shape[1]], i32(ring), i32(lengths), i32(added)
    queue = torch.tensor([head, tail, 99, 99], dtype=torch.int64, device=device)
    plan = hm.PagePlan(len(lengths), rows, page_size, device)
    print(f"plan: {len(lengths)} requests, {rows} rows, pages of {page_size}, table width {table.shape[1]}", flush=True)
    out = (n, queue) if in_place else (plan.lengths, plan.queue)
    hm.page_plan(plan, n, a, t, r, queue, *(out if in_place else ()))
    torch.cuda.synchronize()
    got = {"slots": plan.slots, "positions": plan.positions, "requests": plan.requests, "starts": plan.starts, "lengths": out[0], "queue": out[1],
           "table": t, "ring": r}
    for name, v in got.items():
        np.testing.assert_array_equal(v.cpu().numpy().astype(np.int64), want[name], err_msg=name)
    if pad:
        assert (wide[:, table.shape[1]:] == -5).all()
    if not in_place:
        np.testing.assert_array_equal(n.cpu().numpy(), np.asarray(lengths))
    return want


@pytest.mark.parametrize("requests", [1, 2, 63, 64, 65, 1000, 1024, 1025, 4095, 4096])
@pytest.mark.parametrize("in_place", [False, True])
def test_one_token_of_each_request(hm, device, requests, in_place):
    rng = np.random.default_rng(requests)
    lengths = rng.integers(0, 255, requests)
    table, ring, head = _state(rng, lengths, 16, 16, requests)
    _check(hm, device, lengths, np.ones(requests, np.int64), table, ring, head, head + requests, requests, 16, in_place)


@pytest.mark.parametrize("page_size", [16, 64, 1024])
@pytest.mark.parametrize("rows", [100, 4096, 4097, 20000])
@pytest.mark.parametrize("requests", [7, 300, 2500])
def test_prompts_decodes_idle_and_ended_requests(hm, device, page_size, rows, requests):
    rng = np.random.default_rng([page_size, rows, requests])
    width = max(2, 2048 // page_size)
    lengths = rng.integers(0, width * page_size // 2, requests)
    added = np.where(rng.random(requests) < 0.3, rng.integers(-1, 2, requests), rng.integers(0, max(2, 2 * rows // requests), requests))
    lengths[rng.random(requests) < 0.2] = 0
    table, ring, head = _state(rng, lengths, width, page_size, 3 + int(np.maximum(added, 0).sum() // page_size + requests), extra=5)
    free = int((ring >= 0).sum())
    for in_place in (False, True):
        _check(hm, device, lengths, added, table, ring, head, head + free, rows, page_size, in_place, pad=3)


def test_what_a_step_refuses(hm, device):
    rng = np.random.default_rng(5)
    lengths = np.array([0, 64, 63, -3, 70, 10, 0, 20, 31, 2 ** 31 - 1, 5])
    added = np.array([0, 1, 2, 4, 1, 100, 2 ** 31 - 1, -1, 1, 2 ** 31 - 1, 3])
    for rows in (0, 1, 3, 50, 5000):
        for free in (0, 1, 2, 9):
            table, ring, head = _state(rng, np.clip(lengths, 0, 64), 4, 16, free)
            want = _check(hm, device, lengths, added, table, ring, head, head + free, rows, 16)
            assert want["queue"][2] >= 6


def test_pages_run_out_in_the_middle(hm, device):
    rng = np.random.default_rng(6)
    lengths, added = np.full(200, 16), np.where(np.arange(200) % 3 == 0, 40, 1)
    lengths[1::2] = 17
    for free in (0, 1, 50, 51, 52, 10 ** 3):
        table, ring, head = _state(rng, lengths, 8, 16, free)
        for rows in (200, 6000):
            _check(hm, device, lengths, added, table, ring, head, head + free, rows, 16)


def test_a_full_ring_and_counters_that_make_no_sense(hm, device):
    # the queue's counters only bound what is handed out: nothing is read outside the ring
    rng = np.random.default_rng(7)
    lengths, added = np.array([0, 16, 5]), np.array([16, 16, -1])
    table, ring, head = _state(rng, lengths, 4, 16, 2)
    for queue in ((head, head - 4), (0, 0), (5, 5 + len(ring))):
        want = ref.plan(lengths, added, table, ring, *queue, 40, 16)
        plan = hm.PagePlan(3, 40, 16, device)
        i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device=device)
        q = torch.tensor([*queue, 0, 0], dtype=torch.int64, device=device)
        hm.page_plan(plan, i32(lengths), i32(added), i32(table), i32(ring), q)
        np.testing.assert_array_equal(plan.lengths.cpu().numpy(), want["lengths"])
        np.testing.assert_array_equal(plan.queue.cpu().numpy(), want["queue"])


def test_a_loop_in_a_graph_takes_and_gives_back_pages(hm, device):
    # the captured step advances its own lengths and counters; requests end and start again between replays
    ps, width, requests, rows = 16, 8, 12, 64
    rng = np.random.default_rng(8)
    pages = requests * width
    table = torch.full((requests, width), -1, dtype=torch.int32, device=device)
    ring = torch.tensor(rng.permutation(pages), dtype=torch.int32, device=device)
    lengths = torch.zeros(requests, dtype=torch.int32, device=device)
    added = torch.zeros(requests, dtype=torch.int32, device=device)
    queue = torch.tensor([0, pages, 0, 0], dtype=torch.int64, device=device)
    plan = hm.PagePlan(requests, rows, ps, device)
    hm.page_plan(plan, lengths, added, table, ring, queue, lengths, queue)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        hm.page_plan(plan, lengths, added, table, ring, queue, lengths, queue)
    host = {"table": table.cpu().numpy().astype(np.int64), "ring": ring.cpu().numpy().astype(np.int64), "lengths": np.zeros(requests, np.int64),
            "queue": np.array([0, pages, 0, 0])}
    for step in range(60):
        a = np.where(rng.random(requests) < 0.15, -1, rng.integers(0, 9, requests))
        added.copy_(torch.tensor(a, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        host = ref.plan(host["lengths"], a, host["table"], host["ring"], int(host["queue"][0]), int(host["queue"][1]), rows, ps)
        for name, t in (("slots", plan.slots), ("positions", plan.positions), ("requests", plan.requests), ("lengths", lengths), ("queue", queue),
                        ("table", table), ("ring", ring)):
            np.testing.assert_array_equal(t.cpu().numpy().astype(np.int64), host[name], err_msg=f"step {step} {name}")
        live = [p for r in range(requests) for p in host["table"][r, :ref.pages_of(int(host["lengths"][r]), ps)]]
        free = [host["ring"][i % pages] for i in range(int(host["queue"][0]), int(host["queue"][1]))]
        assert sorted(live + free) == list(range(pages)), "every page is held once or free once"


def _plan_in_a_small_ring(lengths, added, table, ring, head, tail, rows, page_size):
    """The plan made request by request, where ended requests keep their pages that the ring has no room for behind this step's."""
    args = (table, ring, head, tail, rows, page_size)
    taken = int(ref.plan(lengths, added, *args)["queue"][0]) - head
    room = len(ring) - min(max(tail - head, 0), len(ring)) + taken
    kept, at, limited = 0, 0, np.array(added)
    for r, (n, a) in enumerate(zip(lengths, added)):
        if a < 0:
            pages = ref.pages_of(min(max(int(n), 0), table.shape[1] * page_size), page_size)
            at += pages
            if pages and at > room:
                kept, limited[r] = kept + 1, 0
    want = ref.plan(lengths, limited, *args)
    want["queue"][2] += kept
    return want, kept


@pytest.mark.parametrize("rows", [60, 1024, 3000])
@pytest.mark.parametrize("requests", [6, 500, 2500])
@pytest.mark.parametrize("in_place", [False, True])
def test_a_ring_smaller_than_the_pages_in_circulation(hm, device, requests, rows, in_place):
    rng = np.random.default_rng([requests, rows])
    ps, width = 16, 6
    i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device=device)
    some = 0
    for size in (1, requests // 2 + 1, requests + 1, 3 * requests):
        lengths = rng.integers(0, width * ps, requests)
        free = int(rng.integers(size // 2, size + 1))
        held = [ref.pages_of(n, ps) for n in lengths]
        ids = rng.permutation(sum(held) + free)
        table = np.full((requests, width), -7, np.int64)
        at = 0
        for r, h in enumerate(held):
            table[r, :h] = ids[at:at + h]
            at += h
        ring, head = np.full(size, -9, np.int64), int(rng.integers(0, 1 << 40))
        ring[(head + np.arange(free)) % size] = ids[at:]
        added = np.where(rng.random(requests) < 0.4, -1, rng.integers(0, max(2, 2 * rows // requests), requests))
        want, kept = _plan_in_a_small_ring(lengths, added, table, ring, head, head + free, rows, ps)
        some += kept
        t, r, n, q = i32(table), i32(ring), i32(lengths), torch.tensor([head, head + free, 99, 99], dtype=torch.int64, device=device)
        plan = hm.PagePlan(requests, rows, ps, device)
        print(f"{requests} requests, {rows} rows, a ring of {size} with {free} free: {kept} keep their pages", flush=True)
        out = (n, q) if in_place else (plan.lengths, plan.queue)
        hm.page_plan(plan, n, i32(added), t, r, q, *out)
        torch.cuda.synchronize()
        for name, v in {"slots": plan.slots, "positions": plan.positions, "requests": plan.requests, "starts": plan.starts, "lengths": out[0],
                        "queue": out[1], "table": t, "ring": r}.items():
            np.testing.assert_array_equal(v.cpu().numpy().astype(np.int64), want[name], err_msg=name)
    assert some > 0


def test_no_page_is_lost_in_a_small_ring(hm, device):
    # requests that could not end are asked to end again in the next step, as a serving loop would
    ps, width, requests, rows = 16, 8, 12, 64
    rng = np.random.default_rng(9)
    pages, size = 50, 14
    table = torch.full((requests, width), -1, dtype=torch.int32, device=device)
    ids = rng.permutation(pages)
    lengths = torch.tensor([48] * requests, dtype=torch.int32, device=device)
    table[:, :3] = torch.tensor(ids[:36].reshape(12, 3), dtype=torch.int32)
    ring = torch.tensor(ids[36:], dtype=torch.int32, device=device)
    assert len(ring) == size
    queue = torch.tensor([0, size, 0, 0], dtype=torch.int64, device=device)
    plan = hm.PagePlan(requests, rows, ps, device)
    ending, refused = set(), 0
    for step in range(80):
        a = np.where(rng.random(requests) < 0.25, -1, rng.integers(0, 9, requests))
        a[list(ending)] = -1
        hm.page_plan(plan, lengths, torch.tensor(a, dtype=torch.int32, device=device), table, ring, queue, lengths, queue)
        torch.cuda.synchronize()
        n, t, f, q = (v.cpu().numpy().astype(np.int64) for v in (lengths, table, ring, queue))
        ending = {r for r in range(requests) if a[r] < 0 and n[r] > 0}
        refused += len(ending)
        live = [p for r in range(requests) for p in t[r, :ref.pages_of(int(n[r]), ps)]]
        free = [f[i % size] for i in range(int(q[0]), int(q[1]))]
        assert q[1] - q[0] <= size and sorted(live + free) == list(range(pages)), f"step {step}: every page is held once or free once"
    assert refused > 0
