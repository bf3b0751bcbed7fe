"""GPU: requests that become copies of others, compacted caches and copied pages, against the plain forms made request by request."""

import numpy as np
import pytest
import torch

import branch_ref as ref
from attention_ref import pages_of

pytestmark = pytest.mark.gpu

I32 = lambda v, device: torch.tensor(np.asarray(v, np.int64), device=device).to(torch.int32)


def _state(rng, requests, width, ps, free, ring_extra=0):
    """(lengths, table, ring, head): requests that share the first blocks of the one before, now and then, and a ring of `free` pages from somewhere on."""
    lengths, rows, pages = [], [], 0
    for r in range(requests):
        n = int(rng.integers(0, width * ps + 1)) if rng.random() < 0.9 else int(rng.choice([0, 1, ps, width * ps]))
        both = int(rng.integers(0, min(n, lengths[-1]) // ps + 1)) if r and rng.random() < 0.7 else 0
        held = pages_of(n, ps)
        rows.append(rows[-1][:both] + list(range(pages, pages + held - both)) if both else list(range(pages, pages + held)))
        pages += held - both
        lengths.append(n)
    ids = rng.permutation(pages + free)
    table = np.full((requests, width), -7, np.int64)
    for r, row in enumerate(rows):
        table[r, :len(row)] = ids[row] if row else []
    ring = np.full(pages + free + ring_extra, -9, np.int64)
    head = int(rng.integers(0, 1 << 40))
    ring[(head + np.arange(free)) % len(ring)] = ids[pages:]
    return np.array(lengths), table, ring, head


def _moves(rng, lengths, ps):
    count = len(lengths)
    u = rng.random(count)
    sources = np.where(u < 0.35, np.arange(count), np.where(u < 0.5, -1, rng.integers(0, count, count)))
    some = np.where(sources < 0, 0, np.asarray(lengths)[np.maximum(sources, 0)])
    cut = np.where(rng.random(count) < 0.5, rng.integers(0, some + 1), some // ps * ps)
    return sources, np.where(rng.random(count) < 0.5, 2 ** 31 - 1, cut)


def _fork(hm, device, lengths, table, ring, head, tail, sources, keep, ps, in_place=False, pad=0):
    other = None if in_place else np.full(table.shape, -3, np.int64)
    want = ref.fork(sources, keep, lengths, table, ring, head, tail, ps, other)
    wide = torch.full((len(lengths), table.shape[1] + pad), -5, dtype=torch.int32, device=device)
    wide[:, :table.shape[1]] = I32(table, device)
    t, f, n = wide[:, :table.shape[1]], I32(ring, device), I32(lengths, device)
    q = torch.tensor([head, tail, 99, 99], dtype=torch.int64, device=device)
    to = None if in_place else I32(other, device)
    fork = hm.PageFork(*table.shape, ps, device)
    print(f"fork: {len(lengths)} requests, width {table.shape[1]}, pages of {ps}, in place {in_place}: {want['queue'].tolist()}", flush=True)
    hm.page_fork(fork, I32(sources, device), n, t, f, q, keep=None if keep is None else I32(keep, device), table_out=to,
                 lengths_out=n if in_place else None, queue_out=q if in_place else None)
    torch.cuda.synchronize()
    got = {"copies": fork.copies, "lengths": n if in_place else fork.lengths, "queue": q if in_place else fork.queue, "table": t if in_place else to, "ring": f}
    for name, v in got.items():
        np.testing.assert_array_equal(v.cpu().numpy().astype(np.int64), want[name], err_msg=name)
    assert pad == 0 or (wide[:, table.shape[1]:] == -5).all()
    if not in_place:
        np.testing.assert_array_equal(t.cpu().numpy(), table)
    return want


@pytest.mark.parametrize("requests", [1, 2, 5, 63, 64, 65, 300, 1024, 1025, 4096])
@pytest.mark.parametrize("width,ps", [(1, 16), (5, 16), (37, 64)])
def test_requests_become_others(hm, device, requests, width, ps):
    rng = np.random.default_rng([requests, width, ps])
    for in_place in (False, True):
        lengths, table, ring, head = _state(rng, requests, width, ps, requests + 3)
        sources, keep = _moves(rng, lengths, ps)
        for k in (None, keep):
            want = _fork(hm, device, lengths, table, ring, head, head + requests + 3, sources, k, ps, in_place, pad=3)
            assert want["queue"][2] == 0


@pytest.mark.parametrize("width", [1500, 9000])
def test_wide_tables(hm, device, width):
    # more columns than workgroups
    rng = np.random.default_rng(width)
    for requests in (3, 70):
        lengths, table, ring, head = _state(rng, requests, width, 16, requests)
        sources, keep = _moves(rng, lengths, 16)
        _fork(hm, device, lengths, table, ring, head, head + requests, sources, keep, 16)
        _fork(hm, device, lengths, table, ring, head, head + requests, sources, None, 16, in_place=True)


def test_every_request_becomes_the_same_one(hm, device):
    rng = np.random.default_rng(3)
    for requests in (2, 64, 500, 4096):
        for n in (0, 1, 16, 40, 64):
            lengths, table, ring, head = _state(rng, requests, 4, 16, requests)
            lengths[requests // 2] = n
            table[requests // 2, :pages_of(n, 16)] = len(ring) + 10 + np.arange(pages_of(n, 16))  # ids are taken as they stand
            ring = np.concatenate([ring, np.full(8, -9)])
            ring[(head + np.arange(requests)) % len(ring)] = 5000 + np.arange(requests)
            _fork(hm, device, lengths, table, ring, head, head + requests, np.full(requests, requests // 2), None, 16)


def test_what_is_refused_and_negative_entries(hm, device):
    rng = np.random.default_rng(4)
    for requests in (6, 90, 1100):
        lengths, table, ring, head = _state(rng, requests, 6, 16, requests)
        sources, keep = _moves(rng, lengths, 16)
        good = _fork(hm, device, lengths, table, ring, head, head + requests, sources, keep, 16)
        fresh = int(good["queue"][3])
        for change in (dict(sources=requests), dict(keep=-1), dict(lengths=97), dict(lengths=-1), dict(tail=head + fresh - 1), dict(tail=head - 5)):
            args = {"lengths": lengths.copy(), "sources": sources.copy(), "keep": keep.copy(), "tail": head + requests}
            for k, v in change.items():
                if k == "tail":
                    args[k] = v
                else:
                    args[k][requests // 2] = v
            for in_place in (False, True):
                want = _fork(hm, device, args["lengths"], table, ring, head, args["tail"], args["sources"], args["keep"], 16, in_place)
                assert want["queue"][2] == (fresh > 0 or "tail" not in change)
        exact = _fork(hm, device, lengths, table, ring, head, head + fresh, sources, keep, 16)
        assert exact["queue"][2] == 0
        freed = int(good["queue"][1]) - head - requests
        if freed > 0:
            # a ring with no room for all that comes back, and one with just enough
            for size in (requests + freed - 1, requests + freed):
                small = np.full(size, -9)
                small[(head + np.arange(requests)) % size] = ring[(head + np.arange(requests)) % len(ring)]
                want = _fork(hm, device, lengths, table, small, head, head + requests, sources, keep, 16)
                assert want["queue"][2] == (size < requests + freed)
        holes = table.copy()
        holes[rng.random(table.shape) < 0.2] = -1
        _fork(hm, device, lengths, holes, ring, head, head + requests, sources, keep, 16)


class Loop:
    """A cache and its requests, with each request's tokens kept on the host; token x is written as the value x in each head and layer."""

    def __init__(self, hm, device, seed, requests, width, ps, pages, layers=2, dtype=torch.float16, swapped=False):
        self.hm, self.device, self.rng, self.ps, self.width = hm, device, np.random.default_rng(seed), ps, width
        self.table = torch.full((requests, width), -1, dtype=torch.int32, device=device)
        self.ring = I32(self.rng.permutation(pages), device)
        self.lengths, self.added = (torch.zeros(requests, dtype=torch.int32, device=device) for _ in range(2))
        self.sources = torch.arange(requests, dtype=torch.int32, device=device)
        self.keep = torch.full((requests,), 2 ** 31 - 1, dtype=torch.int32, device=device)
        self.queue = torch.tensor([0, pages, 0, 0], dtype=torch.int64, device=device)
        self.plan = hm.PagePlan(requests, 64, ps, device)
        self.fork = hm.PageFork(requests, width, ps, device)
        self.pages, self.kv_heads, self.d = pages, 2, 64
        shape = (pages, ps, 2, 64) if swapped else (pages, 2, ps, 64)
        make = lambda: torch.full(shape, float("nan"), dtype=dtype, device=device)
        view = lambda t: t.transpose(1, 2) if swapped else t
        self.caches = [hm.PagedCache(view(make()), view(make())) for _ in range(layers)]
        self.values = torch.zeros(64, dtype=dtype, device=device)
        self.q, self.qkv = torch.zeros((64, 128), dtype=dtype, device=device), torch.zeros((64, 6 * 64), dtype=dtype, device=device)
        self.parts = torch.tensor([0.0] * 256 + [0.25] * 128, dtype=dtype, device=device)  # of queries and keys, and of values
        self.no_rotation = torch.zeros(0, dtype=torch.float64, device=device)
        self.tokens = [[] for _ in range(requests)]
        self.next = 1

    def step(self):
        """One step on the device: fork, copies, plan, and the new tokens' values to their slots."""
        hm = self.hm
        hm.page_fork(self.fork, self.sources, self.lengths, self.table, self.ring, self.queue, keep=self.keep, lengths_out=self.lengths, queue_out=self.queue)
        hm.copy_pages(self.caches, self.fork.copies)
        hm.page_plan(self.plan, self.lengths, self.added, self.table, self.ring, self.queue, self.lengths, self.queue)
        for i, c in enumerate(self.caches):  # no rotation and no norm: keys and values are written as they are
            self.qkv.copy_(self.values[:, None] + self.parts + 0.5 * i)
            hm.qk_norm_rope(self.q, self.qkv, self.no_rotation, self.plan.positions, cache=c, slots=self.plan.slots)

    def ask(self, sources, keep, added):
        self.sources.copy_(I32(sources, self.device))
        self.keep.copy_(I32(keep, self.device))
        self.added.copy_(I32(added, self.device))
        before = [list(t) for t in self.tokens]
        values = np.zeros(64)
        at = 0
        for r, (s, k, a) in enumerate(zip(sources, keep, added)):
            self.tokens[r] = [] if s < 0 else before[s][:k]
            for _ in range(a):
                self.tokens[r].append(self.next)
                values[at] = self.next
                self.next = self.next % 500 + 1  # exact next to quarters
                at += 1
        self.values.copy_(torch.tensor(values).to(self.values.dtype))

    def check(self, tag):
        torch.cuda.synchronize()
        assert int(self.queue[2]) == 0 and self.lengths.tolist() == [len(t) for t in self.tokens], tag
        table = self.table.cpu().numpy()
        held, owner = set(), {}
        for r, tokens in enumerate(self.tokens):
            for b in range(pages_of(len(tokens), self.ps)):
                page = int(table[r, b])
                held.add(page)
                owner.setdefault(page, []).append((r, b))
        for page, who in owner.items():
            assert len({b for _, b in who}) == 1, "a shared page is the same block of all"
            assert len(who) == 1 or all(len(self.tokens[r]) >= (b + 1) * self.ps for r, b in who), "a page that is not full is one request's own"
        queue, ring = self.queue.tolist(), self.ring.cpu().numpy()
        free = [int(ring[i % self.pages]) for i in range(queue[0], queue[1])]
        assert sorted(free + list(held)) == list(range(self.pages)), f"{tag}: every page is held or free, once"
        for i, c in enumerate(self.caches):
            for j, x in enumerate((c.k, c.v)):
                x = x.float().cpu().numpy()
                for r, tokens in enumerate(self.tokens):
                    at = np.arange(len(tokens))
                    got = x[table[r, at // self.ps], :, at % self.ps] if len(tokens) else np.zeros((0, 2, 64))
                    np.testing.assert_array_equal(got, np.broadcast_to((np.array(tokens) + (2 * i + j) * 0.25)[:, None, None], got.shape), err_msg=f"{tag} request {r}")

    def random(self):
        count, rng = len(self.tokens), self.rng
        u = rng.random(count)
        sources = [r if u[r] < 0.5 else -1 if u[r] < 0.6 else int(rng.integers(0, count)) for r in range(count)]
        keep = [2 ** 31 - 1 if s < 0 or rng.random() < 0.6 else int(rng.integers(0, len(self.tokens[s]) + 1)) for s in sources]
        after = [0 if s < 0 else min(k, len(self.tokens[s])) for s, k in zip(sources, keep)]
        added = [int(min(rng.integers(0, 64 // count + 1), self.width * self.ps - n)) for n in after]
        return sources, keep, added


@pytest.mark.parametrize("swapped", [False, True])
@pytest.mark.parametrize("ps", [16, 64])
def test_tokens_follow_their_requests(hm, device, ps, swapped):
    s = Loop(hm, device, ps, 7, 5, ps, 60, dtype=torch.float16, swapped=swapped)
    for step in range(40):
        s.ask(*s.random())
        s.step()
        s.check(f"step {step}")


def test_a_loop_in_a_graph(hm, device):
    s = Loop(hm, device, 5, 12, 8, 16, 200)
    s.step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        s.step()
    for step in range(25):
        s.ask(*s.random())
        if step % 5 == 4:
            s.step()  # an eager one in between
        else:
            g.replay()
        s.check(f"step {step}")


@pytest.mark.parametrize("pages,limit,requests,width", [(1, 1, 1, 1), (40, 20, 3, 8), (100, 64, 9, 8), (1000, 500, 70, 9), (1000, 1000, 70, 9), (1000, 31, 5, 6), (5000, 2048, 300, 9),
                                                        (300000, 70000, 2000, 40)])
@pytest.mark.parametrize("in_place", [False, True])
def test_pages_move_below_a_limit(hm, device, pages, limit, requests, width, in_place):
    rng = np.random.default_rng([pages, limit, in_place])
    ps = 16
    lengths, table, _, head = _state(rng, requests, width, ps, 0)
    ids = rng.permutation(pages)
    for r in range(requests):  # renumbered over the whole cache, dropping what the limit has no room for
        held = pages_of(lengths[r], ps)
        if table[r, :held].max(initial=0) >= min(limit, pages):
            lengths[r] = 0
        else:
            table[r, :held] = ids[table[r, :held]]
    if requests > 3:
        lengths[1], lengths[2] = -5, 2 ** 31 - 1  # as page_plan takes them: none, and the whole row
        table[2] = table[0, 0] if lengths[0] > 0 else -1
    ring = np.full(pages, -9, np.int64)
    other = None if in_place else np.full(table.shape, -3, np.int64)
    want = ref.compact(pages, limit, lengths, table, ring, head, head + 7, ps, max(1, pages // 2), other)
    assert want["queue"][2] == 0
    t, f, q = I32(table, device), I32(ring, device), torch.tensor([head, head + 7, 99, 99], dtype=torch.int64, device=device)
    to = None if in_place else I32(other, device)
    compact = hm.PageCompact(pages, ps, device)
    compact._workspace.fill_(0xAB)
    print(f"compact: {pages} pages below {limit}, {requests} requests: {want['queue'].tolist()}", flush=True)
    hm.page_compact(compact, limit, I32(lengths, device), t, f, q, table_out=to, queue_out=q if in_place else None)
    torch.cuda.synchronize()
    for name, v in {"copies": compact.copies, "queue": q if in_place else compact.queue, "table": t if in_place else to, "ring": f}.items():
        np.testing.assert_array_equal(v.cpu().numpy().astype(np.int64), want[name], err_msg=name)


def test_compactions_that_are_refused_on_the_device(hm, device):
    table = np.array([[3, 9, 1], [3, 4, -1]])
    for limit, size, refused in ((3, 9, 1), (4, 9, 0), (9, 5, 0), (9, 4, 1), (0, 9, 1)):
        ring = np.full(size, -9)
        want = ref.compact(10, limit, [48, 20], table, ring, 5, 6, 16, 5)
        assert want["queue"][2] == refused
        t, f, q = I32(table, device), I32(ring, device), torch.tensor([5, 6, 0, 0], dtype=torch.int64, device=device)
        c = hm.PageCompact(10, 16, device)
        hm.page_compact(c, limit, I32([48, 20], device), t, f, q)
        for name, v in {"copies": c.copies, "queue": c.queue, "table": t, "ring": f}.items():
            np.testing.assert_array_equal(v.cpu().numpy().astype(np.int64), want[name], err_msg=f"{name} {limit} {size}")


def test_a_loop_whose_cache_is_cut_and_grown(hm, device):
    s = Loop(hm, device, 9, 6, 5, 16, 64)
    compact = hm.PageCompact(64, 16, device)
    for step in range(24):
        s.ask(*s.random())
        s.step()
        if step % 4 == 3:
            limit = [64, 40, 33, 36][step // 4 % 4]  # of up to 30 pages held
            hm.page_compact(compact, limit, s.lengths, s.table, s.ring, s.queue, queue_out=s.queue)
            hm.copy_pages(s.caches, compact.copies)
            torch.cuda.synchronize()
            assert int(s.queue[2]) == 0 and int(s.table.max()) < limit
            hm.page_compact(compact, 64, s.lengths, s.table, s.ring, s.queue, queue_out=s.queue)  # and grown again
            torch.cuda.synchronize()
            assert int(s.queue[3]) == 0 and compact.copies.max() == -1
        s.check(f"step {step}")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("heads,ps,d", [(1, 16, 16), (3, 16, 48), (8, 32, 64), (2, 128, 96), (5, 64, 128), (2, 256, 256), (1, 16, 512)])
def test_copies_of_pages(hm, device, dtype, heads, ps, d):
    rng = np.random.default_rng([heads, ps, d])
    gen = torch.Generator(device=device).manual_seed(d)
    layers, pages = 3, 23
    base = [torch.randn((2, pages, heads, ps, d + 8), generator=gen, device=device).to(dtype) for _ in range(layers)]
    wide = [t[..., :d] for t in base]  # rows that do not follow each other
    caches = [hm.PagedCache(t[0], t[1]) for t in wide]
    other = [torch.randn((2, 2 * pages, ps, heads, d), generator=gen, device=device).to(dtype) for _ in range(layers)]
    others = [hm.PagedCache(t[0].transpose(1, 2), t[1].transpose(1, 2)) for t in other]
    ids = rng.permutation(pages)
    tokens = [0, 1, ps // 2 + 1, ps - 1, ps, ps + 9, -4, 15, 16]
    copies = np.array([(ids[i], ids[9 + i], n) for i, n in enumerate(tokens)] + [(pages, ids[18], ps), (ids[0], 2 * pages, ps), (ids[0], -2, ps), (2 ** 31 - 1, ids[18], ps), (-1, -1, -1),
                                                                              (ids[1], ids[19], ps)])
    for to in (None, others):
        want = [t.clone() for t in (wide if to is None else other)]
        for w, src in zip(want, [t.clone() for t in wide]):
            for a, b, n in copies.tolist()[:len(tokens)] + copies.tolist()[-1:]:
                n = max(0, min(n, ps))
                if to is None:
                    w[:, b, :, :n] = src[:, a, :, :n]
                else:
                    w[:, b, :n] = src[:, a, :, :n].transpose(1, 2)
        gap = [t[..., d:].clone() for t in base]
        hm.copy_pages(caches, I32(copies, device), to=to)
        torch.cuda.synchronize()
        for w, t, g, b in zip(want, wide if to is None else other, gap, base):
            assert torch.equal(w.view(torch.int16), t.contiguous().view(torch.int16)) and torch.equal(g, b[..., d:])
    hm.copy_pages(caches[0], I32(np.zeros((0, 3)), device))
    hm.copy_pages(caches[0], torch.full((5, 3), -1, dtype=torch.int32, device=device))


@pytest.mark.parametrize("d", [16, 32, 48, 80, 112, 144, 256, 272, 512, 528, 1040])
def test_copies_of_rows_of_any_width(hm, device, d):
    test_copies_of_pages(hm, device, torch.bfloat16, 2, 32, d)


def test_copies_of_many_layers_and_entries(hm, device):
    layers, pages, ps = 70, 40, 16
    caches = [hm.PagedCache.empty(pages, ps, 1, 64, torch.float16, device) for _ in range(layers)]
    for i, c in enumerate(caches):
        c.k.copy_(torch.arange(pages, device=device).view(-1, 1, 1, 1) + 100.0 * (i % 7))
        c.v.copy_(c.k + 50)
    copies = torch.stack([torch.arange(20), torch.arange(20, 40), torch.full((20,), ps)], 1).to(torch.int32).to(device)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    hm.copy_pages(caches, copies, stream=stream)
    torch.cuda.synchronize()
    for c in caches:
        assert torch.equal(c.k[20:], c.k[:20]) and torch.equal(c.v[20:], c.v[:20])
    with pytest.raises(ValueError, match="alike"):
        hm.copy_pages([caches[0], hm.PagedCache.empty(41, ps, 1, 64, torch.float16, device)], copies)
    with pytest.raises(ValueError, match="as many"):
        hm.copy_pages(caches[:2], copies, to=caches[0])
    with pytest.raises(ValueError, match="Int"):
        hm.copy_pages(caches[0], copies.long())


def test_calls_that_python_refuses(hm, device):
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=device)
    q = torch.zeros(4, dtype=torch.int64, device=device)
    fork, compact = hm.PageFork(3, 4, 16, device), hm.PageCompact(9, 16, device)
    good = dict(sources=i(3), lengths=i(3), block_table=i(3, 4), free_pages=i(9), queue=q)
    for name, bad in (("sources", i(2)), ("sources", i(3).long()), ("lengths", i(4)), ("block_table", i(2, 4)), ("block_table", i(3, 4).long()), ("free_pages", i(0)), ("queue", q[:3]),
                      ("keep", i(2)), ("table_out", i(3, 5)), ("lengths_out", i(2)), ("queue_out", q.int())):
        with pytest.raises(ValueError):
            hm.page_fork(fork, **{**good, name: bad})
    with pytest.raises(Exception, match="too small"):
        hm.page_fork(hm.PageFork(3, 1, 16, device), **{**good, "block_table": i(3, 4000)})
    good = dict(limit=4, lengths=i(3), block_table=i(3, 4), free_pages=i(9), queue=q)
    for name, bad in (("limit", 10), ("limit", -1), ("lengths", i(4)), ("block_table", i(2, 4)), ("free_pages", i(3, 3)), ("queue", q[:3]), ("table_out", i(4, 4)), ("queue_out", q[:2])):
        with pytest.raises(ValueError):
            hm.page_compact(compact, **{**good, name: bad})
