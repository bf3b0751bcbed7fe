"""GPU: attention over a paged cache for prompts: calls with enough rows for the kernel whose waves share tiles of keys, next to rows that go the
other way, against the float64 form."""

import math

import numpy as np
import pytest
import torch

import attention_ref as ref
from test_gpu_paged_attention import DT, Case, _check, _queries

pytestmark = pytest.mark.gpu


def _blocks(c, positions, requests):
    """How many blocks of rows the launch rule lets the prompts' kernel take, of how many (one card: 256 CUs)."""
    d, kv = c.k.size(3), c.k.size(1)
    group = c.q_heads // kv
    grouped = max(1, 16 // group)
    rows = (64 * (2 if d <= 128 else 1) // group) // grouped * grouped
    groups = 256 * (2 if d <= 128 else 1)
    count = len(positions) // rows
    if 8 * count * kv <= groups:
        return 0, count
    ends = [positions[b * rows + rows - 1] + 1 if requests[b * rows] >= 0 and requests[b * rows] == requests[b * rows + rows - 1] else 0 for b in range(count)]
    return sum(0 < e * max(1, groups // kv) < 8 * sum(ends) for e in ends), count


def _rows(c, seed):
    """Rows of prompts: a whole one, chunks with a context, drafts, single tokens, empty rows, another request inside a block, rows that
    see nothing."""
    rng = np.random.default_rng(seed)
    n = c.lengths
    rows = [(p, 0) for p in range(n[0])] + [(p, 1) for p in range(n[1] - 90, n[1])] + [(n[2] - 1, 2)] + [(p, 3) for p in range(n[3] - 5, n[3])]
    rows += [(-1, -1)] * 7 + [(p, 2) for p in range(n[2] - 200, n[2])]
    at = len(rows) - 150
    rows[at:at + 3] = [(n[1] - 1, 1), (-1, -1), (-1, 2)]
    rows += [(int(p), 1) for p in rng.integers(-1, n[1], 70)] + [(-1, -1)] * 3 + [(p, 0) for p in range(n[0] - 130, n[0])]
    return [r[0] for r in rows], [r[1] for r in rows]


def _case(seed, heads, d, dtype, page_size=16):
    return Case(seed, [150, 260, 333, 40], heads[0], heads[1], d, page_size, dtype)


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("heads", [(64, 64), (64, 32), (64, 16), (80, 16), (112, 16), (128, 16), (144, 12), (192, 12)])
def test_head_layouts(hm, device, heads, d):
    c = _case(40, heads, d, torch.float16 if heads[1] == 16 else torch.bfloat16)
    positions, requests = _rows(c, 41)
    taken, of = _blocks(c, positions, requests)
    assert 0 < taken < of, "both kernels have work"
    got = _check(hm, device, c, positions, requests, _queries(c, len(positions), 42), tag=f"{taken} of {of} blocks")
    for t, p in enumerate(positions):
        if requests[t] >= 0 and p < 0:
            assert (got[t] == 0).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("window", [1, 16, 37, 100, 1000])
def test_windows(hm, device, window, dtype):
    c = _case(43, (64, 16), 128, DT[dtype])
    positions, requests = _rows(c, 44)
    assert _blocks(c, positions, requests)[0] > 0
    _check(hm, device, c, positions, requests, _queries(c, len(positions), 45), window=window, tag="windows")


@pytest.mark.parametrize("page_size,layout", [(16, "sliced"), (32, "page_token_head"), (64, "page_head_token"), (256, "sliced")])
def test_pages_and_strides(hm, device, page_size, layout):
    c = _case(46, (64, 16), 64, torch.bfloat16, page_size)
    c.layout = layout
    positions, requests = _rows(c, 47)
    _check(hm, device, c, positions, requests, _queries(c, len(positions), 48), tag="pages and strides")


@pytest.mark.parametrize("scale", [0.0, -0.09, 1e-30, 2.0])
def test_scales(hm, device, scale):
    c = _case(49, (64, 16), 64, torch.bfloat16)
    positions, requests = _rows(c, 50)
    assert _blocks(c, positions, requests)[0] > 0
    _check(hm, device, c, positions, requests, _queries(c, len(positions), 51), scale=scale, tag="scales")


@pytest.mark.parametrize("length", [1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200])
def test_prompts_around_the_tiles(hm, device, length):
    # whole prompts of a length, one after the other: blocks that hold parts of one, and several
    c = Case(52, [length] * (700 // length), 64, 32, 64, 16, torch.float16)
    rows = [(p, r) for r in range(len(c.lengths)) for p in range(length)]
    positions, requests = zip(*rows)
    _check(hm, device, c, list(positions), list(requests), _queries(c, len(rows), 53), tag="around the tiles")


@pytest.mark.parametrize("window", [0, 64])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d", [128, 256])
def test_later_tokens_do_not_show_in_earlier_rows(hm, device, d, dtype, window):
    c = Case(54, [40, 400], 64, 16, d, 16, DT[dtype])
    at = lambda t, p: t[int(c.table[1, p // 16]), :, p % 16]
    clean = [t.clone() for t in (c.k, c.v)]
    at(c.v, 230)[0, 5] = float("inf")
    at(c.v, 233)[1, 7] = float("nan")
    at(c.k, 281)[2, 3] = float("nan")
    positions = list(range(144, 400))
    assert _blocks(c, positions, [1] * len(positions))[0] > 0
    q = _queries(c, len(positions), 55)
    pos, req = torch.tensor(positions, dtype=torch.int32), torch.full((len(positions),), 1, dtype=torch.int32)
    out = torch.zeros(q.shape, dtype=c.dtype, device=device)
    got = hm.paged_attention(out, q.to(device), c.cache(hm, device), c.table.to(device), pos.to(device), req.to(device), window=window).cpu()
    c.k, c.v = clean
    want, bound = ref.attention(q, c.k, c.v, c.table, pos, req, 1 / math.sqrt(d), window, 16)
    sees = lambda p: torch.tensor([x >= p and (not window or x < p + window) for x in positions])
    hit = torch.zeros(q.shape, dtype=torch.bool)
    hit[sees(230), :4, 5] = True
    hit[sees(233), 4:8, 7] = True
    assert torch.isposinf(got[sees(230)][:, :4, 5]).all()
    assert torch.isnan(got[sees(233)][:, 4:8, 7]).all()
    assert torch.isnan(got[sees(281)][:, 8:12]).all()
    hit[sees(281), 8:12] = True
    assert torch.isfinite(got[~hit]).all()
    ref.assert_within(torch.where(hit, 0, got), torch.where(hit, 0.0, want), bound, c.dtype, "the others")


@pytest.mark.parametrize("window", [0, 40])
def test_rows_outside_the_table_or_cache_are_nan(hm, device, window):
    c = Case(56, [300, 40], 64, 16, 64, 16, torch.bfloat16)
    table = c.table.clone()
    table[0, 9] = c.k.size(0)  # tokens 144..159
    rows = [(p, 0) for p in range(300)] + [(39, 1)]
    rows[70], rows[100], rows[130] = (16 * table.size(1), 0), (100, 2), (-2, 0)
    positions, requests = zip(*rows)
    assert _blocks(c, positions, requests)[0] > 0
    q = _queries(c, len(rows), 57)
    pos, req = torch.tensor(positions, dtype=torch.int32), torch.tensor(requests, dtype=torch.int32)
    got = hm.paged_attention(torch.zeros(q.shape, dtype=c.dtype, device=device), q.to(device), c.cache(hm, device), table.to(device), pos.to(device), req.to(device),
                             window=window).cpu()
    sees = torch.tensor([(r == 0 and p >= 144 and (not window or p - window < 159)) or r == 2 or p in (-2, 16 * table.size(1)) for p, r in rows])
    assert torch.isnan(got[sees]).all()
    want, bound = ref.attention(q[~sees], c.k, c.v, c.table, pos[~sees], req[~sees], 1 / 8, window, 16)
    ref.assert_within(got[~sees], want, bound, c.dtype, "rows that do not see it")


def test_small_weights_add_up(hm, device):
    # a key of weight 1 next to a thousand of weight 2^-26 with values 2^9 times as large
    n, d, heads = 1000, 64, 32
    c = Case(58, [n], heads, heads, d, 16, torch.float16)
    q = torch.zeros((512, heads, d), dtype=torch.float16)
    q[..., 0] = 26.0
    at = torch.arange(n)
    where = (c.table[0, at // 16].long(), slice(None), at % 16)
    c.k[where] = 0.0
    c.v[where] = 512.0
    k0 = torch.full((n, heads), -1.0, dtype=torch.float16)
    k0[100] = 0.0
    c.k[where[0], :, where[2], 0] = k0
    c.v[int(c.table[0, 100 // 16]), :, 100 % 16] = 1.0
    positions = list(range(n - 512, n))
    assert _blocks(c, positions, [0] * 512)[0] > 0
    got = _check(hm, device, c, positions, [0] * 512, q, scale=math.log(2.0), tag="small weights")
    assert float(got[-1].float().mean()) > 1.005


def test_a_long_request_among_short_ones_is_split(hm, device):
    # the block of the long request is above the limit, and goes to the other kernel
    c = Case(59, [30000, 150, 150, 150, 150], 64, 16, 64, 16, torch.bfloat16)
    rows = [(p, 0) for p in range(30000 - 32, 30000)] + [(p, r) for r in range(1, 5) for p in range(150)]
    positions, requests = zip(*rows)
    taken, of = _blocks(c, positions, requests)
    _check(hm, device, c, list(positions), list(requests), _queries(c, len(rows), 60), tag=f"{taken} of {of} blocks")


def test_a_replayed_graph_follows_its_rows(hm, device):
    c = _case(61, (64, 16), 64, torch.bfloat16)
    rows = 320
    cache, table = c.cache(hm, device), c.table.to(device)
    pos, req = (torch.zeros(rows, dtype=torch.int32, device=device) for _ in range(2))
    q, out, ws = _queries(c, rows, 62).to(device), torch.zeros((rows, 64, 64), dtype=c.dtype, device=device), cache.attention_workspace(64)
    hm.paged_attention(out, q, cache, table, pos, req, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        hm.paged_attention(out, q, cache, table, pos, req, workspace=ws)
    full = [(p, 2) for p in range(13, 333)]
    mixed = ([(p, 0) for p in range(150)] + [(p, 1) for p in range(120, 260)] + [(-1, -1)] * 30)
    single = [(n - 1, r) for r, n in enumerate(c.lengths)] + [(-1, -1)] * (rows - 4)
    for case in (full, single, mixed, [(-1, -1)] * rows, full):
        p, r = zip(*case)
        pos.copy_(torch.tensor(p, dtype=torch.int32))
        req.copy_(torch.tensor(r, dtype=torch.int32))
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        live = torch.tensor(r) >= 0
        want, bound = ref.attention(q.cpu(), c.k, c.v, c.table, p, r, 1 / 8, 0, 16)
        if live.any():
            ref.assert_within(out[live.to(device)], want[live], bound[live], c.dtype, "replay")
        assert (out[~live.to(device)] == 7.0).all()


def test_the_same_bits_on_every_call(hm, device):
    c = _case(63, (64, 16), 128, torch.bfloat16)
    positions, requests = _rows(c, 64)
    q, cache, table = _queries(c, len(positions), 65).to(device), c.cache(hm, device), c.table.to(device)
    pos, req = torch.tensor(positions, dtype=torch.int32, device=device), torch.tensor(requests, dtype=torch.int32, device=device)
    first = hm.paged_attention(torch.zeros_like(q), q, cache, table, pos, req)
    for _ in range(3):
        assert torch.equal(hm.paged_attention(torch.zeros_like(q), q, cache, table, pos, req), first)


@pytest.mark.parametrize("rows", [1024, 1025, 1300, 3000])
@pytest.mark.parametrize("kind", ["single", "drafts", "prompts", "empty"])
def test_many_rows(hm, device, rows, kind):
    # around the number of rows from which they are counted in a launch of their own, and chunks of several rows
    rng = np.random.default_rng(66)
    if kind == "single":
        c = Case(67, [int(n) for n in rng.integers(1, 60, rows)], 8, 2, 64, 16, torch.float16)
        _check(hm, device, c, tag="single tokens")
        return
    c = Case(68, [int(n) for n in rng.integers(100, 200, 40)], 16, 4, 64, 16, torch.bfloat16)
    at = []
    while len(at) < rows:
        r = int(rng.integers(0, 40))
        n = c.lengths[r]
        if kind == "drafts":
            at += [(p, r) for p in range(n - int(rng.integers(1, 6)), n)] + [(-1, -1)] * int(rng.integers(0, 2))
        elif kind == "prompts":
            at += [(p, r) for p in range(n)]
        else:
            at += [(-1, -1)] * 900 + [(n - 1, r)]
    positions, requests = zip(*at[:rows])
    _check(hm, device, c, list(positions), list(requests), _queries(c, rows, 69), tag=f"{kind}")


@pytest.mark.parametrize("scale,order", [(1.0, "rising"), (1.0, "falling"), (-1.0, "rising")])
@pytest.mark.parametrize("window", [0, 37])
@pytest.mark.parametrize("dtype,k_log,q_size", [("fp16", 9, 500.0), ("fp16", 13, 8000.0), ("fp16", 16, 60000.0), ("bf16", 16, 60000.0), ("bf16", 40, 1e12)])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_scores_far_from_zero(hm, device, d, dtype, k_log, q_size, window, scale, order):
    # Scores up to 2^80 of which a row's largest is ahead of the next by more than 2^6 in base 2, so that each other weight is zero in fp32 and
    # the output is one key's value, exactly: a weight is hi + lo to 2^-16, far less than half a step of the output.
    n, kv, heads = 256, 16, 64
    c = Case(70, [n], heads, kv, d, 16, DT[dtype])
    at = torch.arange(n)
    size = ((at + 1) / n - 0.5) * 2.0 ** k_log  # distinct, of 8 bits: exact in both types
    where = (c.table[0, at // 16].long(), slice(None), at % 16)
    k = torch.zeros((n, kv, d), dtype=c.dtype)
    k[..., 0] = (size if order == "rising" else -size).to(c.dtype)[:, None]
    c.k[where] = k
    values = c.v[where]
    q = torch.zeros((n, heads, d), dtype=c.dtype)
    q[..., 0] = (q_size * (0.5 + 0.5 * torch.rand((n, heads), generator=torch.Generator().manual_seed(71)))).to(c.dtype)
    assert _blocks(c, list(range(n)), [0] * n)[0] > 0
    pos = torch.arange(n, dtype=torch.int32, device=device)
    got = hm.paged_attention(torch.zeros(q.shape, dtype=c.dtype, device=device), q.to(device), c.cache(hm, device), c.table.to(device), pos, torch.zeros_like(pos),
                             scale=scale, window=window).cpu()
    first = (at - window + 1).clamp(min=0) if window else torch.zeros_like(at)
    top = at if (scale > 0) == (order == "rising") else first
    want = values[top].repeat_interleave(heads // kv, 1)
    wrong = (got != want).any(-1)
    print(f"{dtype} d={d} window={window}: {int(wrong.sum())} of {wrong.numel()} heads are wrong", flush=True)
    assert not wrong.any()


def test_the_limit_keeps_a_long_request_out(hm, device):
    # Above 1024 rows the launch that counts tiles leaves the limit of prompt blocks behind 256 counts in the workspace: eight times what all blocks take
    # on average per place on the card (256 CUs with two workgroups each, over the key heads).
    c = Case(72, [30000] + [150] * 7, 64, 16, 64, 16, torch.bfloat16)
    rows = [(p, 0) for p in range(30000 - 32, 30000)] + [(p, r) for r in range(1, 8) for p in range(150)]
    positions, requests = zip(*rows)
    assert len(rows) > 1024
    cache, q = c.cache(hm, device), _queries(c, len(rows), 73)
    ws = torch.zeros(cache.attention_workspace_bytes(64) + 256, dtype=torch.uint8, device=device)
    ws = ws[-ws.data_ptr() % 256:]
    _check(hm, device, c, list(positions), list(requests), q, tag="a long request among short ones", workspace=ws)
    ends = [positions[b + 31] + 1 if requests[b] == requests[b + 31] else 0 for b in range(0, len(rows) - 31, 32)]
    runs = 2048  # one per wave: more units than three for every four waves
    left = int(ws[16 * runs + 4 * 256:16 * runs + 4 * 256 + 4].view(torch.int32))
    print(f"limit {left}, blocks of {sorted(set(ends))} keys", flush=True)
    assert left == (8 * sum(ends) - 1) // (512 // 16)
    assert ends[0] == 30000 > left > max(ends[1:]) > 0
