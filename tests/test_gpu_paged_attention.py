"""GPU: one-token attention over a paged cache against its float64 form."""

import math

import numpy as np
import pytest
import torch

import attention_ref as ref

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


class Case:
    """A cache of shuffled pages holding `lengths` tokens of each request; what no request holds is NaN."""

    def __init__(self, seed, lengths, q_heads, kv_heads, d, page_size, dtype, width=None, layout="page_head_token", q_scale=1.5):
        rng = np.random.default_rng(seed)
        gen = torch.Generator().manual_seed(seed)
        self.dtype, self.page_size, self.q_heads = dtype, page_size, q_heads
        held = [ref.pages_of(n, page_size) for n in lengths]
        pages = sum(held) + 3
        ids = rng.permutation(pages)
        width = max(max(held), 1) if width is None else width
        self.table = torch.full((len(lengths), width), -1, dtype=torch.int32)
        self.k = torch.full((pages, kv_heads, page_size, d), float("nan"), dtype=dtype)
        self.v = self.k.clone()
        at = 0
        for r, (n, h) in enumerate(zip(lengths, held)):
            self.table[r, :h] = torch.from_numpy(ids[at:at + h].astype(np.int32))
            at += h
            pos = torch.arange(n)
            for c in (self.k, self.v):
                c[self.table[r, pos // page_size].long(), :, pos % page_size] = torch.randn((n, kv_heads, d), generator=gen).to(dtype)
        self.q = (q_scale * torch.randn((len(lengths), q_heads, d), generator=gen)).to(dtype)
        self.lengths, self.layout = lengths, layout

    def cache(self, hm, device):
        if self.layout == "page_token_head":
            k, v = (c.transpose(1, 2).contiguous().to(device).transpose(1, 2) for c in (self.k, self.v))
        elif self.layout == "sliced":  # one allocation for k and v, with room between the tokens and heads
            both = torch.full((self.k.size(0), 2, self.k.size(1) + 1, self.page_size, self.k.size(3) + 8), float("nan"), dtype=self.dtype, device=device)
            for i, c in enumerate((self.k, self.v)):
                both[:, i, :-1, :, :-8] = c.to(device)
            k, v = both[:, 0, :-1, :, :-8], both[:, 1, :-1, :, :-8]
        else:
            k, v = self.k.to(device), self.v.to(device)
        return hm.PagedCache(k, v)


def _check(hm, device, c, positions=None, requests=None, q=None, scale=None, window=0, tag="", **kw):
    q = c.q if q is None else q
    pos = torch.tensor([n - 1 for n in c.lengths] if positions is None else positions, dtype=torch.int32)
    req = None if requests is None else torch.tensor(requests, dtype=torch.int32)
    scale = 1 / math.sqrt(q.size(2)) if scale is None else scale
    want, bound = ref.attention(q, c.k, c.v, c.table, pos, req, scale, window, c.page_size)
    out = torch.full(q.shape, 7.0, dtype=c.dtype, device=device)
    print(f"{tag}: rows={q.size(0)} heads={c.q_heads}/{c.k.size(1)} d={q.size(2)} page={c.page_size} window={window} longest={int(pos.max()) + 1}", flush=True)
    got = hm.paged_attention(out, q.to(device), c.cache(hm, device), c.table.to(device), pos.to(device), None if req is None else req.to(device),
                             scale=scale, window=window, **kw)
    torch.cuda.synchronize()
    live = torch.ones(q.size(0), dtype=torch.bool) if req is None else req >= 0
    ref.assert_within(got[live.to(device)], want[live], bound[live], c.dtype, tag)
    assert (got[~live.to(device)] == 7.0).all(), "rows of no request are left as they are"
    return got


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_lengths_around_the_tiles(hm, device, d, dtype):
    lengths = [1, 2, 15, 16, 17, 31, 32, 33, 47, 64, 127, 128, 129, 160, 255, 256, 257, 1000]
    _check(hm, device, Case(d, lengths, 8, 2, d, 16, DT[dtype]), tag="lengths")


@pytest.mark.parametrize("heads", [(1, 1), (2, 2), (5, 1), (12, 4), (16, 1), (17, 1), (40, 1), (28, 4), (40, 8), (64, 8), (32, 32)])
def test_head_layouts(hm, device, heads):
    _check(hm, device, Case(2, [70, 1, 333], heads[0], heads[1], 128, 16, torch.bfloat16), tag="heads")


@pytest.mark.parametrize("page_size", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("layout", ["page_head_token", "page_token_head", "sliced"])
def test_pages_and_strides(hm, device, page_size, layout):
    _check(hm, device, Case(3, [5, 777, 64, 1500], 8, 4, 64, page_size, torch.float16, layout=layout), tag=layout)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 100, 128, 129, 1000, 5000])
def test_windows(hm, device, window):
    lengths = [1, 16, 17, 100, 129, 300, 1023, 2000]
    c = Case(4, lengths, 8, 2, 128, 32, torch.bfloat16)
    # what lies before the window may hold anything
    for r, n in enumerate(lengths):
        for at in range(0, max(0, n - window)):
            for t in (c.k, c.v):
                t[int(c.table[r, at // 32]), :, at % 32] = float("nan") if at % 2 else float("inf")
    _check(hm, device, c, window=window, tag="window")


@pytest.mark.parametrize("d", [64, 128])
def test_one_long_row_split_over_the_card(hm, device, d):
    _check(hm, device, Case(5, [20011], 8, 2, d, 16, torch.float16), tag="long row")


def test_ragged_batch_with_shared_parts(hm, device):
    rng = np.random.default_rng(6)
    lengths = [int(v) for v in np.exp(rng.uniform(0, np.log(6000), 40))] + [9001]
    _check(hm, device, Case(6, lengths, 20, 4, 128, 16, torch.bfloat16), tag="ragged")


def test_many_short_rows(hm, device):
    rng = np.random.default_rng(7)
    _check(hm, device, Case(7, [int(v) for v in rng.integers(1, 40, 700)], 4, 2, 64, 16, torch.float16), tag="short rows")


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("window", [0, 50])
def test_rows_enough_for_a_run_per_wave(hm, device, d, window):
    # 2050 and more units: runs of single waves, that end inside long rows; with empty rows, rows of no request and rows outside the cache
    rng = np.random.default_rng(d)
    lengths = [int(v) for v in rng.integers(1, 70, 1025)]
    for r in (0, 3, 500, 1024):
        lengths[r] = int(rng.integers(1000, 3000))
    c = Case(d, lengths, 4, 2, d, 16, torch.bfloat16)
    if window:  # what lies before the window may hold anything
        for r in (0, 500):
            at = torch.arange(lengths[r] - window)
            for t in (c.k, c.v):
                t[c.table[r, at // 16].long(), :, at % 16] = float("nan")
    positions = [n - 1 for n in lengths]
    requests = list(range(1025))
    for r in range(700, 900):
        requests[r] = -1
    positions[10] = positions[901] = -1
    _check(hm, device, c, positions, requests, window=window, tag="a run per wave")
    c.table[20, (lengths[20] - 1) // 16] = c.k.size(0) + 7  # the page of its last key, which every window holds
    positions[30] = 16 * c.table.size(1)
    pos, req = (torch.tensor(v, dtype=torch.int32) for v in (positions, requests))
    got = hm.paged_attention(torch.zeros(c.q.shape, dtype=c.dtype, device=device), c.q.to(device), c.cache(hm, device), c.table.to(device), pos.to(device),
                             req.to(device), window=window).cpu()
    assert torch.isnan(got[[20, 30]]).all() and torch.isfinite(got[:20]).all() and torch.isfinite(got[21:30]).all() and torch.isfinite(got[31:]).all()


@pytest.mark.parametrize("heads", [(24, 1), (32, 1), (33, 1), (64, 2), (100, 1)])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_many_query_heads_of_a_key_head(hm, device, heads, d):
    _check(hm, device, Case(22, [1, 100, 2500, 31], heads[0], heads[1], d, 32, torch.float16), tag="many query heads")


@pytest.mark.parametrize("lengths", [[1], [129], [128 * 512], [3, 70000], [1, 2, 40000, 5, 3000]])
def test_few_rows(hm, device, lengths):
    _check(hm, device, Case(23, lengths, 6, 2, 64, 256, torch.bfloat16), tag="few rows")


def _prompt_rows(seed):
    """(positions, requests) of more rows than requests: chunks of prompts, drafted tokens, decodes, positions out of order and twice, empty
    rows and rows of no request, at places that fall in and across blocks of 2 to 16 rows."""
    rng = np.random.default_rng(seed)
    rows = [(p, 2) for p in range(800, 1025)] + [(p, 1) for p in range(40)] + [(299, 0), (298, 0), (299, 0)] + [(-1, 0), (5, 0)] + [(0, 3)] * 2
    rows += [(-1, -1)] * 5 + [(int(p), 2) for p in rng.integers(-1, 1025, 30)] + [(6, 3), (39, 1), (299, 0), (1024, 2)] * 3 + [(-1, -1)] * 100 + [(250, 0)]
    return [r[0] for r in rows], [r[1] for r in rows]


def _group_case(seed, heads, d, dtype):
    return Case(seed, [300, 40, 1025, 7], heads[0], heads[1], d, 16, dtype)


def _queries(c, rows, seed=30):
    return (1.5 * torch.randn((rows, c.q_heads, c.k.size(3)), generator=torch.Generator().manual_seed(seed))).to(c.dtype)


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("heads", [(4, 4), (6, 2), (8, 2), (7, 1), (16, 1), (20, 1)])
@pytest.mark.parametrize("window", [0, 37])
def test_prompts_and_drafts(hm, device, heads, d, window):
    c = _group_case(24, heads, d, torch.float16 if d == 96 else torch.bfloat16)
    positions, requests = _prompt_rows(25)
    got = _check(hm, device, c, positions, requests, _queries(c, len(positions)), window=window, tag="prompts and drafts")
    for t, p in enumerate(positions):
        if requests[t] >= 0 and p < 0:
            assert (got[t] == 0).all()


@pytest.mark.parametrize("d", [64, 128])
def test_prompts_enough_for_a_run_per_wave(hm, device, d):
    # as many blocks of rows and heads as waves fit the card
    rng = np.random.default_rng(26)
    c = Case(26, [int(v) for v in rng.integers(20, 90, 60)], 32, 16, d, 16, torch.bfloat16)
    rows = [(p, r) for r, n in enumerate(c.lengths) for p in range(0 if r % 3 else n - 1, n)]
    rows += [(-1, -1)] * 20
    assert len(rows) >= 1040
    positions, requests = zip(*rows)
    _check(hm, device, c, list(positions), list(requests), _queries(c, len(rows)), tag="prompts, a run per wave")


@pytest.mark.parametrize("window", [0, 64])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_later_tokens_do_not_show_in_earlier_rows(hm, device, dtype, window):
    # an infinite value, a NaN value and a NaN key in the middle of a prompt: the rows before them, and behind their window, know nothing of them
    c = _group_case(27, (8, 2), 128, DT[dtype])
    at = lambda t, p: t[int(c.table[2, p // 16]), :, p % 16]
    clean = [t.clone() for t in (c.k, c.v)]
    at(c.v, 850)[0, 5] = float("inf")
    at(c.v, 853)[1, 7] = float("nan")
    at(c.k, 901)[0, 3] = float("nan")
    positions = list(range(800, 1025))
    q = _queries(c, len(positions))
    pos, req = torch.tensor(positions, dtype=torch.int32), torch.full((len(positions),), 2, dtype=torch.int32)
    out = torch.zeros(q.shape, dtype=c.dtype, device=device)
    got = hm.paged_attention(out, q.to(device), c.cache(hm, device), c.table.to(device), pos.to(device), req.to(device), window=window).cpu()
    c.k, c.v = clean
    want, bound = ref.attention(q, c.k, c.v, c.table, pos, req, 1 / math.sqrt(128), window, 16)
    sees = lambda p: torch.tensor([x >= p and (not window or x < p + window) for x in positions])
    hit = torch.zeros(q.shape, dtype=torch.bool)
    hit[sees(850), :4, 5] = True
    hit[sees(853), 4:, 7] = True
    assert torch.isposinf(got[sees(850) & ~sees(901)][:, :4, 5]).all()
    assert torch.isnan(got[sees(853)][:, 4:, 7]).all()
    assert torch.isnan(got[sees(901)][:, :4]).all()
    hit[sees(901), :4] = True
    assert torch.isfinite(got[~hit]).all()
    ref.assert_within(torch.where(hit, 0, got), torch.where(hit, 0.0, want), bound, c.dtype, "the others")


@pytest.mark.parametrize("window", [0, 40])
def test_rows_that_see_a_bad_page_are_nan_and_their_neighbours_not(hm, device, window):
    c = _group_case(28, (8, 2), 64, torch.bfloat16)
    table = c.table.clone()
    table[2, 52] = -3  # tokens 832..847
    rows = [(p, 2) for p in range(801, 900)] + [(100, 0), (16 * table.size(1), 0), (101, 0), (-2, 0), (102, 0), (103, 4), (103, 0)]
    positions, requests = zip(*rows)
    q = _queries(c, len(rows))
    pos, req = torch.tensor(positions, dtype=torch.int32), torch.tensor(requests, dtype=torch.int32)
    got = hm.paged_attention(torch.zeros(q.shape, dtype=c.dtype, device=device), q.to(device), c.cache(hm, device), table.to(device), pos.to(device), req.to(device),
                             window=window).cpu()
    sees = torch.tensor([(r == 2 and p >= 832 and (not window or p - window < 847)) or r == 4 or p in (-2, 16 * table.size(1)) for p, r in rows])
    assert torch.isnan(got[sees]).all()
    fine = ~sees
    want, bound = ref.attention(q[fine], c.k, c.v, c.table, pos[fine], req[fine], 1 / 8, window, 16)
    ref.assert_within(got[fine], want, bound, c.dtype, "rows that do not see it")


def test_prompts_in_a_replayed_graph(hm, device):
    c = _group_case(29, (8, 2), 128, torch.bfloat16)
    cache, table = c.cache(hm, device), c.table.to(device)
    pos, req = (torch.zeros(64, dtype=torch.int32, device=device) for _ in range(2))
    q, out, ws = _queries(c, 64).to(device), torch.zeros((64, 8, 128), dtype=c.dtype, device=device), cache.attention_workspace(8)
    hm.paged_attention(out, q, cache, table, pos, req, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        hm.paged_attention(out, q, cache, table, pos, req, workspace=ws)
    rng = np.random.default_rng(29)
    for _ in range(4):
        r = np.sort(rng.integers(-1, 4, 64))
        p = np.array([rng.integers(-1, c.lengths[x]) if x >= 0 else -1 for x in r])
        pos.copy_(torch.tensor(p, dtype=torch.int32))
        req.copy_(torch.tensor(r, dtype=torch.int32))
        out.fill_(7.0)
        g.replay()
        torch.cuda.synchronize()
        live = torch.tensor(r >= 0)
        want, bound = ref.attention(q.cpu(), c.k, c.v, c.table, p, r, 1 / math.sqrt(128), 0, 16)
        ref.assert_within(out[live.to(device)], want[live], bound[live], c.dtype, "replay")
        assert (out[~live.to(device)] == 7.0).all()


def test_rows_of_requests(hm, device):
    # several rows of one request (drafted tokens), empty rows, rows of no request in runs longer than a wave, requests out of order
    c = Case(8, [300, 40, 1025], 8, 2, 128, 16, torch.bfloat16)
    requests = [2, 2, 2, 0, 0] + [-1] * 200 + [1, 1, 0] + [-1] * 70
    positions = [1022, 1023, 1024, 0, 299] + [-1] * 200 + [39, -1, 17] + [-1] * 70
    q = torch.randn((len(requests), 8, 128), generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)
    got = _check(hm, device, c, positions, requests, q, tag="rows of requests")
    assert (got[206] == 0).all(), "a row that sees no key is zero"


def test_no_rows_to_work_on(hm, device):
    c = Case(10, [40], 8, 2, 64, 16, torch.float16)
    q = torch.zeros((3, 8, 64), dtype=torch.float16)
    _check(hm, device, c, [-1, -1, -1], [-1, -1, -1], q, tag="only rows of no request")
    _check(hm, device, c, [-1, -1, -1], [0, 0, 0], q, tag="only empty rows")
    out = torch.empty((0, 8, 64), dtype=torch.float16, device=device)
    assert hm.paged_attention(out, out, c.cache(hm, device), c.table.to(device), torch.empty(0, dtype=torch.int32, device=device)).numel() == 0


def test_extreme_scores(hm, device):
    # one key that outweighs the rest, scores far apart and far below zero, a zero scale
    for dtype in (torch.float16, torch.bfloat16):
        c = Case(11, [600, 600, 600], 4, 2, 64, 16, dtype, q_scale=12.0)
        c.k[int(c.table[0, 3]), :, 5] *= 8
        _check(hm, device, c, scale=1.0, tag="large scores")
        _check(hm, device, c, scale=-1.0, tag="negative scale")
        _check(hm, device, c, scale=0.0, tag="zero scale")


def test_small_weights_add_up(hm, device):
    # a key of weight 1 next to thousands of weight 2^-26 with values 2^9 times as large: fp16 weights would lose them all
    n, d = 4097, 64
    c = Case(12, [n], 1, 1, d, 16, torch.float16)
    q = torch.zeros((1, 1, d), dtype=torch.float16)
    q[..., 0] = 26.0
    for at in range(n):
        page, o = int(c.table[0, at // 16]), at % 16
        c.k[page, 0, o] = 0.0
        c.k[page, 0, o, 0] = 0.0 if at == 1000 else -1.0
        c.v[page, 0, o] = 1.0 if at == 1000 else 512.0
    got = _check(hm, device, c, q=q, scale=math.log(2.0), tag="small weights")
    assert float(got.float().mean()) > 1.02


def test_infinities_and_nan_stay_in_their_row(hm, device):
    c = Case(13, [100, 200, 300], 4, 2, 128, 16, torch.float16)
    c.k[int(c.table[1, 3]), 0, 4, 7] = float("nan")
    c.v[int(c.table[2, 5]), 1, 2, 9] = float("inf")
    want, bound = ref.attention(c.q, c.k, c.v, c.table, torch.tensor([99, 199, 299]), None, 0.1, 0, 16)
    out = torch.zeros(c.q.shape, dtype=c.dtype, device=device)
    got = hm.paged_attention(out, c.q.to(device), c.cache(hm, device), c.table.to(device), torch.tensor([99, 199, 299], dtype=torch.int32, device=device),
                             scale=0.1).cpu().double()
    assert torch.isnan(got[1, :2]).all() and torch.isposinf(got[2, 2:, 9]).all()
    fine = torch.isfinite(want)
    assert torch.isfinite(got[fine]).all()
    ref.assert_within(got[0], want[0], bound[0], c.dtype, "row without them")


def test_rows_outside_the_table_or_cache_are_nan(hm, device):
    c = Case(14, [100, 200, 300, 400], 4, 2, 64, 16, torch.bfloat16)
    table = c.table.clone()
    table[1, 4] = c.k.size(0)
    table[2, 18] = -1
    pos = torch.tensor([99, 199, 299, 399, 399, 16 * table.size(1), -2], dtype=torch.int32, device=device)
    req = torch.tensor([0, 1, 2, 3, 4, 3, 3], dtype=torch.int32, device=device)
    q = torch.randn((7, 4, 64)).to(c.dtype)
    out = torch.zeros(q.shape, dtype=c.dtype, device=device)
    got = hm.paged_attention(out, q.to(device), c.cache(hm, device), table.to(device), pos, req).cpu()
    for t in (1, 2, 4, 5, 6):
        assert torch.isnan(got[t]).all(), t
    want, bound = ref.attention(q[[0, 3]], c.k, c.v, c.table, [99, 399], [0, 3], 1 / 8, 0, 16)
    ref.assert_within(got[[0, 3]], want, bound, c.dtype, "rows inside")


def test_strided_queries_and_outputs(hm, device):
    c = Case(15, [90, 33], 8, 2, 64, 16, torch.float16)
    want, bound = ref.attention(c.q, c.k, c.v, c.table, [89, 32], None, 0.125, 0, 16)
    qkv = torch.full((2, 12 * 64), float("nan"), dtype=c.dtype, device=device)
    qkv[:, :512] = c.q.view(2, 512).to(device)
    out = torch.full((2, 1024), 3.0, dtype=c.dtype, device=device)
    hm.paged_attention(out[:, 8:520], qkv[:, :512], c.cache(hm, device), c.table.to(device), torch.tensor([89, 32], dtype=torch.int32, device=device))
    ref.assert_within(out[:, 8:520].reshape(2, 8, 64), want, bound, c.dtype, "strided")
    assert (out[:, :8] == 3.0).all() and (out[:, 520:] == 3.0).all()


def test_a_replayed_graph_follows_lengths_and_pages(hm, device):
    c = Case(16, [1500, 700, 90], 8, 2, 128, 16, torch.bfloat16)
    cache, table = c.cache(hm, device), c.table.to(device)
    q, pos = c.q.to(device), torch.tensor([1499, 699, 89], dtype=torch.int32, device=device)
    out = torch.zeros(c.q.shape, dtype=c.dtype, device=device)
    ws = cache.attention_workspace(8)
    hm.paged_attention(out, q, cache, table, pos, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        hm.paged_attention(out, q, cache, table, pos, workspace=ws)
    for positions in ([1499, 699, 89], [0, 1, 2], [777, -1, 60], [1499, 699, 89]):
        pos.copy_(torch.tensor(positions, dtype=torch.int32))
        out.fill_(float("nan"))
        g.replay()
        torch.cuda.synchronize()
        eager = hm.paged_attention(torch.zeros_like(out), q, cache, table, pos)
        assert torch.equal(out, eager)
        want, bound = ref.attention(c.q, c.k, c.v, c.table, positions, None, 1 / math.sqrt(128), 0, 16)
        ref.assert_within(out, want, bound, c.dtype, f"replay at {positions}")


def test_two_streams_with_their_own_workspaces(hm, device):
    a, b = Case(17, [5000], 8, 2, 128, 16, torch.float16), Case(18, [3000, 41], 8, 2, 128, 16, torch.float16)
    runs = []
    for c in (a, b):
        s = torch.cuda.Stream()
        cache, table, q = c.cache(hm, device), c.table.to(device), c.q.to(device)
        pos = torch.tensor([n - 1 for n in c.lengths], dtype=torch.int32, device=device)
        runs.append((c, s, cache, table, q, pos, torch.zeros(q.shape, dtype=q.dtype, device=device)))
    torch.cuda.synchronize()
    for _ in range(10):
        for c, s, cache, table, q, pos, out in runs:
            hm.paged_attention(out, q, cache, table, pos, stream=s)
    torch.cuda.synchronize()
    for c, s, cache, table, q, pos, out in runs:
        want, bound = ref.attention(c.q, c.k, c.v, c.table, pos.cpu(), None, 1 / math.sqrt(128), 0, 16)
        ref.assert_within(out, want, bound, c.dtype, "on its stream")


def test_the_same_bits_on_every_call(hm, device):
    c = Case(19, [3000, 17, 800], 8, 2, 128, 16, torch.bfloat16)
    cache, table, q = c.cache(hm, device), c.table.to(device), c.q.to(device)
    pos = torch.tensor([2999, 16, 799], dtype=torch.int32, device=device)
    first = hm.paged_attention(torch.zeros_like(q), q, cache, table, pos)
    for _ in range(5):
        assert torch.equal(first, hm.paged_attention(torch.zeros_like(q), q, cache, table, pos))


def test_a_cache_past_32_bits_of_elements(hm, device):
    # pages at both ends of a cache of 2^32 + elements per tensor (8.6 GB each)
    pages = (1 << 32) // (16 * 8 * 128) + 64
    k = torch.zeros((pages, 8, 16, 128), dtype=torch.float16, device=device)
    v = torch.zeros((pages, 8, 16, 128), dtype=torch.float16, device=device)
    cache = hm.PagedCache(k, v)
    gen = torch.Generator().manual_seed(20)
    table = torch.tensor([[pages - 1, 0, pages - 40, 1]], dtype=torch.int32)
    small_k, small_v = (torch.randn((4, 8, 16, 128), generator=gen).half() for _ in range(2))
    for i, p in enumerate(table[0].tolist()):
        k[p], v[p] = small_k[i].to(device), small_v[i].to(device)
    q = torch.randn((1, 32, 128), generator=gen).half()
    got = hm.paged_attention(torch.zeros((1, 32, 128), dtype=torch.float16, device=device), q.to(device), cache, table.to(device),
                             torch.tensor([60], dtype=torch.int32, device=device))
    want, bound = ref.attention(q, small_k, small_v, torch.arange(4)[None], [60], None, 1 / math.sqrt(128), 0, 16)
    ref.assert_within(got, want, bound, torch.float16, "far pages")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_the_halves_of_a_weight_fit_together(hm, device, dtype):
    # two keys of about the same weight, a hundred thousand times: a weight whose lower half belongs to another rounding of its upper one is
    # 2^-10 (fp16) off, which shows where the two values nearly cancel
    c = Case(19, [2] * 2000, 64, 16, 64, 16, DT[dtype], q_scale=0.5)
    _check(hm, device, c, tag="two keys")


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("window", [0, 25000])
def test_drafts_of_a_long_request(hm, device, d, dtype, window):
    # few units of several rows, each split over the card: drafted tokens of one request and of two, an empty row among them
    c = Case(31, [30000], 8, 2, d, 16, DT[dtype])
    q = _queries(c, 4)
    _check(hm, device, c, list(range(29996, 30000)), [0] * 4, q, window=window, tag="four drafts")
    got = _check(hm, device, c, [29996, -1, 29998, 29999], [0] * 4, q, window=window, tag="drafts and an empty row")
    assert (got[1] == 0).all()
    c = Case(32, [20001, 9000], 8, 2, d, 32, DT[dtype])
    rows = [(p, 0) for p in range(19997, 20001)] + [(p, 1) for p in range(8995, 9000)] + [(-1, -1), (3, 1)]
    positions, requests = zip(*rows)
    _check(hm, device, c, list(positions), list(requests), _queries(c, len(rows)), window=window and 7000, tag="drafts of two")


@pytest.mark.parametrize("height", [4, 64, 400])
def test_the_tables_height(hm, device, height):
    # the same rows in tables with few and many other requests
    c = _group_case(33, (8, 2), 128, torch.bfloat16)
    c.table = torch.cat([c.table, torch.full((height - 4, c.table.size(1)), -1, dtype=torch.int32)])
    positions, requests = _prompt_rows(34)
    _check(hm, device, c, positions, requests, _queries(c, len(positions)), tag=f"a table of {height} requests")
