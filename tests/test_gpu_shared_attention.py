"""GPU: attention over shared pages against float64, and against paged_attention's own form of the same call."""

import math

import numpy as np
import pytest
import torch

import attention_ref as ref
from test_gpu_share_plan import I32, as_table, tree

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


class Call:
    """Rows over a cache of random pages, and the plan of what they share."""

    def __init__(self, hm, device, seed, rows, ends, ps, heads, d, dtype, requests=None, positions=None, window=0, scale=None, swapped=False, spread=1.5, width=None):
        self.hm, self.device, self.ps, self.window = hm, device, ps, window
        self.scale = 1 / math.sqrt(d) if scale is None else scale
        hq, hkv = heads
        pages = max((max(r) for r in rows if r), default=0) + 1
        rng = np.random.default_rng(seed)
        table = as_table(rows, (max(map(len, rows)) + 1) if width is None else width, rng.permutation(pages + 3))
        self.table, self.requests = torch.from_numpy(table), requests
        self.positions = np.asarray(ends) - 1 if positions is None else positions
        gen = torch.Generator(device=device).manual_seed(seed)
        randn = lambda *s: torch.randn(s, generator=gen, device=device).to(TYPES[dtype])
        shape = (pages + 3, ps, hkv, d) if swapped else (pages + 3, hkv, ps, d)
        self.cache = hm.PagedCache(*(t.transpose(1, 2) if swapped else t for t in (randn(*shape), randn(*shape))))
        self.q = (spread * randn(len(self.positions), hq, d)).to(TYPES[dtype])
        self.share = hm.SharePlan(len(self.positions), ps, hq, hkv, device, window=window)
        self.on = [I32(table, device), I32(self.positions, device), None if requests is None else I32(requests, device)]

    def __call__(self, out=None, stream=None):
        hm, (table, positions, requests) = self.hm, self.on
        print(f"shared attention: {tuple(self.q.shape)}, {self.cache.kv_heads} key heads, pages of {self.ps}, window {self.window}, {self.q.dtype}", flush=True)
        hm.share_plan(self.share, table, positions, requests, stream=stream)
        out = torch.full_like(self.q, 7.0) if out is None else out
        return hm.shared_attention(out, self.q, self.cache, table, positions, self.share, requests, self.scale, stream=stream)

    def check(self, tag, out=None):
        got = self() if out is None else out
        torch.cuda.synchronize()
        want, bound = ref.attention(self.q.cpu(), self.cache.k.cpu(), self.cache.v.cpu(), self.table, self.positions, self.requests, self.scale, self.window, self.ps)
        skipped = np.zeros(len(self.positions), bool) if self.requests is None else np.asarray(self.requests) < 0
        assert (got.cpu()[skipped] == 7.0).all(), "rows of no request stay as they are"
        # The parts of a row are joined by factors 2^(m - M) of maxima that were rounded once more: within the bound's share of 4 u for each weight's exponent,
        # which has 2 u (d + 4) of the largest score besides.
        ref.assert_within(got.cpu()[~skipped], want[~skipped], bound[~skipped], self.q.dtype, tag)


def prompts(groups, rows, common, prompt, tail, ps):
    """Table rows and ends: a common part, prompts of groups and tails of rows, in tokens."""
    out, ends, pages = [], [], common // ps
    for g in range(groups):
        path = list(range(common // ps)) + list(range(pages, pages + prompt // ps))
        pages += prompt // ps
        for r in range(rows):
            n = 1 + (37 * g + 11 * r) % tail
            more = -(-n // ps)
            out.append(path + list(range(pages, pages + more)))
            pages += more
            ends.append(len(path) * ps + n)
    return out, ends


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("heads", [(8, 2), (5, 1), (3, 3), (24, 1), (32, 4)])
def test_heads(hm, device, dtype, d, heads):
    for seed, shape in enumerate([(1, 4, 0, 130, 40), (3, 5, 256, 192, 100), (1, 40, 200, 0, 30), (2, 17, 64, 64, 1)]):
        rows, ends = prompts(*shape, 16)
        Call(hm, device, seed, rows, ends, 16, heads, d, dtype).check(f"{heads} heads of {d}, {shape}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ps", [16, 64, 256])
@pytest.mark.parametrize("window", [0, 1, 50, 700])
def test_trees(hm, device, dtype, ps, window):
    rng = np.random.default_rng([ps, window])
    for rows, depth, fan in ((1, 5, 1), (2, 300, 5), (9, 1500, 30), (33, 900, 8), (100, 400, 50)):
        table, ends, _ = tree(rng, rows, ps, depth, fan)
        Call(hm, device, rows, table, ends, ps, (8, 2), 64, dtype, window=window).check(f"{rows} rows to {depth} keys")


@pytest.mark.parametrize("dtype", TYPES)
def test_lengths_from_one_token_on(hm, device, dtype):
    for n in (1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 191, 192, 193, 256, 1000):
        same = [list(range(-(-n // 16)))] * 3
        Call(hm, device, n, same, [n, max(1, n - 1), n], 16, (8, 2), 128, dtype).check(f"{n} keys three times")
        for rows in (5, 30):  # narrow and wide
            deep = [list(range(-(-n // 16))) + [1000 + t] for t in range(rows)]
            Call(hm, device, n, deep, [16 * len(r) - t % 16 for t, r in enumerate(deep)], 16, (8, 2), 64, dtype).check(f"{rows} rows on {n} keys")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,rows", [((8, 2), 16), ((8, 2), 17), ((8, 2), 32), ((8, 2), 33), ((8, 2), 65), ((5, 1), 26), ((5, 1), 100), ((128, 1), 3), ((48, 1), 7), ((1, 1), 200)])
def test_columns_of_wide_units(hm, device, dtype, heads, rows):
    table, ends = prompts(1, rows, 320, 0, 60, 16)
    Call(hm, device, rows, table, ends, 16, heads, 64, dtype).check(f"{rows} rows, {heads} heads")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,rows", [((8, 2), 5), ((5, 1), 6), ((32, 4), 4), ((17, 1), 1), ((24, 1), 1), ((3, 3), 30)])
def test_units_of_17_to_32_columns(hm, device, dtype, d, heads, rows):
    for window in (0, 90):
        table, ends = prompts(2, rows, 64, 320, 50, 16)
        Call(hm, device, rows, table, ends, 16, heads, d, dtype, window=window).check(f"{rows} rows, {heads} heads of {d}, window {window}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [6, 8])
def test_infinities_and_nan_in_units_of_24_and_32_columns(hm, device, dtype, rows):
    test_infinities_and_nan(hm, device, dtype, rows)


@pytest.mark.parametrize("dtype,d,heads,rows,keys", [("bf16", 64, (32, 8), 128, 37000), ("fp16", 128, (64, 8), 120, 20016), ("bf16", 256, (32, 8), 100, 20000)])
def test_wide_runs_of_many_tiles(hm, device, dtype, d, heads, rows, keys):
    # about 150 tiles for each of 256 runs, of which the pages of 64 are read at a time
    table, ends = prompts(1, rows, keys // 16 * 16, 0, 200, 16)
    c = Call(hm, device, 4, table, ends, 16, heads, d, dtype)
    got = c()
    same = hm.paged_attention(torch.zeros_like(c.q), c.q, c.cache, *c.on[:2])
    torch.cuda.synchronize()
    step = 2 * ref.half_step(c.q.dtype) * (same.float().abs().amax(-1, keepdim=True) + 1e-3)  # as below
    assert ((got.float() - same.float()).abs() <= step).all()


def test_long_keys_are_split_over_the_card(hm, device):
    for dtype, rows, heads, d in (("bf16", 2, (8, 2), 128), ("fp16", 30, (8, 2), 64), ("bf16", 40, (4, 1), 128), ("fp16", 3, (2, 1), 256)):
        table, ends = prompts(1, rows, 20000, 0, 300, 16)
        Call(hm, device, rows, table, ends, 16, heads, d, dtype).check(f"{rows} rows of 20000 keys")


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_requests_padding_and_no_keys(hm, device, dtype):
    rng = np.random.default_rng(5)
    table, ends, _ = tree(rng, 20, 16, 900, 40)
    requests = np.array([0, 0, 0, 1, 1, 2, -1, 3, 3, 4, 4, 5, 6, 7, -1, -1])
    positions = np.array([min(ends[r], 500 - i) - 1 if r >= 0 else 5 for i, r in enumerate(requests)])
    positions[4] = positions[9] = -1
    for window in (0, 64):
        Call(hm, device, window, table, ends, 16, (8, 2), 64, dtype, requests=requests, positions=positions, window=window).check(f"window {window}")
    none = Call(hm, device, 1, table, ends, 16, (8, 2), 64, dtype, positions=np.full(20, -1))
    assert (none() == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("swapped", [False, True])
def test_strides_and_scales(hm, device, dtype, swapped):
    rows, ends = prompts(2, 9, 128, 128, 40, 32)
    for scale in (0.0, -0.2, 1.0, 1e-30):
        Call(hm, device, 3, rows, ends, 32, (8, 2), 64, dtype, scale=scale, swapped=swapped).check(f"scale {scale}")
    c = Call(hm, device, 4, rows, ends, 32, (8, 2), 64, dtype, swapped=swapped)
    wide = torch.full((len(ends), 12 * 64 + 8), 3.0, dtype=TYPES[dtype], device=device)
    wide[:, 64:64 + 512] = c.q.view(len(ends), 512)
    c.q = wide[:, 64:64 + 512].unflatten(1, (8, 64))
    to = torch.full((len(ends), 600), 7.0, dtype=TYPES[dtype], device=device)
    c.check("columns of wider rows", c(to[:, 8:520].unflatten(1, (8, 64))))
    assert (to[:, :8] == 7).all() and (to[:, 520:] == 7).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_large_scores(hm, device, dtype):
    rows, ends = prompts(2, 20, 256, 64, 40, 16)
    for spread in (30.0, 1000.0 if dtype == "fp16" else 1e5):
        c = Call(hm, device, 3, rows, ends, 16, (8, 2), 64, dtype, spread=spread)
        got = c()
        torch.cuda.synchronize()
        want, bound = ref.attention(c.q.cpu(), c.cache.k.cpu(), c.cache.v.cpu(), c.table, c.positions, None, c.scale, 0, 16)
        sure = bound <= 0.05 * want.abs().amax()  # where the scores' own rounding leaves the weights known
        assert torch.isfinite(got).all()
        ref.assert_within(torch.where(sure.to(device), got, 0), torch.where(sure, want, 0), bound, c.q.dtype, f"queries of {spread}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [3, 40])
def test_infinities_and_nan(hm, device, dtype, rows):
    # behind the rows' ends and before their windows they do not show; where some rows see them they show in those only
    table, ends = prompts(1, rows, 192, 0, 30, 16)
    for window in (0, 100):
        c = Call(hm, device, 5, table, ends, 16, (8, 2), 64, dtype, window=window)
        k, v = c.cache.k, c.cache.v
        for t, (row, end) in enumerate(zip(table, ends)):
            last = c.table[t, len(row) - 1]
            for x, value in ((k, math.nan), (v, math.inf if t % 2 else math.nan)):
                x[last, :, (end - 1) % 16 + 1:] = value
        if window:
            early = [int(c.table[0, b]) for b in range((min(ends) - window) // 16)]
            k[early], v[early] = math.nan, math.inf
        clean_k, clean_v = torch.nan_to_num(k.float(), 0, 0, 0).to(k.dtype), torch.nan_to_num(v.float(), 0, 0, 0).to(k.dtype)
        got = c()
        torch.cuda.synchronize()
        want, bound = ref.attention(c.q.cpu(), clean_k.cpu(), clean_v.cpu(), c.table, c.positions, None, c.scale, window, 16)
        ref.assert_within(got, want, bound, c.q.dtype, f"{rows} rows, window {window}")
    c = Call(hm, device, 6, table, ends, 16, (8, 2), 64, dtype)
    plain = c().clone()
    own, shared = int(c.table[1, len(table[1]) - 1]), int(c.table[0, 2])
    for page, value, who in ((own, math.inf, [1]), (own, math.nan, [1]), (shared, -math.inf, list(range(rows))), (shared, math.nan, list(range(rows)))):
        c = Call(hm, device, 6, table, ends, 16, (8, 2), 64, dtype)
        c.cache.v[page, 1, 0, 5] = value
        got = c()
        torch.cuda.synchronize()
        odd = torch.zeros_like(got, dtype=torch.bool)
        odd[who, 4:, 5] = True
        assert torch.equal(got[~odd], plain[~odd])
        assert torch.isnan(got[odd]).all() if math.isnan(value) else (got[odd] == value).all()
        c.cache.v.copy_(c.cache.v.nan_to_num(0, 0, 0))
        c.cache.k[page, 1, 0, 5] = math.nan
        got = c()
        torch.cuda.synchronize()
        assert torch.isnan(got[who, 4:]).all() and torch.isfinite(got[:, :4]).all()


def test_pages_and_rows_outside(hm, device):
    for rows in (3, 40):
        table, ends = prompts(1, rows, 192, 0, 30, 16)
        for page, who in ((-1, [0]), (10 ** 6, [0]), (-1, None)):
            c = Call(hm, device, 6, table, ends, 16, (8, 2), 64, "bf16")
            plain = c().clone()
            if who is None:  # a page that all share
                c.table[:, 3] = page
                who = list(range(rows))
            else:
                c.table[0, len(table[0]) - 1] = page
            c.on[0] = c.table.to(torch.int32).to(device)
            got = c()
            torch.cuda.synchronize()
            rest = [t for t in range(rows) if t not in who]
            assert torch.isnan(got[who]).all() and torch.equal(got[rest], plain[rest])
        requests, positions = np.arange(rows), np.asarray(ends) - 1
        requests[1], positions[2] = rows + 5, 10 ** 6
        c = Call(hm, device, 6, table, ends, 16, (8, 2), 64, "bf16", requests=requests, positions=positions)
        got = c()
        torch.cuda.synchronize()
        assert torch.isnan(got[1:3]).all()
        c.requests, c.positions = np.delete(requests, [1, 2]), np.delete(positions, [1, 2])
        keep = [t for t in range(rows) if t not in (1, 2)]
        c.q = c.q[keep]
        c.check("the other rows", got[keep])


def test_a_plan_that_is_not_the_calls(hm, device):
    # not made, of other rows' or of a wider table: nothing outside the arrays is read, rows are NaN or wrong
    table, ends = prompts(2, 9, 192, 64, 30, 16)
    c = Call(hm, device, 6, table, ends, 16, (8, 2), 64, "bf16")
    out = torch.zeros_like(c.q)
    hm.shared_attention(out, c.q, c.cache, c.on[0], c.on[1], c.share)
    torch.cuda.synchronize()
    assert torch.isnan(out).all()
    c()
    narrow = c.on[0][:, :5].contiguous()
    hm.shared_attention(out, c.q, c.cache, narrow, c.on[1].clamp(max=79), c.share)
    hm.shared_attention(out, c.q, c.cache, narrow[:4], c.on[1].clamp(max=79), c.share, I32(np.arange(18) % 4, device))
    torch.cuda.synchronize()
    c.check("again")


def test_the_same_as_paged_attention(hm, device):
    for dtype, groups, rows, common, prompt, tail, heads, d, window in (("bf16", 16, 4, 0, 1024, 200, (40, 8), 128, 0), ("fp16", 4, 32, 1024, 512, 200, (32, 8), 64, 0),
                                                                        ("bf16", 64, 1, 8000, 0, 900, (32, 8), 128, 0), ("fp16", 8, 8, 500, 3000, 64, (16, 2), 96, 1111),
                                                                        ("bf16", 3, 5, 2000, 400, 64, (64, 8), 256, 0), ("fp16", 500, 2, 64, 64, 40, (8, 2), 64, 0)):
        table, ends = prompts(groups, rows, common, prompt, tail, 16)
        c = Call(hm, device, rows, table, ends, 16, heads, d, dtype, window=window)
        got = c()
        same = hm.paged_attention(torch.zeros_like(c.q), c.q, c.cache, *c.on[:2], window=window)
        torch.cuda.synchronize()
        # both are off by at most half a step and the fp32 work before it, well below another half
        step = 2 * ref.half_step(c.q.dtype) * (same.float().abs().amax(-1, keepdim=True) + 1e-3)
        assert ((got.float() - same.float()).abs() <= step).all()
        assert torch.equal(c(), got), "the same call gives the same bits"


def test_a_captured_step_is_replayed_with_other_lengths(hm, device):
    table, ends = prompts(3, 10, 512, 256, 60, 16)
    c = Call(hm, device, 9, table, ends, 16, (8, 2), 64, "bf16", width=60)
    out = torch.zeros_like(c.q)
    ws = c.cache.shared_attention_workspace(8, 30)
    t, p, _ = c.on

    def step():
        hm.share_plan(c.share, t, p)
        hm.shared_attention(out, c.q, c.cache, t, p, c.share, workspace=ws)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    rng = np.random.default_rng(3)
    pages = c.cache.pages
    for i in range(6):
        rows, new_ends, used = tree(rng, 30, 16, 900, [2, 30, 1000][i % 3])
        fold = [[x % pages for x in r] for r in rows]
        for r in range(1, 30):  # what is shared stays so
            fold[r] = [fold[r - 1][b] if b < len(rows[r - 1]) and rows[r][b] == rows[r - 1][b] else x for b, x in enumerate(fold[r])]
        c.table = torch.from_numpy(as_table(fold, 60))
        c.positions = np.asarray(new_ends) - 1
        t.copy_(c.table.to(torch.int32))
        p.copy_(I32(c.positions, device))
        if i == 4:
            step()
        else:
            g.replay()
        c.check(f"replay {i}", out)
        print(float(out.abs().sum()), flush=True)  # work of the program's own between replays


def test_streams(hm, device):
    table, ends = prompts(3, 10, 512, 256, 60, 16)
    calls = [Call(hm, device, s, table, ends, 16, (8, 2), 64, "fp16") for s in range(3)]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    outs = [torch.full_like(c.q, 7.0) for c in calls]
    torch.cuda.synchronize()
    for _ in range(3):
        for c, s, o in zip(calls, streams, outs):
            c(o, stream=s)
    for c, o in zip(calls, outs):
        c.check("on a stream", o)


def test_calls_that_python_refuses(hm, device):
    table, ends = prompts(1, 4, 64, 0, 20, 16)
    c = Call(hm, device, 6, table, ends, 16, (8, 2), 64, "bf16")
    out = torch.zeros_like(c.q)
    good = dict(out=out, q=c.q, cache=c.cache, block_table=c.on[0], positions=c.on[1], share=c.share)
    other = hm.PagedCache.empty(9, 32, 2, 64, torch.bfloat16, device)
    for name, bad in (("out", out[:3]), ("q", c.q[:3]), ("q", c.q.half()), ("cache", other), ("block_table", c.on[0].long()), ("block_table", c.on[0][:3]), ("positions", c.on[1][:3]),
                      ("requests", c.on[1][:2]), ("share", hm.SharePlan(5, 16, 8, 2, device)), ("share", hm.SharePlan(4, 16, 4, 2, device)), ("scale", math.nan),
                      ("workspace", torch.zeros(5, device="cpu"))):
        with pytest.raises(ValueError):
            hm.shared_attention(**{**good, name: bad})
    with pytest.raises(hm.HMError, match="workspace"):
        hm.shared_attention(**good, workspace=torch.zeros(100, device=device))
