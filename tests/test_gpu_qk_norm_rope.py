"""GPU: Q/K/V rows made ready for attention (bias, head norms, rotation, cache write) against their float64 form."""

import numpy as np
import pytest
import torch

import attention_ref as ref

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _check(hm, device, seed, rows, q_heads, kv_heads, d, rotary, dtype, norm="qk", bias=True, interleaved=False, page_size=16, base=10000.0,
           farthest=4096, cached=True, in_place=False, pad=0, layout="page_head_token", skip=()):
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(s, generator=gen).to(dtype)
    heads = q_heads + 2 * kv_heads
    qkv = randn(rows, heads * d)
    weights = {n: 1 + 0.3 * randn(d) if n in norm else None for n in "qk"}
    b = randn(heads * d) if bias else None
    freq = hm.rope_frequencies(rotary, base)
    pos = torch.randint(0, farthest, (rows,), generator=gen, dtype=torch.int32)
    pages = ref.pages_of(rows, page_size) + 2
    slots = torch.randperm(pages * page_size, generator=gen)[:rows]
    for t in skip:
        pos[t], slots[t] = -1, -1
    # the float64 form
    x = qkv.double().view(rows, heads, d)
    if b is not None:
        x = x + b.double().view(heads, d)
    q64, qb = ref.norm_rope(x[:, :q_heads], pos, freq, weights["q"], 1e-6, rotary, interleaved)
    k64, kb = ref.norm_rope(x[:, q_heads:q_heads + kv_heads], pos, freq, weights["k"], 1e-6, rotary, interleaved)
    v64, vb = x[:, q_heads + kv_heads:], ref.U * x[:, q_heads + kv_heads:].abs()
    live = pos >= 0
    to = lambda t: None if t is None else t.to(device)
    wide = torch.full((rows, heads * d + pad), 5.0, dtype=dtype, device=device)
    wide[:, :heads * d] = qkv.to(device)
    dev_qkv = wide[:, :heads * d]
    q = dev_qkv[:, :q_heads * d] if in_place else torch.full((rows, q_heads, d), 7.0, dtype=dtype, device=device)
    print(f"rope: rows={rows} heads={q_heads}/{kv_heads} d={d} rotary={rotary} {dtype} norm={norm} cached={cached} in_place={in_place}", flush=True)
    args = dict(q_weight=to(weights["q"]), k_weight=to(weights["k"]), bias=to(b), eps=1e-6, interleaved=interleaved)
    if cached:
        shape = (pages, kv_heads, page_size, d) if layout == "page_head_token" else (pages, page_size, kv_heads, d)
        k, v = (torch.full(shape, 9.0, dtype=dtype, device=device) for _ in range(2))
        if layout != "page_head_token":
            k, v = k.transpose(1, 2), v.transpose(1, 2)
        hm.qk_norm_rope(q, dev_qkv, freq.to(device), pos.to(device), cache=hm.PagedCache(k, v), slots=slots.to(device), **args)
    else:
        k = dev_qkv[:, q_heads * d:(q_heads + kv_heads) * d] if in_place else torch.full((rows, kv_heads, d), 7.0, dtype=dtype, device=device)
        hm.qk_norm_rope(q, dev_qkv, freq.to(device), pos.to(device), k_out=k, kv_heads=kv_heads, head_dim=d, **args)
    torch.cuda.synchronize()
    ref.assert_within(q.reshape(rows, q_heads, d)[live.to(device)], q64[live], qb[live], dtype, "q")
    kept = qkv.view(rows, heads, d)
    if in_place:
        assert torch.equal(q.reshape(rows, q_heads, d).cpu()[~live], kept[:, :q_heads][~live])
    else:
        assert (q.cpu()[~live] == 7.0).all()
    if cached:
        page, off = slots[live] // page_size, slots[live] % page_size
        ref.assert_within(k.cpu()[page, :, off], k64[live], kb[live], dtype, "k in the cache")
        ref.assert_within(v.cpu()[page, :, off], v64[live], vb[live], dtype, "v in the cache")
        mark = torch.ones((pages, page_size), dtype=torch.bool)
        mark[page, off] = False
        for c in (k, v):
            assert (c.cpu().transpose(1, 2)[mark] == 9.0).all(), "slots of no row are left as they are"
    else:
        ref.assert_within(k.reshape(rows, kv_heads, d)[live.to(device)], k64[live], kb[live], dtype, "k")
        assert torch.equal(dev_qkv.cpu().view(rows, heads, d)[:, q_heads + kv_heads:], kept[:, q_heads + kv_heads:]), "values stay where they are"
    if pad:
        assert (wide[:, heads * d:] == 5.0).all()


@pytest.mark.parametrize("d,rotary", [(16, 16), (32, 32), (64, 64), (64, 32), (80, 32), (96, 96), (112, 112), (128, 128), (128, 64), (128, 0), (256, 256), (256, 64),
                                      (512, 512)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_head_sizes(hm, device, d, rotary, interleaved, dtype):
    _check(hm, device, d + rotary, 9, 6, 2, d, rotary, DT[dtype], interleaved=interleaved, skip=(4,))


@pytest.mark.parametrize("norm", ["", "q", "k", "qk"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("cached", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
def test_forms(hm, device, norm, bias, cached, in_place):
    _check(hm, device, 3, 21, 5, 1, 128, 128, torch.bfloat16, norm=norm, bias=bias, cached=cached, in_place=in_place, pad=8, skip=(0, 7, 20))


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 63, 64, 65, 1000, 4099])
def test_row_counts(hm, device, rows):
    _check(hm, device, rows, rows, 8, 2, 128, 128, torch.float16, bias=False, skip=(rows // 2,) if rows > 1 else ())


@pytest.mark.parametrize("heads", [(1, 1), (3, 1), (32, 8), (40, 8), (32, 32), (71, 1), (200, 3)])
def test_head_counts(hm, device, heads):
    for rows in (2, 300):
        _check(hm, device, 11, rows, heads[0], heads[1], 64, 64, torch.float16, bias=rows == 2)


@pytest.mark.parametrize("page_size", [16, 64, 1024])
@pytest.mark.parametrize("layout", ["page_head_token", "page_token_head"])
def test_cache_layouts(hm, device, page_size, layout):
    _check(hm, device, 12, 200, 4, 2, 96, 96, torch.bfloat16, page_size=page_size, layout=layout)


@pytest.mark.parametrize("farthest", [131072, 2 ** 31 - 1])
def test_far_positions(hm, device, farthest):
    _check(hm, device, 13, 500, 4, 1, 128, 128, torch.float16, base=500000.0, farthest=farthest)


def test_large_and_zero_rows(hm, device):
    # a row of zeros has no direction to keep; large values must not overflow on the way
    x = torch.zeros((3, 3 * 64), dtype=torch.float16, device=device)
    x[1] = 60000.0
    x[2, 0] = 6e-8
    q, k = (torch.full((3, 1, 64), 7.0, dtype=torch.float16, device=device) for _ in range(2))
    pos = torch.zeros(3, dtype=torch.int32, device=device)
    ones = torch.ones(64, dtype=torch.float16, device=device)
    hm.qk_norm_rope(q, x, hm.rope_frequencies(64, device=device), pos, k_out=k, kv_heads=1, head_dim=64, q_weight=ones, k_weight=ones, eps=1e-6)
    assert (q[0] == 0).all() and (k[0] == 0).all()
    assert (q[1] == 1).all() and (k[1] == 1).all()
    assert torch.isfinite(q[2]).all()


def test_slots_outside_the_cache_are_not_written(hm, device):
    rows, ps, pages = 6, 16, 4
    k, v = (torch.full((pages, 2, ps, 64), 9.0, dtype=torch.float16, device=device) for _ in range(2))
    slots = torch.tensor([-1, pages * ps, 2 ** 40, -2 ** 40, 5, pages * ps - 1], device=device)
    qkv = torch.randn((rows, 8 * 64), device=device).half()
    q = torch.zeros((rows, 4, 64), dtype=torch.float16, device=device)
    pos = torch.arange(rows, dtype=torch.int32, device=device)
    hm.qk_norm_rope(q, qkv, hm.rope_frequencies(64, device=device), pos, cache=hm.PagedCache(k, v), slots=slots)
    torch.cuda.synchronize()
    written = (v != 9.0).any(-1).any(1).cpu().nonzero().tolist()
    assert written == [[0, 5], [pages - 1, ps - 1]]
    assert torch.equal(v[0, :, 5], qkv[4].view(8, 64)[6:]) and (q != 0).any(-1).all()


def test_a_replayed_graph_follows_positions_and_slots(hm, device):
    rows, d = 5, 128
    qkv = torch.randn((rows, 8 * d), device=device).half()
    pos, slots = torch.arange(rows, dtype=torch.int32, device=device), torch.arange(rows, device=device)
    k, v = (torch.zeros((4, 2, 16, d), dtype=torch.float16, device=device) for _ in range(2))
    cache, q, freq = hm.PagedCache(k, v), torch.zeros((rows, 4, d), dtype=torch.float16, device=device), hm.rope_frequencies(d, device=device)
    hm.qk_norm_rope(q, qkv, freq, pos, cache=cache, slots=slots)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        hm.qk_norm_rope(q, qkv, freq, pos, cache=cache, slots=slots)
    for i in range(4):
        pos.add_(3)
        slots.add_(7)
        pos[i] = -1
        for t in (q, k, v):
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        k2, v2, q2 = torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(q)
        hm.qk_norm_rope(q2, qkv, freq, pos, cache=hm.PagedCache(k2, v2), slots=slots)
        assert torch.equal(q, q2) and torch.equal(k, k2) and torch.equal(v, v2)
        assert (q[i] == 0).all() and (q != 0).any()


# From 2048 rows of one pass on, a workgroup takes two rows of all heads and results are stored past the caches: each form of that kernel, with rows left out
# first and second of their pair and alone in the last.
MANY = dict(skip=(0, 7, 20, 1001, 2050))


@pytest.mark.parametrize("d,rotary", [(16, 16), (64, 64), (64, 32), (80, 32), (96, 96), (128, 128), (128, 0), (256, 64), (512, 512)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_head_sizes_of_many_rows(hm, device, d, rotary, interleaved, dtype):
    _check(hm, device, d + rotary, 2051, 3, 1, d, rotary, DT[dtype], interleaved=interleaved, **MANY)


@pytest.mark.parametrize("norm,bias", [("", False), ("", True), ("q", False), ("k", True), ("qk", True), ("qk", False)])
@pytest.mark.parametrize("cached", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("dtype,interleaved", [("bf16", False), ("fp16", True)])
def test_forms_of_many_rows(hm, device, norm, bias, cached, in_place, dtype, interleaved):
    _check(hm, device, 14, 2051, 5, 1, 64, 64, DT[dtype], norm=norm, bias=bias, interleaved=interleaved, cached=cached, in_place=in_place, pad=8, **MANY)


@pytest.mark.parametrize("rows", [2047, 2048, 2049, 6001])
@pytest.mark.parametrize("page_size,layout", [(16, "page_token_head"), (64, "page_head_token"), (1024, "page_token_head")])
def test_row_counts_and_layouts_of_many_rows(hm, device, rows, page_size, layout):
    _check(hm, device, rows, rows, 4, 2, 64, 64, torch.bfloat16, page_size=page_size, layout=layout, skip=(rows - 1,))
