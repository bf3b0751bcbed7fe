"""CPU checks of the attention operators' refusals: every call here is turned down before anything reaches a GPU."""

import ctypes
import math

import numpy as np
import pytest
import torch

import attention_ref as ref

FAKE = 0x1000  # an aligned address that is never read


def _cache(hm, **over):
    f = dict(k=FAKE, v=FAKE, pages=4, page_size=16, page_stride=2 * 16 * 64, head_stride=16 * 64, token_stride=64, kv_heads=2, head_dim=64, dtype=0)
    f.update(over)
    return hm._lib.KvCache(**f)


def _attention(hm, cache=None, **over):
    f = dict(out=FAKE, ldo=512, q=FAKE, ldq=512, rows=3, q_heads=8, table=FAKE, ld=5, R=3, W=5, positions=FAKE, requests=None, scale=0.125, window=0, ws=FAKE,
             wb=1 << 40, stream=None)
    f.update(over)
    return hm._lib.load().hm_paged_attention(ctypes.byref(_cache(hm)) if cache is None else cache, *f.values())


BAD_CACHES = [
    dict(k=None), dict(v=None), dict(k=FAKE + 2), dict(v=FAKE + 8), dict(pages=0), dict(pages=2 ** 31), dict(page_size=0), dict(page_size=8), dict(page_size=24),
    dict(page_size=-16), dict(page_stride=8), dict(head_stride=0), dict(token_stride=56), dict(token_stride=68), dict(page_stride=2052), dict(kv_heads=0),
    dict(head_dim=0), dict(head_dim=40), dict(dtype=2), dict(dtype=-1),
]


@pytest.mark.parametrize("over", BAD_CACHES, ids=str)
def test_caches_that_are_refused(hm, over):
    c = ctypes.byref(_cache(hm, **over))
    assert _attention(hm, c) == hm._lib.HM_INVALID_ARGUMENT
    assert "hm_paged_attention" in hm._lib.last_error()
    a = _rope_args(hm)
    assert hm._lib.load().hm_qk_norm_rope(ctypes.byref(a), c, None) == hm._lib.HM_INVALID_ARGUMENT


@pytest.mark.parametrize("over,status", [
    (dict(out=None), 1), (dict(out=FAKE + 8), 1), (dict(ldo=504), 1), (dict(ldo=516), 1), (dict(q=None), 1), (dict(ldq=511), 1), (dict(rows=-1), 1),
    (dict(rows=2 ** 31), 1), (dict(q_heads=0), 1), (dict(q_heads=7), 1), (dict(q_heads=65538), 1), (dict(table=None), 1), (dict(ld=4), 1), (dict(R=0), 1),
    (dict(W=0), 1), (dict(positions=None), 1), (dict(rows=4), 1), (dict(scale=float("nan")), 1), (dict(scale=float("inf")), 1), (dict(window=-1), 1),
    (dict(W=2 ** 27, ld=2 ** 27), 2), (dict(ws=None), 5), (dict(wb=100), 5), (dict(ws=FAKE + 4), 1),
], ids=str)
def test_attention_calls_that_are_refused(hm, over, status):
    assert _attention(hm, **over) == status
    assert "hm_paged_attention" in hm._lib.last_error()


def test_attention_shapes_that_are_unsupported(hm):
    for over in (dict(head_dim=80, token_stride=80), dict(head_dim=512, token_stride=512, head_stride=16 * 512, page_stride=32 * 512),
                 dict(token_stride=2 ** 27)):
        assert _attention(hm, ctypes.byref(_cache(hm, **over)), ldq=1 << 20, ldo=1 << 20) == hm._lib.HM_UNSUPPORTED, over
    c = ctypes.byref(_cache(hm, kv_heads=65536))
    assert _attention(hm, c, q_heads=65536, W=2 ** 26, ld=2 ** 26) == hm._lib.HM_UNSUPPORTED
    assert hm._lib.load().hm_paged_attention(None, *([FAKE, 512] * 2), 1, 8, FAKE, 5, 3, 5, FAKE, None, 1.0, 0, FAKE, 1 << 40, None) == hm._lib.HM_INVALID_ARGUMENT


def test_workspace_bytes(hm):
    lib = hm._lib.load()
    assert lib.hm_paged_attention_workspace_bytes(None, 8) == 0
    assert lib.hm_paged_attention_workspace_bytes(ctypes.byref(_cache(hm)), 7) == 0
    size = lambda h, **over: lib.hm_paged_attention_workspace_bytes(ctypes.byref(_cache(hm, **over)), h)
    assert size(2) > 0 and size(2) == size(32) == size(16)  # units of 16 columns: rows of a request, or query heads
    assert size(80) > 0 and size(8, head_dim=128) > size(8)


def _rope_args(hm, **over):
    a = hm._lib.QkNormRopeArgs(qkv=FAKE, ldqkv=768, q=FAKE, ldq=512, k=None, ldk=0, bias=None, q_weight=None, k_weight=None, frequencies=FAKE, positions=FAKE,
                               slots=FAKE, rows=3, q_heads=8, kv_heads=2, head_dim=64, rotary_dim=64, eps=1e-6, interleaved=0, dtype=0)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("over", [
    dict(qkv=None), dict(qkv=FAKE + 8), dict(ldqkv=760), dict(ldqkv=772), dict(q=None), dict(ldq=508), dict(bias=FAKE + 2), dict(q_weight=FAKE + 8),
    dict(k_weight=FAKE + 4), dict(frequencies=None), dict(positions=None), dict(slots=None), dict(rows=-1), dict(rows=2 ** 31), dict(q_heads=0), dict(kv_heads=0),
    dict(kv_heads=3), dict(head_dim=128), dict(head_dim=72), dict(rotary_dim=72), dict(rotary_dim=-16), dict(rotary_dim=24), dict(eps=-1.0),
    dict(eps=float("nan")), dict(dtype=5), dict(dtype=1),
], ids=str)
def test_rope_calls_that_are_refused(hm, over):
    assert hm._lib.load().hm_qk_norm_rope(ctypes.byref(_rope_args(hm, **over)), ctypes.byref(_cache(hm)), None) == hm._lib.HM_INVALID_ARGUMENT
    assert "hm_qk_norm_rope" in hm._lib.last_error()


@pytest.mark.parametrize("rows", [2 ** 24 + 1, 2 ** 31 - 1])
def test_rope_rows_beyond_a_launch(hm, rows):
    assert hm._lib.load().hm_qk_norm_rope(ctypes.byref(_rope_args(hm, rows=rows)), ctypes.byref(_cache(hm)), None) == hm._lib.HM_UNSUPPORTED
    assert "2^24 rows" in hm._lib.last_error()


def test_rope_without_a_cache(hm):
    lib = hm._lib.load()
    assert lib.hm_qk_norm_rope(None, None, None) == hm._lib.HM_INVALID_ARGUMENT
    for over in (dict(k=None), dict(k=FAKE, ldk=120), dict(k=FAKE, ldk=132), dict(k=FAKE, ldk=128, head_dim=528, rotary_dim=0)):
        assert lib.hm_qk_norm_rope(ctypes.byref(_rope_args(hm, **over)), None, None) == hm._lib.HM_INVALID_ARGUMENT, over
    assert lib.hm_qk_norm_rope(ctypes.byref(_rope_args(hm, rows=0, qkv=None)), None, None) == hm._lib.HM_OK


def _plan_args(**over):
    f = dict(lengths=FAKE, added=FAKE, R=3, table=FAKE, ld=5, W=5, page_size=16, free_pages=FAKE, Q=9, queue_in=FAKE, slots=FAKE, positions=FAKE, requests=FAKE,
             rows=7, starts=FAKE, lengths_out=FAKE, queue_out=FAKE, stream=None)
    f.update(over)
    return tuple(f.values())


@pytest.mark.parametrize("over,status", [
    *[({k: None}, 1) for k in ("lengths", "added", "table", "free_pages", "queue_in", "slots", "positions", "requests", "starts", "lengths_out", "queue_out")],
    (dict(R=0), 1), (dict(R=4097), 2), (dict(ld=4), 1), (dict(W=0), 1), (dict(page_size=17), 1), (dict(page_size=8), 1), (dict(Q=0), 1), (dict(Q=2 ** 31), 1),
    (dict(rows=-1), 1), (dict(rows=2 ** 31), 1), (dict(W=2 ** 27, ld=2 ** 27), 2),
], ids=str)
def test_plans_that_are_refused(hm, over, status):
    assert hm._lib.load().hm_page_plan(*_plan_args(**over)) == status
    assert "hm_page_plan" in hm._lib.last_error()


def test_host_tensors_are_refused(hm):
    z = torch.zeros((2, 2, 16, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="device tensors"):
        hm.PagedCache(z, z)
    i = torch.zeros(2, dtype=torch.int32)
    plan = hm.PagePlan(2, 4, 16, "cpu")
    with pytest.raises(ValueError, match="device tensors"):
        hm.page_plan(plan, i, i, torch.zeros((2, 3), dtype=torch.int32), i, torch.zeros(4, dtype=torch.int64))
    q = torch.zeros((2, 12 * 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="device tensors"):
        hm.qk_norm_rope(q[:, :512], q, hm.rope_frequencies(64), i, k_out=q[:, 512:640], kv_heads=2, head_dim=64)


@pytest.mark.parametrize("shape", [(0, 2, 16, 64), (4, 0, 16, 64), (4, 2, 0, 64), (4, 2, 16, 0)])
def test_empty_caches_are_refused(hm, shape):
    # before the device is looked at: heads of no elements would be divided by
    k = torch.zeros(shape, dtype=torch.float16)
    with pytest.raises(ValueError, match="must not be empty"):
        hm.PagedCache(k, k.clone())


def test_rope_frequencies(hm):
    f = hm.rope_frequencies(128, 500000.0).numpy()
    np.testing.assert_allclose(f, 500000.0 ** (-np.arange(64) / 64), rtol=1e-15)
    s = hm.rope_frequencies(128, 500000.0, llama3_scaling=(8.0, 1.0, 4.0, 8192)).numpy()
    turns = 8192 * f / (2 * np.pi)
    np.testing.assert_array_equal(s[turns >= 4], f[turns >= 4])
    np.testing.assert_allclose(s[turns <= 1], f[turns <= 1] / 8, rtol=1e-15)
    between = (turns > 1) & (turns < 4)
    assert between.any() and (s[between] < f[between]).all() and (s[between] > f[between] / 8).all()
    assert hm.rope_frequencies(0).numel() == 0


def test_the_request_by_request_plan():
    # known answers: two decodes (one into a new page), a prompt over two pages, an ended request, one refused for pages
    p = ref.plan([15, 16, 0, 20, 0], [1, 1, 18, -1, 16], [[4, -1], [2, -1], [-1, -1], [7, 3], [-1, -1]], [9, 8, 5, -1, -1, -1], 0, 3, 40, 16)
    assert p["slots"][:20].tolist() == [4 * 16 + 15, 9 * 16] + list(range(8 * 16, 9 * 16)) + [5 * 16, 5 * 16 + 1]
    assert (p["slots"][20:] == -1).all() and (p["requests"][20:] == -1).all()
    assert p["positions"][:5].tolist() == [15, 16, 0, 1, 2] and p["starts"].tolist() == [0, 1, 2, 20, 20, 36]
    assert p["lengths"].tolist() == [16, 17, 18, 0, 0] and p["queue"].tolist() == [3, 5, 1, 36]
    assert p["table"].tolist() == [[4, -1], [2, 9], [8, 5], [7, 3], [-1, -1]] and p["ring"].tolist() == [9, 8, 5, 7, 3, -1]


def _layer(hm, q_heads=8, kv_heads=2, head_dim=64, wo_device="cuda:0", **kw):
    from types import SimpleNamespace

    cuda = torch.device("cuda", 0)
    wqkv = SimpleNamespace(k=512, n=(q_heads + 2 * kv_heads) * head_dim, dtype=torch.float16, device=cuda)
    wo = SimpleNamespace(k=q_heads * head_dim, n=512, dtype=torch.float16, device=torch.device(wo_device))
    return hm.AttnLayer(wqkv, wo, q_heads, kv_heads, head_dim, hm.rope_frequencies(64), **kw)


@pytest.mark.parametrize("kw,match", [
    *[(dict(head_dim=d), "heads of 64, 96, 128 or 256") for d in (16, 32, 80, 112, 160, 512)],
    (dict(kv_heads=0), "multiple"), (dict(q_heads=0), "multiple"), (dict(q_heads=7), "multiple"), (dict(q_heads=65538), "65536"),
    *[(dict(scale=s), "scale") for s in (math.nan, math.inf, 1e39)], (dict(window=-1), "window"), (dict(wo_device="cuda:1"), "device"),
], ids=str)
def test_layers_that_no_call_would_take_are_refused_when_made(hm, kw, match):
    # they used to fail in their first call, when keys and values had been written to the cache (or, on two devices, not at all)
    with pytest.raises(ValueError, match=match):
        _layer(hm, **kw)


def test_layers_of_every_head_size(hm):
    for d in (64, 96, 128, 256):
        assert _layer(hm, head_dim=d, scale=0.0, window=5).head_dim == d
