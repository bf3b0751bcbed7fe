"""CPU checks of the refusals of the operators for requests that branch: every call here is turned down before anything reaches a GPU; and known answers of their
plain forms."""

import ctypes

import numpy as np
import pytest
import torch

import branch_ref as ref
from test_attention_args import BAD_CACHES, FAKE, _cache


def _call(name, defaults, over):
    import heteromega_amd as hm

    f = dict(defaults)
    f.update(over)
    status = getattr(hm._lib.load(), name)(*f.values())
    if status != hm._lib.HM_OK:
        assert name in hm._lib.last_error()
    return status


FORK = dict(sources=FAKE, keep=None, lengths=FAKE, R=3, table=FAKE, ld=5, table_out=FAKE, ld_out=5, W=5, page_size=16, ring=FAKE, Q=9, queue=FAKE, copies=FAKE,
            lengths_out=FAKE, queue_out=FAKE, ws=FAKE, bytes=1 << 30, stream=None)
COMPACT = dict(pages=9, limit=4, lengths=FAKE, R=3, table=FAKE, ld=5, table_out=FAKE, ld_out=5, W=5, page_size=16, ring=FAKE, Q=9, queue=FAKE, copies=FAKE, n=4,
               queue_out=FAKE, ws=FAKE, bytes=1 << 30, stream=None)
BEAM = dict(logits=FAKE, ld=100, dtype=0, scores=FAKE, ended=None, end=-1, R=2, beams=4, V=100, k=4, parents=FAKE, tokens=FAKE, scores_out=FAKE, ended_out=FAKE, ws=FAKE,
            bytes=1 << 30, stream=None)
SHARE = dict(table=FAKE, ld=5, R=3, W=5, page_size=16, positions=FAKE, requests=None, rows=3, q_heads=8, kv_heads=2, window=0, shared=FAKE, plan=FAKE, bytes=1 << 20,
             stream=None)
TABLES = [(dict(table=None), 1), (dict(R=0), 1), (dict(W=0), 1), (dict(ld=4), 1), (dict(page_size=8), 1), (dict(page_size=48), 1), (dict(W=2 ** 27, ld=2 ** 27, ld_out=2 ** 27), 2)]
RINGS = [(dict(ring=None), 1), (dict(Q=0), 1), (dict(Q=2 ** 31), 1), (dict(queue=None), 1), (dict(queue_out=None), 1)]
SPACES = [(dict(ws=None), 5), (dict(bytes=16), 5), (dict(ws=FAKE + 8), 1)]


@pytest.mark.parametrize("over,status", [
    *TABLES, *RINGS, *SPACES, (dict(sources=None), 1), (dict(lengths=None), 1), (dict(copies=None), 1), (dict(lengths_out=None), 1), (dict(table_out=None), 1),
    (dict(ld_out=4), 1), (dict(ld=7, ld_out=5), 1), (dict(R=4097), 2),
], ids=str)
def test_forks_that_are_refused(hm, over, status):
    assert _call("hm_page_fork", FORK, over) == status


@pytest.mark.parametrize("over,status", [
    *TABLES, *RINGS, *SPACES, (dict(lengths=None), 1), (dict(copies=None), 1), (dict(n=3), 1), (dict(limit=0, n=0), 1), (dict(limit=-1), 1), (dict(limit=10), 1), (dict(pages=0), 1),
    (dict(pages=2 ** 31 - 1), 1), (dict(table_out=None), 1), (dict(ld_out=6), 1),
], ids=str)
def test_compactions_that_are_refused(hm, over, status):
    assert _call("hm_page_compact", COMPACT, over) == status


@pytest.mark.parametrize("over,status", [
    *SPACES, *[({k: None}, 1) for k in ("logits", "scores", "parents", "tokens", "scores_out", "ended_out")], (dict(ld=99), 1), (dict(dtype=3), 1), (dict(dtype=-1), 1),
    (dict(logits=FAKE + 1), 1), (dict(logits=FAKE + 2, dtype=2), 1), (dict(R=0), 1), (dict(beams=0), 1), (dict(beams=257), 1), (dict(V=0), 1), (dict(k=0), 1), (dict(k=65), 1),
    (dict(end=100), 1), (dict(end=-2), 1), (dict(ended=FAKE + 64, end=-1), 1), (dict(k=3, scores_out=FAKE), 1), (dict(R=20000), 2), (dict(V=2 ** 24 + 1, ld=2 ** 25), 2),
], ids=str)
def test_selections_that_are_refused(hm, over, status):
    assert _call("hm_beam_select", BEAM, over) == status


@pytest.mark.parametrize("over,status", [
    *TABLES, (dict(positions=None), 1), (dict(shared=None), 1), (dict(plan=None), 5), (dict(bytes=100), 5), (dict(plan=FAKE + 8), 1), (dict(rows=-1), 1), (dict(rows=4), 1),
    (dict(rows=4097, requests=FAKE), 2), (dict(q_heads=7), 1), (dict(kv_heads=0), 1), (dict(q_heads=0), 1), (dict(q_heads=258), 2), (dict(window=-1), 1),
    (dict(W=2 ** 26, ld=2 ** 26, q_heads=64, kv_heads=64), 2),
], ids=str)
def test_share_plans_that_are_refused(hm, over, status):
    assert _call("hm_share_plan", SHARE, over) == status


def test_share_plans_count_tiles_of_32_keys_in_31_bits(hm):
    # 5 * rows * key heads * (W * page_size / 32 + 2) is 2^31 and more from W = 104856 on: 52429 tiles and two, 2 heads, 4096 rows
    assert _call("hm_share_plan", SHARE, dict(rows=4096, R=4096, W=104856, ld=104856, bytes=1 << 30)) == hm._lib.HM_UNSUPPORTED


def _shared(hm, cache=None, **over):
    f = dict(out=FAKE, ldo=512, q=FAKE, ldq=512, rows=3, q_heads=8, table=FAKE, ld=5, R=3, W=5, positions=FAKE, requests=None, scale=0.125, plan=FAKE, plan_bytes=1 << 20,
             ws=FAKE, wb=1 << 40, stream=None)
    f.update(over)
    status = hm._lib.load().hm_shared_attention(ctypes.byref(_cache(hm)) if cache is None else cache, *f.values())
    assert status == hm._lib.HM_OK or "hm_shared_attention" in hm._lib.last_error()
    return status


@pytest.mark.parametrize("over,status", [
    (dict(out=None), 1), (dict(out=FAKE + 8), 1), (dict(ldo=504), 1), (dict(q=None), 1), (dict(ldq=511), 1), (dict(rows=-1), 1), (dict(rows=4097, requests=FAKE), 2), (dict(q_heads=7), 1),
    (dict(q_heads=0), 1), (dict(q_heads=258), 2), (dict(table=None), 1), (dict(ld=4), 1), (dict(R=0), 1), (dict(positions=None), 1), (dict(rows=4), 1), (dict(scale=float("nan")), 1),
    (dict(scale=float("inf")), 1), (dict(plan=None), 1), (dict(plan_bytes=100), 1), (dict(plan=FAKE + 8), 1), (dict(ws=None), 5), (dict(wb=100), 5), (dict(ws=FAKE + 4), 1),
], ids=str)
def test_shared_attention_calls_that_are_refused(hm, over, status):
    assert _shared(hm, **over) == status


@pytest.mark.parametrize("over", BAD_CACHES, ids=str)
def test_caches_that_are_refused(hm, over):
    c = _cache(hm, **over)
    assert _shared(hm, ctypes.byref(c)) == hm._lib.HM_INVALID_ARGUMENT
    for pair in ((c, _cache(hm)), (_cache(hm), c)):
        assert hm._lib.load().hm_copy_pages(ctypes.byref(pair[0]), ctypes.byref(pair[1]), 1, FAKE, 3, None) == hm._lib.HM_INVALID_ARGUMENT


def test_copies_that_are_refused(hm):
    copy, good = hm._lib.load().hm_copy_pages, _cache(hm)
    two = (hm._lib.KvCache * 2)
    assert copy(None, None, 1, FAKE, 3, None) == copy(ctypes.byref(good), None, 0, FAKE, 3, None) == copy(ctypes.byref(good), None, 1, None, 3, None) == 1
    assert copy(ctypes.byref(good), None, 1, FAKE, -1, None) == 1 and copy(ctypes.byref(good), None, 1, None, 0, None) == hm._lib.HM_OK
    for over in (dict(pages=5), dict(page_stride=4096), dict(token_stride=72, head_stride=2048, page_stride=4096), dict(dtype=1), dict(page_size=32), dict(kv_heads=1), dict(head_dim=48)):
        assert copy(two(good, _cache(hm, **over)), None, 2, FAKE, 3, None) == hm._lib.HM_INVALID_ARGUMENT, over
    for over in (dict(dtype=1), dict(page_size=32), dict(kv_heads=1), dict(head_dim=48)):  # pages and strides may differ between the two sides
        assert copy(ctypes.byref(good), ctypes.byref(_cache(hm, **over)), 1, FAKE, 3, None) == hm._lib.HM_INVALID_ARGUMENT, over


def test_shapes_that_are_unsupported(hm):
    for over in (dict(head_dim=80, token_stride=80), dict(head_dim=512, token_stride=512, head_stride=16 * 512, page_stride=32 * 512)):
        assert _shared(hm, ctypes.byref(_cache(hm, **over)), ldq=1 << 20, ldo=1 << 20) == hm._lib.HM_UNSUPPORTED
    c = ctypes.byref(_cache(hm, kv_heads=65536))
    assert _shared(hm, c, q_heads=65536, W=2 ** 26, ld=2 ** 26) == hm._lib.HM_UNSUPPORTED


def test_a_workspace_for_many_requests_is_enough_for_fewer(hm):
    of = hm._lib.load().hm_beam_select_workspace_bytes
    for dtype in (hm._lib.HM_FP16, hm._lib.HM_BF16, hm._lib.HM_LOGITS_FP32):
        for v in (1, 1000, 32003, 152064, 2 ** 22 + 1):
            sizes = [of(r, 4, v, 8, dtype) for r in range(1, 300)]
            assert sizes[0] > 0 and sizes == sorted(sizes)


def test_workspace_bytes(hm):
    lib = hm._lib.load()
    assert lib.hm_page_fork_workspace_bytes(0, 5) == lib.hm_page_fork_workspace_bytes(5, 0) == lib.hm_page_compact_workspace_bytes(0) == 0
    assert lib.hm_beam_select_workspace_bytes(2, 4, 100, 65, 0) == 0 and lib.hm_beam_select_workspace_bytes(2, 4, 100, 4, 0) > 0
    assert lib.hm_share_plan_bytes(-1) == lib.hm_share_plan_bytes(4097) == 0 and lib.hm_share_plan_bytes(4096) > lib.hm_share_plan_bytes(1) > 0
    c = ctypes.byref(_cache(hm))
    assert lib.hm_shared_attention_workspace_bytes(None, 8, 3) == lib.hm_shared_attention_workspace_bytes(c, 7, 3) == lib.hm_shared_attention_workspace_bytes(c, 8, 4097) == 0
    assert lib.hm_shared_attention_workspace_bytes(c, 8, 30) > lib.hm_shared_attention_workspace_bytes(c, 8, 3)


def test_objects_that_no_call_would_take_are_refused_when_made(hm):
    for args in ((0, 4, 4, 100), (2, 0, 4, 100), (2, 257, 4, 100), (2, 4, 0, 100), (2, 4, 65, 100), (2, 4, 4, 0)):
        with pytest.raises(ValueError, match="BeamStep"):
            hm.BeamStep(*args, "cpu")
    for args in ((0, 16, 8, 2), (4097, 16, 8, 2), (4, 16, 7, 2), (4, 16, 8, 0), (4, 16, 0, 2), (4, 16, 258, 2)):
        with pytest.raises(ValueError, match="SharePlan"):
            hm.SharePlan(*args, "cpu")
    with pytest.raises(ValueError, match="window"):
        hm.SharePlan(4, 16, 8, 2, "cpu", window=-1)
    for make in (lambda: hm.PageFork(0, 4, 16, "cpu"), lambda: hm.PageFork(4, 0, 16, "cpu"), lambda: hm.PageCompact(0, 16, "cpu")):
        with pytest.raises(ValueError):
            make()


def test_host_tensors_are_refused(hm):
    i = lambda *s: torch.zeros(s, dtype=torch.int32)
    q = torch.zeros(4, dtype=torch.int64)
    for call in (lambda: hm.beam_select(hm.BeamStep(1, 2, 2, 10, "cpu"), torch.zeros(2, 10), torch.zeros(2)),
                 lambda: hm.page_fork(hm.PageFork(2, 3, 16, "cpu"), i(2), i(2), i(2, 3), i(9), q),
                 lambda: hm.page_compact(hm.PageCompact(9, 16, "cpu"), 4, i(2), i(2, 3), i(9), q),
                 lambda: hm.share_plan(hm.SharePlan(2, 16, 8, 2, "cpu"), i(2, 3), i(2))):
        with pytest.raises(ValueError, match="device tensors"):
            call()
    with pytest.raises(ValueError, match="needs caches"):
        hm.copy_pages([], i(2, 3))


def test_the_request_by_request_fork():
    # pages of 16: 0 and 1 share page 5 and end in 6 and 7; 1 becomes 0, 2 becomes the first 20 tokens of 0, 3 ends, 4 is cut to 10
    f = ref.fork([0, 0, 0, -1, 4], [99, 99, 20, 0, 10], [40, 35, 3, 16, 33], [[5, 8, 6], [5, 9, 7], [1, -1, -1], [2, -1, -1], [3, 4, 10]],
                 [20, 21, 22, -1, -1, -1, -1, -1, -1, -1, -1, -1], 0, 3, 16)
    # request 1's last page is a copy of 6 (8 tokens), request 2's of page 8, which 0 and 1 hold in full (4 tokens)
    assert f["copies"].tolist() == [[6, 20, 8], [8, 21, 4], [-1, -1, -1], [-1, -1, -1], [-1, -1, -1]]
    assert f["table"].tolist() == [[5, 8, 6], [5, 8, 20], [5, 21, -1], [2, -1, -1], [3, 4, 10]] and f["lengths"].tolist() == [40, 40, 20, 0, 10]
    assert f["queue"].tolist() == [2, 9, 0, 2] and f["ring"].tolist()[3:9] == [1, 2, 9, 4, 7, 10]
    # beams that all leave their parent's place: the first child keeps its last page
    f = ref.fork([1, 1], None, [20, 20], [[0, 1], [0, 2]], [7, 8, -1, -1], 0, 2, 16)
    assert f["copies"].tolist() == [[2, 7, 4], [-1, -1, -1]] and f["table"].tolist() == [[0, 7], [0, 2]] and f["ring"].tolist() == [7, 8, 1, -1]
    for bad in (dict(sources=[2, 0]), dict(keep=[-1, 4]), dict(lengths=[33, 20]), dict(lengths=[-1, 20]), dict(tail=0)):
        args = dict(sources=[1, 1], keep=None, lengths=[20, 20], table=[[0, 1], [0, 2]], ring=[7, 8, -1, -1], head=0, tail=2, page_size=16)
        assert ref.fork(**{**args, **bad})["queue"][2] == 1, bad


def test_the_request_by_request_compaction():
    c = ref.compact(10, 5, [20, 40, 0], [[1, 9, -1], [1, 7, 4], [3, 3, 3]], [0, 2, 3, 5, 6, 8, -1], 2, 8, 16, 5)
    assert c["copies"].tolist() == [[7, 0, 16], [9, 2, 16]] + [[-1] * 3] * 3
    assert c["table"].tolist() == [[1, 2, -1], [1, 0, 4], [3, 3, 3]] and c["queue"].tolist() == [2, 3, 0, 2] and c["ring"][2] == 3
    assert ref.compact(10, 3, [20, 40, 0], [[1, 9, -1], [1, 7, 4], [3, 3, 3]], [0] * 7, 2, 8, 16, 5)["queue"].tolist() == [2, 8, 1, 0]


def test_the_row_by_row_selection_and_sharing():
    x = torch.tensor([[0.0, 1.0, 1.0], [3.0, -np.inf, 0.0], [0.0, 0.0, 0.0], [5.0, 5.0, np.nan]])
    p, t, s, e = ref.beam(x, [0.0, -1.0, -0.5, 0.0], [False, False, True, False], 2, 2, 3)
    assert p.tolist() == [[0, 0, 1], [2, -1, -1]] and t.tolist() == [[1, 2, 0], [2, -1, -1]] and e.tolist() == [[False, True, False], [True, True, True]]
    assert s[1, 0] == -0.5 and abs(s[0, 0] - (1 - np.log(1 + 2 * np.e))) < 1e-12
    table = np.array([[1, 2, 3], [1, 2, 4], [1, 2, 4]])
    assert ref.shared_tokens(table, [40, 40, 20], None, 16).tolist() == [0, 32, 21]
    assert ref.shared_tokens(table, [5, 7, 40, 3], [0, 0, -1, 2], 16).tolist() == [0, 6, 0, 0]
