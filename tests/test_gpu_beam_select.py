"""GPU: beam search's selection against float64."""

import math

import numpy as np
import pytest
import torch

import branch_ref as ref

pytestmark = pytest.mark.gpu

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _check(hm, device, logits, scores, ended, end_token, beams, k, step=None):
    rows, v = logits.shape
    requests = rows // beams
    want = ref.beam(logits, scores.tolist(), None if ended is None else ended.tolist(), end_token, beams, k)
    step = hm.BeamStep(requests, beams, k, v, device) if step is None else step
    step._workspace.fill_(0xFF)
    print(f"beam: {requests} x {beams}, {v} tokens, k {k}, {logits.dtype}, strides {logits.stride()}", flush=True)
    hm.beam_select(step, logits, scores, ended=ended, end_token=end_token)
    torch.cuda.synchronize()
    got, best = step.scores.cpu().double().numpy(), want[2]
    assert (np.isinf(got) == np.isinf(best)).all() and (got[np.isinf(got)] == -np.inf).all()
    some = np.isfinite(best)
    # fp32 output (2^-24 of it), and of the log of the sum: terms' exponents rounded at up to 2^-24 of 88 log2(e) and exp2 itself 2^-23, sums of 32 to 64 terms
    # and of 64 lanes 40 x 2^-24
    sums = (127 + 2 + 40) * 2.0 ** -24
    off = np.abs(got[some] - best[some])
    assert (off <= 2.0 ** -24 * np.abs(best[some]) + sums).all(), off.max()
    parents, tokens, done = (t.cpu().numpy() for t in (step.parents, step.tokens, step.ended))
    differ = np.argwhere((parents != want[0]) | (tokens != want[1]))
    for q, j in differ:
        # Two rows' sums are off by `sums` at most each, so candidates of different rows whose scores lie within twice that may come in either order. (Rows of i / v
        # and of -i / v even tie in real numbers: sum of exp(i / v) is exp((v - 1) / v) times that of exp(-i / v).)
        row, token = int(parents[q, j]), int(tokens[q, j])
        near = np.argwhere(np.abs(best[q] - best[q, j]) <= 2 * sums).flatten()
        assert len({int(want[0][q, i]) for i in near} | {row}) > 1, (q, j)
        exact = float(scores[row]) + float(logits[row, token].double() - torch.logsumexp(logits[row].double(), 0))
        assert not (ended is not None and ended[row]) and abs(exact - best[q, j]) <= 2 * sums, (q, j)
    for q in {int(q) for q, _ in differ}:
        assert len(set(zip(parents[q], tokens[q]))) == k
    same = np.ones(parents.shape, bool)
    same[tuple(differ.T)] = False
    np.testing.assert_array_equal(done[same], want[3][same])
    return step


def _inputs(device, seed, rows, v, dtype, spread=2.5):
    gen = torch.Generator(device=device).manual_seed(seed)
    return (spread * torch.randn((rows, v), generator=gen, device=device)).to(DTYPES[dtype]), -2 * torch.rand(rows, generator=gen, device=device) - 5


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocabulary", [1, 2, 7, 8, 63, 1000, 2047, 2048, 2049, 8192, 50257, 128256])
def test_vocabularies(hm, device, dtype, vocabulary):
    logits, scores = _inputs(device, vocabulary, 6, vocabulary, dtype)
    _check(hm, device, logits, scores, None, -1, 3, 6)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("requests,beams,k", [(1, 1, 1), (1, 1, 64), (3, 2, 2), (5, 4, 8), (2, 16, 16), (1, 64, 64), (1, 256, 64), (70, 5, 10)])
def test_beams(hm, device, dtype, requests, beams, k):
    logits, scores = _inputs(device, beams, requests * beams, 3001, dtype)
    gen = torch.Generator(device=device).manual_seed(1)
    ended = torch.rand(requests * beams, generator=gen, device=device) < 0.3
    _check(hm, device, logits, scores, ended, 17, beams, k)
    _check(hm, device, logits, scores, None, 17, beams, k)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("requests,beams,k,vocabulary", [(300, 2, 4, 30001), (150, 1, 8, 131075), (1, 256, 16, 66000), (9, 64, 64, 32000), (128, 4, 1, 40003)])
def test_many_logits(hm, device, dtype, requests, beams, k, vocabulary):
    logits, scores = _inputs(device, k, requests * beams, vocabulary, dtype)
    ended = torch.rand(requests * beams, device=device, generator=torch.Generator(device=device).manual_seed(2)) < 0.3
    _check(hm, device, logits, scores, ended, 5, beams, k)


@pytest.mark.parametrize("beams,vocabulary", [(256, 70), (256, 1000), (200, 1025), (37, 64)])
@pytest.mark.parametrize("k", [16, 64])
def test_many_beams_of_few_logits(hm, device, beams, vocabulary, k):
    logits, scores = _inputs(device, beams, beams, vocabulary, "fp16")
    _check(hm, device, logits, scores, None, -1, beams, k)
    _check(hm, device, logits, torch.zeros_like(scores), None, -1, beams, k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_any_alignment(hm, device, dtype):
    for ld, at in ((5003, 0), (5003, 1), (5001, 3), (5016, 7), (5000, 0)):
        big, scores = _inputs(device, at, 8, ld, dtype)
        logits = big[:, at:at + 4990]
        big[:, :at] = math.nan  # what lies next to a row is not its
        big[:, at + 4990:] = math.nan
        _check(hm, device, logits, scores, None, -1, 4, 8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_equal_logits(hm, device, dtype):
    # whole rows of one value, few values, and the best all in one lane's registers: lists overflow
    v = 9000
    logits = torch.zeros((8, v), device=device)
    logits[1] = 1.5
    logits[2] = (torch.arange(v, device=device) % 3).float()
    logits[3] = (torch.arange(v, device=device) // 8 % 64 == 5).float() * 4
    logits[4, 5000:] = 2
    logits[5] = torch.arange(v, device=device).float() / v * 16
    logits[6] = -logits[5]
    scores = torch.tensor([0, -1.0, -2, -3, 0, 0, 0, 0], device=device)
    for beams, k in ((1, 64), (2, 64), (8, 64), (4, 3), (8, 1)):
        _check(hm, device, logits.to(DTYPES[dtype]), scores, None, -1, beams, k)


def test_equal_rows_and_scores(hm, device):
    logits, scores = _inputs(device, 3, 4, 5000, "bf16")
    same = logits[:1].repeat(4, 1)
    _check(hm, device, same, torch.zeros(4, device=device), None, -1, 4, 12)
    _check(hm, device, same, torch.full((4,), -3.25, device=device), torch.tensor([False, True, False, True], device=device), 9, 4, 12)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_without_candidates(hm, device, dtype):
    inf, nan = math.inf, math.nan
    logits, scores = _inputs(device, 4, 12, 4100, dtype)
    logits[0, 3000] = nan
    logits[1, 5] = inf
    logits[2] = -inf
    logits[3, 1:] = -inf  # one token
    logits[4, 100:] = -inf
    logits[7, 4099] = nan
    scores[5], scores[6], scores[8] = -inf, nan, inf
    ended = torch.zeros(12, dtype=torch.bool, device=device)
    ended[7] = True  # its logits are not looked at
    for k in (1, 5, 64):
        _check(hm, device, logits, scores, ended, 4099, 12, k)
        _check(hm, device, logits, scores, ended, 0, 3, k)
        _check(hm, device, logits, scores, ended, 0, 1, k)
    scores[:] = -inf
    scores[0::4] = 0  # the first step of a search: one beam in use
    _check(hm, device, _inputs(device, 5, 12, 4100, dtype)[0], scores, None, -1, 4, 4)


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_largest_vocabulary(hm, device, dtype):
    v = 2 ** 24
    logits = torch.full((2, v), -math.inf, dtype=DTYPES[dtype], device=device)
    logits[0, 0] = logits[0, v - 1] = logits[1, 12345] = 1
    step = hm.BeamStep(1, 2, 4, v, device)
    hm.beam_select(step, logits, torch.zeros(2, device=device), end_token=v - 1)
    torch.cuda.synchronize()
    assert step.parents.tolist() == [[1, 0, 0, -1]] and step.tokens.tolist() == [[12345, 0, v - 1, -1]] and step.ended.tolist() == [[False, False, True, True]]
    want = torch.tensor([0, -math.log(2), -math.log(2), -math.inf])
    assert torch.equal(step.scores.cpu()[0, 3], want[3]) and (step.scores.cpu()[0, :3] - want[:3]).abs().max() <= 4 * 2.0 ** -24


def test_extreme_logits(hm, device):
    for dtype in DTYPES:
        logits, scores = _inputs(device, 6, 4, 3000, dtype, 100.0)
        _check(hm, device, logits, scores, None, -1, 2, 8)
        big = torch.finfo(DTYPES[dtype]).max
        logits[:, 7], logits[:, 9] = big, -big
        _check(hm, device, logits, torch.zeros(4, device=device), None, -1, 1, 3)


def test_a_search_in_a_graph_on_its_own_state(hm, device):
    requests, beams, v, end = 3, 4, 4001, 11
    step = hm.BeamStep(requests, beams, beams, v, device)
    logits = torch.zeros((requests * beams, v), dtype=torch.bfloat16, device=device)
    start = torch.full((requests, beams), -math.inf, device=device)
    start[:, 0] = 0
    scores, ended = step.scores.view(-1), step.ended.view(-1)
    call = lambda: hm.beam_select(step, logits, scores, ended=ended, end_token=end)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        call()
    step.scores.copy_(start)
    step.ended.fill_(False)
    s, e = start.view(-1).tolist(), [False] * (requests * beams)
    gen = torch.Generator(device=device).manual_seed(8)
    for i in range(12):
        logits.copy_(2 * torch.randn((requests * beams, v), generator=gen, device=device))
        logits[:, end] += 6 if i % 3 == 1 else 0
        torch.cuda.synchronize()
        if i % 4 == 3:
            call()
        else:
            g.replay()
        torch.cuda.synchronize()
        want = ref.beam(logits, s, e, end, beams, beams)
        np.testing.assert_array_equal(step.parents.cpu().numpy(), want[0])
        np.testing.assert_array_equal(step.tokens.cpu().numpy(), want[1])
        np.testing.assert_array_equal(step.ended.cpu().numpy(), want[3])
        s, e = step.scores.view(-1).tolist(), step.ended.view(-1).tolist()
    assert any(e)


def test_calls_that_python_refuses(hm, device):
    step = hm.BeamStep(2, 3, 3, 50, device)
    good = dict(logits=torch.zeros((6, 50), device=device), scores=torch.zeros(6, device=device))
    for name, bad in (("logits", torch.zeros((5, 50), device=device)), ("logits", torch.zeros((6, 51), device=device)), ("logits", torch.zeros((6, 50), device=device).double()),
                      ("logits", torch.zeros((50, 6), device=device).T), ("scores", torch.zeros(5, device=device)), ("scores", torch.zeros(6, device=device).double()),
                      ("ended", torch.zeros(6, device=device)), ("ended", torch.zeros(5, dtype=torch.bool, device=device)), ("end_token", 50), ("end_token", -2)):
        with pytest.raises(ValueError):
            hm.beam_select(step, **{**good, name: bad})
    with pytest.raises(ValueError):
        hm.beam_select(step, **good, ended=torch.zeros(6, dtype=torch.bool, device=device))  # needs an end token
