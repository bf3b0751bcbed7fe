"""GPU: beam search's selection among equal scores, whose order is by beam and token and no other."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _in_order(row, beams, k):
    """(beam, token) of the k best of `beams` equal rows: by logit, then beam, then token. The rows' sums are one number, and fp64 keeps the scores of unequal logits apart."""
    x = row.double().cpu().numpy()
    best = np.argsort(-x, kind="stable")[:k]
    found = sorted((-x[t], beam, int(t)) for beam in range(beams) for t in best)
    return [(beam, t) for _, beam, t in found[:k]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("beams,vocabulary", [(2, 2049), (3, 5000), (4, 5003), (5, 32001), (8, 50256), (16, 50257), (4, 128256), (7, 128261), (4, 152064), (64, 9001), (256, 4100)])
def test_equal_rows(hm, device, dtype, beams, vocabulary):
    for seed in range(4):
        gen = torch.Generator(device=device).manual_seed(100 * beams + seed)
        row = (2.5 * torch.randn(vocabulary, generator=gen, device=device)).to(DTYPES[dtype])
        requests = 3 if beams <= 16 else 1
        logits = row.repeat(requests * beams, 1)  # an odd vocabulary begins each row at another alignment
        k = min(64, 3 * beams)
        print(f"equal rows: {requests} x {beams}, {vocabulary} tokens, k {k}, {dtype}, seed {seed}", flush=True)
        step = hm.BeamStep(requests, beams, k, vocabulary, device)
        hm.beam_select(step, logits, torch.full((requests * beams,), -3.25, device=device))
        torch.cuda.synchronize()
        want = _in_order(row, beams, k)
        for q in range(requests):
            assert [(p - q * beams, t) for p, t in zip(step.parents[q].tolist(), step.tokens[q].tolist())] == want, q
        # one sum for all rows: a logit's score is the same number in each
        of = {}
        for (_, t), s in zip(want, step.scores[0].tolist()):
            assert of.setdefault(float(row[t]), s) == s


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ld,at", [(5003, 0), (5003, 1), (5001, 3), (5016, 7), (5000, 0)])
def test_equal_rows_within_wider_ones(hm, device, dtype, ld, at):
    gen = torch.Generator(device=device).manual_seed(ld + at)
    row = (2.5 * torch.randn(4990, generator=gen, device=device)).to(DTYPES[dtype])
    wide = torch.full((8, ld), math.nan, dtype=DTYPES[dtype], device=device)
    wide[:, at:at + 4990] = row
    step = hm.BeamStep(1, 8, 40, 4990, device)
    hm.beam_select(step, wide[:, at:at + 4990], torch.zeros(8, device=device))
    torch.cuda.synchronize()
    assert list(zip(step.parents[0].tolist(), step.tokens[0].tolist())) == _in_order(row, 8, 40)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_row_has_one_score_wherever_it_lies(hm, device, dtype):
    # as any beam of any number, at any alignment
    gen = torch.Generator(device=device).manual_seed(7)
    row = (2.5 * torch.randn(6001, generator=gen, device=device)).to(DTYPES[dtype])
    seen = set()
    for beams in (1, 2, 3, 7, 20):
        step = hm.BeamStep(1, beams, beams, 6001, device)
        hm.beam_select(step, row.repeat(beams, 1), torch.full((beams,), -1.5, device=device))
        torch.cuda.synchronize()
        seen.add(step.scores[0, 0].item())
    assert len(seen) == 1


def test_scores_below_the_range_of_fp32(hm, device):
    # Two beams that went on with a masked token, of the type's lowest value, and have one token each that is not: the next ones are masked again, the lowest first
    lowest = torch.finfo(torch.float32).min
    for v, token in ((5000, 3000), (9001, 0), (140000, 139999)):
        for beams in (2, 3, 70):
            logits = torch.full((beams, v), lowest, device=device)
            logits[:, token] = 1.0
            step = hm.BeamStep(1, beams, beams + 4, v, device) if beams < 60 else hm.BeamStep(1, beams, 64, v, device)
            hm.beam_select(step, logits, torch.full((beams,), -3e38, device=device))
            torch.cuda.synchronize()
            print(f"below the range: {beams} beams, {v} tokens", flush=True)
            masked = [t for t in range(6) if t != token]
            want = ([(b, token) for b in range(beams)] + [(0, t) for t in masked])[:step.k]
            assert list(zip(step.parents[0].tolist(), step.tokens[0].tolist())) == want
            assert (step.scores[0, :min(beams, step.k)].double() + 3e38).abs().max() <= 2.0 ** -23 * 3e38 and (step.scores[0, beams:] == -math.inf).all()
