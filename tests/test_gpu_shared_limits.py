"""GPU: attention over shared pages at the ends of what it accepts: keys at the end of 31 bits."""

import math

import numpy as np
import pytest
import torch

import attention_ref as ref
from test_gpu_shared_attention import Call, prompts

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
PS = 64
MOST = (2 ** 31 - 320) // PS  # blocks of a table: 2^31 - 320 tokens


def _call(hm, cache, q, table, positions, requests, window):
    rows, heads, _ = q.shape
    device = q.device
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    share = hm.SharePlan(rows, PS, heads, cache.kv_heads, device, window=window)
    print(f"shared attention: {tuple(q.shape)}, table {tuple(table.shape)}, window {window}, {q.dtype}", flush=True)
    hm.share_plan(share, table, i32(positions), i32(requests))
    out = hm.shared_attention(torch.full_like(q, 7.0), q, cache, table, i32(positions), share, i32(requests))
    torch.cuda.synchronize()
    return out, share.shared.tolist()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,d", [((40, 1), 64), ((8, 1), 64), ((40, 1), 128), ((12, 2), 128)])
def test_the_last_keys_of_the_longest_table(hm, device, dtype, heads, d):
    # Page numbers are read ahead of the keys, past 2^31 here. The same pages in a short table are the same call: its blocks are a multiple of 64 tokens earlier.
    gen = torch.Generator(device=device).manual_seed(d + heads[0])
    randn = lambda *s: torch.randn(s, generator=gen, device=device).to(TYPES[dtype])
    cache = hm.PagedCache(randn(160, heads[1], PS, d), randn(160, heads[1], PS, d))
    q = 1.5 * randn(3, heads[0], d)
    last = np.random.default_rng(3).permutation(160)[:140].astype(np.int32)
    ends = np.stack([last[:100], np.concatenate([last[:60], last[100:]])])  # two requests that share 60 of the last 100 pages
    requests, window = [0, 0, 1], 4000
    tables = []
    for width in (MOST, 200):
        t = torch.full((2, width), -1, dtype=torch.int32, device=device)
        t[:, -100:] = torch.from_numpy(ends).to(device)
        tables.append(t)
    far, shared = _call(hm, cache, q, tables[0], [MOST * PS - 1 - n for n in (0, 2, 5)], requests, window)
    near, shared_near = _call(hm, cache, q, tables[1], [200 * PS - 1 - n for n in (0, 2, 5)], requests, window)
    assert [s - (MOST - 200) * PS for s in shared[1:]] == shared_near[1:]
    assert torch.equal(far, near)
    want, bound = ref.attention(q.cpu(), cache.k.cpu(), cache.v.cpu(), tables[1].cpu(), np.array([200 * PS - 1 - n for n in (0, 2, 5)]), np.array(requests), 1 / math.sqrt(d),
                                window, PS)
    ref.assert_within(near.cpu(), want, bound, q.dtype, f"{heads} heads of {d}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads", [(40, 1), (8, 1)])
def test_all_keys_of_the_longest_table(hm, device, dtype, heads):
    # Two pages in turn, of equal scores: weights and their sums within a run are exact, so the outputs are the values' mean but for the join of at most 2048 parts
    # (2048 x 2^-24) and the last rounding.
    k = torch.zeros((2, 1, PS, 64), dtype=TYPES[dtype], device=device)
    v = torch.zeros_like(k)
    v[:] = 2.0 ** (torch.arange(64, device=device) % 3)
    v[1] *= 3
    table = (torch.arange(MOST, device=device) % 2).to(torch.int32).view(1, MOST)
    q = torch.randn((2, heads[0], 64), device=device).to(TYPES[dtype])
    out, shared = _call(hm, hm.PagedCache(k, v), q, table, [(MOST - 1) * PS - 1] * 2, [0, 0], 0)
    assert shared == [0, (MOST - 1) * PS]
    want = 2 * 2.0 ** (torch.arange(64, device=device) % 3)
    off = (out.double() - want).abs() / want
    assert off.max() <= ref.half_step(TYPES[dtype]) + 2048 * 2.0 ** -24


@pytest.mark.parametrize("d", [64, 96, 128, 256])
@pytest.mark.parametrize("rows", [3, 40])
def test_values_near_the_end_of_bf16(hm, device, d, rows):
    # Scores rise by 15 powers of two behind the first keys, which is less than the maximum has to follow at once; weights times values stay below 2^128 all the same.
    table, ends = prompts(1, rows, 320, 0, 60, 16)
    c = Call(hm, device, rows, table, ends, 16, (8, 2), d, "bf16", scale=math.log(2.0))
    c.cache.k.zero_()
    c.cache.k[[int(p) for p in c.table[0, 2:20]], :, :, 0] = 15
    c.cache.v.mul_(2.0 ** 116)  # of 380 normal numbers: sums below 2^127
    c.q.zero_()
    c.q[..., 0] = 1
    c.check(f"{rows} rows, heads of {d}")
