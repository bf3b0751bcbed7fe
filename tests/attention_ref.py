"""Plain float64 forms of the attention operators for their tests, on the CPU, and the tolerances of the kernels against them.

Tolerances count roundings: an output off by half a step of its type (eps / 2 relative), plus what the fp32 work before
the rounding can lose, elementwise."""

import math

import numpy as np
import torch

U = 2.0 ** -24  # half a step of fp32
# Half a step of a result next to zero: half the smallest subnormal of fp16; bf16 reaches as low as fp32.
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def pages_of(n, page_size):
    return -(-n // page_size)


def gather(cache, table_row, first, end, page_size):
    """Tokens [first, end) of one request, float64 [kv_heads, tokens, head_dim], from a cache on the CPU."""
    at = np.arange(first, end)
    return cache[table_row[at // page_size].long(), :, torch.from_numpy(at % page_size)].double().transpose(0, 1)


def attention(q, k, v, table, positions, requests, scale, window, page_size):
    """(out, bound) float64 [rows, q_heads, d]: softmax(scale q K^T) V, and the most that a kernel's output may be off before its rounding.

    With A = max_j scale sum_d |q_d k_jd|: a score's products and sums are fp32, at most 2 u (d + 4) A off (u of each operation, doubled for
    sums that the matrix unit truncates); so each weight is off by at most twice that, relative, with the maximum's own error,
    and its exp2 by 4 u. The weight enters the second product as hi + lo in 16 bits: hi is at most
    2^-8 + 2^-9 of it below (bf16), and lo's rounding is half a step, 2^-9 of that: 2^-16 in all (fp16 less). The weighted sum
    over n keys adds 2 u (n / 32 + 64) of sum_j p_j |v_j|; the division by their sum doubles what is common."""
    rows, q_heads, d = q.shape
    kv_heads = k.shape[1]
    group = q_heads // kv_heads
    out = torch.zeros((rows, q_heads, d), dtype=torch.float64)
    bound = torch.zeros_like(out)
    for t in range(rows):
        r = t if requests is None else int(requests[t])
        pos = int(positions[t])
        if r < 0 or pos < 0:
            continue
        first = max(0, pos + 1 - window) if window else 0
        kk, vv = (gather(c, table[r], first, pos + 1, page_size) for c in (k, v))
        qq = q[t].double().view(kv_heads, group, d)
        s = qq @ kk.transpose(1, 2) * scale
        p = torch.softmax(s, -1)
        out[t] = (p @ vv).reshape(q_heads, d)
        a = float((qq.abs() @ kk.abs().transpose(1, 2) * abs(scale)).max())
        n = pos + 1 - first
        rel = 2 * (2 * 2 * U * (d + 4) * a + 4 * U + 2.0 ** -16) + 2 * U * (n / 32 + 64)
        bound[t] = rel * (p @ vv.abs()).reshape(q_heads, d)
    return out, bound


def assert_within(got, ref, bound, dtype, tag):
    got = got.detach().cpu().double()
    tol = half_step(dtype) * (ref.abs() + bound) + bound + TINY[dtype]
    off = (got - ref).abs()
    worst = float((off / tol).max()) if off.numel() else 0.0
    print(f"{tag} {dtype}: worst error / tolerance {worst:.3f}", flush=True)
    assert torch.isfinite(got).all(), tag
    assert worst <= 1.0, (tag, worst)


def norm_rope(x, positions, frequencies, weight, eps, rotary, interleaved):
    """(y, bound) float64 of heads x [rows, heads, d] (float64, bias added): norm with weight (None: none), rotation of the first
    `rotary` elements. fp32 work: a bias sum, a sum of d squares, a root, a quotient and three products, 2 u (d + 16) relative in
    all; a pair's rotation adds products and a sum, and cos and sin are 2^-22 off: relative to |a| + |b|."""
    d = x.shape[-1]
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    size = x.abs()
    y = x.clone()
    half = rotary // 2
    if half:
        ang = positions.double()[:, None, None] * frequencies.double().cpu()
        cos, sin = torch.cos(ang), torch.sin(ang)
        i = torch.arange(half)
        lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        a, b = x[..., lo], x[..., hi]
        y[..., lo], y[..., hi] = a * cos - b * sin, b * cos + a * sin
        both = a.abs() + b.abs()
        size = size.clone()
        size[..., lo], size[..., hi] = both, both
    return y, (2 * U * (d + 16) + 2.0 ** -22) * size


def plan(lengths, added, table, ring, head, tail, rows, page_size):
    """One step's page plan, request by request: a dict of int64 arrays (slots, positions, requests, starts, lengths, queue, table, ring)."""
    lengths, added, table, ring = (np.array(v, np.int64) for v in (lengths, added, table, ring))
    width, size = table.shape[1], len(ring)
    slots, positions, requests = (np.full(rows, -1, np.int64) for _ in range(3))
    starts, after, fresh, back = [], lengths.copy(), 0, []
    row, refused, dry = 0, 0, False
    old_ring = ring.copy()
    for r, (n, a) in enumerate(zip(lengths.tolist(), added.tolist())):
        starts.append(min(row, rows))
        if a < 0:
            back += table[r, :pages_of(min(max(n, 0), width * page_size), page_size)].tolist()
            after[r] = 0
        if a <= 0:
            continue
        first, row = row, row + a
        if n < 0 or n + a > width * page_size or row > rows:
            refused += 1
            continue
        need = pages_of(n + a, page_size) - pages_of(n, page_size)
        if need and (dry or fresh + need > min(max(tail - head, 0), size)):
            dry = True
            refused += 1
            continue
        for b in range(pages_of(n, page_size), pages_of(n + a, page_size)):
            table[r, b] = old_ring[(head + fresh) % size]
            fresh += 1
        for i in range(a):
            slots[first + i] = table[r, (n + i) // page_size] * page_size + (n + i) % page_size
            positions[first + i], requests[first + i] = n + i, r
        after[r] = n + a
    for i, page in enumerate(back):
        ring[(tail + i) % size] = page
    starts.append(min(row, rows))
    return {"slots": slots, "positions": positions, "requests": requests, "starts": np.array(starts), "lengths": after,
            "queue": np.array([head + fresh, tail + len(back), refused, row]), "table": table, "ring": ring}
