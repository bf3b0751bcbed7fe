"""Performance cases of the attention operators over a paged key-value cache.

A pass is one call of one operator, as a model's layer (or, for the page plan, a serving loop's step) makes it:

  plan       page_plan: pages, cache slots and positions of a step's new tokens, from the requests' lengths
  rope       qk_norm_rope: the rows of a Q/K/V projection; bias, norms of the query and key heads, position rotation, and
             the keys and values written to their slots of the cache
  attention  paged_attention: one new token of each request over its cached keys and values

Head layouts are those of Llama-3.2-1B, Llama-3-8B, Phi-3.5-mini and Qwen2.5-14B and others between them, pages hold 16 to
256 tokens and lie in the cache in no order, contexts run from one token to 131072, fp16 and bf16. Without `own` a pass
computes the operator from elementary torch operations in fp32 (angles in fp64) and rounds once at the end.
"""

import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_LARGEST_ATTENTION = 64 * 8192 * 8 * 128  # cached elements of K that the largest listed case reads


def _plan(name, requests, rows, longest, page_size, kind, mix):
    return {"name": name, "op": "plan", "requests": requests, "rows": rows, "longest": longest, "page_size": page_size, "kind": kind, "mix": mix}


def _rope(name, rows, used, q_heads, kv_heads, head_dim, rotary, norm, bias, interleaved, base, farthest, page_size, dtype):
    return {"name": name, "op": "rope", "rows": rows, "used": used, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "rotary": rotary, "norm": norm, "bias": bias, "interleaved": interleaved, "base": base, "farthest": farthest,
            "page_size": page_size, "dtype": dtype}


def _attention(name, rows, longest, spread, q_heads, kv_heads, head_dim, page_size, window, dtype, mix):
    return {"name": name, "op": "attention", "rows": rows, "longest": longest, "spread": spread, "q_heads": q_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page_size": page_size, "window": window, "dtype": dtype, "mix": mix}


def listed():
    return [
        # One decoded token of each of 64 requests: the smallest plan, a launch's latency.
        _plan("plan_decode_64", 64, 64, 8192, 16, "decode", 1),
        # Continuous batching: decoding requests, prompt chunks, idle and finished requests in one padded step.
        _plan("plan_mixed_256", 256, 8192, 16384, 16, "mixed", 2),
        # A large offline batch takes in its prompts.
        _plan("plan_prompts_2048", 2048, 65536, 32768, 64, "mixed", 3),
        # One decoded token, Llama-3-8B: rotation and cache write alone.
        _rope("rope_8b_m1_fp16", 1, 1, 32, 8, 128, 128, False, False, False, 500000.0, 8192, 16, "fp16"),
        # A decode batch with Qwen2.5-14B's heads and biases, and norms of queries and keys.
        _rope("rope_norm_14b_m64_bf16", 64, 61, 40, 8, 128, 128, True, True, False, 1000000.0, 32768, 16, "bf16"),
        # A prompt chunk of Llama-3.2-1B, an odd number of rows in a padded step.
        _rope("rope_1b_m2048_fp16", 2048, 2011, 32, 8, 64, 64, False, False, False, 500000.0, 131072, 64, "fp16"),
        # A large step of prompt chunks with normed queries and keys at far positions.
        _rope("rope_norm_8b_m8192_bf16", 8192, 8192, 32, 8, 128, 128, True, False, False, 500000.0, 131072, 16, "bf16"),
        # One request, a short context: latency.
        _attention("attn_8b_r1_fp16", 1, 1037, 1, 32, 8, 128, 16, 0, "fp16", 1),
        # A decode batch with ragged contexts, Qwen2.5-14B heads (five queries to a key head).
        _attention("attn_14b_r32_bf16", 32, 8192, 64, 40, 8, 128, 16, 0, "bf16", 2),
        # Many requests with medium contexts, Llama-3.2-1B heads, larger pages.
        _attention("attn_1b_r128_fp16", 128, 2040, 3, 32, 8, 64, 64, 0, "fp16", 3),
        # One request with a very long context: few rows, the work is all along one axis.
        _attention("attn_8b_r1_long_bf16", 1, 130987, 1, 32, 8, 128, 16, 0, "bf16", 4),
        # A full decode batch with long contexts: the largest call, all of it cache reads.
        _attention("attn_8b_r64_bf16", 64, 8192, 1, 32, 8, 128, 16, 0, "bf16", 5),
    ]


def _log_between(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "rope", "attention", "attention"])
    dtype = rng.choice(["fp16", "bf16"])
    page_size = rng.choice([16, 32, 64, 128, 256])
    if op == "plan":
        requests = _log_between(rng, 1, 2048)
        kind = rng.choice(["decode", "mixed"])
        rows = requests if kind == "decode" else _log_between(rng, requests, 65536)
        return {k: v for k, v in _plan("", requests, rows, _log_between(rng, 64, 32768), page_size, kind, rng.randrange(1 << 30)).items() if k != "name"}
    q_heads, kv_heads = rng.choice([(32, 8), (40, 8), (32, 32), (28, 4), (16, 2), (24, 1), (64, 8)])
    head_dim = rng.choice([64, 96, 128, 128, 256])
    if op == "rope":
        most = 8192 * 48 * 128 // ((q_heads + 2 * kv_heads) * head_dim)
        rows = _log_between(rng, 1, most)
        used = rows if rng.random() < 0.5 else rng.randint(max(1, rows - rows // 8), rows)
        rotary = head_dim if rng.random() < 0.7 else head_dim // 2
        case = _rope("", rows, used, q_heads, kv_heads, head_dim, rotary, rng.random() < 0.6, rng.random() < 0.4, rng.random() < 0.3,
                     rng.choice([10000.0, 500000.0, 1000000.0]), _log_between(rng, 256, 131072), page_size, dtype)
    else:
        rows = _log_between(rng, 1, 256)
        most = min(131072, _LARGEST_ATTENTION // (kv_heads * head_dim * rows))
        longest = _log_between(rng, 1, max(2, most))
        window = _log_between(rng, 16, longest) if longest > 64 and rng.random() < 0.25 else 0
        case = _attention("", rows, longest, rng.choice([1, 4, 64, 1024]), q_heads, kv_heads, head_dim, page_size, window, dtype,
                          rng.randrange(1 << 30))
    return {k: v for k, v in case.items() if k != "name"}


def _attention_lengths(case):
    """Keys that each row sees, the new token's among them: between longest / spread and longest, evenly over the logarithm."""
    rng = random.Random(case["mix"])
    lo = max(1, case["longest"] // case["spread"])
    lengths = [_log_between(rng, lo, case["longest"]) for _ in range(case["rows"])]
    if case["spread"] == 1:  # a batch of like contexts, up to a 16th shorter
        lengths = [max(1, case["longest"] - rng.randint(0, case["longest"] // 16)) if case["rows"] > 1 else case["longest"] for _ in lengths]
    lengths[rng.randrange(case["rows"])] = case["longest"]
    return lengths


def _plan_requests(case):
    """(lengths, added) of the requests: cached tokens, and the new tokens of this step (0: idle, -1: the request has ended)."""
    rng = random.Random(case["mix"])
    r, longest = case["requests"], case["longest"]
    if case["kind"] == "decode":
        return [_log_between(rng, 1, longest - 1) for _ in range(r)], [1] * r
    lengths, added, room = [], [], case["rows"]
    for i in range(r):
        u = rng.random()
        left = r - 1 - i  # at least one row for each that may follow
        if u < 0.1:
            lengths.append(_log_between(rng, 1, longest))
            added.append(rng.choice([0, -1]))
        elif u < 0.55 and room > left:
            lengths.append(_log_between(rng, 1, longest - 1))
            added.append(1)
        elif room > left:
            n = 0 if rng.random() < 0.5 else _log_between(rng, 1, max(1, longest // 2))
            a = max(1, min(_log_between(rng, 1, max(1, 4 * case["rows"] // r)), longest - n, room - left))
            lengths.append(n)
            added.append(a)
        else:
            lengths.append(0)
            added.append(0)
        room -= max(added[-1], 0)
    return lengths, added


def _pages_of(n, page_size):
    return -(-n // page_size)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _inputs(case, seed):
    rng = random.Random(seed)
    gen = _generator(seed)
    dev = "cuda"
    ps = case["page_size"]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    if case["op"] == "plan":
        lengths, added = _plan_requests(case)
        order = list(range(case["requests"]))
        rng.shuffle(order)
        lengths, added = [lengths[i] for i in order], [added[i] for i in order]
        width = _pages_of(case["longest"], ps)
        held = [_pages_of(n, ps) for n in lengths]
        need = sum(_pages_of(n + max(a, 0), ps) - h for n, a, h in zip(lengths, added, held))
        spare = need + case["mix"] % 64
        pages = sum(held) + spare
        ids = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
        table = torch.full((case["requests"], width), -1, dtype=torch.int32, device=dev)
        at = 0
        for r, h in enumerate(held):
            table[r, :h] = ids[at:at + h]
            at += h
        head = rng.randrange(1 << 20)
        ring = torch.full((pages,), -1, dtype=torch.int32, device=dev)
        ring[(head + torch.arange(spare, device=dev)) % pages] = ids[at:]
        return {"lengths": i32(lengths), "added": i32(added), "table": table, "ring": ring,
                "queue": torch.tensor([head, head + spare, 0, 0], dtype=torch.int64, device=dev)}
    dtype = _DTYPES[case["dtype"]]
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    randn = lambda *shape: torch.randn(shape, generator=gen, device=dev, dtype=torch.float32).to(dtype)
    if case["op"] == "rope":
        rows, used = case["rows"], case["used"]
        half = case["rotary"] // 2
        freq = torch.tensor([case["base"] ** (-i / half) for i in range(half)], dtype=torch.float64, device=dev)
        pages = _pages_of(used, ps) + 3
        slots = torch.randperm(pages * ps, generator=gen, device=dev)[:used]  # a batch's tokens end in pages all over the cache
        if used > 4 * ps:  # prompts fill whole pages in order
            first = torch.randperm(pages, generator=gen, device=dev)[:_pages_of(used, ps)]
            slots = (first[:, None] * ps + torch.arange(ps, device=dev)).reshape(-1)[:used]
        pad = torch.full((rows - used,), -1, dtype=torch.int64, device=dev)
        start = rng.randint(0, case["farthest"] - 1)
        pos = (start + torch.arange(used, device=dev)) % case["farthest"] if used > 4 * ps else \
            torch.randint(0, case["farthest"], (used,), generator=gen, device=dev)
        return {"qkv": randn(rows, (hq + 2 * hkv) * d), "freq": freq, "slots": torch.cat([slots, pad]),
                "positions": torch.cat([pos, pad]).to(torch.int32),
                "q_weight": 1 + 0.2 * randn(d) if case["norm"] else None, "k_weight": 1 + 0.2 * randn(d) if case["norm"] else None,
                "bias": randn((hq + 2 * hkv) * d) if case["bias"] else None, "q": torch.zeros((rows, hq, d), dtype=dtype, device=dev),
                "k": torch.zeros((pages, hkv, ps, d), dtype=dtype, device=dev), "v": torch.zeros((pages, hkv, ps, d), dtype=dtype, device=dev)}
    lengths = _attention_lengths(case)
    rng.shuffle(lengths)
    held = [_pages_of(n, ps) for n in lengths]
    pages = sum(held) + 5
    ids = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
    table = torch.full((case["rows"], max(held)), -1, dtype=torch.int32, device=dev)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = ids[at:at + h]
        at += h
    kv = [torch.empty((pages, hkv, ps, d), dtype=dtype, device=dev) for _ in range(2)]
    for t in kv:
        for part in t.split(max(1, (1 << 27) // (hkv * ps * d))):
            part.copy_(torch.randn(part.shape, generator=gen, device=dev, dtype=torch.float32))
    return {"q": 1.5 * randn(case["rows"], hq, d), "k": kv[0], "v": kv[1], "table": table, "positions": i32([n - 1 for n in lengths]),
            "lengths": lengths, "scale": 1.0 / math.sqrt(d), "out": torch.zeros((case["rows"], hq, d), dtype=dtype, device=dev)}


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        import heteromega_amd as hm

        s["hm"] = hm
        if case["op"] == "plan":
            s["plan"] = hm.PagePlan(case["requests"], case["rows"], case["page_size"], s["lengths"].device)
        else:
            s["cache"] = hm.PagedCache(s["k"], s["v"])
        if case["op"] == "attention":
            s["workspace"] = s["cache"].attention_workspace(case["q_heads"])
    return s


def run(state):
    return {"plan": _run_plan, "rope": _run_rope, "attention": _run_attention}[state["case"]["op"]](state)


def _run_plan(s):
    if own:
        p = s["hm"].page_plan(s["plan"], s["lengths"], s["added"], s["table"], s["ring"], s["queue"])
        return [p.slots, p.positions, p.requests, p.starts, p.lengths, p.queue, s["table"], s["ring"]]
    ps, rows = s["case"]["page_size"], s["case"]["rows"]
    table, ring, queue = s["table"], s["ring"], s["queue"]
    width, size, count = table.size(1), ring.size(0), table.size(0)
    n, added = s["lengths"].long(), s["added"].long()
    new = added.clamp(min=0)
    end = torch.cumsum(new, 0)
    start = end - new
    known = n.clamp(0, width * ps)
    held = (known + ps - 1) // ps
    fits = (new > 0) & (known == n) & (n + new <= width * ps) & (end <= rows)
    need = torch.where(fits, (known + new + ps - 1) // ps - held, 0)
    upto = torch.cumsum(need, 0)
    served = fits & ((need == 0) | (upto <= queue[1] - queue[0]))
    # the step's rows
    t = torch.arange(rows, device=n.device)
    r = (t[:, None] >= end).sum(1) if rows * count <= 1 << 24 else torch.searchsorted(end, t, right=True)
    rr = r.clamp(max=count - 1)
    real = (r < count) & served[rr]
    pos = n[rr] + t - start[rr]
    block = pos // ps
    fresh = block >= held[rr]
    page = torch.where(fresh, ring[(queue[0] + (upto - need)[rr] + block - held[rr]) % size].long(),
                       table[rr, block.clamp(0, width - 1)].long())
    slots = torch.where(real, page * ps + pos % ps, -1)
    positions = torch.where(real, pos, -1).int()
    requests = torch.where(real, rr, -1).int()
    # the queue: pages of ended requests behind its tail, in the requests' order
    back = torch.where(added < 0, held, 0)
    back_end = torch.cumsum(back, 0)
    o = (torch.arange(size, device=n.device) - queue[1]) % size
    br = torch.searchsorted(back_end, o, right=True).clamp(max=count - 1)
    block_back = (o - (back_end - back)[br]).clamp(0, width - 1)
    ring.copy_(torch.where(o < back_end[-1], table[br, block_back], ring))
    # the table: fresh pages of the requests that are served
    b = torch.arange(width, device=n.device)
    mine = served[:, None] & (b >= held[:, None]) & (b < (held + need)[:, None])
    table.copy_(torch.where(mine, ring[(queue[0] + (upto - need - held)[:, None] + b) % size], table))
    lengths = torch.where(added < 0, 0, torch.where(served, n + new, n)).int()
    state = torch.stack([queue[0] + (need * served).sum(), queue[1] + back_end[-1], ((new > 0) & ~served).sum(), end[-1]])
    starts = torch.cat([start, end[-1:]]).clamp(max=rows).int()
    return [slots, positions, requests, starts, lengths, state, table, ring]


def _run_rope(s):
    c = s["case"]
    if own:
        s["hm"].qk_norm_rope(s["q"], s["qkv"], s["freq"], s["positions"], cache=s["cache"], slots=s["slots"], q_weight=s["q_weight"],
                             k_weight=s["k_weight"], bias=s["bias"], eps=1e-6, interleaved=c["interleaved"])
        return [s["q"], s["k"], s["v"]]
    used, hq, hkv, d, rd, ps = c["used"], c["q_heads"], c["kv_heads"], c["head_dim"], c["rotary"], c["page_size"]
    x = s["qkv"][:used].float()
    if s["bias"] is not None:
        x = x + s["bias"].float()
    x = x.view(used, hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if c["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-6) * s["q_weight"].float()
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-6) * s["k_weight"].float()
    angle = s["positions"][:used].double()[:, None, None] * s["freq"]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()

    def rotate(h):
        if c["interleaved"]:
            a, b = h[..., 0:rd:2], h[..., 1:rd:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = h[..., :rd // 2], h[..., rd // 2:rd]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([turned, h[..., rd:]], -1)

    page, offset = s["slots"][:used] // ps, s["slots"][:used] % ps
    s["q"][:used] = rotate(q).to(s["q"].dtype)
    s["k"][page, :, offset] = rotate(k).to(s["k"].dtype)
    s["v"][page, :, offset] = v.to(s["v"].dtype)
    return [s["q"], s["k"], s["v"]]


def _run_attention(s):
    c = s["case"]
    if own:
        return s["hm"].paged_attention(s["out"], s["q"], s["cache"], s["table"], s["positions"], scale=s["scale"], window=c["window"],
                                       workspace=s["workspace"])
    hq, hkv, d, ps, window = c["q_heads"], c["kv_heads"], c["head_dim"], c["page_size"], c["window"]
    out = s["out"]
    # as many rows at a time as fit 2^30 gathered elements, padded to their longest
    rows, most = c["rows"], max(s["lengths"])
    step = max(1, (1 << 30) // (_pages_of(most, ps) * ps * hkv * d))
    for at in range(0, rows, step):
        n = max(s["lengths"][at:at + step])
        table = s["table"][at:at + step, :_pages_of(n, ps)].clamp(min=0).long()
        m = table.size(0)
        k, v = (s[x][table].transpose(1, 2).reshape(m, hkv, -1, d).float() for x in ("k", "v"))
        q = s["q"][at:at + step].float().view(m, hkv, hq // hkv, d)
        score = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
        pos = s["positions"][at:at + step, None].long()
        key = torch.arange(k.size(2), device=q.device)
        seen = key <= pos
        if window:
            seen = seen & (key > pos - window)
        score = torch.where(seen[:, None, None], score, -math.inf)
        p = torch.exp(score - score.amax(-1, keepdim=True))
        v = torch.where(seen[:, None, :, None], v, 0)
        out[at:at + step] = (torch.matmul(p, v) / p.sum(-1, keepdim=True)).view(m, hq, d).to(out.dtype)
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    return {"plan": _exact_plan, "rope": _exact_rope, "attention": _exact_attention}[case["op"]](case, s)


def _exact_plan(case, s):
    ps, rows = case["page_size"], case["rows"]
    lengths, added, table, ring = (s[k].cpu().numpy().astype(np.int64) for k in ("lengths", "added", "table", "ring"))
    head, tail = (int(v) for v in s["queue"][:2].cpu())
    size, width = len(ring), table.shape[1]
    slots, positions, requests = (np.full(rows, -1, np.int64) for _ in range(3))
    starts, after = [], lengths.copy()
    row = taken = pushed = refused = 0
    left = tail - head
    out_of_pages = False
    for r in range(len(lengths)):
        starts.append(min(row, rows))
        n, a = int(lengths[r]), int(added[r])
        if a < 0:
            for b in range(_pages_of(min(max(n, 0), width * ps), ps)):
                ring[(tail + pushed) % size] = table[r, b]
                pushed += 1
            after[r] = 0
        if a <= 0:
            continue
        first, row = row, row + a
        if not 0 <= n <= width * ps or n + a > width * ps or row > rows:
            refused += 1
            continue
        need = _pages_of(n + a, ps) - _pages_of(n, ps)
        out_of_pages = out_of_pages or need > left - taken
        if need and out_of_pages:
            refused += 1
            continue
        for b in range(_pages_of(n, ps), _pages_of(n + a, ps)):
            table[r, b] = ring[(head + taken) % size]
            taken += 1
        at = np.arange(n, n + a)
        slots[first:row] = table[r, at // ps] * ps + at % ps
        positions[first:row] = at
        requests[first:row] = r
        after[r] = n + a
    starts.append(min(row, rows))
    i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")
    return [torch.from_numpy(slots).cuda(), i32(positions), i32(requests), i32(starts), i32(after),
            torch.tensor([head + taken, tail + pushed, refused, row], dtype=torch.int64, device="cuda"), i32(table), i32(ring)]


def _exact_rope(case, s):
    hq, hkv, d, rd, ps = case["q_heads"], case["kv_heads"], case["head_dim"], case["rotary"], case["page_size"]
    out = [s[k].double() for k in ("q", "k", "v")]
    half = rd // 2
    # a pair of elements as a complex number, turned by e^(i angle)
    lo = torch.arange(half, device="cuda") * 2 if case["interleaved"] else torch.arange(half, device="cuda")
    hi = lo + 1 if case["interleaved"] else lo + half
    valid = torch.nonzero(s["positions"] >= 0).flatten()
    for rows in valid.split(1024):
        turn = torch.exp(1j * s["positions"][rows].double()[:, None] * s["freq"])[:, None]
        x = s["qkv"][rows].double()
        if s["bias"] is not None:
            x += s["bias"].double()
        heads = x.unflatten(1, (hq + 2 * hkv, d)).clone()
        for part, weight in ((slice(0, hq), s["q_weight"]), (slice(hq, hq + hkv), s["k_weight"])):
            h = heads[:, part]
            if weight is not None:
                h = h / torch.sqrt(h.square().sum(-1, keepdim=True) / d + 1e-6) * weight.double()
            z = torch.complex(h[..., lo], h[..., hi]) * turn
            h = h.clone()
            h[..., lo], h[..., hi] = z.real, z.imag
            heads[:, part] = h
        out[0][rows] = heads[:, :hq]
        for dest, part in ((out[1], heads[:, hq:hq + hkv]), (out[2], heads[:, hq + hkv:])):
            dest[s["slots"][rows] // ps, :, s["slots"][rows] % ps] = part
    return out


def _exact_attention(case, s):
    hq, hkv, d, ps = case["q_heads"], case["kv_heads"], case["head_dim"], case["page_size"]
    out = torch.zeros((case["rows"], hq, d), dtype=torch.float64, device="cuda")
    for r, n in enumerate(s["lengths"]):
        first = max(0, n - case["window"]) if case["window"] else 0
        at = torch.arange(first, n, device="cuda")
        page, offset = s["table"][r].long()[at // ps], at % ps
        for h in range(hkv):
            k, v = s["k"][page, h, offset].double(), s["v"][page, h, offset].double()
            q = s["q"][r, h * (hq // hkv):(h + 1) * (hq // hkv)].double()
            out[r, h * (hq // hkv):(h + 1) * (hq // hkv)] = torch.softmax(q @ k.T * s["scale"], -1) @ v
    return out


def work(case):
    ps = case["page_size"]
    if case["op"] == "plan":
        lengths, added = _plan_requests(case)
        rows = sum(max(a, 0) for a in added)
        need = sum(_pages_of(n + max(a, 0), ps) - _pages_of(n, ps) for n, a in zip(lengths, added))
        back = sum(_pages_of(n, ps) for n, a in zip(lengths, added) if a < 0)
        partial = sum(1 for n, a in zip(lengths, added) if a > 0 and n % ps)
        # lengths and new tokens in; slots, positions, requests, starts and lengths out; pages from or to the queue and the table
        return {"bytes": 16 * len(lengths) + 16 * case["rows"] + 8 * (need + back) + 4 * partial + 64, "flops": 4 * rows}
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "rope":
        elements = case["used"] * (hq + 2 * hkv) * d
        turned = case["used"] * (hq + hkv)
        return {"bytes": 4 * elements + 12 * case["rows"] + 8 * (case["rotary"] // 2) + (4 * d if case["norm"] else 0) +
                (2 * (hq + 2 * hkv) * d if case["bias"] else 0),
                "flops": turned * (3 * case["rotary"] + (4 * d if case["norm"] else 0)) + (elements if case["bias"] else 0)}
    lengths = _attention_lengths(case)
    seen = sum(min(n, case["window"]) if case["window"] else n for n in lengths)
    pages = sum(_pages_of(n, ps) - ((max(0, n - case["window"]) // ps) if case["window"] else 0) for n in lengths)
    return {"bytes": 4 * seen * hkv * d + 4 * case["rows"] * hq * d + 4 * pages + 4 * case["rows"], "flops": 4 * seen * hq * d}
