"""Performance cases of the operators for requests that branch over a paged key-value cache.

A pass is one call of one operator, as a serving loop's step or a model's layer makes it:

  beam     beam_select: the best continuations of each request's beams, from a step's logits
  fork     page_fork and copy_pages: requests become copies (or prefixes) of others, and the pages that they cannot share are copied in some
           layers' caches
  compact  page_compact and copy_pages: the pages in use move to the front of some layers' caches
  share    share_plan: what neighbouring rows of a step share of their pages
  shared   shared_attention: one new token of each request over its cached keys and values, shared pages read once

Head layouts are those of Llama-3.2-1B, Llama-3-8B and Qwen2.5-14B and others between them, vocabularies those of Llama 3 and Qwen2.5. Pages hold 16 to
256 tokens and lie in the cache in no order. Without `own` a pass computes the operator from elementary torch operations (attention in fp32, rounded once
at the end; the beams' scores in fp64, since candidates of different beams lie next to each other).
"""

import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _beam(name, requests, beams, k, vocabulary, ended, dtype):
    return {"name": name, "op": "beam", "requests": requests, "beams": beams, "k": k, "vocabulary": vocabulary, "ended": ended, "dtype": dtype}


def _fork(name, groups, beams, prompt, tail, kind, page_size, layers, kv_heads, head_dim, dtype, mix):
    return {"name": name, "op": "fork", "groups": groups, "beams": beams, "prompt": prompt, "tail": tail, "kind": kind, "page_size": page_size,
            "layers": layers, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "mix": mix}


def _compact(name, requests, longest, used, page_size, layers, kv_heads, head_dim, dtype, mix):
    return {"name": name, "op": "compact", "requests": requests, "longest": longest, "used": used, "page_size": page_size, "layers": layers,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "mix": mix}


def _shared(name, op, groups, beams, common, prompt, tail, q_heads, kv_heads, head_dim, page_size, window, dtype, mix):
    return {"name": name, "op": op, "groups": groups, "beams": beams, "common": common, "prompt": prompt, "tail": tail, "q_heads": q_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page_size": page_size, "window": window, "dtype": dtype, "mix": mix}


def listed():
    return [
        # One request's beam search: the smallest selection, latency.
        _beam("beam_1x4_fp16", 1, 4, 4, 128256, 0.0, "fp16"),
        # A batch of beam searches that asks for twice the beams, as loops do that set finished hypotheses aside.
        _beam("beam_64x4_bf16", 64, 4, 8, 152064, 0.1, "bf16"),
        # Beams reordered after a selection: every slot may change, some layers' partial pages are copied.
        _fork("fork_beams_64_fp16", 16, 4, 2048, 256, "beams", 16, 4, 8, 128, "fp16", 1),
        # A large batch of agents: requests end, start from prefixes of others, or go back to an earlier token; large pages.
        _fork("fork_mixed_512_bf16", 64, 8, 8192, 1024, "mixed", 128, 2, 8, 64, "bf16", 2),
        # A small cache is made smaller.
        _compact("compact_32_fp16", 32, 2048, 0.5, 16, 2, 8, 128, "fp16", 3),
        # A large one.
        _compact("compact_256_bf16", 256, 8192, 0.6, 64, 2, 8, 64, "bf16", 4),
        # What the rows of a decode step share, once per step: a beam search's batch, and a large batch on a system prompt.
        _shared("share_64", "share", 16, 4, 0, 2048, 256, 32, 8, 128, 16, 0, "bf16", 5),
        _shared("share_1024", "share", 256, 4, 2048, 4096, 512, 32, 8, 128, 16, 0, "bf16", 6),
        # Four beams of one prompt: latency.
        _shared("shared_8b_1x4_fp16", "shared", 1, 4, 0, 1024, 64, 32, 8, 128, 16, 0, "fp16", 7),
        # A batch of beam searches, Qwen2.5-14B heads (five queries to a key head).
        _shared("shared_14b_16x4_bf16", "shared", 16, 4, 0, 2048, 256, 40, 8, 128, 16, 0, "bf16", 8),
        # A system prompt, under it prompts with eight samples each, Llama-3.2-1B heads, larger pages.
        _shared("shared_1b_32x8_fp16", "shared", 32, 8, 2048, 4096, 256, 32, 8, 64, 64, 0, "fp16", 9),
        # A full decode batch on a long common document: the largest call.
        _shared("shared_8b_128_bf16", "shared", 128, 1, 16384, 0, 1024, 32, 8, 128, 16, 0, "bf16", 10),
    ]


def _log_between(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["beam", "fork", "compact", "share", "shared", "shared", "shared"])
    dtype = rng.choice(["fp16", "bf16"])
    page_size = rng.choice([16, 32, 64, 128, 256])
    mix = rng.randrange(1 << 30)
    if op == "beam":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
        vocabulary = _log_between(rng, 1000, 160000)
        requests = _log_between(rng, 1, max(2, min(1024, 256 * 152064 // (beams * vocabulary))))
        case = _beam("", requests, beams, rng.choice([beams, 2 * beams, rng.randint(1, 32)]), vocabulary, rng.choice([0.0, 0.1, 0.5]),
                     rng.choice(["fp16", "bf16", "fp32"]))
    elif op == "fork":
        groups, beams = _log_between(rng, 1, 128), rng.choice([1, 2, 3, 4, 5, 8])
        case = _fork("", groups, beams, _log_between(rng, 16, 512 * 1024 // (groups * beams) if groups * beams > 64 else 8192), _log_between(rng, 1, 1024),
                     rng.choice(["beams", "mixed"]), page_size, rng.randint(1, 2), rng.choice([1, 2, 8]), rng.choice([64, 128]), dtype, mix)
    elif op == "compact":
        requests = _log_between(rng, 1, 256)
        case = _compact("", requests, _log_between(rng, 16, 8192), rng.uniform(0.3, 0.95), page_size, rng.randint(1, 2), rng.choice([1, 2, 8]), 64, dtype, mix)
    else:
        groups, beams = _log_between(rng, 1, 128), rng.choice([1, 1, 2, 3, 4, 5, 8, 16])
        if groups * beams > 256:
            groups = max(1, 256 // beams)
        q_heads, kv_heads = rng.choice([(32, 8), (40, 8), (32, 32), (28, 4), (16, 2), (24, 1), (64, 8)])
        head_dim = rng.choice([64, 96, 128, 128, 256])
        most = max(64, 128 * 16384 * 32 * 128 // (groups * beams * q_heads * head_dim))  # keys of a row
        common = 0 if rng.random() < 0.4 else _log_between(rng, 16, min(32768, max(17, most // 2)))
        prompt = 0 if rng.random() < 0.2 else _log_between(rng, 1, min(16384, max(2, most // 4)))
        tail = _log_between(rng, 1, min(2048, max(2, most // 4)))
        window = _log_between(rng, 16, common + prompt + tail) if common + prompt > 64 and rng.random() < 0.2 else 0
        case = _shared("", op, groups, beams, common, prompt, tail, q_heads, kv_heads, head_dim, page_size, window, dtype, mix)
    return {k: v for k, v in case.items() if k != "name"}


def _pages_of(n, page_size):
    return -(-n // page_size)


# ---- requests and their pages, from a case alone: tables of page numbers that `_inputs` deals out in a random order ----


def _fork_requests(case):
    """(lengths, rows of page numbers, pages, sources, keep or None). The beams of a group share their prompt and, with the one before, some of what followed."""
    rng = random.Random(case["mix"])
    ps, m = case["page_size"], case["beams"]
    lengths, table, pages = [], [], 0
    for _ in range(case["groups"]):
        prompt = _log_between(rng, max(1, case["prompt"] // 4), case["prompt"])
        n = prompt + rng.randint(0, case["tail"])
        for i in range(m):
            mine = n if case["kind"] == "beams" else max(0, n - rng.randint(0, min(n, case["tail"])) * rng.randint(0, 1))
            both = 0 if i == 0 else min(rng.randint(prompt, n), mine, lengths[-1]) // ps
            held = _pages_of(mine, ps)
            table.append((table[-1][:both] if i else []) + list(range(pages, pages + held - both)))
            pages += held - both
            lengths.append(mine)
    count = len(lengths)
    if case["kind"] == "beams":
        return lengths, table, pages, [g * m + rng.randrange(m) for g in range(case["groups"]) for _ in range(m)], None
    sources, keep = [], []
    for r in range(count):
        u = rng.random()
        s = r if u < 0.5 else -1 if u < 0.65 else rng.randrange(count)
        some = lengths[s] if s >= 0 else 0
        sources.append(s)
        keep.append(rng.randint(0, some) if 0.35 < u < 0.5 or u > 0.8 else 2 ** 31 - 1)
    return lengths, table, pages, sources, keep


def _compact_requests(case):
    """(lengths, rows of page numbers, pages in use, pages of the cache, limit)."""
    rng = random.Random(case["mix"])
    ps = case["page_size"]
    lengths, table, pages = [], [], 0
    for r in range(case["requests"]):
        n = _log_between(rng, max(1, case["longest"] // 16), case["longest"])
        both = 0 if r == 0 or rng.random() < 0.5 else rng.randint(0, min(n, lengths[-1])) // ps
        held = _pages_of(n, ps)
        table.append((table[-1][:both] if r else []) + list(range(pages, pages + held - both)))
        pages += held - both
        lengths.append(n)
    total = max(pages, int(pages / case["used"]))
    return lengths, table, pages, total, min(total, pages + pages // 16)


def _shared_requests(case):
    """(lengths with the new token, rows of page numbers, pages): all rows begin with the common part, those of a group go on with its prompt."""
    rng = random.Random(case["mix"])
    ps = case["page_size"]
    common = case["common"] // ps
    pages = common
    lengths, table = [], []
    for _ in range(case["groups"]):
        prompt = 0 if case["prompt"] == 0 else _log_between(rng, max(1, case["prompt"] // 4), case["prompt"]) // ps
        path = list(range(common)) + list(range(pages, pages + prompt))
        pages += prompt
        for _ in range(case["beams"]):
            tail = rng.randint(1, case["tail"])
            more = _pages_of(tail, ps)
            table.append(path + list(range(pages, pages + more)))
            pages += more
            lengths.append(len(path) * ps + tail)
    return lengths, table, pages


def _table_of(rows, width, ids, fill=-1):
    table = np.full((len(rows), max(width, 1)), fill, np.int32)
    for r, held in enumerate(rows):
        if held:
            table[r, :len(held)] = ids[np.asarray(held)]
    return table


def _randn(gen, shape, dtype):
    t = torch.empty(shape, dtype=dtype, device="cuda")
    flat = t.view(-1)
    for part in flat.split(1 << 27):
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda", dtype=torch.float32))
    return t


def _inputs(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    i32 = lambda v: torch.tensor(np.asarray(v, np.int64), device="cuda").to(torch.int32)
    if case["op"] == "beam":
        rows = case["requests"] * case["beams"]
        # a language model's logits: most tokens far below a few that compete
        logits = 2.5 * torch.randn((rows, case["vocabulary"]), generator=gen, device="cuda", dtype=torch.float32)
        scores = -2 * torch.rand(rows, generator=gen, device="cuda") - 20
        ended = torch.rand(rows, generator=gen, device="cuda") < case["ended"]
        return {"logits": logits.to(_DTYPES[case["dtype"]]), "scores": scores, "ended": ended, "end_token": case["vocabulary"] - 7}
    ps, dtype = case["page_size"], _DTYPES[case["dtype"]]
    caches = lambda pages, layers: [[_randn(gen, (pages, case["kv_heads"], ps, case["head_dim"]), dtype) for _ in range(2)] for _ in range(layers)]
    if case["op"] == "fork":
        lengths, rows, held, sources, keep = _fork_requests(case)
        spare = len(lengths) + 5
        pages = held + spare
        ids = rng.permutation(pages).astype(np.int32)
        head = int(rng.integers(1 << 20))
        ring = np.full(pages, -1, np.int32)
        ring[(head + np.arange(spare)) % pages] = ids[held:]
        table = i32(_table_of(rows, max(map(len, rows)) + 1, ids))
        return {"lengths": i32(lengths), "sources": i32(sources), "keep": None if keep is None else i32(keep), "table": table, "table_out": table.clone(),
                "ring": i32(ring), "queue": torch.tensor([head, head + spare, 0, 0], dtype=torch.int64, device="cuda"), "caches": caches(pages, case["layers"])}
    if case["op"] == "compact":
        lengths, rows, held, pages, limit = _compact_requests(case)
        ids = rng.permutation(pages).astype(np.int32)
        head = int(rng.integers(1 << 20))
        ring = np.full(pages, -1, np.int32)
        ring[(head + np.arange(pages - held)) % pages] = ids[held:]
        table = i32(_table_of(rows, max(map(len, rows)), ids))
        return {"lengths": i32(lengths), "table": table, "table_out": table.clone(), "ring": i32(ring), "pages": pages, "limit": limit,
                "queue": torch.tensor([head, head + pages - held, 0, 0], dtype=torch.int64, device="cuda"), "caches": caches(pages, case["layers"])}
    lengths, rows, held = _shared_requests(case)
    groups = [g * case["beams"] + i for g in rng.permutation(case["groups"]) for i in range(case["beams"])]  # the prompts in any order
    lengths, rows = [lengths[r] for r in groups], [rows[r] for r in groups]
    pages = held + 5
    table = i32(_table_of(rows, max(map(len, rows)), rng.permutation(pages).astype(np.int32)))
    s = {"table": table, "positions": i32(np.asarray(lengths) - 1), "lengths": lengths}
    if case["op"] == "shared":
        hq, d = case["q_heads"], case["head_dim"]
        (s["k"], s["v"]), = caches(pages, 1)
        s["q"] = (1.5 * torch.randn((len(lengths), hq, d), generator=gen, device="cuda")).to(dtype)
        s["out"] = torch.zeros((len(lengths), hq, d), dtype=dtype, device="cuda")
        s["scale"] = 1.0 / math.sqrt(d)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        import heteromega_amd as hm

        s["hm"] = hm
        op = case["op"]
        if op == "beam":
            s["step"] = hm.BeamStep(case["requests"], case["beams"], case["k"], case["vocabulary"], "cuda")
        elif op in ("fork", "compact"):
            count, width = s["table"].shape
            s["paged"] = [hm.PagedCache(k, v) for k, v in s["caches"]]
            s["plan"] = hm.PageFork(count, width, case["page_size"], "cuda") if op == "fork" else hm.PageCompact(s["pages"], case["page_size"], "cuda")
        else:
            s["share"] = hm.SharePlan(len(s["lengths"]), case["page_size"], case["q_heads"], case["kv_heads"], "cuda", window=case["window"])
        if op == "shared":
            s["cache"] = hm.PagedCache(s["k"], s["v"])
            hm.share_plan(s["share"], s["table"], s["positions"])  # once per step, for all layers
            s["workspace"] = s["cache"].shared_attention_workspace(case["q_heads"], len(s["lengths"]))
    return s


def run(state):
    return {"beam": _run_beam, "fork": _run_fork, "compact": _run_compact, "share": _run_share, "shared": _run_shared}[state["case"]["op"]](state)


def _run_beam(s):
    c = s["case"]
    if own:
        p = s["hm"].beam_select(s["step"], s["logits"], s["scores"], ended=s["ended"], end_token=s["end_token"])
        return [p.parents, p.tokens, p.scores, p.ended]
    requests, beams, k, v = c["requests"], c["beams"], c["k"], c["vocabulary"]
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    norm = top + torch.log(torch.exp(x - top).sum(1, keepdim=True))
    score = s["scores"].double()[:, None] + (x - norm)
    token = torch.arange(v, device=x.device)
    score = torch.where(s["ended"][:, None], torch.where(token == s["end_token"], s["scores"].double()[:, None], -math.inf), score)
    best, at = torch.sort(score.view(requests, beams * v), dim=1, descending=True, stable=True)
    best, at = best[:, :k], at[:, :k]
    row = torch.arange(requests, device=x.device)[:, None] * beams + at // v
    some = best > -math.inf
    tokens = torch.where(some, at % v, -1)
    return [torch.where(some, row, -1).int(), tokens.int(), best.float(), ~some | s["ended"][row] | (tokens == s["end_token"])]


def _copy(caches, copies):
    """The first `tokens` tokens of page `source` to page `to`, for each (source, to, tokens) of `copies`."""
    for layer in caches:
        for x in layer:
            t = torch.arange(x.size(2), device=x.device)
            source, to, tokens = copies.long().unbind(1)
            for i in range(0, len(source), 4096):
                a, b = source[i:i + 4096], to[i:i + 4096]
                new = (t < tokens[i:i + 4096, None])[:, None, :, None]
                x[b] = torch.where(new, x[a], x[b])


def _run_fork(s):
    ps, caches = s["case"]["page_size"], [x for layer in s["caches"] for x in layer]
    if own:
        p = s["hm"].page_fork(s["plan"], s["sources"], s["lengths"], s["table"], s["ring"], s["queue"], keep=s["keep"], table_out=s["table_out"])
        s["hm"].copy_pages(s["paged"], p.copies)
        return [p.copies, p.lengths, p.queue, s["table_out"], s["ring"], *caches]
    table, ring, queue, n = s["table"].long(), s["ring"], s["queue"], s["lengths"].long()
    count, width = table.shape
    r, b = torch.arange(count, device=n.device), torch.arange(width, device=n.device)
    source = s["sources"].long()
    after = torch.where(source < 0, 0, n[source.clamp(min=0)])
    if s["keep"] is not None:
        after = torch.minimum(after, s["keep"].long())
    new = torch.where(b < ((after + ps - 1) // ps)[:, None], table[source.clamp(min=0)], -1)
    # a last page that is not full belongs to one request: of those that hold it, to none if one holds it in full, else to one that had it, else to the first
    last = after // ps
    part = after % ps > 0
    page = new[r, last.clamp(max=width - 1)]
    both = (new[:, last.clamp(max=width - 1)].T == page[:, None]) & part[:, None] & (page >= 0)[:, None]  # [r, other]
    whole = (both & (after[None, :] >= ((last + 1) * ps)[:, None])).any(1)
    rank = torch.where(source == r, r, count + r)
    heir = torch.where(both, rank, 2 * count).amin(1)
    fresh = part & (page >= 0) & (both.sum(1) > 1) & (whole | (heir != rank))
    order = torch.cumsum(fresh, 0)
    wanted = order[-1]
    given = ring[(queue[0] + order - 1) % ring.size(0)].long()
    new[r[fresh], last[fresh]] = given[fresh]
    # pages that nobody holds any more, by blocks and then by the first request that held them
    old = torch.where(b < ((n + ps - 1) // ps)[:, None], table, -1).T.reshape(-1)
    held = torch.zeros(int(ring.size(0)) + 1, dtype=torch.bool, device=n.device)
    held[new[new >= 0]] = True
    first = torch.full((held.numel(),), old.numel(), device=n.device).scatter_reduce_(0, old.clamp(min=0), torch.where(old >= 0, torch.arange(old.numel(), device=n.device), old.numel()), "amin")
    gone = (old >= 0) & ~held[old.clamp(min=0)] & (first[old.clamp(min=0)] == torch.arange(old.numel(), device=n.device))
    freed = old[gone]
    ring[(queue[1] + torch.arange(len(freed), device=n.device)) % ring.size(0)] = freed.int()
    s["table_out"].copy_(torch.where(new >= 0, new, s["table_out"]))
    copies = torch.full((count, 3), -1, dtype=torch.int32, device=n.device)
    copies[:int(wanted)] = torch.stack([page, given, after % ps], 1)[fresh].int()
    _copy(s["caches"], copies[:int(wanted)])
    return [copies, after.int(), torch.stack([queue[0] + wanted, queue[1] + len(freed), wanted * 0, wanted]), s["table_out"], ring, *caches]


def _run_compact(s):
    ps, caches = s["case"]["page_size"], [x for layer in s["caches"] for x in layer]
    if own:
        p = s["hm"].page_compact(s["plan"], s["limit"], s["lengths"], s["table"], s["ring"], s["queue"], table_out=s["table_out"])
        s["hm"].copy_pages(s["paged"], p.copies)
        return [p.copies, p.queue, s["table_out"], s["ring"], *caches]
    table, ring, queue, pages, limit = s["table"].long(), s["ring"], s["queue"], s["pages"], s["limit"]
    held = torch.arange(table.size(1), device=table.device) < ((s["lengths"].long() + ps - 1) // ps)[:, None]
    live = torch.zeros(pages, dtype=torch.bool, device=table.device)
    live[table[held]] = True
    source, to = torch.nonzero(live[limit:]).flatten() + limit, torch.nonzero(~live[:limit]).flatten()
    moves = len(source)
    place = torch.arange(pages, device=table.device)
    place[source] = to[:moves]
    s["table_out"].copy_(torch.where(held, place[table.clamp(min=0)], s["table_out"]))
    free = to[moves:]
    ring[(queue[0] + torch.arange(len(free), device=table.device)) % ring.size(0)] = free.int()
    copies = torch.full((max(1, pages // 2), 3), -1, dtype=torch.int32, device=table.device)
    copies[:moves] = torch.stack([source, to[:moves], torch.full_like(source, ps)], 1).int()
    _copy(s["caches"], copies[:moves])
    zero = torch.zeros_like(queue[0])
    return [copies, torch.stack([queue[0], queue[0] + len(free), zero, zero + moves]), s["table_out"], ring, *caches]


def _run_share(s):
    if own:
        return s["hm"].share_plan(s["share"], s["table"], s["positions"]).shared
    table, n = s["table"], s["positions"].long() + 1
    same = torch.cumprod((table[1:] == table[:-1]).to(torch.int32), 1).sum(1) * s["case"]["page_size"]
    shared = torch.zeros_like(s["positions"])
    shared[1:] = torch.minimum(same, torch.minimum(n[1:], n[:-1])).int()
    return shared


def _run_shared(s):
    c = s["case"]
    if own:
        return s["hm"].shared_attention(s["out"], s["q"], s["cache"], s["table"], s["positions"], s["share"], scale=s["scale"], workspace=s["workspace"])
    hq, hkv, d, ps, window = c["q_heads"], c["kv_heads"], c["head_dim"], c["page_size"], c["window"]
    out = s["out"]
    # as many rows at a time as fit 2^30 gathered elements, padded to their longest
    rows, most = out.size(0), max(s["lengths"])
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
    return {"beam": _exact_beam, "fork": _exact_fork, "compact": _exact_compact, "share": _exact_share, "shared": _exact_shared}[case["op"]](case, s)


def _exact_beam(case, s):
    requests, beams, k, v = case["requests"], case["beams"], case["k"], case["vocabulary"]
    out = [np.full((requests, k), -1, np.int32), np.full((requests, k), -1, np.int32), np.full((requests, k), -np.inf), np.ones((requests, k), bool)]
    scores, ended, end = s["scores"].cpu().double().numpy(), s["ended"].cpu().numpy(), s["end_token"]
    for q in range(requests):
        rows = range(q * beams, (q + 1) * beams)
        x = torch.log_softmax(s["logits"][q * beams:(q + 1) * beams].double(), 1)
        least = torch.topk(x, min(k, v), 1).values[:, -1]
        found = []
        for i, row in enumerate(rows):
            if ended[row]:
                found.append((-scores[row], i * v + end))
                continue
            token = torch.nonzero(x[i] >= least[i]).flatten()
            found += [(-(scores[row] + a), i * v + t) for a, t in zip(x[i, token].tolist(), token.tolist())]
        for j, (score, at) in enumerate(sorted(found)[:k]):
            row = q * beams + at // v
            out[0][q, j], out[1][q, j], out[2][q, j], out[3][q, j] = row, at % v, -score, bool(ended[row]) or at % v == end
    return [torch.from_numpy(t).cuda() for t in out]


def _exact_copies(s, copies):
    for source, to, tokens in copies:
        for layer in s["caches"]:
            for x in layer:
                x[to, :, :tokens] = x[source, :, :tokens]
    return [x for layer in s["caches"] for x in layer]


def _exact_fork(case, s):
    ps = case["page_size"]
    table, ring = s["table"].cpu().numpy(), s["ring"].cpu().numpy().copy()
    n, sources = s["lengths"].tolist(), s["sources"].tolist()
    keep = [2 ** 31 - 1] * len(n) if s["keep"] is None else s["keep"].tolist()
    head, tail = s["queue"][:2].tolist()
    count = len(n)
    after = [0 if q < 0 else min(k, n[q]) for q, k in zip(sources, keep)]
    new = [[] if q < 0 else table[q, :_pages_of(a, ps)].tolist() for q, a in zip(sources, after)]
    holders = {}
    for r in range(count):
        for b, page in enumerate(new[r]):
            holders.setdefault(page, []).append((after[r] < (b + 1) * ps, sources[r] != r, r))  # who keeps it first: those that have it in full
    copies = []
    for r in range(count):
        if after[r] % ps == 0:
            continue
        page = new[r][-1]
        first = min(holders[page])
        if not first[0] or first[2] != r:
            to = int(ring[(head + len(copies)) % len(ring)])
            copies.append((page, to, after[r] % ps))
            new[r][-1] = to
    left = {page for row in new for page in row}
    out = s["table_out"].cpu().numpy().copy()
    freed = []
    for b in range(table.shape[1]):
        for r in range(count):
            if b < _pages_of(n[r], ps) and int(table[r, b]) not in left:
                left.add(int(table[r, b]))
                freed.append(int(table[r, b]))
    for i, page in enumerate(freed):
        ring[(tail + i) % len(ring)] = page
    for r in range(count):
        out[r, :len(new[r])] = new[r]
    all_copies = np.full((count, 3), -1, np.int32)
    all_copies[:len(copies)] = np.asarray(copies, np.int32).reshape(-1, 3)
    i32 = lambda v: torch.tensor(np.asarray(v, np.int32), device="cuda")
    return [i32(all_copies), i32(after), torch.tensor([head + len(copies), tail + len(freed), 0, len(copies)], dtype=torch.int64, device="cuda"), i32(out),
            i32(ring), *_exact_copies(s, copies)]


def _exact_compact(case, s):
    ps, limit = case["page_size"], s["limit"]
    table, ring, lengths = s["table"].cpu().numpy().copy(), s["ring"].cpu().numpy().copy(), s["lengths"].tolist()
    head = int(s["queue"][0])
    live = sorted({int(p) for r, n in enumerate(lengths) for p in table[r, :_pages_of(n, ps)]})
    below = set(p for p in live if p < limit)
    to = [p for p in range(limit) if p not in below]
    moved = dict(zip([p for p in live if p >= limit], to))
    free = to[len(moved):]
    for r, n in enumerate(lengths):
        for b in range(_pages_of(n, ps)):
            table[r, b] = moved.get(int(table[r, b]), table[r, b])
    for i, p in enumerate(free):
        ring[(head + i) % len(ring)] = p
    copies = np.full((max(1, s["pages"] // 2), 3), -1, np.int32)
    for i, (a, b) in enumerate(moved.items()):
        copies[i] = a, b, ps
    i32 = lambda v: torch.tensor(np.asarray(v, np.int32), device="cuda")
    return [i32(copies), torch.tensor([head, head + len(free), 0, len(moved)], dtype=torch.int64, device="cuda"), i32(table), i32(ring),
            *_exact_copies(s, [(a, b, ps) for a, b in moved.items()])]


def _exact_share(case, s):
    table, shared = s["table"].cpu().numpy(), [0]
    for t in range(1, len(s["lengths"])):
        n = min(s["lengths"][t - 1:t + 1])
        b = 0
        while b * case["page_size"] < n and table[t, b] == table[t - 1, b]:
            b += 1
        shared.append(min(n, b * case["page_size"]))
    return torch.tensor(shared, dtype=torch.int32, device="cuda")


def _exact_shared(case, s):
    hq, hkv, d, ps = case["q_heads"], case["kv_heads"], case["head_dim"], case["page_size"]
    out = torch.zeros((len(s["lengths"]), hq, d), dtype=torch.float64, device="cuda")
    for r, n in enumerate(s["lengths"]):
        at = torch.arange(max(0, n - case["window"]) if case["window"] else 0, n, device="cuda")
        page, offset = s["table"][r].long()[at // ps], at % ps
        for h in range(hkv):
            k, v = s["k"][page, h, offset].double(), s["v"][page, h, offset].double()
            q = s["q"][r, h * (hq // hkv):(h + 1) * (hq // hkv)].double()
            out[r, h * (hq // hkv):(h + 1) * (hq // hkv)] = torch.softmax(q @ k.T * s["scale"], -1) @ v
    return out


def work(case):
    op = case["op"]
    if op == "beam":
        rows, k = case["requests"] * case["beams"], case["requests"] * case["k"]
        elements = rows * case["vocabulary"]
        # an addition, an exponential and a comparison of each logit
        return {"bytes": elements * (4 if case["dtype"] == "fp32" else 2) + 5 * rows + 13 * k, "flops": 3 * elements}
    ps = case["page_size"]
    if op in ("fork", "compact"):
        token = 2 * case["layers"] * case["kv_heads"] * case["head_dim"] * 2  # of all caches
    if op == "fork":
        lengths, _, _, sources, keep = _fork_requests(case)
        after = [0 if q < 0 else min(lengths[q], 2 ** 31 if keep is None else keep[r]) for r, q in enumerate(sources)]
        entries = sum(_pages_of(n, ps) for n in after) + sum(_pages_of(n, ps) for n in lengths)
        # the partial pages that several requests end in, but for one of each
        ends = {}
        for q, n in zip(sources, after):
            if n % ps:
                ends.setdefault(q, []).append(n % ps)
        copied = sum(sum(v) - max(v) for v in ends.values())
        return {"bytes": 4 * entries + 12 * len(lengths) + 2 * token * copied, "flops": entries}
    if op == "compact":
        lengths, _, held, pages, limit = _compact_requests(case)
        entries = sum(_pages_of(n, ps) for n in lengths)
        moved = int(held * (pages - limit) / pages)  # about: the pages lie in no order
        return {"bytes": 8 * entries + 4 * len(lengths) + 12 * moved + 4 * max(0, limit - held) + 2 * token * ps * moved, "flops": entries + pages}
    lengths, table, _ = _shared_requests(case)
    if op == "share":
        return {"bytes": 4 * sum(map(len, table)) + 8 * len(lengths), "flops": sum(map(len, table))}
    hq, hkv, d, window = case["q_heads"], case["kv_heads"], case["head_dim"], case["window"]
    seen, first = 0, {}
    for n, row in zip(lengths, table):
        begin = max(0, n - window) if window else 0
        seen += n - begin
        for b in range(begin // ps, len(row)):  # tokens of each page that some row sees
            lo, hi = first.get(row[b], (ps, 0))
            first[row[b]] = min(lo, max(0, begin - b * ps)), max(hi, min(ps, n - b * ps))
    distinct = sum(hi - lo for lo, hi in first.values())
    return {"bytes": 4 * distinct * hkv * d + 4 * len(lengths) * hq * d + 4 * len(first) + 4 * len(lengths), "flops": 4 * seen * hq * d}
