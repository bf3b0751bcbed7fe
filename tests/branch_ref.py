"""Plain forms of the operators for requests that branch, request by request on the CPU, for their tests."""

import math

import numpy as np
import torch

from attention_ref import pages_of


def fork(sources, keep, lengths, table, ring, head, tail, page_size, table_out=None):
    """page_fork: a dict of int64 arrays (copies, lengths, queue, table, ring)."""
    table, ring = np.array(table, np.int64), np.array(ring, np.int64)
    out = table.copy() if table_out is None else np.array(table_out, np.int64)
    count, width = table.shape
    n, s = [int(v) for v in lengths], [int(v) for v in sources]
    k = [2 ** 31 - 1] * count if keep is None else [int(v) for v in keep]
    size = len(ring)
    bad = any(not 0 <= v <= width * page_size for v in n) or any(v >= count for v in s) or any(v < 0 for v in k)
    copies = np.full((count, 3), -1, np.int64)

    def refused(wanted):
        for r in range(count):  # another table gets what the old one has
            held = pages_of(min(max(n[r], 0), width * page_size), page_size)
            if table_out is not None:
                out[r, :held] = table[r, :held]
        return {"copies": copies, "lengths": np.array(n), "queue": np.array([head, tail, 1, wanted]), "table": out, "ring": ring}

    if bad:
        return refused(0)
    after = [0 if s[r] < 0 else min(k[r], n[s[r]]) for r in range(count)]
    new = [[int(v) for v in table[s[r], :pages_of(after[r], page_size)]] for r in range(count)]
    old = [[int(v) for v in table[r, :pages_of(n[r], page_size)]] for r in range(count)]
    by_page = {}
    for r in range(count):
        for b, page in enumerate(new[r]):
            by_page.setdefault((b, page), []).append(r)
    wanted = []  # (request, page)
    for r in range(count):
        if after[r] % page_size == 0 or new[r][-1] < 0:
            continue
        b, page = len(new[r]) - 1, new[r][-1]
        holders = by_page[b, page]
        full = [t for t in holders if after[t] >= (b + 1) * page_size]
        stay = [t for t in holders if s[t] == t]
        heir = None if full else (stay or holders)[0]
        if heir != r:
            wanted.append((r, page))
    left = min(max(tail - head, 0), size)
    held = set()
    fresh = {r: i for i, (r, _) in enumerate(wanted)}
    for r in range(count):
        held.update(p for b, p in enumerate(new[r]) if not (r in fresh and b == len(new[r]) - 1))
    freed = []
    for b in range(width):
        for r in range(count):
            if b < len(old[r]) and old[r][b] >= 0 and old[r][b] not in held:
                held.add(old[r][b])
                freed.append(old[r][b])
    if len(wanted) > left or left + len(freed) > size:
        return refused(len(wanted))
    given = [int(ring[(head + i) % size]) for i in range(len(wanted))]
    for i, (r, page) in enumerate(wanted):
        copies[i] = page, given[i], after[r] % page_size
        new[r][-1] = given[i]
    for i, page in enumerate(freed):
        ring[(tail + i) % size] = page
    for r in range(count):
        out[r, :len(new[r])] = new[r]
    return {"copies": copies, "lengths": np.array(after), "queue": np.array([head + len(wanted), tail + len(freed), 0, len(wanted)]), "table": out, "ring": ring}


def compact(pages, limit, lengths, table, ring, head, tail, page_size, most, table_out=None):
    """page_compact: a dict of int64 arrays (copies [most, 3], queue, table, ring)."""
    table, ring = np.array(table, np.int64), np.array(ring, np.int64)
    out = table.copy() if table_out is None else np.array(table_out, np.int64)
    width = table.shape[1]
    held = [pages_of(min(max(int(n), 0), width * page_size), page_size) for n in lengths]
    used = sorted({int(p) for r, h in enumerate(held) for p in table[r, :h] if 0 <= p < pages})
    copies = np.full((most, 3), -1, np.int64)
    refused = len(used) > limit or limit - len(used) > len(ring)
    below = {p for p in used if p < limit}
    to = [p for p in range(limit) if p not in below]
    moved = {} if refused else dict(zip([p for p in used if p >= limit], to))
    for r, h in enumerate(held):
        for b in range(h):
            out[r, b] = moved.get(int(table[r, b]), table[r, b])
    if refused:
        return {"copies": copies, "queue": np.array([head, tail, 1, 0]), "table": out, "ring": ring}
    for i, (a, b) in enumerate(moved.items()):
        copies[i] = a, b, page_size
    free = to[len(moved):]
    for i, p in enumerate(free):
        ring[(head + i) % len(ring)] = p
    return {"copies": copies, "queue": np.array([head, head + len(free), 0, len(moved)]), "table": out, "ring": ring}


def shared_tokens(table, positions, requests, page_size):
    """share_plan's shared, row by row."""
    count, width = table.shape

    def end(t):
        r = t if requests is None else int(requests[t])
        return (r, int(positions[t]) + 1) if 0 <= r < count and 0 <= positions[t] < width * page_size else (r, 0)

    out = [0]
    for t in range(1, len(positions)):
        (r, n), (q, m) = end(t), end(t - 1)
        most = min(n, m)
        b = 0
        while b * page_size < most and table[r, b] == table[q, b]:
            b += 1
        out.append(min(most, b * page_size))
    return np.array(out[:len(positions)])


def beam(logits, scores, ended, end_token, beams, k):
    """beam_select in float64, row by row: parents, tokens, scores, ended [requests, k]."""
    rows, v = logits.shape
    requests = rows // beams
    parents, tokens, best, done = (np.full((requests, k), -1, np.int64), np.full((requests, k), -1, np.int64), np.full((requests, k), -np.inf),
                                   np.ones((requests, k), bool))
    x = logits.double().cpu()
    for q in range(requests):
        found = []
        for i in range(beams):
            row = q * beams + i
            score = float(scores[row])
            if not math.isfinite(score):
                continue
            if ended is not None and ended[row]:
                found.append((-score, i, 0.0, end_token))
                continue
            y = x[row]
            if torch.isnan(y).any() or (y == math.inf).any() or (y == -math.inf).all():
                continue
            a = score + (y - torch.logsumexp(y, 0))
            # the row's k best, equal ones by their token; by their logits, which tell more apart than their rounded scores
            order = torch.sort(y, descending=True, stable=True).indices[:k]
            found += [(-float(a[t]), i, -float(y[t]), int(t)) for t in order if y[t] > -math.inf]
        for j, (score, beam, _, token) in enumerate(sorted(found)[:k]):
            row = q * beams + beam
            parents[q, j], tokens[q, j], best[q, j] = row, token, -score
            done[q, j] = bool(ended is not None and ended[row]) or token == end_token
    return parents, tokens, best, done
