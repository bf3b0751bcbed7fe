"""GPU: what rows share, against a row-by-row form, and the plan that attention works on: each row's segments have its keys once each."""

import numpy as np
import pytest
import torch

import branch_ref as ref

pytestmark = pytest.mark.gpu

I32 = lambda v, device: torch.tensor(np.asarray(v, np.int64), device=device).to(torch.int32)
STEP, LEVELS = 64, 3


def tree(rng, rows, ps, depth_tokens, fan):
    """(table rows, ends): requests that branch from each other at random depths, neighbours most alike."""
    table, ends, pages = [], [], 0
    for r in range(rows):
        n = int(rng.integers(1, depth_tokens + 1))
        both = 0 if r == 0 or rng.random() < 1.0 / fan else int(rng.integers(0, min(n - 1, ends[-1]) // ps + 1))
        held = -(-n // ps)
        table.append((table[-1][:both] if r else []) + list(range(pages, pages + held - both)))
        pages += held - both
        ends.append(n)
    return table, ends, pages


def as_table(rows, width, ids=None):
    t = np.full((len(rows), width), -1, np.int64)
    for r, row in enumerate(rows):
        t[r, :len(row)] = row if ids is None else ids[row]
    return t


def decode(share):
    """(segments of the narrow and the wide line, their tiles, paths [rows, 5, 8], where the runs begin) of a plan, from its memory."""
    raw = share._plan
    words = raw[(-raw.data_ptr()) % 256:].cpu().numpy()
    words = words[:len(words) // 4 * 4].view(np.int32)
    rows, head = share.rows, words[:8]
    assert head[2:5].tolist() == [rows, share.q_heads // share.kv_heads, share.kv_heads]
    lines = words[8:8 + 48 * rows].reshape(2, 3 * rows, 8)
    paths = words[8 + 48 * rows:8 + 88 * rows].reshape(5, rows, 8).transpose(1, 0, 2)
    groups, wide, narrow = head[5:8].tolist()
    starts = words[8 + 88 * rows:8 + 88 * rows + 5 * groups]
    assert 0 <= wide <= groups // 2 and (wide > 0) == (head[1] > 0) and 0 < narrow <= 4 * (groups - wide)
    counts = []
    for i in range(2):  # as many as have the line's tiles
        at = n = 0
        while at < head[i]:
            at += int(lines[i, n, 5]) * share.kv_heads * -(-int(lines[i, n, 1]) // int(lines[i, n, 7]))
            n += 1
        counts.append(n)
    return [lines[i, :counts[i]] for i in range(2)], head[:2].tolist(), paths, [starts[:narrow], starts[4 * groups:4 * groups + wide]]


def check_plan(share, table, positions, requests, ps):
    lines, tiles, paths, starts = decode(share)
    group, window = share.q_heads // share.kv_heads, share.window
    slots, begins = [], []
    for i, line in enumerate(lines):
        at, begin = 0, []
        for row0, rows, lo, hi, tile0, n, slot0, chunk in line.tolist():
            assert 0 <= row0 and rows > 0 and row0 + rows <= share.rows and 0 <= lo < hi and tile0 == at
            assert (rows * group > 32) == (i == 1) and n == -(-(hi - lo // 16 * 16) // 32)
            assert rows == 1 or lo % 16 == 0
            assert chunk >= 1 and (chunk * group <= 128 if i else chunk == rows)
            begin.append(at)
            at += n * share.kv_heads * -(-rows // chunk)
            for u in range(row0 + 1, row0 + rows):  # all rows have these pages
                q, r = (u, row0) if requests is None else (int(requests[u]), int(requests[row0]))
                np.testing.assert_array_equal(table[q, lo // ps:-(-hi // ps)], table[r, lo // ps:-(-hi // ps)])
            slots.append((slot0, rows))
        assert at == tiles[i]
        runs = max(1, len(starts[i]))
        per, longer = divmod(tiles[i], runs)
        w = np.arange(len(starts[i]))
        x = w * per + np.minimum(w, longer)
        some = x < tiles[i]
        np.testing.assert_array_equal(starts[i][some], np.searchsorted(begin, x[some], side="right") - 1)
    slots.sort()
    at = 0
    for slot0, rows in slots:
        assert slot0 == at
        at += rows
    assert at <= 5 * share.rows
    by_slot = {int(s[6]): s for line in lines for s in line}
    for t in range(share.rows):
        r = t if requests is None else int(requests[t])
        good = 0 <= r < table.shape[0] and 0 <= positions[t] < table.shape[1] * ps
        end = int(positions[t]) + 1 if good else 0
        first = max(0, end - window) if window else 0
        keys = []
        for n, line, tile, per_head, slot0, rows, row, in_chunk in paths[t].tolist():
            if n == 0:
                continue
            row0, count, lo, hi, tile0, tiles_of, _, chunk = by_slot[slot0].tolist()
            assert (n, rows, row, line) == (tiles_of, count, t - row0, int(count * group > 32)) and 0 <= row < rows and in_chunk == row % chunk
            assert tile == tile0 + row // chunk * n and per_head == n * -(-rows // chunk)
            keys.append((lo, hi))
        keys.sort()
        at = first
        for lo, hi in keys:
            assert lo == at, (t, keys, first, end)
            at = hi
        assert at == end or (end == 0 and not keys), (t, keys, first, end)
        if not window and good and paths[t, 0, 0] > 0:  # what the row keeps for itself
            assert by_slot[int(paths[t, 0, 4])][2] % STEP == 0


def run(hm, device, rows, ends, ps, heads, requests=None, window=0, positions=None):
    width = max(map(len, rows)) + 1
    table = as_table(rows, width)
    positions = np.asarray(ends) - 1 if positions is None else positions
    count = len(positions)
    share = hm.SharePlan(count, ps, *heads, device, window=window)
    print(f"share: {count} rows, pages of {ps}, {heads} heads, window {window}", flush=True)
    got = hm.share_plan(share, I32(table, device), I32(positions, device), None if requests is None else I32(requests, device)).shared
    torch.cuda.synchronize()
    np.testing.assert_array_equal(got.cpu().numpy(), ref.shared_tokens(table, positions, requests, ps))
    check_plan(share, table, positions, requests, ps)
    return share


@pytest.mark.parametrize("rows", [1, 2, 3, 16, 63, 64, 65, 300, 1024])
@pytest.mark.parametrize("ps,depth", [(16, 40), (16, 3000), (64, 2000), (256, 5000)])
def test_trees(hm, device, rows, ps, depth):
    rng = np.random.default_rng([rows, ps, depth])
    for fan, heads, window in ((2, (8, 2), 0), (50, (32, 8), 0), (50, (24, 1), 0), (8, (16, 16), 100), (1000, (40, 8), 700), (30, (128, 1), 0)):
        table, ends, _ = tree(rng, rows, ps, depth, fan)
        run(hm, device, table, ends, ps, heads, window=window)


@pytest.mark.parametrize("rows", [1025, 2048, 4095, 4096])
def test_many_rows(hm, device, rows):
    rng = np.random.default_rng(rows)
    for fan in (3, 100):
        table, ends, _ = tree(rng, rows, 16, 700, fan)
        run(hm, device, table, ends, 16, (8, 2))
    run(hm, device, [list(range(40))] * rows, [640] * rows, 16, (8, 2))


def test_stairs_deeper_than_the_levels(hm, device):
    # row t shares all but its last pages with the one before: a segment within a segment, many times
    for rows in (4, 5, 30, 200):
        for step in (4, 1, 9):
            up = [list(range(step * (t + 1))) for t in range(rows)]
            ends = [16 * len(r) for r in up]
            for order in (up, up[::-1], up[::2] + up[1::2][::-1]):
                e = [16 * len(r) for r in order]
                run(hm, device, order, e, 16, (8, 2))
                run(hm, device, order, e, 16, (8, 2), window=200)
            assert ends[-1] == 16 * step * rows


def test_nested_prompts(hm, device):
    rows, pages = [], 100
    for _ in range(6):
        prompt = list(range(pages, pages + 30))
        pages += 30
        for _ in range(3):
            inner = list(range(pages, pages + 8))
            pages += 8
            for _ in range(4):
                rows.append(list(range(100))[:64] + prompt + inner + [pages])
                pages += 1
    share = run(hm, device, rows, [16 * len(r) - 5 for r in rows], 16, (32, 8))
    lines, _, paths, _ = decode(share)
    assert (paths[:, 2:, 0] > 0).all() and len(lines[1]) == 1 + 6 and len(lines[0]) == 18 + 72


def test_rows_of_requests_padding_and_bad_rows(hm, device):
    rng = np.random.default_rng(5)
    table, ends, _ = tree(rng, 20, 16, 900, 40)
    width = max(map(len, table)) + 1
    requests = np.array([0, 0, 0, 1, 1, 2, -1, 3, 3, 25, 4, 4, 5, 2 ** 30, 6, 7, -1, -1])
    positions = np.array([min(ends[r], 500 - i) - 1 if 0 <= r < 20 else 5 for i, r in enumerate(requests)])
    positions[4], positions[11], positions[12] = -1, width * 16, -7
    run(hm, device, table, ends, 16, (8, 2), requests=requests, positions=positions)
    run(hm, device, table, ends, 16, (8, 2), requests=requests, positions=positions, window=64)
    none = run(hm, device, table, ends, 16, (8, 2), positions=np.full(20, -1))
    assert decode(none)[1] == [0, 0]


def test_windows_over_rows_of_different_lengths(hm, device):
    rows = [list(range(60)) + [100 + 10 * t + i for i in range(1 + t % 7)] for t in range(40)]
    ends = [16 * len(r) - (5 * t) % 16 for t, r in enumerate(rows)]
    for window in (1, 16, 60, 64, 130, 500, 960, 100000):
        run(hm, device, rows, ends, 16, (8, 2), window=window)


def test_calls_that_python_refuses(hm, device):
    i = lambda *s: torch.zeros(s, dtype=torch.int32, device=device)
    share = hm.SharePlan(3, 16, 8, 2, device)
    for args in ((i(3, 4).long(), i(3)), (i(2, 4), i(3)), (i(3, 4), i(2)), (i(3, 4), i(3).long()), (i(3, 4), i(3), i(2))):
        with pytest.raises(ValueError):
            hm.share_plan(share, *args)
