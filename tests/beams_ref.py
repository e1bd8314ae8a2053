"""The operators for several continuations of a text in plain numpy, 64 bits, from their definitions."""
import math

import numpy as np


def select(logits, scores, ended, beams, n_out, end):
    """logits [rows, vocab] as float64; scores float32 [rows]; ended int [rows] or None."""
    rows, vocab = logits.shape
    batch = rows // beams
    out = [np.full((batch, n_out), -np.inf), np.full((batch, n_out), -1), np.full((batch, n_out), -1), np.zeros((batch, n_out), int)]
    for b in range(batch):
        found = []
        for k in range(beams):
            row = b * beams + k
            base = float(scores[row])
            if ended is not None and ended[row]:
                if math.isfinite(base):
                    found.append((-base, k * vocab + end))
                continue
            x = logits[row]
            if np.isnan(x).any() or np.isposinf(x).any() or np.isneginf(x).all():
                continue
            top = x.max()
            base -= top + math.log(np.exp(x - top).sum())
            if not math.isfinite(base):
                continue
            at = np.where(np.isfinite(x))[0]
            at = at[np.argsort(-x[at], kind="stable")][:n_out]
            found += [(-(base + float(x[t])), k * vocab + int(t)) for t in at]
        for j, (s, at) in enumerate(sorted(found)[:n_out]):
            out[0][b, j], out[1][b, j], out[2][b, j] = -s, at % vocab, b * beams + at // vocab
            out[3][b, j] = int(at % vocab == end)
    return out


def row_lens(lens, width, page):
    return [int(min(max(int(n), 0), width * page)) for n in lens]


def fork(table, lens, parents, shares, free, pool, page, width, moves, free_after):
    """The outputs of a fork; `moves` and `free_after` as they were before it."""
    pages, n, rows = len(shares), len(lens), len(parents)
    lens = row_lens(lens, width, page)
    held = [-(-x // page) for x in lens]
    head, count = int(pool[0]), int(pool[1])
    shares = shares.astype(np.int64).copy()
    children = {p for p in parents if 0 <= p < n}
    for p in range(n):
        if p not in children:
            for x in table[p, :held[p]]:
                if 0 <= x < pages:
                    shares[x] -= 1
    freed = np.where(shares < 0)[0]
    shares[freed] = 0
    have = [int(x) for x in freed] + [int(x) for x in free[head:head + count]]
    after, lens_after = np.full((rows, width), -1, np.int32), np.zeros(rows, np.int32)
    moves, free_after = moves.copy(), free_after.copy()
    seen, taken, asked = set(), 0, 0
    for r, p in enumerate(parents):
        p = int(p)
        if not 0 <= p < n:
            continue
        full, rest = lens[p] // page, lens[p] % page
        row = table[p, :held[p]].copy()
        if p in seen:
            if rest:
                asked += 1
                if asked > len(have):
                    continue
                moves[taken] = (row[full], have[taken], rest, 0)
                row[full] = have[taken]
                taken += 1
            for x in row[:full]:
                if 0 <= x < pages:
                    shares[x] += 1
        seen.add(p)
        after[r, :held[p]] = row
        lens_after[r] = lens[p]
    free_after[:len(have) - taken] = have[taken:]
    return (after, lens_after, shares.astype(np.int32), free_after, np.array([0, len(have) - taken, taken, asked - taken], np.int32),
            moves)


def compact(table, lens, shares, free, pool, limit, page, width, moves, free_after):
    pages = len(shares)
    held = [-(-x // page) for x in row_lens(lens, width, page)]
    is_free = np.zeros(pages, bool)
    is_free[free[int(pool[0]):int(pool[0]) + int(pool[1])]] = True
    used = int((~is_free).sum())
    limit = min(max(limit, used), pages)
    src = [x for x in range(limit, pages) if not is_free[x]]
    dst = [x for x in range(limit) if is_free[x]][:len(src)]
    numbers, after = np.arange(pages, dtype=np.int32), np.zeros(pages, np.int32)
    numbers[src] = dst
    after[numbers[~is_free]] = shares[~is_free]
    left = np.setdiff1d(np.arange(pages), numbers[~is_free])
    moves, free_after = moves.copy(), free_after.copy()
    free_after[:len(left)] = left
    for j, x in enumerate(src):
        moves[j] = (x, dst[j], page, 0)
    table_after = np.full((len(lens), width), -1, np.int32)
    for r in range(len(lens)):
        row = table[r, :held[r]]
        table_after[r, :held[r]] = [numbers[x] if 0 <= x < pages else x for x in row]
    return table_after, after, free_after, np.array([0, len(left), len(src), 0], np.int32), numbers, moves


def copy(cache, moves, page, order):
    """cache: an array of the layout's shape; the moves carried out in place."""
    pages = cache.shape[0]
    for src, dst, tokens, _ in moves.tolist():
        if not (0 <= src < pages and 0 <= dst < pages):
            continue
        tokens = min(max(tokens, 0), page)
        if order == "HND":
            cache[dst, :, :tokens] = cache[src, :, :tokens]
        else:
            cache[dst, :tokens] = cache[src, :tokens]
    return cache
