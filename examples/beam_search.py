"""Beam search for a few prompts over a paged key-value cache that the beams share.

Every step runs, on the device:

  1. pages, slots and positions of the beams' new tokens      (PageAssigner.assign)
  2. rotary positions, keys and values into their slots       (RopeAppend.run)
  3. attention; a prompt's whole pages are read once for its beams (PrefixAttention.run)
  4. the best continuations of each prompt                    (BeamSelect.run)
  5. page tables reordered by the chosen parents              (PageBook.fork)
  6. the partly filled pages that beams no longer share       (PageCopy.run)

and in the middle of the way the pages in use are moved together (PageBook.compact).
Queries, keys, values and logits are synthetic (a model would compute them; here the logits
are a fixed projection of the attention's result, made on the host); every step's attention is
compared with float64 attention over each beam's own history, and its choice with the host's.

    python examples/beam_search.py [--steps 6] [--beams 4] [--cache bf16|f8_e4m3]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

import numpy as np

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from examples.paged_decode import attended, bf16_values, turned  # noqa: E402
from manifesto_b200 import COMPAT_OCP, CUDABackend, DeviceBuffer, Stream, beams as beam, paged, synthetic  # noqa: E402
from manifesto_b200._abi import call  # noqa: E402
from manifesto_b200.dtype import DType, parse  # noqa: E402


def chosen(logits: np.ndarray, scores: np.ndarray, beams: int):
    """The `beams` best of each prompt in float64, ties to the lowest beam and token: scores, tokens, parents."""
    x = logits.astype(np.float64)
    top = x.max(1, keepdims=True)
    all_scores = scores.astype(np.float64)[:, None] + x - top - np.log(np.exp(x - top).sum(1, keepdims=True))
    out = []
    for p in range(len(scores) // beams):
        flat = all_scores[p * beams:(p + 1) * beams].reshape(-1)
        at = np.argsort(-flat, kind="stable")[:beams]
        out += [(flat[i], i % x.shape[1], p * beams + i // x.shape[1]) for i in at]
    return [np.array(v) for v in zip(*out)]


def run(prompts=(37, 5, 64), beams: int = 4, steps: int = 6, heads: int = 8, kv_heads: int = 2, dim: int = 64, page: int = 16,
        vocab: int = 501, cache_dtype: str = "bf16", seed: int = 23) -> list[float]:
    """`steps` tokens for every prompt; returns each step's largest difference of the attention from float64."""
    CUDABackend(0)
    stream, code = Stream(), parse(cache_dtype)
    n, rows = len(prompts), len(prompts) * beams
    width = -(-(max(prompts) + steps + 1) // page)
    pages = rows * width + 5
    rng = np.random.default_rng(seed)

    def device(a: np.ndarray) -> DeviceBuffer:
        b = DeviceBuffer(max(a.nbytes, 16))
        b.upload(np.ascontiguousarray(a))
        return b

    def twice(a: np.ndarray) -> list[DeviceBuffer]:
        return [device(a), device(a)]

    layout = paged.CacheLayout(pages, page, kv_heads, dim, code)
    fp8, per_token = code.size == 1, (heads + 2 * kv_heads) * dim
    cache = [device(np.zeros(int(np.prod(layout.shape)) * code.size, np.uint8)) for _ in range(2)]
    scale = device(np.full(2 * kv_heads, 0.0625, np.float32))  # of an FP8 cache's codes: powers of two
    scales = {"k_scale_inv": scale.ptr if fp8 else 0, "v_scale_inv": scale.ptr + 4 * kv_heads if fp8 else 0}
    freq = device(paged.rope_frequencies(dim))

    # the books: [0] is the state, [1] where the next one goes
    table, lens = twice(np.full((rows, width), -1, np.int32)), twice(np.zeros(rows, np.int32))
    shares, free = twice(np.zeros(pages, np.int32)), twice(rng.permutation(pages).astype(np.int32))
    pool = twice(np.array([0, pages, 0, 0], np.int32))
    moves, numbers = device(np.zeros((max(rows, pages // 2), 4), np.int32)), device(np.zeros(pages, np.int32))
    most = sum(prompts) + rows
    slots, positions, owner = (device(np.zeros(s * most, np.uint8)) for s in (8, 4, 4))
    begins, fresh = device(np.zeros(rows + 1, np.int32)), device(np.zeros(rows, np.int32))
    qkv, q = (device(np.zeros(most * w, np.uint16)) for w in (per_token, heads * dim))
    queries, out = (device(np.zeros(rows * heads * dim, np.uint16)) for _ in range(2))
    lse = device(np.zeros(rows * heads, np.float32))
    # the beams of a prompt are a group; they share its whole pages
    starts = device(np.arange(0, rows + 1, beams, dtype=np.int32))
    shared = device(np.array([p // page * page for p in prompts], np.int32))
    # of the beams only the first is in use before the first choice
    scores = twice(np.where(np.arange(rows) % beams == 0, 0.0, -np.inf).astype(np.float32))
    logits = device(np.zeros((rows, vocab), np.float32))
    tokens, parents = device(np.zeros(rows, np.int32)), device(np.zeros(rows, np.int32))

    assign = paged.PageAssigner(page, width)
    append = paged.RopeAppend(paged.Rope(freq.ptr, DType.BFLOAT16, dim), layout, heads, compat=COMPAT_OCP, token_stride=per_token, **scales)
    # shared always: prompts as short as these would be read beam by beam
    attend = paged.PrefixAttention(layout, heads, DType.BFLOAT16, width, rows, always=True, **scales)
    select = beam.BeamSelect(DType.FLOAT32, vocab, beams, beams, n)
    book = paged.PageBook(page, width, pages, rows)
    copy = paged.PageCopy(layout, [c.ptr for c in cache])

    projection = rng.normal(0, 0.4, (heads * dim, vocab))
    none = np.zeros((0, kv_heads, dim))
    past = [(none, none) for _ in range(rows)]
    have, worst = np.zeros(rows, np.int64), []
    for step in range(steps + 1):
        new = np.array([prompts[r // beams] if r % beams == 0 else 0 for r in range(rows)] if step == 0 else [1] * rows, np.int32)
        total = int(new.sum())
        bits = synthetic.normal_bf16(seed + 100 + step, total * per_token)
        fresh.upload(new, stream)
        qkv.upload(bits, stream)
        assign.assign(lens[0].ptr, fresh.ptr, rows, table[0].ptr, free[0].ptr, pool[0].ptr, total, slots.ptr, positions.ptr, owner.ptr,
                      begins.ptr, lens[1].ptr, pool[1].ptr, stream)
        lens.reverse()
        pool.reverse()
        append.run(qkv.ptr, qkv.ptr + 2 * heads * dim, qkv.ptr + 2 * (heads + kv_heads) * dim, q.ptr, cache[0].ptr, cache[1].ptr,
                   positions.ptr, slots.ptr, total, stream)
        ends = np.cumsum(new) - 1
        row = 2 * heads * dim
        for r in range(rows):  # the newest token of each row
            if new[r]:
                call("mf_memcpy_d2d_async", queries.ptr + r * row, q.ptr + int(ends[r]) * row, row, stream.handle)
        attend.run(queries.ptr, cache[0].ptr, cache[1].ptr, table[0].ptr, lens[0].ptr, rows, starts.ptr, shared.ptr, n if step else 0,
                   out.ptr, lse.ptr, stream)
        stream.sync()
        got = bf16_values(out.download(rows * row).view(np.uint16)).reshape(rows, heads, dim)

        # the same in float64 over each beam's own history
        x, inv_freq = bf16_values(bits).reshape(total, heads + 2 * kv_heads, dim), paged.rope_frequencies(dim)
        off = 0.0
        for r in range(rows):
            if not new[r]:
                continue
            mine = slice(int(ends[r]) + 1 - int(new[r]), int(ends[r]) + 1)
            at = have[r] + np.arange(new[r])
            past[r] = (np.concatenate([past[r][0], turned(x[mine, heads:heads + kv_heads], at, inv_freq)]),
                       np.concatenate([past[r][1], x[mine, heads + kv_heads:].astype(np.float64)]))
            off = max(off, float(np.abs(attended(turned(x[mine, :heads], at, inv_freq)[-1], *past[r]) - got[r]).max()))
        have += new
        worst.append(off)
        if step == steps:
            break

        made = (got.reshape(rows, -1) @ projection).astype(np.float32)
        want = chosen(made, scores[0].download(4 * rows).view(np.float32), beams)
        logits.upload(made, stream)
        select.run(logits.ptr, scores[0].ptr, n, scores[1].ptr, tokens.ptr, parents.ptr, stream=stream)
        book.fork(table[0].ptr, lens[0].ptr, rows, parents.ptr, rows, shares[0].ptr, free[0].ptr, pool[0].ptr, table[1].ptr, lens[1].ptr,
                  shares[1].ptr, free[1].ptr, pool[1].ptr, moves.ptr, stream)
        for both in (scores, table, lens, shares, free, pool):
            both.reverse()
        copy.run(moves.ptr, rows, count=pool[0].ptr + 8, stream=stream)
        if step == steps // 2:
            book.compact(table[0].ptr, lens[0].ptr, rows, shares[0].ptr, free[0].ptr, pool[0].ptr, 0, table[1].ptr, shares[1].ptr,
                         free[1].ptr, pool[1].ptr, numbers.ptr, moves.ptr, stream)
            for both in (table, shares, free, pool):
                both.reverse()
            copy.run(moves.ptr, pages // 2, count=pool[0].ptr + 8, stream=stream)
        stream.sync()
        picked = parents.download(4 * rows).view(np.int32)
        if not (np.array_equal(picked, want[2]) and np.array_equal(tokens.download(4 * rows).view(np.int32), want[1])):
            raise RuntimeError(f"step {step}: chose other continuations than the host")
        if pool[0].download(16).view(np.int32)[3]:
            raise RuntimeError(f"step {step}: the pool ran out of pages")
        past, have = [past[p] for p in picked], have[picked]

    # every beam ends: all pages come back
    parents.upload(np.full(rows, -1, np.int32), stream)
    book.fork(table[0].ptr, lens[0].ptr, rows, parents.ptr, rows, shares[0].ptr, free[0].ptr, pool[0].ptr, table[1].ptr, lens[1].ptr,
              shares[1].ptr, free[1].ptr, pool[1].ptr, moves.ptr, stream)
    stream.sync()
    if pool[1].download(16).view(np.int32)[1] != pages:
        raise RuntimeError("pages were lost")
    for h in (attend, select, book):
        h.close()
    for b in (*cache, scale, freq, *table, *lens, *shares, *free, *pool, moves, numbers, slots, positions, owner, begins, fresh, qkv, q,
              queries, out, lse, starts, shared, *scores, logits, tokens, parents):
        b.free()
    stream.close()
    return worst


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=6)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--cache", default="bf16", choices=["bf16", "f8_e4m3", "f8_e5m2"])
    args = ap.parse_args()
    for step, off in enumerate(run(steps=args.steps, beams=args.beams, cache_dtype=args.cache)):
        print(f"step {step}: largest difference from float64 attention {off:.4f}")
    return 0


if __name__ == "__main__":
    sys.exit(main())
