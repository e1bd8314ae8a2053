"""Decode a few tokens for several requests over a paged key-value cache.

The state is declared and materialised the way a program declares it (a
``page_table`` and two ``paged_tensor`` entries); then every step runs, on the
device and without waiting for it:

  1. pages, slots and positions of the step's new tokens  (PageAssigner.assign)
  2. rotary positions, keys and values into their slots   (RopeAppend.run)
  3. attention of each request's newest token             (PagedAttention.run)

The first step takes the requests' prompts, the following ones a token each.
Queries, keys and values are synthetic (a model would compute them); every
step's result is compared with attention computed in float64 on the host.

    python examples/paged_decode.py [--steps 4] [--cache bf16|f8_e4m3]
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import numpy as np

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from manifesto_b200 import COMPAT_OCP, CUDABackend, DeviceBuffer, Stream, paged, state, synthetic  # noqa: E402
from manifesto_b200._abi import call  # noqa: E402
from manifesto_b200.dtype import DType, parse  # noqa: E402


def bf16_values(bits: np.ndarray) -> np.ndarray:
    return (bits.astype(np.uint32) << 16).view(np.float32)


def turned(x: np.ndarray, positions: np.ndarray, inv_freq: np.ndarray) -> np.ndarray:
    """Rotary positions in float64, half layout, of [tokens, heads, dim]."""
    half = x.shape[-1] // 2
    angle = positions[:, None].astype(np.float64) * inv_freq.astype(np.float64)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = x[..., :half].astype(np.float64), x[..., half:].astype(np.float64)
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


def attended(q: np.ndarray, k: np.ndarray, v: np.ndarray) -> np.ndarray:
    """softmax(q k / sqrt(dim)) v in float64: q [heads, dim], k and v [tokens, kv_heads, dim]."""
    group, out = q.shape[0] // k.shape[1], np.zeros(q.shape)
    for h in range(q.shape[0]):
        s = k[:, h // group] @ q[h] / math.sqrt(q.shape[1])
        p = np.exp(s - s.max())
        out[h] = p @ v[:, h // group] / p.sum()
    return out


def run(prompts=(37, 5, 64, 1), steps: int = 4, heads: int = 8, kv_heads: int = 2, dim: int = 64, page: int = 16,
        cache_dtype: str = "bf16", seed: int = 11) -> list[float]:
    """Decodes `steps` tokens after the prompts; returns each step's largest difference from the float64 result."""
    backend, stream = CUDABackend(0), Stream()
    n, code = len(prompts), parse(cache_dtype)
    longest = max(prompts) + steps
    width = -(-longest // page)
    pages = sum(-(-(p + steps) // page) for p in prompts) + 1

    # state, as a program declares it: a page table and the cache's two paged tensors
    layout = paged.CacheLayout(pages, page, kv_heads, dim, code)
    store = state.StateStore({"table": state.PageTableState(n * width), "keys": state.PagedTensorState(list(layout.shape)),
                              "values": state.PagedTensorState(list(layout.shape))})
    state.materialize_state_tensors(store, [state.StateDeclaration("table", "page_table"),
                                            state.StateDeclaration("keys", "paged_tensor", config={"dtype": cache_dtype}),
                                            state.StateDeclaration("values", "paged_tensor", config={"dtype": cache_dtype})],
                                    backend, DType.BFLOAT16)
    table, keys, values = (store.get(name)[0].storage.dispatch_pointer() for name in ("table", "keys", "values"))

    def device(a: np.ndarray) -> DeviceBuffer:
        b = DeviceBuffer(max(a.nbytes, 4))
        b.upload(a)
        return b

    rng = np.random.default_rng(seed)
    inv_freq = paged.rope_frequencies(dim)
    scale = np.full(2 * kv_heads, 0.0625, np.float32)  # of an FP8 cache's codes: powers of two
    most = sum(prompts)
    width_qkv = (heads + 2 * kv_heads) * dim
    free, freq, scales = device(rng.permutation(pages).astype(np.int32)), device(inv_freq), device(scale)
    lens = [device(np.zeros(n, np.int32)) for _ in range(2)]
    pool = [device(np.array([0, pages], np.int32)), device(np.zeros(4, np.int32))]
    fresh, slots, positions, owner, starts = (DeviceBuffer(s) for s in (4 * n, 8 * most, 4 * most, 4 * most, 4 * (n + 1)))
    qkv, q_out, q_last, out = (DeviceBuffer(2 * s) for s in (most * width_qkv, most * heads * dim, n * heads * dim,
                                                             n * heads * dim))
    fp8 = code.size == 1
    rope = paged.Rope(freq.ptr, DType.BFLOAT16, dim)
    assign = paged.PageAssigner(page, width)
    append = paged.RopeAppend(rope, layout, heads, k_scale_inv=scales.ptr if fp8 else 0,
                              v_scale_inv=scales.ptr + 4 * kv_heads if fp8 else 0, compat=COMPAT_OCP, token_stride=width_qkv)
    attend = paged.PagedAttention(layout, heads, DType.BFLOAT16, width, k_scale_inv=scales.ptr if fp8 else 0,
                                  v_scale_inv=scales.ptr + 4 * kv_heads if fp8 else 0)

    past = [(np.zeros((0, kv_heads, dim)), np.zeros((0, kv_heads, dim))) for _ in range(n)]
    have, worst = np.zeros(n, np.int64), []
    for step in range(steps + 1):
        new = np.array(prompts if step == 0 else [1] * n, np.int32)
        tokens = int(new.sum())
        bits = synthetic.normal_bf16(seed + 100 + step, tokens * width_qkv)
        fresh.upload(new, stream)
        qkv.upload(bits, stream)

        assign.assign(lens[0].ptr, fresh.ptr, n, table, free.ptr, pool[0].ptr, tokens, slots.ptr, positions.ptr, owner.ptr,
                      starts.ptr, lens[1].ptr, pool[1].ptr, stream)
        append.run(qkv.ptr, qkv.ptr + 2 * heads * dim, qkv.ptr + 2 * (heads + kv_heads) * dim, q_out.ptr, keys, values,
                   positions.ptr, slots.ptr, tokens, stream)
        ends = np.cumsum(new) - 1
        queries = q_out.ptr
        if step == 0:  # of a prompt, the newest token's
            row, queries = 2 * heads * dim, q_last.ptr
            for r, at in enumerate(ends):
                call("mf_memcpy_d2d_async", q_last.ptr + r * row, q_out.ptr + int(at) * row, row, stream.handle)
        attend.run(queries, keys, values, table, lens[1].ptr, n, out.ptr, stream=stream)
        stream.sync()

        got = bf16_values(out.download(2 * n * heads * dim).view(np.uint16)).reshape(n, heads, dim)
        lens.reverse()
        pool.reverse()

        # the same in float64 from the same inputs
        x = bf16_values(bits).reshape(tokens, heads + 2 * kv_heads, dim)
        off = 0.0
        for r in range(n):
            rows = slice(int(ends[r]) + 1 - int(new[r]), int(ends[r]) + 1)
            at = have[r] + np.arange(new[r])
            k, v = past[r]
            past[r] = (np.concatenate([k, turned(x[rows, heads:heads + kv_heads], at, inv_freq)]),
                       np.concatenate([v, x[rows, heads + kv_heads:].astype(np.float64)]))
            q = turned(x[rows, :heads], at, inv_freq)[-1]
            off = max(off, float(np.abs(attended(q, *past[r]) - got[r]).max()))
        have += new
        worst.append(off)
    attend.close()
    for b in (free, freq, scales, *lens, *pool, fresh, slots, positions, owner, starts, qkv, q_out, q_last, out):
        b.free()
    for name in ("table", "keys", "values"):
        store.get(name)[0].storage.close()
    stream.close()
    return worst


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=4)
    ap.add_argument("--cache", default="bf16", choices=["bf16", "f8_e4m3", "f8_e5m2"])
    args = ap.parse_args()
    for step, off in enumerate(run(steps=args.steps, cache_dtype=args.cache)):
        print(f"step {step}: largest difference from float64 attention {off:.4f}")
    return 0


if __name__ == "__main__":
    sys.exit(main())
