"""Plain 64-bit forms of the paged-cache operators, from their formulas (numpy, a token or request at a time)."""
from __future__ import annotations

import math

import numpy as np

from manifesto_b200 import synthetic
from manifesto_b200.dtype import DType
from oracle import ref

FP8 = (DType.FLOAT8_E4M3, DType.FLOAT8_E5M2)
# half the distance of neighbouring values over the value, at most
UNIT = {DType.BFLOAT16: 2.0 ** -8, DType.FLOAT16: 2.0 ** -11, DType.FLOAT32: 2.0 ** -24,
        DType.FLOAT8_E4M3: 2.0 ** -4, DType.FLOAT8_E5M2: 2.0 ** -3}


def codes(x: np.ndarray, dtype: DType, compat: int = 1) -> np.ndarray:
    """Storage codes of float32 values (the oracle's encoders)."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == DType.FLOAT32:
        return x.view(np.uint32)
    out = ref.convert(x.reshape(-1), ref.F32, int(dtype), compat=compat)
    return np.ascontiguousarray(out).view(dtype.storage_numpy).reshape(x.shape)


def values(c: np.ndarray, dtype: DType) -> np.ndarray:
    """float64 values of storage codes."""
    c = np.ascontiguousarray(c).view(dtype.storage_numpy)
    if dtype == DType.FLOAT32:
        return c.view(np.float32).astype(np.float64)
    return np.ascontiguousarray(ref.convert(c.reshape(-1), int(dtype), ref.F32)).view(np.float32).reshape(c.shape).astype(np.float64)


def normal(seed: int, shape, dtype: DType, sigma: float = 1.0) -> np.ndarray:
    n = int(np.prod(shape))
    return codes(synthetic.normal_f32(seed, n, 0.0, sigma), dtype).reshape(shape)


def assign(lens, new, table, free, pool, page, tokens, max_pages):
    """(table, slots, positions, owner, starts, lens_after, pool_after), a request at a time."""
    table = table.copy()
    slots, positions, owner = (np.full(tokens, fill, t) for fill, t in ((-1, np.int64), (0, np.int32), (-1, np.int32)))
    starts, after = [0], []
    wanted = taken = refused = 0
    for r, (n, m) in enumerate(zip(lens, new)):
        n, m = max(int(n), 0), max(int(m), 0)
        held, all_pages = -(-n // page), -(-(n + m) // page)
        room = all_pages <= max_pages
        need = all_pages - held if room else 0
        fits = room and (need == 0 or wanted + need <= pool[1])
        if fits:
            for i in range(need):
                table[r, held + i] = free[pool[0] + wanted + i]
            if need:
                taken = wanted + need
        refused += not fits
        wanted += need
        for t in range(m):
            i = starts[-1] + t
            if i < tokens:
                positions[i], owner[i] = n + t, r
                slots[i] = int(table[r, (n + t) // page]) * page + (n + t) % page if fits else -1
        starts.append(starts[-1] + m)
        after.append(n + m if fits else n)
    return (table, slots, positions, owner, np.array(starts, np.int32), np.array(after, np.int32),
            np.array([pool[0] + taken, pool[1] - taken, starts[-1], refused], np.int32))


def rope(x: np.ndarray, positions, inv_freq, rot: int, layout: str, magnitude: float, inverse: bool = False) -> np.ndarray:
    """[tokens, heads, dim] float64, each pair turned by position * frequency."""
    y = x.astype(np.float64).copy()
    angle = np.asarray(positions, np.float64)[:, None] * np.asarray(inv_freq, np.float64)[None]
    c, s = magnitude * np.cos(angle)[:, None], magnitude * np.sin(angle)[:, None] * (-1 if inverse else 1)
    i = np.arange(rot // 2)
    ia, ib = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
    a, b = x[..., ia].astype(np.float64), x[..., ib].astype(np.float64)
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    return y


def rope_bound(x: np.ndarray, positions, rot: int, layout: str, magnitude: float, dtype: DType, want: np.ndarray) -> np.ndarray:
    """How far a float32 evaluation rounded to dtype may be off.

    The fraction of a turn is rounded to float32 (an angle error of 2 pi 2^-25 = 1.9e-7), cosine and sine are good to
    2 units in the last place (2.4e-7), times the magnitude, two products and a sum: 6e-7 of |a| + |b| together.  The angle's float64 product
    has two roundings here and one in rope() above, 1.5 * 2^-52 of a frequency of 1 times the position."""
    i = np.arange(rot // 2)
    ia, ib = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
    room = np.zeros(x.shape)
    both = (np.abs(x[..., ia]) + np.abs(x[..., ib])) * abs(magnitude)
    both = both * (6e-7 + 1.5 * 2.0 ** -52 * np.abs(np.asarray(positions, np.float64)))[:, None, None]
    room[..., ia] = room[..., ib] = both
    return room + UNIT[dtype] * 1.01 * np.abs(want) + 1e-30 + (6.2e-8 if dtype == DType.FLOAT16 else 0.0)


def attention(q, k, v, slopes, scale, softcap, window, group):
    """One request: q [heads, dim], k and v [tokens, kv_heads, dim], all float64.  Returns out, lse and the mean |v|
    under the weights (what an error of the weights is multiplied by)."""
    heads, n = q.shape[0], k.shape[0]
    first = max(0, n - window) if window else 0
    out, size, lse = np.zeros_like(q), np.zeros_like(q), np.full(heads, -np.inf)
    if n == first:
        return out, lse, size
    at = np.arange(first, n)
    for h in range(heads):
        kh, vh = k[first:, h // group], v[first:, h // group]
        s = scale * (kh @ q[h])
        if softcap > 0:
            s = softcap * np.tanh(s / softcap)
        if slopes is not None:
            s = s + float(slopes[h]) * (at - (n - 1))
        top = s.max()
        if top == -np.inf:
            continue
        p = np.exp(s - top)
        total = p.sum()
        lse[h] = top + math.log(total)
        out[h], size[h] = p @ vh / total, p @ np.abs(vh) / total
    return out, lse, size
