"""The paged-cache operators on the GPU against plain 64-bit forms, at the sizes and masks where they can go wrong."""
import ctypes
import math

import numpy as np
import pytest

from manifesto_b200 import DeviceBuffer, Stream, paged, sync_device, synthetic
from manifesto_b200._abi import call
from manifesto_b200.dtype import DType
from manifesto_b200.errors import (DeviceStickyError, DTypeMismatch, DTypeUnsupported, InvalidArgument,
                                   LayoutUnsupported, ShapeInvalid, ShapeMismatch, TensorClosed)

from . import paged_ref as plain
from .gpu_util import bits_equal, empty, fetch, to_device

pytestmark = pytest.mark.gpu

BF16, F16, F32, E4M3, E5M2 = DType.BFLOAT16, DType.FLOAT16, DType.FLOAT32, DType.FLOAT8_E4M3, DType.FLOAT8_E5M2
BAD_PAGE = 0x7200


def device_status() -> int:
    code = ctypes.c_int(0)
    try:
        call("mf_device_status", ctypes.byref(code))
    except DeviceStickyError:
        pass
    return code.value


# ------------------------------------------------------------------ page tables

def run_assign(lens, new, page, width, count=None, head=3, tokens=None, stride=None, seed=0, stream=None):
    rng = np.random.default_rng(seed)
    lens, new = np.asarray(lens, np.int32), np.asarray(new, np.int32)
    n = len(lens)
    stride = width if stride is None else stride
    table = np.full((n, stride), -7, np.int32)
    held = np.minimum(-(-np.maximum(lens, 0) // page), width)
    for r in range(n):
        table[r, :held[r]] = rng.integers(0, 1 << 20, held[r])
    needed = int(np.maximum(-(-(np.maximum(lens, 0).astype(np.int64) + np.maximum(new, 0)) // page) - held, 0).sum())
    count = needed if count is None else count
    free = rng.integers(0, 1 << 30, head + count + 1).astype(np.int32)
    total = int(np.maximum(new, 0).astype(np.int64).sum())
    tokens = total if tokens is None else tokens
    pool = np.array([head, count], np.int32)
    want = plain.assign(lens, new, table, free, pool, page, tokens, width)
    ins = [to_device(a) if a.size else empty(4) for a in (lens, new, free, pool)]
    tab = to_device(table) if table.size else empty(4)
    sizes = (8 * tokens, 4 * tokens, 4 * tokens, 4 * (n + 1), 4 * n, 16)
    outs = [empty(s + 16) for s in sizes]
    a = paged.PageAssigner(page, width, stride)
    for _ in range(2):  # a step can be planned again
        a.assign(ins[0].ptr, ins[1].ptr, n, tab.ptr, ins[2].ptr, ins[3].ptr, tokens, *(o.ptr for o in outs), stream=stream)
    sync_device()
    got = [fetch(tab, table.nbytes, np.int32).reshape(table.shape)]
    for o, s, t in zip(outs, sizes, (np.int64, np.int32, np.int32, np.int32, np.int32, np.int32)):
        raw = fetch(o, s + 16)
        assert (raw[s:] == 0xA5).all(), "wrote past an output"
        got.append(raw[:s].view(t))
    for b in [*ins, tab, *outs]:
        b.free()
    for x, y in zip(got, want):
        bits_equal(x, y.astype(x.dtype))


@pytest.mark.parametrize("page", [1, 3, 16, 64])
def test_assign_small_steps(backend, page):
    run_assign([0], [1], page, 8)
    run_assign([7], [0], page, 8)
    run_assign([0, page, page - 1, 5, 2 * page], [1, 1, 1, 1, 1], page, 8)
    run_assign([0, 3, 1, 0], [2 * page, 3 * page + 1, 0, 1], page, 64)


def test_assign_nothing(backend):
    run_assign([], [], 16, 4)
    run_assign([5, 0], [0, 0], 16, 4)
    run_assign([], [], 16, 4, tokens=9)


@pytest.mark.parametrize("n", [511, 2047, 2048, 2049, 5000])
def test_assign_many_requests(backend, n):
    """More than one tile of 2048 requests, idle ones between."""
    rng = np.random.default_rng(n)
    new = rng.integers(0, 40, n) * (rng.random(n) < 0.6)
    run_assign(rng.integers(0, 200, n), new, 16, 15, seed=n)


def test_assign_one_long_prompt(backend):
    run_assign([5, 0, 9], [1, 100003, 1], 16, 6251)


@pytest.mark.parametrize("count", [0, 1, 5, 6, 100])
def test_assign_pool_runs_out(backend, count):
    """Requests in order until the pages are gone; those that need none still fit."""
    run_assign([0, 15, 16, 3, 0, 8], [32, 1, 33, 2, 16, 1], 16, 8, count=count)


def test_assign_table_row_too_short(backend):
    """A request past its table row is refused, takes no pages, and leaves the others theirs."""
    run_assign([60, 0, 64, 10], [10, 20, 1, 3], 16, 4, stride=7)


def test_assign_more_or_fewer_entries_than_tokens(backend):
    run_assign([3, 4], [5, 6], 4, 8, tokens=20)
    run_assign([3, 4], [50, 60], 4, 80, tokens=37)


def test_assign_negative_lengths_count_as_zero(backend):
    run_assign([-5, 4, -1], [3, -2, 2], 4, 8)


def test_assign_on_another_stream(backend):
    s = Stream()
    run_assign([3, 4, 99], [5, 6, 7], 4, 80, stream=s)
    s.close()


def test_assign_refusals(backend):
    a = paged.PageAssigner(16, 8)
    b = [empty(64) for _ in range(11)]
    p = [x.ptr for x in b]
    ok = [p[0], p[1], 1, p[2], p[3], p[4], 1, p[5], p[6], p[7], p[8], p[9], p[10]]

    def refused(error, at, value):
        args = list(ok)
        args[at] = value
        with pytest.raises(error):
            a.assign(*args)

    refused(ShapeInvalid, 2, -1)
    refused(ShapeInvalid, 6, -1)
    refused(ShapeInvalid, 6, 1 << 31)
    for at in (0, 1, 3, 4, 5, 7, 8, 9, 10, 11, 12):
        refused(InvalidArgument, at, 0)
    refused(InvalidArgument, 11, p[0])  # lens_after is lens
    refused(InvalidArgument, 12, p[4])  # pool_after is pool
    with pytest.raises(ShapeInvalid):
        paged.PageAssigner(0, 8).assign(*ok)
    with pytest.raises(ShapeMismatch):
        paged.PageAssigner(16, 8, 7).assign(*ok)
    for x in b:
        x.free()


# ------------------------------------------------------------------ rotary positions

def run_rope(tokens, heads, dim, rot, layout, dtype, inverse=False, far=1000, magnitude=1.0, pad=0, in_place=False,
             offset=0, seed=1, stream=None):
    """Runs on rows of `dim + pad` elements that start `offset` elements into the buffer; what lies between stays."""
    rng = np.random.default_rng(seed)
    width = dim + pad
    x = plain.normal(seed, (tokens, heads, dim), dtype)
    wide = np.full((tokens, heads, width), 0x5A, dtype.storage_numpy)
    wide[..., :dim] = x
    pos = rng.integers(-far if far < 0 else 0, abs(far) + 1, tokens).astype(np.int32)
    freq = paged.rope_frequencies(rot)
    item = dtype.size
    flat = np.concatenate([np.zeros(offset, dtype.storage_numpy), wide.reshape(-1)])
    src, positions, f = to_device(flat), to_device(pos), to_device(freq) if rot else empty(4)
    dst = src if in_place else empty(flat.nbytes)
    r = paged.Rope(f.ptr, dtype, dim, rot, layout, magnitude)
    strides = (heads * width, width)
    (r.backward if inverse else r.forward)(src.ptr + offset * item, dst.ptr + offset * item, positions.ptr, tokens, heads,
                                           strides, strides, stream=stream)
    sync_device()
    raw = fetch(dst, flat.nbytes, dtype.storage_numpy)[offset:].reshape(wide.shape)
    if pad:
        rest = raw[..., dim:]
        assert (rest == (0x5A if in_place else np.frombuffer(b"\xa5" * item, dtype.storage_numpy)[0])).all()
    got, xv = plain.values(raw[..., :dim], dtype), plain.values(x, dtype)
    want = plain.rope(xv, pos, freq, rot, layout, magnitude, inverse)
    bound = plain.rope_bound(xv, pos, rot, layout, magnitude, dtype, want)
    worst = np.abs(got - want) / bound
    assert (worst <= 1).all(), f"{worst.max():.3g} times the bound"
    bits_equal(raw[..., rot:dim], x[..., rot:])  # what does not turn passes through
    for b in {src, dst, positions, f}:
        b.free()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim,rot", [(128, 128), (64, 32), (80, 40), (72, 36), (96, 96), (2, 2), (7, 4), (33, 0), (256, 256)])
def test_rope_layouts_types_and_parts(backend, layout, dtype, dim, rot):
    run_rope(5, 3, dim, rot, layout, dtype)
    run_rope(3, 2, dim, rot, layout, dtype, inverse=True, magnitude=1.25)


@pytest.mark.parametrize("tokens,heads", [(1, 1), (1, 64), (17, 5), (149, 1), (3001, 3), (1, 700)])
def test_rope_token_and_head_counts(backend, tokens, heads):
    run_rope(tokens, heads, 64, 64, "half", BF16)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rope_far_positions(backend, layout):
    run_rope(65, 2, 64, 64, layout, F32, far=2_000_000_000)
    run_rope(65, 2, 64, 64, layout, F32, far=-1_000_000, magnitude=0.5)


@pytest.mark.parametrize("pad,offset", [(8, 0), (4, 0), (3, 0), (0, 1), (0, 4), (8, 8)])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rope_strides_and_alignment(backend, pad, offset, dtype):
    run_rope(9, 3, 64, 64, "half", dtype, pad=pad, offset=offset)
    run_rope(9, 3, 64, 32, "interleaved", dtype, pad=pad, offset=offset, in_place=True)


def test_rope_gradient(backend):
    """<rope(x), g> = <x, backward(g)>, and the gradient against differences of <rope(x), g> in float32."""
    tokens, heads, dim, rot = 6, 2, 16, 12
    n = tokens * heads * dim
    x, gy = synthetic.normal_f32(5, n), synthetic.normal_f32(6, n)
    pos = np.arange(tokens, dtype=np.int32) * 1237
    freq, positions = to_device(paged.rope_frequencies(rot)), to_device(pos)
    src, dst = empty(4 * n), empty(4 * n)
    r = paged.Rope(freq.ptr, F32, dim, rot, "half", 1.5)

    def forward(v):
        src.upload(v)
        r.forward(src.ptr, dst.ptr, positions.ptr, tokens, heads)
        return fetch(dst, 4 * n, np.float32).astype(np.float64)

    src.upload(gy)
    r.backward(src.ptr, dst.ptr, positions.ptr, tokens, heads)
    gx = fetch(dst, 4 * n, np.float32).astype(np.float64)
    y = forward(x)
    # each side is a sum of n terms that are off by 6e-7 of their factors' sizes (times 1.5) at most
    room = 1.5 * 6e-7 * 2 * float(np.abs(x) @ np.abs(gy) + np.abs(gx) @ np.abs(x)) * 2
    assert abs(y @ gy.astype(np.float64) - x.astype(np.float64) @ gx) <= room
    # rope is linear: a difference quotient with step 1 is exact up to the roundings of y (|y| <= 1.5 * 2 * 6)
    for i in (0, 5, 6, 11, 13, n // 2 + 1, n - 1):
        e = x.copy()
        e[i] += 1.0
        quotient = (forward(e) - y) @ gy.astype(np.float64) / (float(e[i]) - float(x[i]))
        assert abs(quotient - gx[i]) <= 4 * 18 * 6e-7 * np.abs(gy).max() * 2
    for b in (src, dst, freq, positions):
        b.free()


def test_rope_on_another_stream(backend):
    s = Stream()
    run_rope(40, 3, 64, 64, "half", BF16, stream=s)
    s.close()


def test_rope_refusals(backend):
    b = [empty(4096) for _ in range(4)]
    x, y, pos, f = (v.ptr for v in b)

    def run(dtype=BF16, dim=64, rot=64, tokens=1, heads=1, src=x, dst=y, positions=pos, freq=f, ss=None, ds=None):
        paged.Rope(freq, dtype, dim, rot).forward(src, dst, positions, tokens, heads, ss, ds)

    with pytest.raises(DTypeUnsupported):
        run(dtype=E4M3)
    for dim, rot in ((64, 63), (64, 66), (64, -2), (0, 0), (4096, 1026)):
        with pytest.raises(ShapeInvalid):
            run(dim=dim, rot=rot)
    with pytest.raises(ShapeInvalid):
        run(tokens=-1)
    with pytest.raises(ShapeInvalid):
        run(heads=-1)
    for bad in ({"src": 0}, {"dst": 0}, {"positions": 0}, {"freq": 0}):
        with pytest.raises(InvalidArgument):
            run(**bad)
    with pytest.raises(ShapeInvalid):
        run(tokens=1 << 31)
    with pytest.raises(LayoutUnsupported):
        run(dst=x, ss=(64, 64), ds=(128, 64))
    with pytest.raises(LayoutUnsupported):
        run(ss=(1 << 31, 64))
    with pytest.raises(InvalidArgument):
        paged.Rope(f, BF16, 64, 64, "spiral")
    run(tokens=0)
    run(heads=0)
    for v in b:
        v.free()


# ------------------------------------------------------------------ the cache write

def run_append(tokens, hq, hkv, dim, dtype, cache, page, order, rot=None, layout="half", compat=1, packed=True, far=5000,
               scaled=True, skip=True, seed=3, stream=None, turning=True):
    rng = np.random.default_rng(seed)
    rot = dim if rot is None else rot
    pages = -(-tokens // page) + 2
    all_heads = hq + 2 * hkv
    x = plain.normal(seed, (tokens, all_heads, dim), dtype, 3.0)
    pos = rng.integers(0, far, tokens).astype(np.int32) if turning else np.zeros(tokens, np.int32)
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    if skip:
        slots[::5] = -1
    freq = paged.rope_frequencies(rot)
    scales = rng.uniform(0.01, 0.05, (2, hkv)).astype(np.float32)
    layout_of = paged.CacheLayout(pages, page, hkv, dim, cache, order)
    nbytes = pages * page * hkv * dim * cache.size
    parts = [x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]]
    bufs = {"f": to_device(freq), "pos": to_device(pos), "slots": to_device(slots), "s": to_device(scales),
            "k": empty(nbytes), "v": empty(nbytes), "q": empty(tokens * hq * dim * dtype.size)}
    if packed:
        bufs["x"] = to_device(x)
        at = [bufs["x"].ptr + h * dim * dtype.size for h in (0, hq, hq + hkv)]
    else:
        for i, p in enumerate(parts):
            bufs[f"x{i}"] = to_device(np.ascontiguousarray(p))
        at = [bufs[f"x{i}"].ptr for i in range(3)]
    use = cache in plain.FP8 and scaled
    r = paged.Rope(bufs["f"].ptr, dtype, dim, rot, layout)
    a = paged.RopeAppend(r, layout_of, hq, bufs["s"].ptr if use else 0, bufs["s"].ptr + 4 * hkv if use else 0, compat,
                         all_heads * dim if packed else None)
    a.run(at[0], at[1], at[2], bufs["q"].ptr, bufs["k"].ptr, bufs["v"].ptr, bufs["pos"].ptr, bufs["slots"].ptr, tokens,
          stream=stream)
    sync_device()
    assert device_status() == 0
    got = {"q": fetch(bufs["q"], bufs["q"].nbytes, dtype.storage_numpy).reshape(tokens, hq, dim)}
    for n in "kv":
        c = fetch(bufs[n], nbytes, cache.storage_numpy).reshape(layout_of.shape)
        got[n] = (c if order == "NHD" else c.transpose(0, 2, 1, 3)).reshape(pages * page, hkv, dim)
    for b in bufs.values():
        b.free()
    # queries
    qv = plain.values(parts[0], dtype)
    want = plain.rope(qv, pos, freq, rot, layout, 1.0)
    assert (np.abs(plain.values(got["q"], dtype) - want) <= plain.rope_bound(qv, pos, rot, layout, 1.0, dtype, want)).all()
    used = np.zeros(pages * page, bool)
    used[slots[slots >= 0]] = True
    canary = np.frombuffer(b"\xa5" * cache.size, cache.storage_numpy)[0]
    for i, n in ((0, "k"), (1, "v")):
        assert (got[n][~used] == canary).all(), "wrote a slot that no token has"
        stored = got[n][slots[slots >= 0]]
        source = parts[1 + i][slots >= 0]
        if n == "v" or not turning:
            f = plain.values(source, dtype).astype(np.float32)
            if use:
                f = f * (np.float32(1.0) / scales[i])[None, :, None]
            bits_equal(stored, plain.codes(f, cache, compat))
            continue
        xv = plain.values(source, dtype)
        kw = plain.rope(xv, pos[slots >= 0], freq, rot, layout, 1.0)
        if cache in plain.FP8:
            inv = (1.0 / scales[i].astype(np.float64))[None, :, None] if use else 1.0
            top = 448.0 if cache == E4M3 else 57344.0
            room = plain.rope_bound(xv, pos[slots >= 0], rot, layout, 1.0, F32, kw) * inv
            least = 2.0 ** -10 if cache == E4M3 else 2.0 ** -17  # half the smallest code
            kw = kw * inv
            off = np.abs(plain.values(stored, cache) - np.clip(kw, -top, top))
            assert (off <= room + np.maximum(plain.UNIT[cache] * 1.01 * np.abs(kw), least)).all()
        else:
            off = np.abs(plain.values(stored, cache) - kw)
            assert (off <= plain.rope_bound(xv, pos[slots >= 0], rot, layout, 1.0, cache, kw)).all()


@pytest.mark.parametrize("order", ["HND", "NHD"])
@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (F32, F32), (BF16, E4M3), (F16, E5M2), (F32, E4M3)])
def test_append_types_and_orders(backend, order, dtype, cache):
    run_append(37, 4, 2, 64, dtype, cache, 16, order)
    run_append(5, 3, 1, 40, dtype, cache, 7, order, rot=20, layout="interleaved", packed=False)


@pytest.mark.parametrize("tokens", [1, 2, 300, 2500])
def test_append_token_counts(backend, tokens):
    run_append(tokens, 8, 2, 128, BF16, BF16, 16, "HND")
    run_append(tokens, 1, 1, 64, BF16, E4M3, 1, "NHD", skip=False)


@pytest.mark.parametrize("compat", [0, 1])
@pytest.mark.parametrize("cache", [E4M3, E5M2])
@pytest.mark.parametrize("dim", [64, 24, 10])
def test_append_codes_are_the_encoders(backend, compat, cache, dim):
    """At position 0 nothing turns: keys and values are the scaled encoders' codes bit for bit."""
    run_append(64, 2, 3, dim, BF16, cache, 16, "HND", compat=compat, turning=False)
    run_append(64, 2, 3, dim, F32, cache, 16, "NHD", compat=compat, turning=False, scaled=False)


def test_append_slot_past_the_cache_is_reported(backend):
    """Such a token's keys and values are dropped, the others' are there, and the status says so."""
    hkv, dim, page, pages = 2, 16, 4, 3
    x = plain.normal(9, (3, 1 + 2 * hkv, dim), BF16)
    slots = np.array([5, pages * page, 2], np.int64)
    layout = paged.CacheLayout(pages, page, hkv, dim, BF16, "NHD")
    nbytes = pages * page * hkv * dim * 2
    b = [to_device(v) for v in (x, np.zeros(3, np.int32), slots, paged.rope_frequencies(dim))]
    k, v, q = empty(nbytes), empty(nbytes), empty(3 * dim * 2)
    a = paged.RopeAppend(paged.Rope(b[3].ptr, BF16, dim), layout, 1, token_stride=(1 + 2 * hkv) * dim)
    a.run(b[0].ptr, b[0].ptr + 2 * dim, b[0].ptr + 2 * dim * (1 + hkv), q.ptr, k.ptr, v.ptr, b[1].ptr, b[2].ptr, 3)
    sync_device()
    assert device_status() == BAD_PAGE and device_status() == 0
    got = fetch(k, nbytes, np.uint16).reshape(pages * page, hkv, dim)
    bits_equal(got[5], x[0, 1:1 + hkv])
    bits_equal(got[2], x[2, 1:1 + hkv])
    rest = np.delete(got, [5, 2], 0)
    assert (rest == 0xA5A5).all()
    for t in (*b, k, v, q):
        t.free()


def test_append_refusals(backend):
    f = empty(1024)
    p = f.ptr

    def run(dtype=BF16, cache=BF16, dim=64, cdim=64, page=16, kv=2, hq=2, compat=1, q=p, k=p, out=p, tokens=1):
        a = paged.RopeAppend(paged.Rope(p, dtype, dim), paged.CacheLayout(4, page, kv, cdim, cache), hq, compat=compat)
        a.run(q, k, p, out, p, p, p, p, tokens)

    with pytest.raises(DTypeMismatch):
        run(cache=F16)
    with pytest.raises(DTypeUnsupported):
        run(dtype=E4M3, cache=E4M3)
    with pytest.raises(ShapeMismatch):
        run(cdim=32)
    for bad in ({"page": 0}, {"kv": 0}, {"hq": -1}, {"tokens": -1}):
        with pytest.raises(ShapeInvalid):
            run(**bad)
    for bad in ({"compat": 2}, {"q": 0}, {"k": 0}, {"out": 0}):
        with pytest.raises(InvalidArgument):
            run(**bad)
    run(tokens=0)
    f.free()


# ------------------------------------------------------------------ attention

def make_attn(lens, hq, hkv, dim, page, order, dtype, cache, seed=7, spare=2, width=None):
    """Inputs with fragmented pages; slots and table entries that no token has hold NaN codes and wild numbers."""
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens, np.int32)
    held = -(-np.maximum(lens, 0) // page)
    pages = int(held.sum()) + spare
    width = max(1, int(held.max(initial=0))) + 1 if width is None else width
    table = np.full((len(lens), width), 1 << 30, np.int32)
    order_of = rng.permutation(pages)
    at = 0
    fp8 = cache in plain.FP8
    nan = {BF16: 0x7FFF, F16: 0x7FFF, E4M3: 0x7F, E5M2: 0x7F}[cache]
    kv = [np.full((pages, page, hkv, dim), nan, cache.storage_numpy) for _ in range(2)]
    for r, n in enumerate(lens):
        table[r, :held[r]] = order_of[at:at + held[r]]
        at += held[r]
        for i, c in enumerate(kv):
            if n > 0:
                rows = plain.normal(seed + 31 * r + i, (int(n), hkv, dim), cache, 40.0 if fp8 else 1.0)
                tok = np.arange(n)
                c[table[r, tok // page], tok % page] = rows
    scales = rng.uniform(0.5, 1.5, (2, hkv)).astype(np.float32) / np.float32(40.0) if fp8 else None
    q = plain.normal(seed + 1, (len(lens), hq, dim), dtype)
    return {"lens": lens, "table": table, "kv": kv, "scales": scales, "q": q, "page": page, "order": order, "dtype": dtype,
            "cache": cache, "hq": hq, "hkv": hkv, "dim": dim, "pages": pages}


def want_attn(s, softcap=0.0, window=0, slopes=None, scale=None):
    dim, page = s["dim"], s["page"]
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    q = plain.values(s["q"], s["dtype"])
    got = []
    for r, n in enumerate(np.maximum(s["lens"], 0)):
        tok = np.arange(n)
        rows = [plain.values(c[s["table"][r, tok // page], tok % page], s["cache"]) if n else
                np.zeros((0, s["hkv"], dim)) for c in s["kv"]]
        if s["scales"] is not None:
            rows = [x * s["scales"][i].astype(np.float64)[None, :, None] for i, x in enumerate(rows)]
        got.append(plain.attention(q[r], rows[0], rows[1], slopes, float(np.float32(scale)), softcap, window, s["hq"] // s["hkv"]))
    return tuple(np.stack(x) for x in zip(*got))


class Running:
    """The case on the device."""

    def __init__(self, s, softcap=0.0, window=0, slopes=None, scale=None, q_pad=0):
        self.s = s
        kv = [c if s["order"] == "NHD" else np.ascontiguousarray(c.transpose(0, 2, 1, 3)) for c in s["kv"]]
        n, hq, dim = s["q"].shape
        wide = np.zeros((n, hq, dim + q_pad), s["q"].dtype)
        wide[..., :dim] = s["q"]
        self.bufs = [to_device(x) for x in (wide, kv[0], kv[1], s["table"], s["lens"])]
        self.extra = [to_device(np.asarray(x, np.float32)) for x in (slopes, s["scales"]) if x is not None]
        sl = self.extra[0].ptr if slopes is not None else 0
        ks = self.extra[-1].ptr if s["scales"] is not None else 0
        self.out_pad = 4 if q_pad else 0
        width = dim + self.out_pad
        self.out, self.lse = empty(n * hq * width * 2 + 16), empty(n * hq * 4 + 16)
        layout = paged.CacheLayout(s["pages"], s["page"], s["hkv"], dim, s["cache"], s["order"])
        self.attn = paged.PagedAttention(layout, hq, s["dtype"], s["table"].shape[1], scale=scale, softcap=softcap,
                                         window=window, slopes=sl, k_scale_inv=ks, v_scale_inv=ks + 4 * s["hkv"] if ks else 0,
                                         q_strides=(hq * (dim + q_pad), dim + q_pad), out_strides=(hq * width, width))

    def run(self, stream=None, lse=True, n=None):
        s = self.s
        n = len(s["lens"]) if n is None else n
        hq, dim, width = s["hq"], s["dim"], s["dim"] + self.out_pad
        self.out.memset(0xA5)
        self.lse.memset(0xA5)
        sync_device()
        p = [b.ptr for b in self.bufs]
        self.attn.run(p[0], p[1], p[2], p[3], p[4], n, self.out.ptr, self.lse.ptr if lse else 0, stream=stream)
        sync_device()
        size = n * hq * width * 2
        raw = fetch(self.out, self.out.nbytes)
        assert (raw[size:] == 0xA5).all(), "wrote past the output"
        out = raw[:size].view(np.uint16).reshape(n, hq, width)
        assert (out[..., dim:] == 0xA5A5).all(), "wrote between the rows"
        low = fetch(self.lse, self.lse.nbytes)
        assert (low[(n * hq * 4 if lse else 0):] == 0xA5).all()
        return out[..., :dim].copy(), low[:n * hq * 4].view(np.float32).reshape(n, hq).copy()

    def close(self):
        self.attn.close()
        for b in (*self.bufs, *self.extra, self.out, self.lse):
            b.free()


def check_attn(s, got, want, weights=1e-4):
    """Bounds: a score of D products summed in float32, |q.k| scale ~ sqrt(D) sums of 1e-6 relative error -> 2e-5
    absolute; the two-term weights 2^-16; exp2 2^-22: weights within `weights` = 1e-4 of themselves (twice that after
    dividing by their sum), times the mean |v|; then one rounding to 16 bits.  lse: `weights`, and 2^-22 of itself."""
    out, lse = got
    w_out, w_lse, size = want
    o = plain.values(out, s["dtype"])
    bound = 2 * weights * size + plain.UNIT[s["dtype"]] * 1.01 * np.abs(w_out) + (3.1e-8 if s["dtype"] == F16 else 0.0)
    assert np.isfinite(o).all()
    worst = np.abs(o - w_out) - bound
    assert (worst <= 0).all(), f"out off by {worst.max():.3g} more than the bound at {np.argwhere(worst > 0)[:4].tolist()}"
    none = np.isneginf(w_lse)
    assert np.array_equal(none, np.isneginf(lse)) and (o[none] == 0).all()
    off = np.abs(lse[~none] - w_lse[~none])
    assert (off <= weights + 2.0 ** -22 * np.abs(w_lse[~none])).all(), f"lse off by {off.max():.3g}"


def run_attn(lens, hq=4, hkv=2, dim=64, page=16, order="HND", dtype=BF16, cache=None, seed=7, q_pad=0, stream=None, weights=1e-4, **rules):
    s = make_attn(lens, hq, hkv, dim, page, order, dtype, dtype if cache is None else cache, seed)
    on = Running(s, q_pad=q_pad, **rules)
    got = on.run(stream)
    again = on.run(stream)
    assert device_status() == 0
    on.close()
    check_attn(s, got, want_attn(s, **rules), weights)
    bits_equal(got[0], again[0])
    bits_equal(got[1].view(np.uint32), again[1].view(np.uint32))


TYPES = [(BF16, BF16), (F16, F16), (BF16, E4M3), (F16, E4M3), (BF16, E5M2), (F16, E5M2)]


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("dim", [16, 64, 80, 96, 128, 192, 256])
def test_attn_types_and_head_dims(backend, dtype, cache, dim):
    run_attn([1, 0, 15, 16, 17, 40, 300], dim=dim, dtype=dtype, cache=cache)
    run_attn([33, 2], hq=12, hkv=1, dim=dim, dtype=dtype, cache=cache, order="NHD", page=5)


@pytest.mark.parametrize("dim", [8, 24, 72, 136])
def test_attn_head_dims_that_are_not_16s(backend, dim):
    run_attn([1, 50], dim=dim)
    run_attn([7, 50], dim=dim, dtype=F16, hq=9, hkv=1)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 1), (5, 1), (9, 1), (16, 1), (17, 1), (40, 1), (14, 2), (32, 32), (64, 4)])
@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_attn_head_groups(backend, hq, hkv, cache):
    run_attn([70, 3], hq=hq, hkv=hkv, cache=cache)


@pytest.mark.parametrize("page", [1, 2, 7, 16, 20, 48, 128])
@pytest.mark.parametrize("order", ["HND", "NHD"])
def test_attn_pages(backend, page, order):
    run_attn([1, page, page + 1, 3 * page - 1, 100], page=page, order=order)
    run_attn([1, page, page + 1, 100], page=page, order=order, cache=E4M3, dim=128)


@pytest.mark.parametrize("n", [1, 2, 255, 256, 257, 700])
def test_attn_request_counts(backend, n):
    """More requests than threads, most of them short, some empty."""
    rng = np.random.default_rng(n)
    run_attn(rng.integers(0, 30, n), hq=2, hkv=1)


def test_attn_all_empty(backend):
    run_attn([0, 0, 0])
    run_attn([-3, 0])


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, E4M3)])
def test_attn_one_long_request(backend, dtype, cache):
    """Every CTA has a part of the same items."""
    run_attn([9001], hq=2, hkv=1, dtype=dtype, cache=cache)
    run_attn([5000], hq=16, hkv=1, dim=256, dtype=dtype, cache=cache)
    run_attn([40000], hq=1, hkv=1, dim=128, dtype=dtype, cache=cache, page=64)


def test_attn_long_among_short(backend):
    run_attn([3, 0, 7001, 1, 1, 64, 0, 3000, 5], hq=8, hkv=2, dim=128)
    run_attn([6000] + [17] * 300, hq=4, hkv=1, dim=64)


@pytest.mark.parametrize("window", [1, 5, 16, 100, 5000])
def test_attn_window(backend, window):
    run_attn([1, 4, 5, 6, 120, 2000, 0], window=window)


@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_attn_softcap_and_slopes(backend, cache):
    slopes = [2.0 ** -(h + 1) for h in range(4)]
    run_attn([1, 90, 1500], cache=cache, softcap=5.0)
    run_attn([1, 90, 1500], cache=cache, slopes=slopes)
    run_attn([1, 90, 1500, 0], cache=cache, slopes=slopes, softcap=20.0, window=200, scale=0.3)


def test_attn_strided_queries_and_outputs(backend):
    run_attn([1, 90, 0], q_pad=4)
    run_attn([1, 90, 0], q_pad=2, cache=E4M3)


def test_attn_on_another_stream(backend):
    s = Stream()
    run_attn([1, 2000, 0], stream=s)
    s.close()


def test_attn_large_scores(backend):
    """Scores of some hundreds: one token has nearly all the weight, and a later one may take it over.  Products of
    |q.k| * 40 up to 1000 in float32 are good to 1000 * 2^-21 = 5e-4."""
    run_attn([1, 300, 2000], scale=40.0, hq=2, hkv=1, dim=16, softcap=300.0, weights=1e-3)


def test_attn_zero_keys_weigh_alike(backend):
    s = make_attn([1000, 3], 2, 1, 64, 16, "HND", BF16, BF16)
    tok = s["kv"][0]
    tok[(tok & 0x7FFF) <= 0x7F80] = 0
    on = Running(s)
    got = on.run()
    on.close()
    check_attn(s, got, want_attn(s))
    assert abs(got[1][0, 0] - math.log(1000)) < 1e-5


def test_attn_keys_that_leave_nothing(backend):
    """Keys of minus infinity give scores of minus infinity: zeros, as for a request without tokens."""
    s = make_attn([40, 20], 2, 1, 16, 16, "HND", BF16, BF16)
    s["q"][:] = 0x3F80  # 1.0
    s["kv"][0][s["table"][0, :3]] = 0xFF80
    on = Running(s)
    out, lse = on.run()
    on.close()
    assert (out[0] & 0x7FFF == 0).all() and np.isneginf(lse[0]).all()
    assert np.isfinite(lse[1]).all()


def test_attn_nan_stays_with_its_request_and_head(backend):
    s = make_attn([40, 20, 33], 4, 2, 16, 16, "HND", BF16, BF16)
    s["q"][0, 1, 3] = 0x7FC0
    s["kv"][1][s["table"][2, 0], 5, 1, 2] = 0x7FC0  # one element of one value head
    on = Running(s)
    out, _ = on.run()
    on.close()
    nan = np.isnan(plain.values(out, BF16))
    want = np.zeros(nan.shape, bool)
    want[0, 1] = True
    want[2, 2:, 2] = True
    assert np.array_equal(nan, want)


def test_attn_page_outside_the_cache_is_masked_and_reported(backend):
    s = make_attn([40, 40], 2, 1, 16, 16, "HND", BF16, BF16)
    want = make_attn([40, 40], 2, 1, 16, 16, "HND", BF16, BF16)
    s["table"][0, 2] = s["pages"]
    s["table"][1, 0] = -1
    on = Running(s)
    got = on.run()
    assert device_status() == BAD_PAGE
    on.close()
    assert device_status() == 0
    q = plain.values(want["q"], BF16)
    for r, keep in ((0, np.arange(32)), (1, np.arange(16, 40))):
        k, v = (plain.values(c[want["table"][r, keep // 16], keep % 16], BF16) for c in want["kv"])
        w = plain.attention(q[r], k, v, None, 0.25, 0.0, 0, 2)
        check_attn(s, (got[0][r:r + 1], got[1][r:r + 1]), tuple(x[None] for x in w))


def test_attn_lengths_past_the_table_are_clamped(backend):
    s = make_attn([64, 30], 2, 1, 16, 16, "HND", BF16, BF16, width=4)
    want = want_attn(s)
    s["lens"] = np.array([1000, 30], np.int32)
    on = Running(s)
    got = on.run()
    assert device_status() == 0
    on.close()
    check_attn(s, got, want)


def test_attn_handle_serves_any_batch(backend):
    """One handle, growing and shrinking batches, with and without lse: each as a fresh one gives it."""
    s = make_attn([500, 3, 0, 2000, 77], 4, 2, 64, 16, "HND", BF16, BF16)
    on = Running(s)
    want = want_attn(s)
    for n in (5, 1, 3, 5, 2):
        got = on.run(n=n)
        check_attn(s, got, tuple(x[:n] for x in want))
    out, _ = on.run(lse=False)
    bits_equal(out, on.run()[0])
    on.close()
    with pytest.raises(TensorClosed):
        on.attn.run(1, 1, 1, 1, 1, 1, 1)


def test_attn_padded_tables_and_caches(backend):
    """Table rows and pages that are longer than what they hold; the gaps hold NaN codes."""
    lens, hq, hkv, dim, page = [1, 45, 0, 130], 4, 2, 64, 16
    s = make_attn(lens, hq, hkv, dim, page, "NHD", BF16, BF16)
    want = want_attn(s)
    n, width = s["table"].shape
    table = np.full((n, width + 5), 1 << 30, np.int32)
    table[:, :width] = s["table"]
    rows, heads = page + 3, hkv + 1  # a page of 16 of 19 rows, 2 of 3 heads, 64 of 72 elements
    kv = []
    for c in s["kv"]:
        wide = np.full((s["pages"], rows, heads, dim + 8), 0x7FFF, np.uint16)
        wide[:, :page, :hkv, :dim] = c
        kv.append(to_device(wide))
    layout = paged.CacheLayout(s["pages"], page, hkv, dim, BF16)
    layout.struct.page_stride, layout.struct.token_stride = rows * heads * (dim + 8), heads * (dim + 8)
    layout.struct.head_stride = dim + 8
    bufs = [to_device(x) for x in (s["q"], table, s["lens"])]
    out, lse = empty(2 * n * hq * dim), empty(4 * n * hq)
    with paged.PagedAttention(layout, hq, BF16, width, table_stride=width + 5) as attn:
        attn.run(bufs[0].ptr, kv[0].ptr, kv[1].ptr, bufs[1].ptr, bufs[2].ptr, n, out.ptr, lse.ptr)
        sync_device()
    got = fetch(out, out.nbytes, np.uint16).reshape(n, hq, dim), fetch(lse, lse.nbytes, np.float32).reshape(n, hq)
    assert device_status() == 0
    check_attn(s, got, want)
    for b in (*bufs, *kv, out, lse):
        b.free()


@pytest.mark.parametrize("page", [16, 20])
def test_offsets_past_32_bits(backend, page):
    """Pages 2^28 bytes apart: the last of 18 lies past 2^32 bytes.  Written by the append, read by the attention."""
    hkv, hq, dim, pages, tokens = 1, 2, 64, 18, 50
    stride = 1 << 27  # elements
    layout = paged.CacheLayout(pages, page, hkv, dim, BF16, "NHD")
    layout.struct.page_stride = stride
    row = (hq + 2 * hkv) * dim
    x = plain.normal(77, (tokens, hq + 2 * hkv, dim), BF16)
    used = np.array([17, 3, 16, 0][:-(-tokens // page)], np.int32)
    tok = np.arange(tokens)
    slots = used[tok // page].astype(np.int64) * page + tok % page
    nbytes = 2 * ((pages - 1) * stride + page * hkv * dim)
    assert nbytes > 1 << 32
    k, v = empty(nbytes, None), empty(nbytes, None)
    b = [to_device(a) for a in (x, np.zeros(tokens, np.int32), slots, paged.rope_frequencies(dim), used, np.array([tokens], np.int32))]
    q_out, out, lse = empty(2 * tokens * hq * dim), empty(2 * hq * dim), empty(4 * hq)
    a = paged.RopeAppend(paged.Rope(b[3].ptr, BF16, dim), layout, hq, token_stride=row)
    a.run(b[0].ptr, b[0].ptr + 2 * hq * dim, b[0].ptr + 2 * (hq + hkv) * dim, q_out.ptr, k.ptr, v.ptr, b[1].ptr, b[2].ptr, tokens)
    sync_device()
    for i, n in enumerate(used):  # nothing turns at position 0: the pages hold the rows as they are
        have = min(page, tokens - i * page)
        for c, at in ((k, hq), (v, hq + hkv)):
            got = fetch(c, 2 * have * dim, np.uint16, offset=2 * int(n) * stride).reshape(have, 1, dim)
            bits_equal(got, x[i * page:i * page + have, at:at + 1])
    with paged.PagedAttention(layout, hq, BF16, len(used)) as attn:
        attn.run(q_out.ptr + 2 * (tokens - 1) * hq * dim, k.ptr, v.ptr, b[4].ptr, b[5].ptr, 1, out.ptr, lse.ptr)
        sync_device()
    assert device_status() == 0
    xv = plain.values(x, BF16)
    want = plain.attention(xv[-1, :hq], xv[:, hq:hq + 1], xv[:, hq + 1:], None, 0.125, 0.0, 0, hq)
    check_attn({"dtype": BF16}, (fetch(out, out.nbytes, np.uint16).reshape(1, hq, dim), fetch(lse, lse.nbytes, np.float32).reshape(1, hq)),
               tuple(w[None] for w in want))
    for t in (k, v, *b, q_out, out, lse):
        t.free()


@pytest.mark.parametrize("lens", [[1999], [1000] * 8, [50, 900, 2000], [300] * 40, [130] * 90, [2000, 1, 1, 1, 1, 1]])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (16, 1)])
def test_attn_ways_to_share_out_the_work(backend, lens, hq, hkv):
    """CTAs of their own for each item, with few or many tiles, and the even cut: up to 148 items and past them."""
    run_attn(lens, hq=hq, hkv=hkv, dim=64)


def test_attn_handles_made_again(backend):
    """A new handle may get an earlier one's workspace: other shapes before and after it change nothing."""
    s = make_attn([3000, 17], 2, 1, 64, 16, "HND", BF16, BF16)
    first = Running(s)
    want = first.run()
    first.close()
    for hq, dim in ((32, 256), (4, 64), (2, 128)):
        run_attn([4000, 3], hq=hq, hkv=1, dim=dim)
    again = Running(s)
    got = again.run()
    again.close()
    bits_equal(got[0], want[0])
    bits_equal(got[1].view(np.uint32), want[1].view(np.uint32))


def test_attn_lengths_that_ask_for_too_much(backend):
    """More than 2^31 - 1 tiles (65536 requests over one shared table row of the longest reach): reported, not computed."""
    n, width = 65536, 1 << 20
    layout = paged.CacheLayout(4, 16, 1, 64, BF16)
    lens = to_device(np.full(n, 16 << 20, np.int32))
    b = [empty(4096) for _ in range(3)]
    out = empty(n * 64 * 2, 0xA5)
    with paged.PagedAttention(layout, 1, BF16, width, table_stride=width) as attn:
        attn.run(b[0].ptr, b[1].ptr, b[1].ptr, b[2].ptr, lens.ptr, n, out.ptr)
        sync_device()
        assert device_status() == 0x7300
    assert (fetch(out, out.nbytes) == 0xA5).all()
    for t in (*b, out, lens):
        t.free()


def test_attn_refusals(backend):
    def make(dtype=BF16, cache=BF16, hq=4, hkv=2, dim=64, page=16, max_pages=4, stride=None, **more):
        paged.PagedAttention(paged.CacheLayout(4, page, hkv, dim, cache), hq, dtype, max_pages, stride, **more).close()

    make()
    for bad in ({"dtype": F32, "cache": F32}, {"dtype": E4M3, "cache": E4M3}):
        with pytest.raises(DTypeUnsupported):
            make(**bad)
    with pytest.raises(DTypeMismatch):
        make(cache=F16)
    for bad in ({"hq": 3}, {"hq": 0}, {"hkv": 0}, {"dim": 0}, {"dim": 264}, {"dim": 12}, {"dim": 72, "cache": E4M3},
                {"page": 0}, {"max_pages": 0}, {"stride": 3}):
        with pytest.raises(ShapeInvalid):
            make(**bad)
    for bad in ({"q_strides": (256, 63)}, {"out_strides": (258, 64)}):
        with pytest.raises(LayoutUnsupported):
            make(**bad)
    for stride in (-64, 1 << 31):
        layout = paged.CacheLayout(4, 16, 2, 64, BF16)
        layout.struct.page_stride = stride
        with pytest.raises(LayoutUnsupported):
            paged.PagedAttention(layout, 4, BF16, 4)
    for bad in ({"window": -1}, {"softcap": -1.0}, {"softcap": float("nan")}):
        with pytest.raises(InvalidArgument):
            make(**bad)
    b = empty(4096)
    p = b.ptr
    a = paged.PagedAttention(paged.CacheLayout(4, 16, 2, 64, BF16), 4, BF16, 4)
    ok = [p, p, p, p, p, 1, p]
    for at in (0, 1, 2, 3, 4, 6):
        args = list(ok)
        args[at] = 0
        with pytest.raises(InvalidArgument):
            a.run(*args)
    for at, by in ((0, 2), (1, 8), (2, 8), (6, 4)):
        args = list(ok)
        args[at] += by
        with pytest.raises(LayoutUnsupported):
            a.run(*args)
    with pytest.raises(ShapeInvalid):
        a.run(p, p, p, p, p, -1, p)
    a.run(0, 0, 0, 0, 0, 0, 0)
    a.close()
    b.free()


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("cache,most", [("bf16", 0.05), ("f8_e4m3", 0.35), ("f8_e5m2", 0.7)])
def test_decoding_steps_of_the_example(backend, cache, most):
    """Prompts, then a token at a time, against float64 attention over what the requests hold.

    A BF16 cache rounds values and rotated keys and queries (2^-9 of themselves on average, |v| up to 4, scores off by
    2^-8 of 3 at most): 0.05.  FP8 keys and values are off by up to 2^-4 (E4M3) or 2^-3 (E5M2) of themselves: a value of 4
    by 0.25 or 0.5, more than what its token's weight changes."""
    import importlib.util
    from pathlib import Path
    spec = importlib.util.spec_from_file_location("paged_decode", Path(__file__).parents[1] / "examples" / "paged_decode.py")
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    worst = example.run(cache_dtype=cache)
    assert len(worst) == 5 and max(worst) <= most


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("softcap", [64.0, 65.0, 1000.0, 1e6])
def test_attn_wide_caps(backend, softcap, cache):
    """A cap far above the scores leaves them as they are: its tanh has to be good relative to the score, not to the
    cap.  Up to 64 an error of 2^-22 of the cap is 1.5e-5, inside the usual bound; above, relative errors of 2^-22."""
    for dim, hq, hkv in ((64, 4, 2), (128, 18, 2), (256, 4, 2)):
        run_attn([1, 90, 1500, 0], cache=cache, softcap=softcap, dim=dim, hq=hq, hkv=hkv)


def test_attn_refuses_an_infinite_cap(backend):
    with pytest.raises(InvalidArgument):
        paged.PagedAttention(paged.CacheLayout(4, 16, 2, 64, BF16), 4, BF16, 4, softcap=float("inf"))


# ------------------------------------------------------------------ a dominant token

# Half the spacing of f16's smallest numbers, 2^-25, over the largest weight that leaves its maximum alone, 2^12.
FLOOR = 2.0 ** -37


def dominant(cache, dtype, lead, n=8192, dim=64, seed=61):
    """One row of keys and values for every request: token 0 leads by `lead` and has the value zero, as a first token
    often does, so that the result is what the others' small weights make of it."""
    rng = np.random.default_rng(seed)
    k = rng.normal(size=(n, 1, dim)).astype(np.float32)
    v = rng.uniform(16.0, 48.0, (n, 1, dim)).astype(np.float32)
    k[0, 0, 0], v[0] = lead, 0.0
    q = np.zeros((2, dim), np.float32)
    q[0, 0], q[1, 0] = 8.0, -8.0  # scores of +-k[:, 0] at a scale of 1/8: the second head sees token 0 last of all
    return plain.codes(q, dtype), plain.codes(k, cache), plain.codes(v, cache)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (F16, E4M3), (F16, E5M2), (BF16, E4M3)])
@pytest.mark.parametrize("lead", [12.0, 16.0, 20.0])
def test_attn_small_weights_beside_a_dominant_one(backend, dtype, cache, lead):
    """2000 requests over the same 8192 tokens: most teams have some thousands of tokens beside the dominant one.

    Beside the usual bound, each f16 weight may be off by FLOOR of the largest (half the spacing of f16's smallest
    numbers, and what the largest weight is at least): as many times the mean |v| as there are tokens."""
    requests, n, page = 2000, 8192, 16
    q, k, v = dominant(cache, dtype, lead, n)
    dim = q.shape[1]
    layout = paged.CacheLayout(n // page, page, 1, dim, cache)
    order = np.random.default_rng(5).permutation(n // page).astype(np.int32)
    kv = [np.empty_like(x) for x in (k, v)]
    for x, y in zip(kv, (k, v)):
        x.reshape(n // page, -1)[order] = y.reshape(n // page, -1)
    bufs = [to_device(a) for a in (np.repeat(q[None], requests, 0), *kv, np.repeat(order[None], requests, 0),
                                   np.full(requests, n, np.int32))]
    out, lse = empty(requests * 2 * dim * 2), empty(requests * 2 * 4)
    with paged.PagedAttention(layout, 2, dtype, n // page) as attn:
        attn.run(*(b.ptr for b in bufs), requests, out.ptr, lse.ptr)
        sync_device()
    got = plain.values(fetch(out, out.nbytes, np.uint16).reshape(requests, 2, dim), dtype)
    got_lse = fetch(lse, lse.nbytes, np.float32).reshape(requests, 2)
    for b in (*bufs, out, lse):
        b.free()
    want, want_lse, size = plain.attention(plain.values(q, dtype), plain.values(k, cache), plain.values(v, cache), None,
                                           0.125, 0.0, 0, 2)
    floor = 0.0 if cache == BF16 else n * FLOOR * np.abs(plain.values(v, cache)).mean(0)
    bound = 2e-4 * size + floor + plain.UNIT[dtype] * 1.01 * np.abs(want) + (3.1e-8 if dtype == F16 else 0.0)
    worst = (np.abs(got - want) / bound).max()
    assert worst <= 1, f"{worst:.3g} times the bound"
    assert (np.abs(got_lse - want_lse) <= 1e-4 + 2.0 ** -22 * np.abs(want_lse)).all()


@pytest.mark.parametrize("cache", [F16, E4M3])
def test_attn_weights_stay_inside_f16_at_coarse_scores(backend, cache):
    """Scores of 2^25 are four apart in float32 (times log2 e): a maximum plus 15 is none of them, and a weight of 2^16,
    which f16 has not, must not come of it.  All values are 1, so every average is."""
    n, dim, page = 200, 64, 16
    k, v, q = np.zeros((n, 1, dim), np.float32), np.ones((n, 1, dim), np.float32), np.zeros((1, 1, dim), np.float32)
    k[:, 0, 0], k[:, 0, 1] = 128.0, np.arange(n) // 13
    q[0, 0, :2] = 32768.0, 0.5
    pages = -(-n // page)
    layout = paged.CacheLayout(pages, page, 1, dim, cache)
    kv = [np.zeros((pages * page, 1, dim), cache.storage_numpy) for _ in range(2)]
    for x, y in zip(kv, (k, v)):
        x[:n] = plain.codes(y, cache)
    bufs = [to_device(a) for a in (plain.codes(q, F16), *kv, np.arange(pages, dtype=np.int32), np.array([n], np.int32))]
    out, lse = empty(2 * dim), empty(4)
    with paged.PagedAttention(layout, 1, F16, pages, scale=8.0) as attn:
        attn.run(*(b.ptr for b in bufs), 1, out.ptr, lse.ptr)
        sync_device()
    got = plain.values(fetch(out, out.nbytes, np.uint16), F16)
    assert (np.abs(got - 1.0) <= 2e-4 + 2.0 ** -11).all()
    assert abs(float(fetch(lse, 4, np.float32)[0]) / 2.0 ** 25 - 1.0) < 1e-5
    for b in (*bufs, out, lse):
        b.free()


@pytest.mark.parametrize("page", [48, 1000])
@pytest.mark.parametrize("dim,cache", [(64, BF16), (128, BF16), (128, E4M3)])
def test_attn_longest_request(backend, page, dim, cache):
    """2^31 - 1 tokens, of which a window sees the last 40: the tile that ends past 2^31 reads neither a table entry past
    the row nor the rows past the length, which hold NaN."""
    n, window, hq, hkv = 2 ** 31 - 1, 40, 4, 2
    width = -(-n // page)
    pages = 4
    tail = np.array([2, 0, 3, 1], np.int32)  # the pages of the row's last entries
    table = DeviceBuffer(4 * width)
    table.memset(0xFF)
    table.upload(tail, offset=4 * (width - len(tail)))
    first = (width - len(tail)) * page
    tok = np.arange(n - window, n)
    kv = [np.full((pages, page, hkv, dim), {BF16: 0x7FFF, E4M3: 0x7F}[cache], cache.storage_numpy) for _ in range(2)]
    rows = [plain.normal(91 + i, (window, hkv, dim), cache) for i in range(2)]
    for c, x in zip(kv, rows):
        c[tail[(tok - first) // page], (tok - first) % page] = x
    q = plain.normal(93, (1, hq, dim), BF16)
    slopes = np.array([0.5, 0.25, 0.125, 0.0625], np.float32)
    bufs = [to_device(a) for a in (q, *kv, np.array([n], np.int32), slopes)]
    out, lse = empty(2 * hq * dim), empty(4 * hq)
    layout = paged.CacheLayout(pages, page, hkv, dim, cache, "NHD")
    with paged.PagedAttention(layout, hq, BF16, width, window=window, slopes=bufs[4].ptr) as attn:
        attn.run(bufs[0].ptr, bufs[1].ptr, bufs[2].ptr, table.ptr, bufs[3].ptr, 1, out.ptr, lse.ptr)
        sync_device()
    assert device_status() == 0
    want = plain.attention(plain.values(q, BF16)[0], *(plain.values(x, cache) for x in rows), slopes,
                           float(np.float32(1.0 / math.sqrt(dim))), 0.0, 0, hq // hkv)
    check_attn({"dtype": BF16}, (fetch(out, out.nbytes, np.uint16).reshape(1, hq, dim), fetch(lse, lse.nbytes, np.float32).reshape(1, hq)),
               tuple(w[None] for w in want))
    for b in (*bufs, table, out, lse):
        b.free()


@pytest.mark.parametrize("n", [2 ** 31 - 1, 2 ** 31 - 2 ** 16 + 1])
def test_request_counts_past_the_loops_are_refused(backend, n):
    """The loops over requests step past the last in 32 bits: counts that would wrap them do not reach the device."""
    b = [empty(4096) for _ in range(4)]
    p = [x.ptr for x in b]
    with pytest.raises(ShapeInvalid):
        paged.PageAssigner(16, 1).assign(p[0], p[0], n, p[1], p[1], p[1], 0, 0, 0, 0, p[2], p[2], p[3])
    with paged.PagedAttention(paged.CacheLayout(4, 16, 1, 16, BF16), 1, BF16, 1) as a:
        with pytest.raises(ShapeInvalid):
            a.run(p[0], p[1], p[1], p[2], p[2], n, p[3])
    for x in b:
        x.free()


# ------------------------------------------------------------------ handles, streams and captured steps

def free_memory() -> int:
    sync_device()
    free, total = ctypes.c_size_t(0), ctypes.c_size_t(0)
    assert ctypes.CDLL("libcuda.so.1").cuMemGetInfo_v2(ctypes.byref(free), ctypes.byref(total)) == 0
    return free.value


def test_attn_destroyed_handles_keep_nothing(backend):
    """A handle's workspace goes with it: nothing is kept by address for handles to come."""
    def make():
        return paged.PagedAttention(paged.CacheLayout(4, 16, 1, 256, BF16), 16, BF16, 4)

    make().close()
    before = free_memory()
    handles = [make() for _ in range(6)]
    assert free_memory() < before - (64 << 20)  # some 22 MB each
    for h in handles:
        h.close()
    assert free_memory() >= before - (4 << 20)


def test_attn_handle_closes_after_shutdown(backend):
    """A handle outlives the library's shutdown: closing it then still frees its workspace."""
    def make():
        return paged.PagedAttention(paged.CacheLayout(4, 16, 1, 256, BF16), 16, BF16, 4)

    make().close()
    before = free_memory()
    a = make()
    call("mf_shutdown")
    try:
        a.close()
    finally:
        call("mf_init", 0)
    assert free_memory() >= before - (4 << 20)
    run_attn([1, 90, 0])


def test_assign_first_refusal_for_pages_stops_the_rest_of_the_step(backend):
    """Page grants are a prefix of the step: behind a request whose pages are not there none gets a page, however few it
    needs; those that need none still fit."""
    run_assign([16, 0, 16, 3, 32], [1, 32, 1, 1, 1], 16, 8, count=2)
    lens, new = [to_device(np.array(a, np.int32)) for a in ([16, 0, 16, 3, 32], [1, 32, 1, 1, 1])]
    table = to_device(np.arange(40, dtype=np.int32).reshape(5, 8))
    free, pool = to_device(np.array([70, 71], np.int32)), to_device(np.array([0, 2], np.int32))
    outs = [empty(s) for s in (8 * 36, 4 * 36, 4 * 36, 4 * 6, 4 * 5, 16)]
    paged.PageAssigner(16, 8).assign(lens.ptr, new.ptr, 5, table.ptr, free.ptr, pool.ptr, 36, *(o.ptr for o in outs))
    after, left = fetch(outs[4], 20, np.int32), fetch(outs[5], 16, np.int32)
    assert after.tolist() == [17, 0, 16, 4, 32]
    assert left.tolist() == [1, 1, 36, 3]
    for b in (lens, new, table, free, pool, *outs):
        b.free()


def queued(on, times, stream):
    """`times` runs of the case on a stream, none waited for."""
    s, p = on.s, [b.ptr for b in on.bufs]
    for _ in range(times):
        on.attn.run(p[0], p[1], p[2], p[3], p[4], len(s["lens"]), on.out.ptr, on.lse.ptr, stream=stream)


def results(on):
    return fetch(on.out, on.out.nbytes), fetch(on.lse, on.lse.nbytes)


def test_attn_two_handles_on_two_streams(backend):
    """Each handle has its own workspace: runs that overlap give what each gives alone."""
    cases = [Running(make_attn([9001, 5, 700], 4, 1, 64, 16, "HND", BF16, BF16)),
             Running(make_attn([3000] * 40, 8, 2, 128, 16, "NHD", F16, E4M3))]
    alone = []
    for on in cases:
        queued(on, 1, None)
        alone.append(results(on))
        on.out.memset(0xA5)
        on.lse.memset(0xA5)
    sync_device()
    streams = [Stream(), Stream()]
    for _ in range(20):
        for on, s in zip(cases, streams):
            queued(on, 2, s)
    for s in streams:
        s.sync()
    for on, want in zip(cases, alone):
        for x, y in zip(results(on), want):
            bits_equal(x, y)
        on.close()
    for s in streams:
        s.close()


def test_attn_destroyed_while_its_runs_are_queued(backend):
    """Destroying waits for the handle's runs; the next handle may get their memory."""
    first = Running(make_attn([30000, 5], 4, 1, 64, 16, "HND", BF16, BF16))
    queued(first, 1, None)
    want = results(first)
    s = Stream()
    queued(first, 30, s)
    first.attn.close()
    second = Running(make_attn([9001, 5, 700], 4, 1, 64, 16, "HND", BF16, BF16, seed=8))
    queued(second, 1, None)
    check_attn(second.s, second.run(), want_attn(second.s))
    for x, y in zip(results(first), want):
        bits_equal(x, y)
    first.close()
    second.close()
    s.close()


@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_a_captured_step_replays_with_other_lengths(backend, cache):
    """Page assignment, append and attention captured once; each replay serves the lengths that are there then, as the
    same calls one by one do."""
    import torch

    n, hq, hkv, dim, page, width, pages = 5, 4, 2, 64, 16, 32, 200
    row = (hq + 2 * hkv) * dim
    layout = paged.CacheLayout(pages, page, hkv, dim, cache)
    nbytes = pages * page * hkv * dim * cache.size
    rng = np.random.default_rng(17)
    freq, free = to_device(paged.rope_frequencies(dim)), to_device(rng.permutation(pages).astype(np.int32))
    rope, assign = paged.Rope(freq.ptr, BF16, dim), paged.PageAssigner(page, width)
    append = paged.RopeAppend(rope, layout, hq, token_stride=row)
    keys, vals = plain.normal(71, (nbytes // cache.size,), cache), plain.normal(72, (nbytes // cache.size,), cache)

    class Step:
        def __init__(self):
            self.k, self.v = to_device(keys), to_device(vals)
            self.table = to_device(np.zeros((n, width), np.int32))
            self.lens, self.new, self.pool = empty(4 * n), empty(4 * n), empty(8)
            self.x, self.q, self.out, self.lse = empty(2 * n * row), empty(2 * n * hq * dim), empty(2 * n * hq * dim), empty(4 * n * hq)
            self.slots, self.pos, self.owner = empty(8 * n), empty(4 * n), empty(4 * n)
            self.starts, self.after, self.pool_after = empty(4 * (n + 1)), empty(4 * n), empty(16)
            self.attn = paged.PagedAttention(layout, hq, BF16, width)

        def run(self, stream):
            assign.assign(self.lens.ptr, self.new.ptr, n, self.table.ptr, free.ptr, self.pool.ptr, n, self.slots.ptr,
                          self.pos.ptr, self.owner.ptr, self.starts.ptr, self.after.ptr, self.pool_after.ptr, stream)
            append.run(self.x.ptr, self.x.ptr + 2 * hq * dim, self.x.ptr + 2 * (hq + hkv) * dim, self.q.ptr, self.k.ptr,
                       self.v.ptr, self.pos.ptr, self.slots.ptr, n, stream)
            self.attn.run(self.q.ptr, self.k.ptr, self.v.ptr, self.table.ptr, self.after.ptr, n, self.out.ptr, self.lse.ptr,
                          stream)

        def load(self, lens, x):
            held = -(-lens // page)
            table = np.zeros((n, width), np.int32)
            table[np.arange(width)[None] < held[:, None]] = pages - 1 - np.arange(held.sum())
            for b, a in ((self.table, table), (self.lens, lens), (self.new, np.ones(n, np.int32)),
                         (self.pool, np.array([0, 8], np.int32)), (self.x, x)):
                b.upload(a)
            sync_device()

        def state(self):
            return [fetch(b, b.nbytes) for b in (self.table, self.k, self.v, self.q, self.out, self.lse, self.slots, self.pos,
                                                 self.owner, self.starts, self.after, self.pool_after)]

        def close(self):
            self.attn.close()
            for b in vars(self).values():
                if hasattr(b, "free"):
                    b.free()

    one, other = Step(), Step()
    one.load(np.full(n, 3, np.int32), plain.normal(73, (n, row), BF16))
    stream = torch.cuda.Stream()
    one.run(stream.cuda_stream)
    stream.synchronize()
    one.k.upload(keys)
    one.v.upload(vals)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        one.run(stream.cuda_stream)
    for i, lens in enumerate(([3, 0, 15, 16, 31], [200, 1, 64, 0, 499], [0, 0, 0, 0, 0], [496, 497, 1, 95, 96])):
        lens, x = np.array(lens, np.int32), plain.normal(80 + i, (n, row), BF16)
        one.load(lens, x)
        other.load(lens, x)
        graph.replay()
        torch.cuda.synchronize()
        other.run(None)
        for a, b in zip(one.state(), other.state()):
            bits_equal(a, b)
    assert device_status() == 0
    del graph
    for b in (one, other, freq, free):
        getattr(b, "close" if isinstance(b, Step) else "free")()


# ------------------------------------------------------------------ precision of single scores

def single_scores(cache, softcap, n=4096, dim=64):
    """lse of `n` requests of one token each is its score; q and k have one element each that is not zero, so the score is
    their product without a rounding.  Returns (lse, the scores in 64 bits)."""
    rng = np.random.default_rng(21)
    k = np.zeros((n, 1, 1, dim), np.float32)
    k[:, 0, 0, 0] = np.exp2(rng.uniform(-4, 4, n)) * rng.choice([-1, 1], n)
    q = np.zeros((n, 1, dim), np.float32)
    q[..., 0] = 8.0
    kc, dtype = plain.codes(k, cache), BF16 if cache == BF16 else F16
    bufs = [to_device(a) for a in (plain.codes(q, dtype), kc, kc, np.arange(n, dtype=np.int32), np.ones(n, np.int32))]
    out, lse = empty(2 * n * dim), empty(4 * n)
    with paged.PagedAttention(paged.CacheLayout(n, 1, 1, dim, cache), 1, dtype, 1, scale=0.125, softcap=softcap) as attn:
        attn.run(*(b.ptr for b in bufs), n, out.ptr, lse.ptr)
        sync_device()
    got = fetch(lse, lse.nbytes, np.float32).astype(np.float64)
    for b in (*bufs, out, lse):
        b.free()
    s = plain.values(kc, cache)[:, 0, 0, 0]
    return got, softcap * np.tanh(s / softcap) if softcap else s


@pytest.mark.parametrize("cache", [BF16, F16, E4M3, E5M2])
@pytest.mark.parametrize("softcap", [2.0, 20.0, 50.0, 64.0, 1000.0])
def test_attn_capped_scores_keep_their_bits(backend, cache, softcap):
    """A capped score is good relative to itself, however far below the cap: the polynomial 1e-7, or at 0.4 of the cap an
    exponential and a reciprocal of 2^-22 each over tanh(0.4), and some six roundings of 2^-24: 2^-20 together.  The
    f16 forms hold the maximum less 12 and its distance to it, 2^-21 each, and a logarithm near 12, 2^-21: 2^-20 absolutely
    after the change of base."""
    got, want = single_scores(cache, softcap)
    assert (np.abs(got - want) <= 2.0 ** -20 * np.abs(want) + (0.0 if cache == BF16 else 2.0 ** -20)).all()


@pytest.mark.parametrize("cache", [BF16, F16, E4M3, E5M2])
def test_attn_lse_of_single_tokens(backend, cache):
    """Without a cap: three roundings of the score, and in the f16 forms those of the maximum less 12 and of its distance
    to it (2^-21 each at most, times ln 2)."""
    got, want = single_scores(cache, 0.0)
    off = np.abs(got - want)
    assert (off <= 2.0 ** -21 * np.abs(want) + (0.0 if cache == BF16 else 2.0 ** -20 * math.log(2.0))).all()
    assert math.sqrt((off ** 2).sum() / (want ** 2).sum()) <= 2.0 ** -21


@pytest.mark.parametrize("cache", [BF16, F16, E4M3, E5M2])
def test_attn_lse_of_equal_scores(backend, cache):
    """Queries of zero: lse = log(n).  What is summed is exact in every form; a float32 log2 (one unit in the last place, up
    to 0.63 of 2^-22 of the result), a constant and a product: 0.75 of 2^-22 of it, for f16 weights of 2^12 as well."""
    dim, dtype, most = 64, BF16 if cache == BF16 else F16, 40
    kv = plain.normal(33, (most, 1, 1, dim), cache)
    lens = np.arange(1, most + 1, dtype=np.int32)
    table = np.tile(np.arange(most, dtype=np.int32), (most, 1))
    bufs = [to_device(a) for a in (np.zeros((most, 1, dim), np.uint16), kv, kv, table, lens)]
    out, lse = empty(2 * most * dim), empty(4 * most)
    with paged.PagedAttention(paged.CacheLayout(most, 1, 1, dim, cache), 1, dtype, most) as attn:
        attn.run(*(b.ptr for b in bufs), most, out.ptr, lse.ptr)
        sync_device()
    got = fetch(lse, lse.nbytes, np.float32).astype(np.float64)
    for b in (*bufs, out, lse):
        b.free()
    assert (np.abs(got - np.log(lens)) <= 0.75 * 2.0 ** -22 * np.log(lens)).all()
