"""Attention over a shared prefix on the GPU against 64-bit attention of every request by itself."""
import numpy as np
import pytest

from manifesto_b200 import Stream, paged, sync_device
from manifesto_b200._abi import call
from manifesto_b200.dtype import DType
from manifesto_b200.errors import (DTypeMismatch, DTypeUnsupported, InvalidArgument, LayoutUnsupported, ShapeInvalid, TensorClosed)

from . import paged_ref as plain
from .gpu_util import bits_equal, empty, fetch, to_device
from .test_gpu_paged import BAD_PAGE, TYPES, check_attn, device_status, make_attn, want_attn

pytestmark = pytest.mark.gpu

BF16, F16, F32, E4M3, E5M2 = DType.BFLOAT16, DType.FLOAT16, DType.FLOAT32, DType.FLOAT8_E4M3, DType.FLOAT8_E5M2


def make_groups(groups, hq, hkv, dim, page, order, dtype, cache, seed, alone=0):
    """groups: (shared tokens, own tokens of each member; negative: that many tokens less than the shared ones)."""
    lens, starts, shared = [5 + 3 * i for i in range(alone)], [alone], []
    for common, own in groups:
        lens += [common + x for x in own]
        starts.append(len(lens))
        shared.append(common)
    full = [max(n, 0) for n in lens]
    for g, common in enumerate(shared):  # the first member's row names every shared page
        if starts[g] < starts[g + 1]:
            full[starts[g]] = max(full[starts[g]], common)
    s = make_attn(full, hq, hkv, dim, page, order, dtype, cache, seed)
    for g, common in enumerate(shared):
        lead = s["table"][starts[g]] if starts[g] < starts[g + 1] else None
        for r in range(starts[g] + 1, starts[g + 1]):
            whole, rest = common // page, common % page
            n = min(whole, -(-full[r] // page))
            s["table"][r, :n] = lead[:n]
            if rest and full[r] > whole * page:  # the page where the members part: equal tokens in pages of their own
                for c in s["kv"]:
                    c[s["table"][r, whole], :min(rest, full[r] - whole * page)] = c[lead[whole], :min(rest, full[r] - whole * page)]
    s["lens"] = np.array(lens, np.int32)
    s["starts"], s["shared"] = np.array(starts, np.int32), np.array(shared, np.int32)
    return s


def check_prefix(s, got, want):
    """The bounds of the attention without sharing (the join adds float32 products of weights that are good to 2^-22).

    Over an FP8 cache with BF16 queries the shared tokens' weights enter the product as one f16 term, off by half a step,
    2^-11 of themselves: 2^-11 of the mean |v| more, which check_attn counts as twice `weights`.  lse knows nothing of it."""
    one_term = s["dtype"] == BF16 and s["cache"] in (E4M3, E5M2)
    check_attn(s, got, want, 1e-4 + 2.0 ** -12 if one_term else 1e-4)
    some = np.isfinite(want[1])
    assert (np.abs(got[1][some] - want[1][some]) <= 1e-4 + 2.0 ** -22 * np.abs(want[1][some])).all()


class Running:
    """The case on the device."""

    def __init__(self, s, softcap=0.0, window=0, slopes=None, scale=None, q_pad=0, max_requests=None, always=True):
        self.s = s
        kv = [c if s["order"] == "NHD" else np.ascontiguousarray(c.transpose(0, 2, 1, 3)) for c in s["kv"]]
        n, hq, dim = s["q"].shape
        wide = np.zeros((n, hq, dim + q_pad), s["q"].dtype)
        wide[..., :dim] = s["q"]
        self.bufs = [to_device(x) if x.size else empty(16) for x in (wide, kv[0], kv[1], s["table"], s["lens"], s["starts"], s["shared"])]
        self.extra = [to_device(np.asarray(x, np.float32)) for x in (slopes, s["scales"]) if x is not None]
        sl = self.extra[0].ptr if slopes is not None else 0
        ks = self.extra[-1].ptr if s["scales"] is not None else 0
        self.out_pad = 4 if q_pad else 0
        width = dim + self.out_pad
        self.out, self.lse = empty(n * hq * width * 2 + 16), empty(n * hq * 4 + 16)
        layout = paged.CacheLayout(s["pages"], s["page"], s["hkv"], dim, s["cache"], s["order"])
        self.attn = paged.PrefixAttention(layout, hq, s["dtype"], s["table"].shape[1], max_requests or n, scale=scale, softcap=softcap,
                                          window=window, slopes=sl, k_scale_inv=ks, v_scale_inv=ks + 4 * s["hkv"] if ks else 0,
                                          q_strides=(hq * (dim + q_pad), dim + q_pad), out_strides=(hq * width, width), always=always)

    def run(self, stream=None, lse=True, groups=None):
        s = self.s
        n, hq, dim, width = len(s["lens"]), s["hq"], s["dim"], s["dim"] + self.out_pad
        self.out.memset(0xA5)
        self.lse.memset(0xA5)
        sync_device()
        p = [b.ptr for b in self.bufs]
        self.attn.run(*p[:5], n, p[5], p[6], len(s["shared"]) if groups is None else groups, self.out.ptr, self.lse.ptr if lse else 0,
                      stream=stream)
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


def run_groups(groups, hq=4, hkv=2, dim=64, page=16, order="HND", dtype=BF16, cache=None, seed=7, alone=0, q_pad=0, stream=None, **rules):
    s = make_groups(groups, hq, hkv, dim, page, order, dtype, dtype if cache is None else cache, seed, alone)
    on = Running(s, q_pad=q_pad, **rules)
    device_status()
    got = on.run(stream)
    again = on.run(stream)
    assert device_status() == 0
    on.close()
    check_prefix(s, got, want_attn(s, **rules))
    bits_equal(got[0], again[0])
    bits_equal(got[1].view(np.uint32), again[1].view(np.uint32))


def test_prefix_one_tile(backend):
    run_groups([(128, [1, 2, 3, 4])])


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("dim", [16, 64, 80, 96, 128, 192, 256])
def test_prefix_types_and_head_dims(backend, dtype, cache, dim):
    run_groups([(200, [3, 17, 1]), (35, [2, 40])], dim=dim, dtype=dtype, cache=cache)


@pytest.mark.parametrize("dim", [8, 24, 72, 136])
def test_prefix_head_dims_that_are_not_16s(backend, dim):
    run_groups([(200, [3, 17, 1])], dim=dim, dtype=F16)


@pytest.mark.parametrize("hq,hkv,members", [(1, 1, 2), (8, 1, 3), (5, 1, 30), (16, 1, 8), (16, 1, 9), (40, 1, 7), (14, 2, 19), (32, 32, 130), (32, 8, 70),
                                            (64, 4, 33), (200, 1, 2)])
@pytest.mark.parametrize("dim,cache", [(64, BF16), (128, BF16), (128, E4M3), (256, BF16)])
def test_prefix_rows(backend, hq, hkv, members, dim, cache):
    """Blocks of one row, of up to 128 (both groups of warps take turns), of up to 256 (each has its own), several blocks."""
    if members * hq * dim > 200_000:
        members = max(2, 200_000 // (hq * dim))
    run_groups([(300, [1 + i % 3 for i in range(members)])], hq=hq, hkv=hkv, dim=dim, cache=cache)


@pytest.mark.parametrize("shared", [0, 1, 15, 16, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000, 4097])
@pytest.mark.parametrize("dim,cache", [(128, BF16), (64, E4M3), (256, F16)])
def test_prefix_lengths(backend, shared, dim, cache):
    run_groups([(shared, [1, 5, 0, 20])], dim=dim, dtype=F16 if cache == F16 else BF16, cache=cache)


@pytest.mark.parametrize("page", [1, 2, 7, 16, 20, 48, 128, 300])
@pytest.mark.parametrize("order", ["HND", "NHD"])
def test_prefix_pages(backend, page, order):
    """Shared lengths that end inside a page, too."""
    run_groups([(page * 5, [1, 3, 9]), (page * 3 + page // 2, [0, 2, page, 3 * page])], page=page, order=order)


@pytest.mark.parametrize("n", [1, 7, 60, 700])
def test_prefix_many_groups(backend, n):
    run_groups([(20 + 17 * (i % 9), [1 + (i + x) % 5 for x in range(2 + i % 4)]) for i in range(n)], hq=2, hkv=2, dim=32)


def test_prefix_groups_of_all_sizes(backend):
    """None, one member, many; requests in front of the groups; long and short ones side by side."""
    run_groups([(100, []), (50, [3]), (700, [1] * 9), (0, [4, 5]), (5, [0, 0]), (2000, [1, 300]), (128, [7] * 150)], alone=4)


def test_prefix_nothing_is_shared(backend):
    run_groups([], alone=5)
    run_groups([(64, [9])], alone=2)
    run_groups([(0, [9, 8, 7])])


def test_prefix_members_shorter_than_the_prefix(backend):
    """Each sees its own length's part of the shared tokens; an idle one nothing."""
    run_groups([(300, [5, -1, -171, -172, -173, -300, 0]), (300, [-300, 4, -299]), (40, [-40, -40])])


@pytest.mark.parametrize("window", [1, 5, 16, 100, 130, 5000])
def test_prefix_window(backend, window):
    run_groups([(300, [1, 20, 90, 140, -30, 0]), (17, [3, 4])], window=window)


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("dim", [64, 256])
def test_prefix_softcap_and_slopes(backend, cache, dim):
    slopes = [2.0 ** (-x) for x in range(1, 5)]
    run_groups([(300, [1, 20, -7])], cache=cache, dim=dim, softcap=20.0)
    run_groups([(300, [1, 20, -7])], cache=cache, dim=dim, slopes=slopes)
    run_groups([(300, [1, 20, -7])], cache=cache, dim=dim, softcap=3.0, slopes=slopes, window=77)


@pytest.mark.parametrize("scale", [-0.1, 0.0, 0.7])
def test_prefix_scales(backend, scale):
    run_groups([(300, [1, 20, 2])], scale=scale)


def test_prefix_strided_queries_and_outputs(backend):
    run_groups([(300, [1, 20, 2])], q_pad=8)
    run_groups([(300, [1, 20, 2])], q_pad=2)
    run_groups([(300, [1, 20, 2])], q_pad=6, cache=E4M3)


def test_prefix_on_another_stream(backend):
    s = Stream()
    run_groups([(300, [1, 20, 2])], stream=s)
    s.close()


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, E4M3)])
def test_prefix_long(backend, dtype, cache):
    """More tiles than CTAs for one item: every CTA has a part, most of them inside it."""
    run_groups([(30011, [1, 2])], hq=2, hkv=1, dim=128, dtype=dtype, cache=cache)
    run_groups([(9000, [1] * 70), (40, [1, 2]), (9000, [3, 4])], hq=4, hkv=1, dim=128, dtype=dtype, cache=cache)


def test_prefix_nan_stays_with_its_request_and_head(backend):
    s = make_groups([(300, [1, 20, 2, 9])], 4, 2, 64, 16, "HND", BF16, BF16, 3)
    want = want_attn(s)
    s["q"][2, 1, 5] = 0x7fc0
    on = Running(s)
    out, lse = on.run()
    on.close()
    o = plain.values(out, BF16)
    assert np.isnan(o[2, 1]).all() and np.isnan(lse[2, 1])
    o[2, 1], lse[2, 1], want[0][2, 1], want[1][2, 1], want[2][2, 1] = 0, 0, 0, 0, 0
    keep = np.ones((4, 4), bool)
    keep[2, 1] = False
    assert np.isfinite(o).all() and (np.abs(o - want[0])[keep] <= 2e-4 * want[2][keep] + 2.0 ** -8 * 1.01 * np.abs(want[0][keep])).all()


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (F16, E4M3)])
def test_prefix_keys_that_leave_nothing(backend, dtype, cache):
    """Scores of -inf for every token: nothing is seen."""
    s = make_groups([(200, [1, 20, 2])], 2, 1, 64, 16, "HND", dtype, dtype, 3)
    s["kv"][0][:] = plain.normal(1, s["kv"][0].shape, dtype, 0.0)
    s["kv"][0][..., 0] = 0xff80 if dtype == BF16 else 0xfc00
    s["q"][..., 0] = 0x3f80 if dtype == BF16 else 0x3c00
    s["kv"][1][:] = 0
    on = Running(s)
    out, lse = on.run()
    on.close()
    assert (out == 0).all() and np.isneginf(lse).all()


def test_prefix_page_outside_the_cache_is_masked_and_reported(backend):
    s = make_groups([(300, [5, 20, 2])], 4, 2, 64, 16, "HND", BF16, BF16, 3)
    for bad in (-1, 1 << 29):
        s["table"][:, 3] = bad
        on = Running(s)
        device_status()
        got = on.run()
        assert device_status() == BAD_PAGE
        on.close()
        # the same without those 16 tokens
        t = dict(s)
        t["table"] = np.delete(s["table"], 3, 1)
        t["lens"] = s["lens"] - 16
        check_prefix(t, got, want_attn(t))


@pytest.mark.parametrize("starts", [[0, 3, 2, 6], [0, 2, 4, 7], [-1, 2, 4, 6], [0, 2 ** 31 - 1, 2, 6]])
def test_prefix_groups_that_are_none_share_nothing(backend, starts):
    s = make_groups([(100, [1, 2]), (100, [3, 4]), (100, [5, 6])], 4, 2, 64, 16, "HND", BF16, BF16, 3)
    s["starts"] = np.array(starts, np.int32)
    on = Running(s)
    device_status()
    got = on.run()
    assert device_status() == 0x7300
    on.close()
    check_prefix(s, got, want_attn(s))


def test_prefix_shared_past_the_table_or_negative(backend):
    s = make_groups([(96, [0, 0, -5]), (64, [1, 2])], 4, 2, 64, 16, "HND", BF16, BF16, 3)
    s["shared"] = np.array([2 ** 31 - 1, -7], np.int32)
    s["table"] = np.ascontiguousarray(s["table"][:, :6])
    s["table"][0, 5] = s["table"][1, 5]
    on = Running(s)
    device_status()
    got = on.run()
    assert device_status() == 0
    on.close()
    check_prefix(s, got, want_attn(s))


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (F16, E4M3), (BF16, E4M3)])
@pytest.mark.parametrize("lead", [12.0, 16.0, 20.0])
def test_prefix_small_weights_beside_a_dominant_one(backend, dtype, cache, lead):
    """A first token of value 0 that leads by `lead`: what the others add up to is all of the result."""
    s = make_groups([(600, [1, 3])], 2, 1, 64, 16, "HND", dtype, cache, 5)
    q = np.zeros(s["q"].shape)
    q[..., 0] = 1.0
    s["q"] = plain.normal(0, s["q"].shape, dtype, 0.0)
    one = 0x3f80 if dtype == BF16 else 0x3c00
    s["q"][..., 0] = one
    keys, values = s["kv"]
    if s["scales"] is not None:
        s["scales"][:] = 1.0
    page0 = s["table"][0, 0]
    code = {BF16: lambda x: np.float32(x).view(np.uint32) >> 16, F16: lambda x: np.float16(x).view(np.uint16),
            E4M3: lambda x: {12.0: 0x54, 16.0: 0x58, 20.0: 0x5a}[x]}[cache](lead)
    held = sorted({int(x) for row, n in zip(s["table"], s["lens"]) for x in row[:-(-int(n) // 16)]})
    keys[held] = 0
    keys[page0, 0, :, 0] = code
    values[page0, 0] = 0
    on = Running(s, scale=1.0)
    got = on.run()
    on.close()
    check_prefix(s, got, want_attn(s, scale=1.0))


def test_prefix_handle_serves_any_batch(backend):
    """Other requests, groups and lengths on one handle; what the run before left does not show."""
    h = None
    for groups in ([(700, [1] * 40)], [(30, [2, 3])], [(200, [1, 2]), (5, [1, 1, 1])], [(700, [1] * 40)]):
        s = make_groups(groups, 4, 2, 128, 16, "HND", BF16, BF16, 11)
        on = Running(s, max_requests=64)
        if h is None:
            h = on.attn
        else:
            on.attn.close()
            # the same description but for the table's width and the cache's pages: those of the widest case
        on_attn, on.attn = on.attn, h
        if on_attn is h:
            first = s
        if s["table"].shape[1] <= first["table"].shape[1]:
            wide = np.full((len(s["lens"]), first["table"].shape[1]), 1 << 30, np.int32)
            wide[:, :s["table"].shape[1]] = s["table"]
            on.bufs[3].free()
            on.bufs[3] = to_device(wide)
        assert s["pages"] <= first["pages"]
        check_prefix(s, on.run(), want_attn(s))
        for b in (*on.bufs, *on.extra, on.out, on.lse):
            b.free()
    h.close()
    with pytest.raises(TensorClosed):
        h.run(*([1] * 5), 1, 1, 1, 1, 1)


def test_prefix_without_lse(backend):
    s = make_groups([(100, [1, 2])], 4, 2, 64, 16, "HND", BF16, BF16, 3)
    on = Running(s)
    with_lse, without = on.run(), on.run(lse=False)
    on.close()
    bits_equal(with_lse[0], without[0])


def test_prefix_two_handles_on_two_streams(backend):
    cases = [make_groups([(900, [3] * 30)], 8, 2, 128, 16, "HND", BF16, BF16, i) for i in (1, 2)]
    on, streams = [Running(s) for s in cases], [Stream(), Stream()]
    for o in on:
        o.out.memset(0)
    sync_device()
    for _ in range(10):
        for o, st in zip(on, streams):
            p = [b.ptr for b in o.bufs]
            o.attn.run(*p[:5], 30, p[5], p[6], 1, o.out.ptr, o.lse.ptr, stream=st)
    sync_device()
    for o, s in zip(on, cases):
        out = fetch(o.out, 30 * 8 * 128 * 2, np.uint16).reshape(30, 8, 128)
        check_prefix(s, (out, fetch(o.lse, 30 * 8 * 4, np.float32).reshape(30, 8)), want_attn(s))
        o.close()
    for st in streams:
        st.close()


def test_prefix_refusals(backend):
    layout = paged.CacheLayout(4, 16, 2, 64, BF16)
    for kwargs, error in (({"max_requests": 0}, ShapeInvalid), ({"max_requests": -1}, ShapeInvalid), ({"max_requests": 2 ** 31 - 1}, ShapeInvalid),
                          ({"dtype": F32}, DTypeUnsupported), ({"dtype": F16}, DTypeMismatch), ({"q_heads": 3}, ShapeInvalid),
                          ({"max_pages": 0}, ShapeInvalid), ({"window": -1}, InvalidArgument), ({"softcap": float("inf")}, InvalidArgument),
                          ({"q_strides": (257, 65)}, LayoutUnsupported)):
        with pytest.raises(error):
            paged.PrefixAttention(**{**dict(cache=layout, q_heads=4, dtype=BF16, max_pages=4, max_requests=4), **kwargs})
    h = paged.PrefixAttention(layout, 4, BF16, 4, 4)
    b = [empty(1 << 16) for _ in range(9)]
    p = [x.ptr for x in b]
    good = [*p[:5], 4, p[5], p[6], 2, p[7], p[8]]

    def refused(error, at, value):
        args = list(good)
        args[at] = value
        with pytest.raises(error):
            h.run(*args)

    for at in (0, 1, 2, 3, 4, 6, 7, 9):
        refused(InvalidArgument, at, 0)
    for at, value in ((5, 5), (5, -1), (8, -1), (8, 2 ** 31 - 1)):
        refused(ShapeInvalid, at, value)
    for at, by in ((0, 2), (1, 8), (2, 8), (9, 4)):
        refused(LayoutUnsupported, at, p[at if at < 5 else 7] + by)
    h.run(*p[:5], 0, p[5], p[6], 2, p[7], p[8])  # nothing to do
    h.close()
    for x in b:
        x.free()


def test_prefix_longer_than_a_row_of_masks_and_stages(backend):
    """Runs of one tile between long ones: stages are released in order whatever the steps of an item."""
    run_groups([(x, [1] * m) for x, m in ((64, 2), (200, 40), (64, 2), (500, 2), (90, 70), (64, 3), (64, 2), (300, 9)) for _ in range(8)], hq=2, hkv=2)


@pytest.mark.parametrize("page,cache", [(16, BF16), (20, BF16), (16, E4M3)])
def test_prefix_offsets_past_32_bits(backend, page, cache):
    """Pages 2^28 bytes apart or more: the last of 18 lies past 2^32 bytes."""
    s = make_groups([(page * 3, [1, 2, 5])], 4, 2, 64, page, "NHD", BF16, cache, 9)
    stride = (1 << 28) // cache.size
    tight = page * 2 * 64
    small = s["pages"]
    number = np.array([17, 3, 16, 0, 9, 15, 2, 12, 5, 7, 11, 14, 1, 4, 6, 8, 10, 13][:small])
    kv = []
    for c in s["kv"]:
        big = empty(cache.size * (17 * stride + tight), None)
        for i in range(small):
            call("mf_memcpy_h2d_async", big.ptr + cache.size * int(number[i]) * stride, c[i].ctypes.data, c[i].nbytes, None)
        sync_device()
        kv.append(big)
    table = np.where((s["table"] >= 0) & (s["table"] < small), number[np.clip(s["table"], 0, small - 1)], s["table"]).astype(np.int32)
    layout = paged.CacheLayout(18, page, 2, 64, cache, "NHD")
    layout.struct.page_stride = stride
    b = [to_device(a) for a in (s["q"], table, s["lens"], s["starts"], s["shared"])]
    sc = to_device(s["scales"]) if s["scales"] is not None else None
    out, lse = empty(2 * 3 * 4 * 64), empty(4 * 3 * 4)
    with paged.PrefixAttention(layout, 4, BF16, table.shape[1], 3, k_scale_inv=sc.ptr if sc else 0, v_scale_inv=sc.ptr + 8 if sc else 0,
                               always=True) as attn:
        attn.run(b[0].ptr, kv[0].ptr, kv[1].ptr, b[1].ptr, b[2].ptr, 3, b[3].ptr, b[4].ptr, 1, out.ptr, lse.ptr)
        sync_device()
    assert device_status() == 0
    check_prefix(s, (fetch(out, out.nbytes, np.uint16).reshape(3, 4, 64), fetch(lse, lse.nbytes, np.float32).reshape(3, 4)), want_attn(s))
    for t in (*kv, *b, out, lse, *([sc] if sc else [])):
        t.free()


def test_prefix_padded_tables_and_caches(backend):
    """Table rows and pages that are longer than what they hold; the gaps hold NaN codes."""
    hq, hkv, dim, page = 4, 2, 64, 16
    s = make_groups([(100, [1, 45, 0]), (30, [3, 4])], hq, hkv, dim, page, "NHD", BF16, BF16, 4)
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
    b = [to_device(x) for x in (s["q"], table, s["lens"], s["starts"], s["shared"])]
    out, lse = empty(2 * n * hq * dim), empty(4 * n * hq)
    with paged.PrefixAttention(layout, hq, BF16, width, n, table_stride=width + 5, always=True) as attn:
        attn.run(b[0].ptr, kv[0].ptr, kv[1].ptr, b[1].ptr, b[2].ptr, n, b[3].ptr, b[4].ptr, 2, out.ptr, lse.ptr)
        sync_device()
    assert device_status() == 0
    check_prefix(s, (fetch(out, out.nbytes, np.uint16).reshape(n, hq, dim), fetch(lse, lse.nbytes, np.float32).reshape(n, hq)), want_attn(s))
    for t in (*b, *kv, out, lse):
        t.free()


@pytest.mark.parametrize("cache", [BF16, E4M3])
def test_prefix_captured_replays_with_other_groups(backend, cache):
    """Captured once; each replay serves the lengths, groups and shared tokens that are there then."""
    import torch

    cases = [make_groups(g, 8, 2, 128, 16, "HND", BF16, cache, 3) for g in
             ([(200, [1, 2, 3]), (40, [4, 5, 6, 7])], [(0, [9, 8, 7, 1]), (260, [1, 2, 0])], [(64, [1] * 2), (100, [2] * 5)])]
    most = max(s["pages"] for s in cases), max(s["table"].shape[1] for s in cases)
    for s in cases:  # one shape for all
        s["table"] = np.pad(s["table"], ((0, 0), (0, most[1] - s["table"].shape[1])), constant_values=1 << 30)
        s["kv"] = [np.concatenate([c, np.zeros((most[0] - len(c), *c.shape[1:]), c.dtype)]) for c in s["kv"]]
        s["pages"], s["scales"] = most[0], cases[0]["scales"]
    on = Running(cases[0])
    stream = torch.cuda.Stream()
    p = [b.ptr for b in on.bufs]

    def launch():
        on.attn.run(*p[:5], 7, p[5], p[6], 2, on.out.ptr, on.lse.ptr, stream=stream.cuda_stream)

    launch()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        launch()
    for s in cases[::-1]:
        kv = [np.ascontiguousarray(c.transpose(0, 2, 1, 3)) for c in s["kv"]]
        for b, x in zip(on.bufs, (s["q"], kv[0], kv[1], s["table"], s["lens"], s["starts"], s["shared"])):
            b.upload(np.ascontiguousarray(x))
        sync_device()
        graph.replay()
        torch.cuda.synchronize()
        check_prefix(s, (fetch(on.out, 7 * 8 * 128 * 2, np.uint16).reshape(7, 8, 128), fetch(on.lse, 7 * 8 * 4, np.float32).reshape(7, 8)), want_attn(s))
    assert device_status() == 0
    del graph
    on.close()


def test_prefix_destroyed_while_its_runs_are_queued(backend):
    s = make_groups([(3000, [1] * 40)], 8, 2, 128, 16, "HND", BF16, BF16, 3)
    on, st = Running(s), Stream()
    p = [b.ptr for b in on.bufs]
    for _ in range(30):
        on.attn.run(*p[:5], 40, p[5], p[6], 1, on.out.ptr, on.lse.ptr, stream=st)
    on.attn.close()
    got = fetch(on.out, 40 * 8 * 128 * 2, np.uint16).reshape(40, 8, 128), fetch(on.lse, 40 * 8 * 4, np.float32).reshape(40, 8)
    check_prefix(s, got, want_attn(s))
    on.close()
    st.close()


NAN = {BF16: 0x7FC0, F16: 0x7E00, E4M3: 0x7F, E5M2: 0x7F}
INF = {BF16: 0x7F80, F16: 0x7C00, E4M3: 0x7F, E5M2: 0x7C}  # E4M3 has none


@pytest.mark.parametrize("hq,hkv,dim", [(4, 2, 64), (16, 1, 72), (16, 2, 128), (32, 1, 128), (4, 2, 256)])
@pytest.mark.parametrize("dtype,cache", TYPES)
def test_prefix_values_that_a_member_does_not_see(backend, hq, hkv, dim, dtype, cache):
    """Infinities and NaN among the shared tokens stay with the members that see them: 4, 2 or 1 warps for a row's tokens,
    both groups of warps with rows of their own, one group."""
    if cache in plain.FP8 and dim % 16:
        dim = 80
    s = make_groups([(300, [5, -1, -171, -300, 0, 20]), (140, [3, 0])], hq, hkv, dim, 16, "HND", dtype, cache, 5)
    head, at = hkv - 1, 2

    def put(part, token, number):
        for r in range(6):  # all of them have the token in the leader's page, or in a copy
            if s["lens"][r] > token or r == 0:
                s["kv"][part][s["table"][r, token // 16], token % 16, head, at] = number[cache]

    put(1, 131, INF)
    put(1, 290, NAN)
    on = Running(s)
    device_status()
    out, lse = on.run()
    again = on.run()
    assert device_status() == 0
    on.close()
    bits_equal(out, again[0])
    bits_equal(lse.view(np.uint32), again[1].view(np.uint32))
    want = [x.copy() for x in want_attn(s)]
    sees = np.zeros(out.shape, bool)
    sees[np.ix_([r for r in range(6) if s["lens"][r] > 131], range(head * (hq // hkv), hq), [at])] = True
    assert not np.isfinite(want[0][sees]).any() and not np.isfinite(plain.values(out, dtype)[sees]).any()
    out[sees] = 0
    want[0][sees] = want[2][sees] = 0
    check_prefix(s, (out, lse), want)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (BF16, E4M3), (F16, E5M2)])
@pytest.mark.parametrize("part", [0, 1])
def test_prefix_values_that_no_member_sees(backend, dtype, cache, part):
    """Behind every member's length, and in front of every member's window: whatever is there."""
    s = make_groups([(300, [-40, -60, -50])], 4, 2, 64, 16, "HND", dtype, cache, 5)
    for token in (260, 299):
        s["kv"][part][s["table"][0, token // 16], token % 16] = NAN[cache]
    for token in (0, 77):
        s["kv"][part][s["table"][0, token // 16], token % 16] = INF[cache]
    on = Running(s, window=100)
    device_status()
    got = on.run()
    assert device_status() == 0
    on.close()
    check_prefix(s, got, want_attn(s, window=100))


def test_prefix_finite_again_after_values_that_were_not(backend):
    """What one call finds counts for that call alone."""
    s = make_groups([(300, [5, -171, 0])], 4, 2, 64, 16, "NHD", BF16, BF16, 5)
    on = Running(s)
    first = on.run()
    page, at = s["table"][0, 200 // 16], 200 % 16
    wild = s["kv"][1].copy()
    wild[page, at, 0, 7] = NAN[BF16]
    on.bufs[2].upload(wild)
    assert np.isnan(plain.values(on.run()[0], BF16)).sum() == 2 * 2  # two members see it, in two heads
    on.bufs[2].upload(s["kv"][1])
    last = on.run()
    on.close()
    bits_equal(first[0], last[0])
    bits_equal(first[1].view(np.uint32), last[1].view(np.uint32))


@pytest.mark.parametrize("rules", [{}, {"window": 40}, {"slopes": [0.5, 0.25, 0.125, 0.0625]}])
def test_prefix_lengths_past_the_table(backend, rules):
    """Lengths count as no more than the table's rows hold, for windows and slopes too."""
    s = make_groups([(64, [32, 32])], 4, 2, 64, 16, "HND", BF16, BF16, 5)
    s["table"] = np.ascontiguousarray(s["table"][:, :6])
    on = Running({**s, "lens": np.array([96, 96 + 500], np.int32)}, **rules)
    got = on.run()
    on.close()
    check_prefix(s, got, want_attn(s, **rules))


WILD = 1 << 30
TIMEOUT = 0x7100


@pytest.mark.parametrize("own", [[-300, 5, -1, 0], [-170, -300, 9], [-40, -60, -50], [-60, -40, -40], [-299, -300], [-300, -300, -300],
                                 [-300] * 40 + [3] * 5, [-1] * 150 + [0] * 2])
@pytest.mark.parametrize("dim,cache", [(64, BF16), (128, E4M3), (256, BF16)])
def test_prefix_rows_of_the_table_name_what_their_request_has(backend, own, dim, cache):
    """Idle and shorter requests in front: nothing behind a request's own length is read of its row."""
    s = make_groups([(300, own), (64, [0, 2])], 4, 2, dim, 16, "HND", BF16, cache, 5)
    want = want_attn(s)
    for r, n in enumerate(s["lens"]):
        s["table"][r, -(-max(n, 0) // 16):] = WILD
    on = Running(s)
    device_status()
    got = on.run()
    assert device_status() == 0
    on.close()
    check_prefix(s, got, want)


@pytest.mark.parametrize("window", [1, 100, 250])
def test_prefix_pages_in_front_of_every_window_are_not_read(backend, window):
    s = make_groups([(300, [-40, 7, -300, 0, 30])], 4, 2, 64, 16, "HND", BF16, BF16, 5)
    want = want_attn(s, window=window)
    s["table"][:, :(260 - window) // 16] = WILD
    s["table"][2] = WILD
    on = Running(s, window=window)
    device_status()
    got = on.run()
    assert device_status() == 0
    on.close()
    check_prefix(s, got, want)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, E4M3)])
def test_prefix_shared_where_it_pays(backend, dtype, cache):
    """Large groups beside small ones; small ones alone; the same where all are shared, or none."""
    for groups in ([(3000, [2] * 60), (20, [1, 2]), (1900, [3] * 70), (700, [1, 0, 5])], [(48, [1, 2])] * 9):
        s = make_groups(groups, 8, 4, 128, 16, "HND", dtype, cache, 3, alone=2)
        want = want_attn(s)
        for always in (True, False):
            on = Running(s, always=always)
            device_status()
            got, none = on.run(), on.run(groups=0)
            assert device_status() == 0
            on.close()
            check_prefix(s, got, want)
            check_prefix(s, none, want)
            if not always and len(groups) == 9:  # too small: as if there were no groups, to the bit
                bits_equal(got[0], none[0])


def test_prefix_share_refusals(backend):
    s = make_groups([(20, [1, 2])], 4, 2, 64, 16, "HND", BF16, BF16, 3)
    on = Running(s)
    for always in (-1, 2):
        with pytest.raises(InvalidArgument):
            call("mf_prefix_attn_share", on.attn._handle, always)
    on.close()
    with pytest.raises(InvalidArgument):
        call("mf_prefix_attn_share", None, 1)


@pytest.mark.parametrize("groups,hq,hkv,dim,dtype,cache",
                         [([(3000, [2] * 40), (700, [1, 0, 5])], 8, 2, 128, BF16, BF16), ([(900, [1] * 9)], 4, 2, 64, F16, E4M3),
                          ([(500, [3] * 70), (64, [1, 2])], 8, 1, 128, BF16, E4M3), ([(900, [1, 2])], 4, 1, 256, F16, F16)])
def test_prefix_waits_that_run_out_are_reported(backend, groups, hq, hkv, dim, dtype, cache):
    """With no time to wait every role goes on at once, the producers before any row is known.  What they copy then are rows of the
    cache or nothing; the status tells, and the next run is right."""
    s = make_groups(groups, hq, hkv, dim, 16, "HND", dtype, cache, 3)
    want = want_attn(s)
    on = Running(s)
    for _ in range(2):
        device_status()
        call("mf_prefix_attn_limit", on.attn._handle, 0)
        on.run()
        assert device_status() == TIMEOUT
        call("mf_prefix_attn_limit", on.attn._handle, 2 * 10 ** 9)
        got = on.run()
        assert device_status() == 0
        check_prefix(s, got, want)
    on.close()


def test_prefix_without_time_to_wait_what_is_not_shared_is_right(backend):
    s = make_groups([(90, [1, 2]), (40, [3])], 4, 2, 64, 16, "HND", BF16, BF16, 3, alone=2)
    for always, groups in ((True, 0), (False, None)):
        on = Running(s, always=always)
        call("mf_prefix_attn_limit", on.attn._handle, 0)
        device_status()
        got = on.run(groups=groups)
        assert device_status() == 0
        on.close()
        check_prefix(s, got, want_attn(s))


def test_prefix_limit_refusals(backend):
    s = make_groups([(20, [1, 2])], 4, 2, 64, 16, "HND", BF16, BF16, 3)
    on = Running(s)
    for ns in (-1, 2 ** 32):
        with pytest.raises(InvalidArgument):
            call("mf_prefix_attn_limit", on.attn._handle, ns)
    on.close()
    with pytest.raises(InvalidArgument):
        call("mf_prefix_attn_limit", None, 1)


# ------------------------------------------------------------------ precision, and the choice of what is shared

def digits(x, n):
    """x, multiples of 8^-(n - 1) below 8, as n digits of 3 bits, the largest first."""
    y = np.round(np.asarray(x) * 8.0 ** (n - 1)).astype(np.int64)
    assert (y / 8.0 ** (n - 1) == x).all() and (y >= 0).all() and (y < 8 ** n).all()
    return np.stack([y >> 3 * (n - 1 - j) & 7 for j in range(n)], -1).astype(np.float32)


def one_for_all(tokens, values, q, keys, requests, hq, dtype, cache, shared):
    """Requests of the same tokens, all in the same pages (one key-value head); each token's value is one number."""
    n, dim = keys.shape
    s = make_attn([n], hq, 1, dim, 16, "HND", dtype, cache, 5)
    tok = np.arange(n)
    s["kv"][0][s["table"][0, tok // 16], tok % 16, 0] = plain.codes(keys, cache)
    s["kv"][1][s["table"][0, tok // 16], tok % 16, 0] = plain.codes(np.repeat(values[:, None], dim, 1), cache)
    if s["scales"] is not None:
        s["scales"][:] = 1.0
    s["q"] = np.ascontiguousarray(np.broadcast_to(plain.codes(q, dtype), (requests, hq, dim)))
    s["table"] = np.repeat(s["table"], requests, 0)
    s["lens"] = np.array(tokens, np.int32)
    s["starts"], s["shared"] = np.array([0, requests], np.int32), np.array([shared], np.int32)
    return s


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("requests", [2, 20, 70])
def test_prefix_weights_are_good_to_the_bound_without_sharing(backend, dtype, cache, requests):
    """63 tokens of value 1 and 63 of -1 whose weights lie on either side of the middle between two f16 numbers, a half of the
    largest: rounded to f16 alone they are 2^-11 off, up and down, and so is the result.  A row's tokens among 4, 2 and 1 warps."""
    n, dim = 129, 64
    middle = 1.0 - np.log(2.0) + np.log1p(2.0 ** -11)
    below, above = np.floor(middle * 2.0 ** 15) / 2.0 ** 15, (np.floor(middle * 2.0 ** 15) + 2) / 2.0 ** 15
    score, value = np.zeros(n), np.zeros(n, np.float32)
    score[0] = 1.0
    score[1:127:2], value[1:127:2] = below, 1.0
    score[2:127:2], value[2:127:2] = above, -1.0
    keys, q = np.zeros((n, dim), np.float32), np.zeros(dim, np.float32)
    keys[:, :6], q[:6] = digits(score, 6), 8.0 ** -np.arange(6)
    s = one_for_all([n] * requests, value, q, keys, requests, 2, dtype, cache, 128)
    on = Running(s, scale=1.0)
    got = on.run()
    on.close()
    want = want_attn(s, scale=1.0)
    assert np.abs(want[0]).max() < 1e-4 and want[2].min() > 0.9
    check_attn(s, got, want)


@pytest.mark.parametrize("dtype,cache", [(BF16, BF16), (F16, F16), (F16, E4M3), (BF16, E5M2)])
def test_prefix_own_tokens_join_at_large_scores(backend, dtype, cache):
    """Scores of 28672 powers of two and a few: exact products (scale * log2(e) is 1), so that only what the parts are joined by can
    lose bits.  Shared tokens have value 1, own ones -1."""
    dim, rng = 64, np.random.default_rng(3)
    lens = [128 + x for x in (100, 128, 37, 77, 1, 112, 90, 63, 128, 120, 99, 101)]
    n = max(lens)
    keys, q = np.zeros((n, dim), np.float32), np.zeros(dim, np.float32)
    keys[:, 0], q[0] = 224.0, 128.0
    keys[:, 1:4], q[1:4] = digits(rng.integers(0, 3 * 64, n) / 64.0, 3), 8.0 ** -np.arange(3)
    value = np.where(np.arange(n) < 128, 1.0, -1.0).astype(np.float32)
    s = one_for_all(lens, value, q, keys, len(lens), 2, dtype, cache, 128)
    scale = float(np.float32(np.log(2.0)))
    on = Running(s, scale=scale)
    got, alone = on.run(), on.run(groups=0)
    on.close()
    want = want_attn(s, scale=scale)
    check_attn(s, alone, want)  # the bound holds where nothing is joined
    check_attn(s, got, want)


def crowd(lens, shared, cache=BF16):
    """Requests over one text of 2000 tokens and some; 4 key-value heads of 64."""
    s = make_attn([2040], 8, 4, 64, 16, "HND", BF16, cache, 9)
    s["table"] = np.repeat(s["table"], len(lens), 0)
    s["lens"] = np.array(lens, np.int32)
    s["q"] = plain.normal(12, (len(lens), 8, 64), BF16)
    s["starts"], s["shared"] = np.array([0, len(lens)], np.int32), np.array([shared], np.int32)
    return s


CROWDS = {"all see it": ([2001 + i % 30 for i in range(160)], 2000, 0, True),
          "a window of half of it": ([2001 + i % 30 for i in range(400)], 2000, 1000, True),
          "a small window": ([2001 + i % 30 for i in range(160)], 2000, 64, False),
          "a window behind it": ([2040] * 160, 1900, 140, False),
          "idle rows": ([0] * 70 + [2010, 2003] + [-1] * 88, 2000, 0, False),
          "ended rows in front": ([40] * 150 + [2010] * 10, 2000, 0, False),
          "shared past every length": ([30 + i % 9 for i in range(160)], 2000, 0, False)}


@pytest.mark.parametrize("which", CROWDS)
def test_prefix_rule_counts_what_requests_see(backend, which):
    """Tokens are shared where that saves reading them, not where few of the requests, or of the tokens, are left."""
    lens, common, window, pays = CROWDS[which]
    s = crowd(lens, common)
    want = want_attn(s, window=window)
    on = Running(s, window=window, always=False)
    device_status()
    got, none = on.run(), on.run(groups=0)
    assert device_status() == 0
    on.close()
    check_attn(s, got, want)
    check_attn(s, none, want)
    same = (got[1].view(np.uint32) == none[1].view(np.uint32)).all()
    assert same != pays  # 64-bit sums in another order: some of a thousand log-sums differ in their last bit
    if not pays:
        bits_equal(got[0], none[0])
