"""Beam selection, page forks, compaction and copies on the GPU against plain forms."""
import ctypes
import math

import numpy as np
import pytest

from manifesto_b200 import DeviceBuffer, Stream, beams, paged, sync_device
from manifesto_b200._abi import call
from manifesto_b200.dtype import DType
from manifesto_b200.errors import (DeviceStickyError, DTypeUnsupported, InvalidArgument, LayoutUnsupported, ShapeInvalid,
                                   ShapeMismatch, TensorClosed)

from . import beams_ref as plain
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


# ------------------------------------------------------------------ selection

def stored(x, dtype):
    """x as the dtype holds it: the bits to upload, and their values in float64."""
    x = np.asarray(x, np.float32)
    if dtype == F32:
        return x, x.astype(np.float64)
    if dtype == F16:
        h = x.astype(np.float16)
        return h, h.astype(np.float64)
    # bf16: to nearest even (NaN stays one)
    u = x.view(np.uint32)
    bits = np.where(np.isnan(x), 0x7fc0, (u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return bits, (bits.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def run_select(logits, scores, beams_, n_out, dtype=BF16, ended=None, end=-1, stride=None, offset=0, stream=None, max_batch=None,
               handle=None):
    logits = np.asarray(logits, np.float32)
    rows, vocab = logits.shape
    batch = rows // beams_
    stride = vocab if stride is None else stride
    bits, values = stored(logits, dtype)
    wide = np.full((rows, stride), np.array(np.nan, np.float32).astype(np.float16) if dtype == F16 else 0x7fc0 if dtype == BF16 else np.nan,
                   bits.dtype)
    wide[:, :vocab] = bits
    flat = np.concatenate([np.zeros(offset, bits.dtype), wide.reshape(-1)])
    scores = np.asarray(scores, np.float32)
    want = plain.select(values, scores, ended, beams_, n_out, end)
    h = handle or beams.BeamSelect(dtype, vocab, beams_, n_out, max_batch or batch, stride, end)
    src, sc = to_device(flat), to_device(scores)
    en = to_device(np.asarray(ended, np.int32)) if ended is not None else None
    outs = [empty(batch * n_out * 4 + 16) for _ in range(4)]
    for _ in range(2):  # the tickets are back at zero
        h.run(src.ptr + offset * bits.itemsize, sc.ptr, batch, outs[0].ptr, outs[1].ptr, outs[2].ptr, en.ptr if en else 0,
              outs[3].ptr, stream)
    sync_device()
    got = []
    for o, t in zip(outs, (np.float32, np.int32, np.int32, np.int32)):
        raw = fetch(o, batch * n_out * 4 + 16)
        assert (raw[-16:] == 0xA5).all(), "wrote past an output"
        got.append(raw[:-16].view(t).reshape(batch, n_out))
    if handle is None:
        h.close()
    for b in (src, sc, *outs, *([en] if en else [])):
        b.free()
    bits_equal(got[1], want[1].astype(np.int32))
    bits_equal(got[2], want[2].astype(np.int32))
    bits_equal(got[3], want[3].astype(np.int32))
    there = np.isfinite(want[0])
    assert np.array_equal(np.isfinite(got[0]), there)
    # one float32 rounding of the score (2^-24 of it), and the sum's relative error: each term is good to 2^-22, its exponent's
    # argument to 2^-23 of up to 2^5 octaves that still count, 2^-18; a sum of up to 2^5 float32 terms adds 2^-19
    bound = np.abs(want[0][there]) * 2.0 ** -24 + 2.0 ** -17
    assert (np.abs(got[0][there] - want[0][there]) <= bound).all()
    return got


def logits_of(rows, vocab, seed, std=2.5, gap=True):
    """Normal logits; `gap`: of values far enough apart that beams' scores do not meet by chance."""
    return np.random.default_rng(seed).normal(0, std, (rows, vocab)).astype(np.float32)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 31, 2048, 2049, 8191, 8193, 20011])
def test_select_vocabularies(backend, dtype, vocab):
    rng = np.random.default_rng(vocab)
    for batch, k in ((1, 1), (3, 4)):
        run_select(logits_of(batch * k, vocab, vocab + k), -rng.random(batch * k) * 3 - 5, k, 2 * k, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("batch,k,n", [(1, 16, 32), (90, 4, 8), (7, 5, 10), (2, 64, 64), (1, 3, 128), (40, 9, 33), (1, 1, 1)])
def test_select_batches_and_beams(backend, dtype, batch, k, n):
    """Both sizes of chunk, lists of up to 32 results and longer ones."""
    rng = np.random.default_rng(batch)
    run_select(logits_of(batch * k, 9001, batch + n), -rng.random(batch * k) * 2 - 30, k, n, dtype)


@pytest.mark.parametrize("batch,k,vocab", [(1, 8, 60000), (3, 4, 30011), (1, 1, 120000), (2, 3, 4100)])
@pytest.mark.parametrize("n", [2, 8, 16, 31, 32, 33, 100, 128])
def test_select_merges_many_lists(backend, batch, k, vocab, n):
    """Rows in many segments; beams near one another, one far ahead, one that has ended."""
    rng = np.random.default_rng(n + k)
    logits = rng.normal(0, 3, (batch * k, vocab))
    run_select(logits, rng.normal(-20, 1, batch * k), k, n, F16)
    scores = rng.normal(-40, 5, batch * k)
    scores[::k] = -3.0
    ended = np.zeros(batch * k, np.int32)
    ended[k - 1::k] = 1
    run_select(logits, scores, k, n, F16, ended=ended, end=5)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("pad,offset", [(0, 1), (1, 0), (5, 3), (8, 8), (3, 7)])
def test_select_row_strides_and_alignment(backend, dtype, pad, offset):
    """What lies between the rows is NaN and not read into them."""
    run_select(logits_of(6, 5003, pad), -np.arange(6) * 0.3, 3, 6, dtype, stride=5003 + pad, offset=offset)


def test_select_equal_logits_go_by_index(backend):
    """All alike: the lowest beams and tokens; the chunk's and the entry's lists are longer than what is ranked at once."""
    for vocab in (50, 20000):
        run_select(np.full((8, vocab), 1.5), np.zeros(8), 4, 8)
        run_select(np.full((8, vocab), 1.5), np.zeros(8), 8, 40)
    run_select(np.full((40, 30000), -2.0), np.zeros(40), 40, 100, F32)


def test_select_few_values(backend):
    """Many ties: logits of four values, and of one value but for a few."""
    rng = np.random.default_rng(3)
    run_select(rng.integers(0, 4, (6, 20000)).astype(np.float32), [0, 0, 0, -1, -1, -1], 3, 20)
    x = np.zeros((4, 20000), np.float32)
    x[:, 17::4000] = 3.0
    run_select(x, [0, 0, -2, -2], 2, 12)
    run_select(x, [0, 0, -2, -2], 2, 50)


@pytest.mark.parametrize("where", ["first", "last", "ascending"])
def test_select_best_tokens_together(backend, where):
    """The best of a row in one thread's logits, or in order."""
    x = logits_of(4, 16384, 9, std=0.5)
    if where == "ascending":
        x[:] = np.linspace(-5, 5, 16384, dtype=np.float32)
        x += np.arange(4, dtype=np.float32)[:, None] * 1e-3
        run_select(x, -np.arange(4.0), 4, 24, F32)
        return
    at = slice(0, 24) if where == "first" else slice(-24, None)
    x[:, at] = 20.0 + np.arange(24) * 0.25
    run_select(x, -np.arange(4) * 1.1, 4, 24)


def test_select_masked_logits(backend):
    """-inf is no candidate; rows without one, and entries with fewer than were asked for."""
    x = logits_of(8, 3000, 4)
    x[:, ::2] = -np.inf
    x[1] = -np.inf
    x[4:8] = -np.inf
    x[5, 77] = 2.0
    x[6, [3, 2999]] = [1.0, -1.0]
    run_select(x, -np.arange(8.0), 4, 8)
    run_select(np.full((4, 100), -np.inf), np.zeros(4), 2, 3)
    lowest = np.where(np.arange(3000)[None] % 5 == 0, logits_of(4, 3000, 5), np.finfo(np.float32).min).astype(np.float32)
    run_select(lowest, np.zeros(4) - 1, 2, 4, F32)


def test_select_rows_that_are_not_finite_offer_nothing(backend):
    for bad in (np.nan, np.inf, -np.nan):
        for at in (0, 1234, 8999):
            x = logits_of(6, 9000, 6)
            x[1, at] = bad
            x[5, at] = bad
            for dtype in (BF16, F16, F32):
                run_select(x, -np.arange(6.0), 3, 6, dtype)


def test_select_scores_that_are_not_finite_offer_nothing(backend):
    """-inf: a beam that is not in use, as at the first step."""
    run_select(logits_of(6, 4000, 7), [0, -np.inf, -np.inf, np.nan, -1, np.inf], 3, 6)
    run_select(logits_of(6, 4000, 8), [0, -np.inf, -np.inf] * 2, 3, 6, ended=[0, 1, 0, 0, 0, 1], end=3)


def test_select_ended_beams(backend):
    """They go on by the end's token alone, with their score; their logits are not read."""
    x = logits_of(9, 5000, 10)
    x[1] = np.nan
    x[4] = np.inf
    x[8] = -np.inf
    got = run_select(x, [-1, -2, -30, -7, -7, -7, -3, -90, -4], 3, 6, ended=[0, 1, 0, 0, 5, 0, 1, 1, 1], end=4999)
    assert (got[3][2] == [1, 1, 1, 0, 0, 0]).all() and (got[1][2] == [4999] * 3 + [-1] * 3).all()
    run_select(logits_of(4, 300, 11), [-1, -1, -1, -1], 2, 4, ended=[1, 1, 1, 1], end=0)  # of equal scores the lowest beam


def test_select_end_token_reached(backend):
    x = logits_of(2, 1000, 12)
    x[0, 5] = 30.0
    got = run_select(x, [0, 0], 2, 3, end=5)
    assert got[3][0, 0] == 1 and got[1][0, 0] == 5


def test_select_large_and_small_logits(backend):
    x = logits_of(4, 6000, 13)
    run_select(x * 1e4, [0, -1e4, 3, 4], 2, 5, F32)
    run_select(x * 1e-6 + 1e3, [0, -1e-3, 3, 4], 2, 5, F32)
    run_select(x + 80, [-1e5, -1e5 - 1, 0, 0], 2, 5)


def test_select_handle_serves_any_batch(backend):
    h = beams.BeamSelect(BF16, 12345, 2, 5, 700)
    for batch in (700, 1, 60, 299, 300, 1):
        run_select(logits_of(batch * 2, 12345, batch), -np.random.default_rng(batch).random(batch * 2) * 4, 2, 5, handle=h)
    h.close()
    with pytest.raises(TensorClosed):
        h.run(1, 1, 1, 1, 1, 1)


def test_select_two_handles_on_two_streams(backend):
    streams, handles = [Stream(), Stream()], [beams.BeamSelect(BF16, 30000, 4, 8, 20) for _ in range(2)]
    inputs = [(to_device(stored(logits_of(80, 30000, i), BF16)[0]), to_device(np.full(80, -1.0, np.float32))) for i in range(2)]
    outs = [[empty(20 * 8 * 4) for _ in range(3)] for _ in range(2)]
    sync_device()
    for _ in range(20):
        for s, h, (x, sc), o in zip(streams, handles, inputs, outs):
            h.run(x.ptr, sc.ptr, 20, *(b.ptr for b in o), stream=s)
    sync_device()
    for i in range(2):
        want = plain.select(stored(logits_of(80, 30000, i), BF16)[1], np.full(80, -1.0), None, 4, 8, -1)
        assert np.array_equal(fetch(outs[i][1], 640, np.int32).reshape(20, 8), want[1])
        assert np.array_equal(fetch(outs[i][2], 640, np.int32).reshape(20, 8), want[2])
    for h in handles:
        h.close()
    for s in streams:
        s.close()


def test_select_refusals(backend):
    ok = dict(dtype=BF16, vocab=100, beams=4, n_out=4, max_batch=2)
    for change, error in (({"dtype": E4M3}, DTypeUnsupported), ({"vocab": 0}, ShapeInvalid), ({"beams": 0}, ShapeInvalid),
                          ({"beams": 1025}, ShapeInvalid), ({"beams": 4, "vocab": 1 << 29}, ShapeInvalid), ({"n_out": 0}, ShapeInvalid),
                          ({"n_out": 129}, ShapeInvalid), ({"max_batch": 0}, ShapeInvalid), ({"row_stride": 99}, ShapeMismatch),
                          ({"end_token": 100}, InvalidArgument), ({"end_token": -2}, InvalidArgument),
                          ({"max_batch": 1 << 30}, ShapeInvalid)):
        with pytest.raises(error):
            beams.BeamSelect(**{**ok, **change})
    h = beams.BeamSelect(**ok)
    b = [empty(4096) for _ in range(6)]
    p = [x.ptr for x in b]
    good = [p[0], p[1], 2, p[2], p[3], p[4]]

    def refused(error, at, value):
        args = list(good)
        args[at] = value
        with pytest.raises(error):
            h.run(*args)

    for at in (0, 1, 3, 4, 5):
        refused(InvalidArgument, at, 0)
    refused(ShapeInvalid, 2, 3)
    refused(ShapeInvalid, 2, -1)
    refused(LayoutUnsupported, 0, p[0] + 1)
    refused(InvalidArgument, 3, p[1])
    with pytest.raises(InvalidArgument):
        h.run(*good, ended=p[5])  # without an end token
    h.run(p[0], p[1], 0, p[2], p[3], p[4])  # nothing to do
    h.close()
    for x in b:
        x.free()


# ------------------------------------------------------------------ page tables

def family_book(n, page, width, pages, longest, seed, spare_head=3, count=None):
    """Rows in families of four that share their first pages, in a shuffled cache."""
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, longest + 1, n)
    table, shares, number, at = np.full((n, width), -1, np.int32), np.zeros(pages, np.int32), rng.permutation(pages), 0
    for r in range(n):
        held, common = -(-int(lens[r]) // page), 0
        if r % 4:
            lead = r - r % 4
            common = int(min(lens[r], lens[lead]) // page) // 2
            table[r, :common] = table[lead, :common]
            shares[table[r, :common]] += 1
        table[r, common:held] = number[at:at + held - common]
        at += held - common
    assert at <= pages
    free = np.full(pages, -5, np.int32)
    left = number[at:]
    count = len(left) if count is None else count
    head = spare_head if spare_head + count <= pages else 0
    free[head:head + count] = left[:count]
    return lens.astype(np.int32), table, shares, free, np.array([head, count], np.int32)


def run_fork(lens, table, shares, free, pool, parents, page, stride=None, stream=None, handle=None):
    n, width = table.shape
    pages, rows = len(shares), len(parents)
    stride = width if stride is None else stride
    wide = np.full((n, stride), 12345678, np.int32)
    wide[:, :width] = table
    moves0, free0 = np.full((max(rows, 1), 4), -9, np.int32), np.full(pages, -9, np.int32)
    want = plain.fork(table, lens, parents, shares, free, pool, page, width, moves0[:rows], free0)
    h = handle or paged.PageBook(page, width, pages, max(n, rows, 1), stride)
    ins = [to_device(np.asarray(a, np.int32)) if np.size(a) else empty(4) for a in (wide, lens, parents, shares, free, pool)]
    outs = [to_device(np.full((rows, stride), -9, np.int32)), empty(4 * rows), empty(4 * pages), to_device(free0), empty(16), to_device(moves0)]
    for _ in range(2):  # a step can be planned again
        h.fork(ins[0].ptr, ins[1].ptr, n, ins[2].ptr, rows, ins[3].ptr, ins[4].ptr, ins[5].ptr, *(o.ptr for o in outs), stream=stream)
    sync_device()
    got = [fetch(o, s, np.int32) for o, s in zip(outs, (4 * rows * stride, 4 * rows, 4 * pages, 4 * pages, 16, 16 * rows))]
    after = got[0].reshape(rows, stride)
    assert (after[:, width:] == -9).all(), "wrote past the rows of the table"
    bits_equal(np.ascontiguousarray(after[:, :width]), want[0])
    for x, y in zip(got[1:5], want[1:5]):
        bits_equal(x, y)
    bits_equal(got[5].reshape(rows, 4), want[5])
    if handle is None:
        h.close()
    for b in (*ins, *outs):
        b.free()
    return want


@pytest.mark.parametrize("page", [1, 4, 16, 24])
def test_fork_small(backend, page):
    table = np.array([[5, 9, -1, -1], [3, -1, -1, -1], [0, 1, 2, 7], [-1, -1, -1, -1]], np.int32)
    lens = np.array([page + 1, 1, 4 * page, 0], np.int32)
    if page == 1:
        lens[0] = 2
    shares, free, pool = np.zeros(12, np.int32), np.array([4, 6, 8, 10, 11] + [0] * 7, np.int32), np.array([0, 5], np.int32)
    for parents in ([0, 1, 2, 3], [0, 0, 0, 2], [2, 2, 2, 2], [-1, -1, 1, 1], [3, 3, 0, 3], [1], [-1], [4, 99, -7], [1, 2, 1, 2, 1, 2, 0]):
        run_fork(lens, table, shares, free, pool, np.array(parents, np.int32), page)


def test_fork_nothing(backend):
    none = np.zeros((0, 4), np.int32)
    run_fork(np.zeros(0, np.int32), none, np.zeros(9, np.int32), np.arange(9, dtype=np.int32), np.array([2, 5], np.int32), np.zeros(0, np.int32), 16)
    run_fork(np.zeros(0, np.int32), none, np.zeros(9, np.int32), np.arange(9, dtype=np.int32), np.array([2, 5], np.int32), np.array([0, -1], np.int32), 16)
    table = np.array([[1, 2]], np.int32)
    run_fork(np.array([20], np.int32), table, np.zeros(9, np.int32), np.array([0, 3, 4, 5, 6, 7, 8, 0, 0], np.int32), np.array([0, 7], np.int32),
             np.zeros(0, np.int32), 16)


@pytest.mark.parametrize("n,rows,width,page", [(64, 64, 20, 16), (300, 257, 33, 7), (1000, 1500, 60, 4), (31, 2000, 100, 32), (2000, 3, 10, 1),
                                               (4000, 4000, 200, 2)])
def test_fork_families(backend, n, rows, width, page):
    """One CTA, a cluster, a grid; many children, few, none."""
    lens, table, shares, free, pool = family_book(n, page, width, n * width + 500, width * page, n)
    rng = np.random.default_rng(rows)
    parents = rng.integers(-1, n, rows)
    run_fork(lens, table, shares, free, pool, parents, page)
    run_fork(lens, table, shares, free, pool, np.sort(rng.integers(0, max(1, n // 3), rows)), page)
    run_fork(lens, table, shares, free, pool, np.arange(rows), page)


@pytest.mark.parametrize("count", [0, 1, 7, 40])
def test_fork_pool_runs_out(backend, count):
    """Pages that this call sets free are given out, too; later rows that find none begin empty and share nothing."""
    lens, table, shares, free, pool = family_book(60, 8, 12, 1000, 96, 5, count=count)
    rng = np.random.default_rng(count)
    run_fork(lens, table, shares, free, pool, rng.integers(0, 60, 60), 8)
    run_fork(lens, table, shares, free, pool, rng.integers(0, 10, 60), 8)
    want = run_fork(lens, table, shares, free, pool, np.repeat(np.arange(60), 2), 8)
    assert want[4][3] > 0


def test_fork_ends_rows(backend):
    """Rows left out: the pages that were theirs alone come back, shared ones stay with the others."""
    lens, table, shares, free, pool = family_book(40, 16, 10, 600, 160, 6)
    keep = np.array([r for r in range(40) if r % 3])
    want = run_fork(lens, table, shares, free, pool, keep, 16)
    assert want[4][1] > pool[1] and want[4][2] == 0
    want = run_fork(lens, table, shares, free, pool, np.full(5, -1), 16)
    assert want[4][1] == 600 and not want[2].any()  # nobody is left: every page is free


def test_fork_strides_streams_and_lengths_past_the_table(backend):
    lens, table, shares, free, pool = family_book(33, 5, 9, 500, 45, 7)
    s = Stream()
    run_fork(lens, table, shares, free, pool, np.random.default_rng(1).integers(0, 33, 50), 5, stride=13, stream=s)
    s.close()
    lens[3], lens[5] = 1 << 30, -4
    table[3, :] = free[pool[0]:pool[0] + 9]
    pool += np.array([9, -9], np.int32)
    run_fork(lens, table, shares, free, pool, np.array([3, 3, 5, 5, 2]), 5)


def test_fork_bad_pages_are_reported(backend):
    """A number outside the cache holds nothing and stays; so does a list of free pages that leaves its buffer."""
    table = np.array([[5, 99, -3], [3, 1, -1]], np.int32)
    lens, shares = np.array([40, 20], np.int32), np.zeros(8, np.int32)
    free, pool = np.array([0, 2, 4, 6, 7, 0, 0, 0], np.int32), np.array([0, 5], np.int32)
    device_status()
    run_fork(lens, table, shares, free, pool, np.array([1, 1]), 16)
    assert device_status() == BAD_PAGE
    run_fork(lens, table, shares, free, pool, np.array([0, 0]), 16)
    assert device_status() == BAD_PAGE
    run_fork(lens, table, shares, free, pool, np.array([1, 1, 1, 0]), 16)
    assert device_status() == 0
    good = np.array([[5, 1, -1], [3, -1, -1]], np.int32)
    run_fork(np.array([20, 16], np.int32), good, shares, free, np.array([6, 5], np.int32), np.array([0, 1, 0, 0]), 16)
    assert device_status() == BAD_PAGE


def test_fork_bad_pages_of_the_list_and_behind_full_ones(backend):
    """A page that is handed out, or the partly filled one that it is a copy of, outside the cache; one that nobody needs."""
    lens, shares = np.array([20, 16], np.int32), np.zeros(8, np.int32)
    table = np.array([[5, 1, -1], [3, -1, -1]], np.int32)
    device_status()
    for at, status in ((0, BAD_PAGE), (1, 0)):
        for wild in (8, 99, -1, -2 ** 31):
            free, pool = np.array([0, 2, 4, 6, 7, 0, 0, 0], np.int32), np.array([0, 5], np.int32)
            free[at] = wild
            run_fork(lens, table, shares, free, pool, np.array([0, 0, 1]), 16)
            assert device_status() == status
    free = np.array([0, 2, 4, 6, 7, 0, 0, 0], np.int32)
    for wild in (8, -1):
        table[0, 1] = wild
        run_fork(lens, table, shares, free, np.array([0, 5], np.int32), np.array([0, 0, 1]), 16)
        assert device_status() == BAD_PAGE
        run_fork(lens, table, shares, free, np.array([0, 5], np.int32), np.array([0, 1]), 16)
        assert device_status() == 0


def run_compact(lens, table, shares, free, pool, limit, page, stream=None, stride=None):
    n, width = table.shape
    pages = len(shares)
    stride = width if stride is None else stride
    wide = np.full((n, stride), 12345678, np.int32)
    wide[:, :width] = table
    moves0, free0 = np.full((max(1, pages // 2), 4), -9, np.int32), np.full(pages, -9, np.int32)
    want = plain.compact(table, lens, shares, free, pool, limit, page, width, moves0, free0)
    h = paged.PageBook(page, width, pages, max(n, 1), stride)
    ins = [to_device(np.asarray(a, np.int32)) if np.size(a) else empty(4) for a in (wide, lens, shares, free, pool)]
    outs = [to_device(np.full((n, stride), -9, np.int32)), empty(4 * pages), to_device(free0), empty(16), empty(4 * pages), to_device(moves0)]
    for _ in range(2):
        h.compact(ins[0].ptr, ins[1].ptr, n, ins[2].ptr, ins[3].ptr, ins[4].ptr, limit, *(o.ptr for o in outs), stream=stream)
    sync_device()
    got = [fetch(o, s, np.int32) for o, s in zip(outs, (4 * n * stride, 4 * pages, 4 * pages, 16, 4 * pages, 16 * len(moves0)))]
    after = got[0].reshape(n, stride)
    assert (after[:, width:] == -9).all(), "wrote past the rows of the table"
    bits_equal(np.ascontiguousarray(after[:, :width]), want[0])
    for x, y in zip(got[1:5], want[1:5]):
        bits_equal(x, y)
    bits_equal(got[5].reshape(-1, 4), want[5])
    h.close()
    for b in (*ins, *outs):
        b.free()
    return want


@pytest.mark.parametrize("n,width,page,pages", [(5, 4, 16, 33), (40, 10, 8, 1000), (300, 33, 7, 10000), (64, 8, 16, 64 * 8 + 1), (3000, 50, 4, 200001),
                                                (1, 1, 1, 1), (1, 1, 4, 2), (50, 20, 3, 70000)])
def test_compact_sizes(backend, n, width, page, pages):
    if n * width > pages:
        pages = n * width
    lens, table, shares, free, pool = family_book(n, page, width, pages, width * page, n)
    want = run_compact(lens, table, shares, free, pool, 0, page)
    used = pages - pool[1]
    assert want[0].max(initial=-1) < used
    for limit in (1, used, used + 1, (used + pages) // 2, pages - 1, pages, pages + 100):
        run_compact(lens, table, shares, free, pool, int(limit), page)


def test_compact_nothing(backend):
    none, lens = np.zeros((0, 4), np.int32), np.zeros(0, np.int32)
    run_compact(lens, none, np.zeros(50, np.int32), np.arange(50, dtype=np.int32)[::-1].copy(), np.array([0, 50], np.int32), 0, 16)
    full = np.arange(8, dtype=np.int32).reshape(2, 4)
    run_compact(np.array([64, 64], np.int32), full, np.zeros(8, np.int32), np.zeros(8, np.int32), np.array([0, 0], np.int32), 0, 16)
    # pages in use that no table names move all the same
    want = run_compact(np.array([16], np.int32), np.array([[9]], np.int32), np.zeros(10, np.int32), np.array([0, 1, 2, 3, 4, 0, 0, 0, 0, 0], np.int32),
                       np.array([0, 5], np.int32), 0, 16)
    assert want[3][2] == 5 and want[0][0, 0] == 4


def test_compact_streams_strides_and_bad_lists(backend):
    lens, table, shares, free, pool = family_book(33, 5, 9, 500, 45, 8)
    s = Stream()
    run_compact(lens, table, shares, free, pool, 0, 5, stream=s, stride=11)
    s.close()
    device_status()
    # a page listed twice counts once
    twice, head = free.copy(), int(pool[0])
    twice[head + 1] = twice[head]
    run_compact(lens, table, shares, twice, pool, 0, 5)
    assert device_status() == BAD_PAGE


def test_book_refusals(backend):
    ok = dict(page_size=16, max_pages=8, n_pages=100, max_requests=4)
    for change, error in (({"page_size": 0}, ShapeInvalid), ({"max_pages": 0}, ShapeInvalid), ({"table_stride": 7}, ShapeMismatch),
                          ({"n_pages": 0}, ShapeInvalid), ({"n_pages": 2 ** 31 - 1}, ShapeInvalid), ({"max_requests": 0}, ShapeInvalid),
                          ({"max_requests": 2 ** 31 - 1}, ShapeInvalid)):
        with pytest.raises(error):
            paged.PageBook(**{**ok, **change})
    h = paged.PageBook(**ok)
    b = [empty(4096) for _ in range(14)]
    p = [x.ptr for x in b]
    good = [p[0], p[1], 4, p[2], 4, *p[3:12]]

    def refused(call_, args, error, at, value):
        args = list(args)
        args[at] = value
        with pytest.raises(error):
            call_(*args)

    for at in (0, 1, 3, 5, 6, 7, 8, 9, 10, 11, 12, 13):
        refused(h.fork, good, InvalidArgument, at, 0)
    for at, value in ((2, 5), (2, -1), (4, 5), (4, -1)):
        refused(h.fork, good, ShapeInvalid, at, value)
    for out, src in ((8, p[0]), (9, p[1]), (10, p[3]), (11, p[4]), (12, p[5])):
        refused(h.fork, good, InvalidArgument, out, src)
    refused(h.fork, good, LayoutUnsupported, 13, p[11] + 4)
    good = [p[0], p[1], 4, p[2], p[3], p[4], 0, *p[5:11]]
    for at in (0, 1, 3, 4, 5, 7, 8, 9, 10, 11, 12):
        refused(h.compact, good, InvalidArgument, at, 0)
    refused(h.compact, good, ShapeInvalid, 2, 5)
    refused(h.compact, good, InvalidArgument, 6, -1)
    for out, src in ((7, p[0]), (8, p[2]), (9, p[3]), (10, p[4])):
        refused(h.compact, good, InvalidArgument, out, src)
    refused(h.compact, good, LayoutUnsupported, 12, p[10] + 8)
    h.close()
    with pytest.raises(TensorClosed):
        h.fork(*good[:13], 1)
    for x in b:
        x.free()


# ------------------------------------------------------------------ copies

def run_copy(dtype, order, page, heads, dim, pages, moves, n_caches=2, count=None, pads=(0, 0, 0), offset=0, stream=None):
    """pads: elements that lie behind a page, a token, a head; offset: bytes in front of the cache."""
    rng = np.random.default_rng(dim + pages)
    size = dtype.size
    layout = paged.CacheLayout(pages, page, heads, dim, dtype, order)
    st = layout.struct
    if order == "HND":
        st.token_stride = dim + pads[1]
        st.head_stride = page * st.token_stride + pads[2]
        st.page_stride = heads * st.head_stride + pads[0]
    else:
        st.head_stride = dim + pads[2]
        st.token_stride = heads * st.head_stride + pads[1]
        st.page_stride = page * st.token_stride + pads[0]
    moves = np.asarray(moves, np.int32).reshape(-1, 4)
    n = len(moves)
    host = [rng.integers(0, 256, offset + pages * st.page_stride * size).astype(np.uint8) for _ in range(n_caches)]
    dev = [to_device(x) for x in host]
    mv, cnt = to_device(moves) if n else empty(16), to_device(np.array([n if count is None else count], np.int32))
    c = paged.PageCopy(layout, [d.ptr + offset for d in dev])
    c.run(mv.ptr, n, 0 if count is None else cnt.ptr, stream)
    sync_device()
    kept = moves if count is None else moves[:max(0, count)]
    for x, d in zip(host, dev):
        body = x[offset:]
        strides = [st.page_stride * size, st.head_stride * size, st.token_stride * size, 1]
        view = np.lib.stride_tricks.as_strided(body, (pages, heads, page, dim * size), strides)
        plain.copy(view, kept, page, "HND")
        bits_equal(fetch(d, x.nbytes), x)
        d.free()
    mv.free()
    cnt.free()


def moves_of(n, pages, page, seed):
    rng = np.random.default_rng(seed)
    number = rng.permutation(pages)
    dst, src = number[:n], number[n:][rng.integers(0, pages - n, n)]
    return np.stack([src, dst, rng.integers(0, page + 1, n), 0 * src], 1)


@pytest.mark.parametrize("dtype", [BF16, F32, E4M3, DType.FLOAT64])
@pytest.mark.parametrize("order", ["HND", "NHD"])
@pytest.mark.parametrize("page,heads,dim", [(16, 8, 128), (1, 1, 64), (20, 3, 80), (7, 5, 33), (128, 2, 256), (4, 1, 1)])
def test_copy_layouts(backend, dtype, order, page, heads, dim):
    run_copy(dtype, order, page, heads, dim, 40, moves_of(17, 40, page, dim))


@pytest.mark.parametrize("order", ["HND", "NHD"])
@pytest.mark.parametrize("pads,offset", [((8, 0, 0), 0), ((0, 8, 0), 0), ((0, 0, 8), 0), ((3, 1, 5), 0), ((0, 0, 0), 2), ((64, 64, 64), 16)])
def test_copy_padded_caches(backend, order, pads, offset):
    """What lies between the rows stays."""
    run_copy(BF16, order, 12, 3, 64, 30, moves_of(11, 30, 12, 1), pads=pads, offset=offset)


@pytest.mark.parametrize("n,caches", [(1, 1), (1, 130), (900, 3), (300, 300)])
def test_copy_counts(backend, n, caches):
    """More caches than one launch takes; many moves, few."""
    run_copy(E4M3, "HND", 8, 2, 32, 2 * n + 3, moves_of(n, 2 * n + 3, 8, n), n_caches=caches)


def test_copy_counts_on_the_device(backend):
    for count in (-1, 0, 1, 9, 10, 50):
        run_copy(BF16, "NHD", 8, 2, 64, 40, moves_of(10, 40, 8, 2), count=count)


def test_copy_bad_moves_are_left_out(backend):
    device_status()
    run_copy(BF16, "HND", 8, 2, 64, 10, [(1, 2, 8, 0), (3, 10, 8, 0), (-1, 4, 8, 0), (5, 6, 99, 0), (7, 8, -3, 0), (2 ** 31 - 1, 9, 1, 0)])
    assert device_status() == BAD_PAGE
    s = Stream()
    run_copy(BF16, "HND", 8, 2, 64, 10, [(1, 2, 8, 0)], stream=s)
    s.close()
    assert device_status() == 0


def test_copy_refusals(backend):
    layout = paged.CacheLayout(4, 8, 2, 64, BF16)
    buf = empty(8 * 2 * 64 * 4 * 2 + 64)
    mv = empty(64)
    paged.PageCopy(layout, []).run(mv.ptr, 1)
    paged.PageCopy(layout, [buf.ptr]).run(0, 0)
    for ptrs, moves, n, error in (([0], mv.ptr, 1, InvalidArgument), ([buf.ptr], 0, 1, InvalidArgument), ([buf.ptr], mv.ptr, -1, InvalidArgument),
                                  ([buf.ptr + 1], mv.ptr, 1, LayoutUnsupported), ([buf.ptr], mv.ptr + 4, 1, LayoutUnsupported)):
        with pytest.raises(error):
            paged.PageCopy(layout, ptrs).run(moves, n)
    for field, value, error in (("dtype", int(DType.INT4), DTypeUnsupported), ("kv_heads", 0, ShapeInvalid), ("head_dim", 0, ShapeInvalid),
                                ("page_size", 0, ShapeInvalid), ("n_pages", -1, ShapeInvalid), ("page_stride", -1, LayoutUnsupported),
                                ("page_size", 1 << 30, ShapeInvalid)):
        bad = paged.CacheLayout(4, 8, 2, 64, BF16)
        setattr(bad.struct, field, value)
        with pytest.raises(error):
            paged.PageCopy(bad, [buf.ptr]).run(mv.ptr, 1)
    buf.free()
    mv.free()


# ------------------------------------------------------------------ together

@pytest.mark.parametrize("cache,most", [("bf16", 0.05), ("f8_e4m3", 0.35), ("f8_e5m2", 0.7)])
@pytest.mark.parametrize("k", [1, 4])
def test_beam_search_of_the_example(backend, cache, most, k):
    """The bounds of an attention over rounded keys and values: as the decoding example's."""
    from examples import beam_search

    device_status()
    assert max(beam_search.run(beams=k, cache_dtype=cache)) < most
    assert device_status() == 0


def test_a_captured_step_replays_with_other_beams(backend):
    """Selection, fork, page copies and compaction captured once; each replay works on the logits and books that are there then,
    as the same calls one by one do."""
    import torch

    n, k, vocab, page, width, pages, dim = 3, 4, 3001, 8, 12, 400, 32
    rows = n * k
    layout = paged.CacheLayout(pages, page, 2, dim, BF16)
    data = np.random.default_rng(5).integers(0, 1 << 16, pages * page * 2 * dim).astype(np.uint16)

    class Step:
        def __init__(self):
            self.cache = [to_device(data), to_device(data[::-1].copy())]
            self.x, self.scores, self.out = empty(4 * rows * vocab), empty(4 * rows), empty(4 * rows)
            self.tokens, self.parents = empty(4 * rows), empty(4 * rows)
            self.table = [empty(4 * rows * width) for _ in range(3)]
            self.lens, self.shares = [empty(4 * rows) for _ in range(2)], [empty(4 * pages) for _ in range(3)]
            self.free, self.pool = [empty(4 * pages) for _ in range(3)], [empty(16) for _ in range(3)]
            self.moves = [empty(16 * rows, 0), empty(16 * (pages // 2), 0)]
            self.numbers = empty(4 * pages)
            self.select, self.book = beams.BeamSelect(F32, vocab, k, k, n), paged.PageBook(page, width, pages, rows)
            self.copy = paged.PageCopy(layout, [c.ptr for c in self.cache])

        def run(self, stream):
            self.select.run(self.x.ptr, self.scores.ptr, n, self.out.ptr, self.tokens.ptr, self.parents.ptr, stream=stream)
            self.book.fork(self.table[0].ptr, self.lens[0].ptr, rows, self.parents.ptr, rows, self.shares[0].ptr, self.free[0].ptr,
                           self.pool[0].ptr, self.table[1].ptr, self.lens[1].ptr, self.shares[1].ptr, self.free[1].ptr,
                           self.pool[1].ptr, self.moves[0].ptr, stream)
            self.copy.run(self.moves[0].ptr, rows, self.pool[1].ptr + 8, stream)
            self.book.compact(self.table[1].ptr, self.lens[1].ptr, rows, self.shares[1].ptr, self.free[1].ptr, self.pool[1].ptr, 0,
                              self.table[2].ptr, self.shares[2].ptr, self.free[2].ptr, self.pool[2].ptr, self.numbers.ptr,
                              self.moves[1].ptr, stream)
            self.copy.run(self.moves[1].ptr, pages // 2, self.pool[2].ptr + 8, stream)

        def load(self, seed):
            rng = np.random.default_rng(seed)
            lens, table, shares, free, pool = family_book(rows, page, width, pages, width * page - 1, seed)
            for b, a in ((self.x, rng.normal(0, 2, (rows, vocab)).astype(np.float32)), (self.scores, -rng.random(rows, np.float32)),
                         (self.table[0], table), (self.lens[0], lens), (self.shares[0], shares), (self.free[0], free), (self.pool[0], pool),
                         (self.cache[0], data), (self.cache[1], data[::-1].copy())):
                b.upload(np.ascontiguousarray(a))
            sync_device()

        def bufs(self):
            return [*self.cache, self.x, self.scores, self.out, self.tokens, self.parents, *self.table, *self.lens, *self.shares,
                    *self.free, *self.pool, *self.moves, self.numbers]

        def state(self):
            valid = int(fetch(self.pool[1], 16, np.int32)[1]), int(fetch(self.pool[2], 16, np.int32)[1])
            return [fetch(b, b.nbytes) for b in (*self.cache, self.out, self.tokens, self.parents, *self.table[1:], self.lens[1],
                                                 *self.shares[1:], *self.pool[1:], self.numbers)] + \
                   [fetch(b, 4 * v) for b, v in zip(self.free[1:], valid)]

        def close(self):
            self.select.close()
            self.book.close()
            for b in self.bufs():
                b.free()

    one, other = Step(), Step()
    one.load(1)
    stream = torch.cuda.Stream()
    one.run(stream.cuda_stream)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        one.run(stream.cuda_stream)
    for seed in (2, 3, 4, 5):
        one.load(seed)
        other.load(seed)
        graph.replay()
        torch.cuda.synchronize()
        other.run(None)
        for a, b in zip(one.state(), other.state()):
            bits_equal(a, b)
    assert device_status() == 0
    del graph
    one.close()
    other.close()


def test_book_two_handles_on_two_streams(backend):
    """Forks of a grid's size that overlap on two streams give what each gives alone."""
    made = [family_book(3000, 2, 200, 3000 * 200 + 500, 400, seed) for seed in (1, 2)]
    parents = [np.random.default_rng(seed).integers(-1, 3000, 3000).astype(np.int32) for seed in (1, 2)]
    streams = [Stream(), Stream()]
    handles = [paged.PageBook(2, 200, 3000 * 200 + 500, 3000) for _ in range(2)]
    ins = [[to_device(a) for a in (m[1], m[0], p, m[2], m[3], m[4])] for m, p in zip(made, parents)]
    pages = 3000 * 200 + 500
    outs = [[empty(4 * s) for s in (3000 * 200, 3000, pages, pages, 4, 4 * 3000)] for _ in range(2)]
    sync_device()
    for _ in range(10):
        for h, i, o, s in zip(handles, ins, outs, streams):
            p = [b.ptr for b in i]
            h.fork(p[0], p[1], 3000, p[2], 3000, p[3], p[4], p[5], *(b.ptr for b in o), stream=s)
    for s in streams:
        s.sync()
    assert device_status() == 0
    for m, p, o in zip(made, parents, outs):
        want = plain.fork(m[1], m[0], p, m[2], m[3], m[4], 2, 200, np.zeros((3000, 4), np.int32), np.zeros(pages, np.int32))
        bits_equal(fetch(o[0], 4 * 3000 * 200, np.int32).reshape(3000, 200), want[0])
        bits_equal(fetch(o[2], 4 * pages, np.int32), want[2])
        bits_equal(fetch(o[4], 16, np.int32), want[4])
    for h in handles:
        h.close()
    for b in (*ins[0], *ins[1], *outs[0], *outs[1]):
        b.free()
    for s in streams:
        s.close()


@pytest.mark.parametrize("make", [lambda: beams.BeamSelect(BF16, 128256, 8, 64, 64), lambda: paged.PageBook(16, 64, 4_000_000, 64),
                                  lambda: paged.PrefixAttention(paged.CacheLayout(4, 16, 1, 256, BF16), 16, BF16, 4, 256)])
def test_handles_close_after_shutdown_and_keep_nothing(backend, make):
    import torch

    make().close()
    before = torch.cuda.mem_get_info()[0]
    held = [make() for _ in range(4)]
    assert torch.cuda.mem_get_info()[0] < before - (8 << 20)
    call("mf_shutdown")
    try:
        for h in held:
            h.close()
    finally:
        call("mf_init", 0)
    assert torch.cuda.mem_get_info()[0] >= before - (4 << 20)


# ------------------------------------------------------------------ selection of rows of many chunks

def many_chunks(rows, chunks, levels):
    """Sums over whole rows, a row in one segment (three CTAs for every SM and more): `levels`(row) gives a row's 16-bit logits, a
    vector for each chunk of 8192 that its other tokens have, and the number of the first token, which leads."""
    import torch

    vocab = chunks * 8192
    x = torch.empty((rows, chunks, 8192), dtype=torch.bfloat16, device="cuda")
    sums = np.empty(rows)
    for r in range(rows):
        level, lead = levels(r)
        x[r] = torch.tensor(level, dtype=torch.bfloat16, device="cuda")[:, None]
        if lead is not None:  # once for every thread: a token of each 8, of the first 2048
            x[r, 0, :2048:8] = lead
        terms = np.exp(np.asarray(level, np.float64))
        sums[r] = math.log((terms.sum() * 8192) + (0 if lead is None else 256 * (math.exp(lead) - terms[0])))
    top = np.array([max(levels(r)[0].max(), -np.inf if levels(r)[1] is None else levels(r)[1]) for r in range(rows)])
    scores = (sums - top).astype(np.float32)  # results near 0, where float32 is fine
    want = scores.astype(np.float64) + top - sums
    out = [torch.empty(rows, dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32)]
    sc = torch.tensor(scores, device="cuda")
    torch.cuda.synchronize()
    with beams.BeamSelect(BF16, vocab, 1, 1, rows) as h:
        h.run(x.data_ptr(), sc.data_ptr(), rows, *[o.data_ptr() for o in out])
        torch.cuda.synchronize()
    got = out[0].cpu().numpy().astype(np.float64)
    assert np.array_equal(out[2].cpu().numpy(), np.arange(rows))
    return np.abs(got - want) - 2.0 ** -24 * np.abs(want), out[1].cpu().numpy()


def test_select_sums_of_many_logits(backend):
    """448 rows of 2 million logits, all but a few alike: a running float32 sum of a thread's 8192 terms is up to 4e-6 off.

    Bound: an exponential 2^-22, its argument 2^-23 for each octave, 32 terms added in float32 in pairs (5 steps, 2^-24 each);
    the rest is float64."""
    steps = np.linspace(0x3d00, 0x3e7f, 448).astype(np.uint32)  # 2^-5 to 2^-2 in BF16
    below = (steps << 16).view(np.float32).astype(np.float64)
    off, tokens = many_chunks(448, 256, lambda r: (np.full(256, -below[r]), 0.0))
    assert (tokens == 0).all()
    assert (off <= 2.0 ** -22 + 5 * 2.0 ** -24 + 2.0 ** -23 * 0.37).all(), off.max()


def test_select_sums_of_rising_logits(backend):
    """The maximum rises with every chunk, by a step of BF16: what was summed is not rounded each time."""
    def levels(r):
        return -2.0 + (np.arange(256) + r % 3) * 2.0 ** -7, None
    off, tokens = many_chunks(448, 256, levels)
    # up to 2 nepers (2.9 octaves) from the first maximum
    assert (off <= 2.0 ** -22 + 5 * 2.0 ** -24 + 2.0 ** -23 * 2.9).all(), off.max()
    # of a step that BF16 does not tell from the next (2^-7 at 1 to 2) the first token counts
    assert all(255 * 8192 >= t >= 253 * 8192 and t % 8192 == 0 for t in tokens)


@pytest.mark.parametrize("dtype,vocab,beams_,n,pad,offset", [(BF16, 70001, 8, 16, 0, 0), (F32, 40001, 4, 8, 3, 1), (F16, 70001, 7, 40, 1, 5),
                                                             (BF16, 131073, 64, 100, 0, 0)])
def test_select_parts_of_several_chunks(backend, dtype, vocab, beams_, n, pad, offset):
    """448 rows are cut into one segment each, of 9 to 17 chunks: several for each part that a thread keeps a maximum of.  Masked tails,
    rows that begin anywhere, ended beams, a best token in every chunk."""
    rng = np.random.default_rng(vocab + n)
    logits = rng.normal(0, 2.5, (448, vocab)).astype(np.float32)
    logits[::3, vocab - 700:] = -np.inf
    chunk = 4096 if dtype == F32 else 8192
    for c in range(-(-vocab // chunk)):  # the best of some rows stand in one chunk, or one in each
        at = np.minimum(c * chunk + rng.integers(0, chunk, 448), vocab - 701)
        logits[np.arange(448), at] = 12.0 + rng.random(448).astype(np.float32)
    for r in range(0, 448, 16):
        first = int(rng.integers(0, vocab - 3000))
        logits[r, first:first + 2 * n] = 20.0 + rng.random(2 * n).astype(np.float32)
    ended = np.zeros(448, np.int32)
    ended[beams_ - 1::beams_] = 1
    run_select(logits, rng.normal(-30, 1, 448), beams_, n, dtype, ended=ended, end=3, stride=vocab + pad, offset=offset)
