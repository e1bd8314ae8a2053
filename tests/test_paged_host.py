"""The paged-cache operators without a device: frequencies, layouts, descriptions, and the plain forms themselves."""
import ctypes
import math

import numpy as np
import pytest

from manifesto_b200 import _abi, paged
from manifesto_b200.dtype import DType
from manifesto_b200.errors import InvalidArgument, ShapeInvalid

from . import paged_ref as plain


def test_frequencies_are_the_formulas():
    i = np.arange(64)
    f = 10000.0 ** (-2.0 * i / 128)
    assert np.array_equal(paged.rope_frequencies(128), f.astype(np.float32))
    assert np.allclose(paged.rope_frequencies(128, 500000.0), 500000.0 ** (-2.0 * i / 128), rtol=2 ** -23, atol=0)
    assert np.allclose(paged.rope_frequencies(128, scaling="linear", factor=8.0), f / 8, rtol=2 ** -23, atol=0)
    base = 10000.0 * 8.0 ** (128 / 126)
    assert np.allclose(paged.rope_frequencies(128, scaling="base", factor=8.0), base ** (-2.0 * i / 128), rtol=2 ** -23, atol=0)


def test_frequency_bands():
    f = paged.rope_frequencies(128).astype(np.float64)
    g = paged.rope_frequencies(128, scaling="bands", factor=8.0, original_length=8192, low_turns=1.0, high_turns=4.0)
    turns = 8192 * f / (2 * math.pi)
    fast, slow = turns >= 4.001, turns <= 0.999
    assert fast.any() and slow.any() and (~fast & ~slow).any()
    assert np.array_equal(g[fast], f[fast].astype(np.float32))
    assert np.allclose(g[slow], f[slow] / 8, rtol=2 ** -22, atol=0)
    between = ~fast & ~slow
    assert (g[between] <= f[between]).all() and (g[between] >= f[between] / 8).all()


def test_frequency_refusals():
    for rot in (-2, 3, 1026):
        with pytest.raises(ShapeInvalid):
            paged.rope_frequencies(rot)
    for bad in ({"scaling": "spiral"}, {"base": 0.0}, {"scaling": "linear", "factor": 0.0},
                {"scaling": "bands", "factor": 2.0, "original_length": 0.0},
                {"scaling": "bands", "factor": 2.0, "original_length": 10.0, "low_turns": 4.0, "high_turns": 4.0}):
        with pytest.raises(InvalidArgument):
            paged.rope_frequencies(8, **bad)
    assert paged.rope_frequencies(0).size == 0


@pytest.mark.parametrize("order", ["HND", "NHD"])
def test_cache_layout_strides_are_the_shape_s(order):
    c = paged.CacheLayout(5, 16, 3, 64, DType.BFLOAT16, order)
    a = np.arange(5 * 16 * 3 * 64).reshape(c.shape)
    s = c.struct
    for page, tok, head in ((0, 0, 0), (4, 15, 2), (2, 7, 1)):
        at = page * s.page_stride + tok * s.token_stride + head * s.head_stride
        assert at == (a[page, head, tok] if order == "HND" else a[page, tok, head])[0]
    with pytest.raises(InvalidArgument):
        paged.CacheLayout(5, 16, 3, 64, DType.BFLOAT16, "DNH")


def test_struct_sizes_match_the_header():
    """The ctypes structures have the C layout (LP64): the sizes that the compiler gives the header's."""
    assert [ctypes.sizeof(t) for t in (_abi.CacheLayout, _abi.PageConfig, _abi.RopeConfig, _abi.RopeAppendConfig,
                                       _abi.PagedAttnConfig)] == [48, 16, 32, 168, 136]


def test_entry_points_refuse_before_init():
    count = ctypes.c_int(0)
    _abi.lib().mf_device_count(ctypes.byref(count))
    if count.value:
        pytest.skip("a GPU is visible; this checks the closed path")
    from manifesto_b200.errors import BackendClosed
    layout = paged.CacheLayout(4, 16, 2, 64, DType.BFLOAT16)
    rope = paged.Rope(0, DType.BFLOAT16, 64)
    with pytest.raises(BackendClosed):
        paged.PagedAttention(layout, 4, DType.BFLOAT16, 4)
    with pytest.raises(BackendClosed):
        rope.forward(0, 0, 0, 0, 0)
    with pytest.raises(BackendClosed):
        paged.RopeAppend(rope, layout, 4).run(0, 0, 0, 0, 0, 0, 0, 0, 0)
    with pytest.raises(BackendClosed):
        paged.PageAssigner(16, 4).assign(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)


def test_plain_rope_turns_and_turns_back():
    rng = np.random.default_rng(1)
    x = rng.normal(size=(5, 2, 12))
    pos = np.array([0, 1, 7, 100, -3])
    f = plain.np.array([1.0, 0.25, 0.01, 1e-4])
    for layout in ("half", "interleaved"):
        y = plain.rope(x, pos, f, 8, layout, 2.0)
        assert np.allclose(plain.rope(y, pos, f, 8, layout, 0.5, inverse=True), x)
        assert np.allclose(y[0, :, :8], 2 * x[0, :, :8]) and np.array_equal(y[..., 8:], x[..., 8:])
        # the score of two turned vectors depends on the distance alone
        a, b = rng.normal(size=(2, 1, 1, 8))
        score = [float((plain.rope(a, [p + 9], f, 8, layout, 1.0) * plain.rope(b, [p], f, 8, layout, 1.0)).sum()) for p in (0, 41)]
        assert abs(score[0] - score[1]) < 1e-9


def test_plain_attention_of_parts():
    """A window of everything is no window; one token gives its value; equal scores give the mean."""
    rng = np.random.default_rng(2)
    q, k, v = rng.normal(size=(2, 8)), rng.normal(size=(9, 1, 8)), rng.normal(size=(9, 1, 8))
    full, lse, _ = plain.attention(q, k, v, None, 0.3, 0.0, 0, 2)
    same, _, _ = plain.attention(q, k, v, None, 0.3, 0.0, 9, 2)
    assert np.array_equal(full, same)
    one, _, _ = plain.attention(q, k, v, None, 0.3, 0.0, 1, 2)
    assert np.allclose(one, v[8, 0])
    flat, l0, _ = plain.attention(0 * q, k, v, None, 0.3, 0.0, 0, 2)
    assert np.allclose(flat, v[:, 0].mean(0)) and np.allclose(l0, math.log(9))


def test_overlapped_kernels_read_with_plain_loads():
    """A kernel that is set up while the one before it still writes must not use the read-only path, which takes its data
    to be constant for the kernel's whole life."""
    from manifesto_b200.build import CSRC
    overlapped = [f for f in sorted(CSRC.glob("*.cu")) if "launch_overlapped(" in f.read_text()]
    assert {f.name for f in overlapped} >= {"pages.cu", "rope.cu", "paged_attn.cu"}
    for f in overlapped:
        text = f.read_text()
        for form in ("__ldg(", "ld.global.nc", "ld_stream(", "load4_stream<", "load_raw<", "__restrict__"):
            assert form not in text, f"{f.name} reads by {form}"
