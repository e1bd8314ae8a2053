"""A decoding step over a paged key-value cache, on device addresses.

manifesto declares paged state (``page_table`` and ``paged_tensor`` declarations,
runtime/session.go:160-205, materialised by ``state.materialize_state_tensors``) and
plans its pages on the host (runtime/paged_plan.go:14-177).  These are the device
operations of a step, in the order in which a step runs them:

* ``PageAssigner.assign``  -- page tables, slots and positions of the new tokens;
* ``Rope.forward`` / ``backward`` -- rotary positions of an array, and their gradient;
* ``RopeAppend.run``       -- queries and keys rotated, keys and values written to the cache;
* ``PagedAttention.run``   -- attention of one new token per request over the cache.

For requests that share pages, the continuations of a text (K11; ``beams.BeamSelect`` chooses
them):

* ``PageBook.fork`` / ``compact`` -- tables continued by parents, and the used pages moved together;
* ``PageCopy.run``                -- the pages that these move, in every cache;
* ``PrefixAttention.run``         -- attention that reads a group's shared tokens once for all of it.

Each object holds a description that a program makes once; the calls take device
addresses (ints, ``DeviceTensor.dispatch_pointer()``) and launch on a stream,
without waiting for the device.  ``include/mfcuda.h`` has the formulas (K10, K11).
"""
from __future__ import annotations

import ctypes
import math

import numpy as np

from . import _abi
from .backend import COMPAT_REFERENCE, stream_handle
from .dtype import DType
from .errors import InvalidArgument, TensorClosed, raise_for_status

ROPE_LAYOUTS = {"half": 0, "interleaved": 1}
ROPE_SCALINGS = {"none": 0, "linear": 1, "base": 2, "bands": 3}


def _raise(name: str, rc: int) -> None:
    raise_for_status(rc, f"{name}: {_abi.last_error()}")


def rope_frequencies(rot_dim: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                     original_length: float = 0.0, low_turns: float = 1.0, high_turns: float = 4.0) -> np.ndarray:
    """float32 [rot_dim / 2] frequencies of rotary positions, scaled for contexts longer than the trained one.

    ``linear`` divides them by ``factor``; ``base`` raises the base instead; ``bands``
    keeps the waves that turn at least ``high_turns`` times in ``original_length``
    tokens, divides those below ``low_turns`` and ramps between."""
    if scaling not in ROPE_SCALINGS:
        raise InvalidArgument(f"rope: unknown scaling {scaling!r}")
    out = np.zeros(max(int(rot_dim), 0) // 2, np.float32)
    _abi.call("mf_rope_frequencies", int(rot_dim), float(base), ROPE_SCALINGS[scaling], float(factor),
              float(original_length), float(low_turns), float(high_turns),
              out.ctypes.data_as(ctypes.POINTER(ctypes.c_float)))
    return out


class CacheLayout:
    """Shape and strides of a paged cache: ``pages`` pages of ``page_size`` tokens.

    ``order`` is "HND" (a head's tokens together: [pages, kv_heads, page_size, head_dim])
    or "NHD" (a token's heads together: [pages, page_size, kv_heads, head_dim])."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: DType, order: str = "HND"):
        if order not in ("HND", "NHD"):
            raise InvalidArgument(f"paged cache: unknown order {order!r}")
        self.shape = ((pages, kv_heads, page_size, head_dim) if order == "HND" else
                      (pages, page_size, kv_heads, head_dim))
        self.dtype = DType(dtype)
        self.order = order
        token, head = (head_dim, page_size * head_dim) if order == "HND" else (kv_heads * head_dim, head_dim)
        self.struct = _abi.CacheLayout(int(self.dtype), int(kv_heads), int(head_dim), int(page_size), int(pages),
                                       int(page_size * kv_heads * head_dim), int(token), int(head))


class PageAssigner:
    """Page tables, slots and positions of a step's new tokens (mf_page_assign)."""

    def __init__(self, page_size: int, max_pages: int, table_stride: int | None = None):
        self.config = _abi.PageConfig(int(page_size), int(max_pages),
                                      int(max_pages if table_stride is None else table_stride))
        self._config = ctypes.byref(self.config)
        self._assign = _abi.lib().mf_page_assign  # looked up once: the calls are on a decoding step's critical path

    def assign(self, lens: int, new_tokens: int, n_requests: int, table: int, free_pages: int, pool: int, tokens: int,
               slots: int, positions: int, owner: int, starts: int, lens_after: int, pool_after: int, stream=None) -> None:
        """Extend the tables in place and write the tokens' slots, positions and owners, the requests' starts and
        lengths after the step, and what is left of the pool."""
        rc = self._assign(self._config, lens, new_tokens, n_requests, table, free_pages, pool, tokens, slots, positions,
                          owner, starts, lens_after, pool_after, stream if stream is None else stream_handle(stream))
        if rc:
            _raise("mf_page_assign", rc)


class Rope:
    """Rotary positions of [tokens, heads, head_dim] arrays (mf_rope); ``inv_freq`` is a device address."""

    def __init__(self, inv_freq: int, dtype: DType, head_dim: int, rot_dim: int | None = None, layout: str = "half",
                 magnitude: float = 1.0):
        if layout not in ROPE_LAYOUTS:
            raise InvalidArgument(f"rope: unknown layout {layout!r}")
        self.config = _abi.RopeConfig(int(dtype), int(head_dim), int(head_dim if rot_dim is None else rot_dim),
                                      ROPE_LAYOUTS[layout], float(magnitude), int(inv_freq))
        self._config = ctypes.byref(self.config)
        self._rope = _abi.lib().mf_rope

    def _run(self, inverse, src, dst, positions, tokens, heads, src_strides, dst_strides, stream) -> None:
        dim = self.config.head_dim
        st, sh = src_strides or (heads * dim, dim)
        dt, dh = dst_strides or (heads * dim, dim)
        rc = self._rope(self._config, inverse, src, st, sh, dst, dt, dh, positions, tokens, heads,
                        stream if stream is None else stream_handle(stream))
        if rc:
            _raise("mf_rope", rc)

    def forward(self, src: int, dst: int, positions: int, tokens: int, heads: int, src_strides=None, dst_strides=None,
                stream=None) -> None:
        """dst = rope(src); strides are (token, head) in elements, contiguous by default."""
        self._run(0, src, dst, positions, tokens, heads, src_strides, dst_strides, stream)

    def backward(self, src: int, dst: int, positions: int, tokens: int, heads: int, src_strides=None, dst_strides=None,
                 stream=None) -> None:
        """dst = the gradient of rope's input, from src = that of its output."""
        self._run(1, src, dst, positions, tokens, heads, src_strides, dst_strides, stream)


class RopeAppend:
    """Queries and keys rotated, keys and values written to their slots (mf_rope_append).

    ``token_stride`` is the elements from one token's heads to the next for queries,
    keys and values alike (a packed projection); None: each is contiguous."""

    def __init__(self, rope: Rope, cache: CacheLayout, q_heads: int, k_scale_inv: int = 0, v_scale_inv: int = 0,
                 compat: int = COMPAT_REFERENCE, token_stride: int | None = None):
        dim, kv = rope.config.head_dim, cache.struct.kv_heads
        qs, ks = (q_heads * dim, kv * dim) if token_stride is None else (token_stride, token_stride)
        self.config = _abi.RopeAppendConfig(rope.config, cache.struct, int(q_heads), int(compat), int(k_scale_inv) or None,
                                            int(v_scale_inv) or None, qs, dim, ks, dim, ks, dim, q_heads * dim, dim)
        self._config = ctypes.byref(self.config)
        self._append = _abi.lib().mf_rope_append

    def run(self, q: int, k: int, v: int, q_out: int, k_cache: int, v_cache: int, positions: int, slots: int, tokens: int,
            stream=None) -> None:
        rc = self._append(self._config, q, k, v, q_out, k_cache, v_cache, positions, slots, tokens,
                          stream if stream is None else stream_handle(stream))
        if rc:
            _raise("mf_rope_append", rc)


def _attn_config(cache: CacheLayout, q_heads, dtype, max_pages, table_stride, scale, softcap, window, slopes, k_scale_inv,
                 v_scale_inv, q_strides, out_strides) -> _abi.PagedAttnConfig:
    dim = cache.struct.head_dim
    qt, qh = q_strides or (q_heads * dim, dim)
    ot, oh = out_strides or (q_heads * dim, dim)
    return _abi.PagedAttnConfig(
        cache.struct, int(dtype), int(q_heads), int(max_pages), int(window),
        int(max_pages if table_stride is None else table_stride),
        float(1.0 / math.sqrt(dim) if scale is None and dim > 0 else scale or 0.0), float(softcap), int(slopes) or None,
        int(k_scale_inv) or None, int(v_scale_inv) or None, qt, qh, ot, oh)


class PagedAttention:
    """Attention of one new token per request over a paged cache (mf_paged_attn_*).

    Holds the workspace of the split, so one object serves one stream at a time; it
    runs any number of requests, steps and layers of its shape."""

    def __init__(self, cache: CacheLayout, q_heads: int, dtype: DType, max_pages: int, table_stride: int | None = None,
                 scale: float | None = None, softcap: float = 0.0, window: int = 0, slopes: int = 0, k_scale_inv: int = 0,
                 v_scale_inv: int = 0, q_strides: tuple[int, int] | None = None,
                 out_strides: tuple[int, int] | None = None):
        self.config = _attn_config(cache, q_heads, dtype, max_pages, table_stride, scale, softcap, window, slopes, k_scale_inv,
                                   v_scale_inv, q_strides, out_strides)
        handle = ctypes.c_void_p()
        _abi.call("mf_paged_attn_create", ctypes.byref(self.config), ctypes.byref(handle))
        self._handle = handle.value
        self._attend = _abi.lib().mf_paged_attn_run

    def run(self, q: int, k_cache: int, v_cache: int, table: int, lens: int, n_requests: int, out: int, lse: int = 0,
            stream=None) -> None:
        if self._handle is None:
            raise TensorClosed("paged attention: closed")
        rc = self._attend(self._handle, q, k_cache, v_cache, table, lens, n_requests, out, lse,
                          stream if stream is None else stream_handle(stream))
        if rc:
            _raise("mf_paged_attn_run", rc)

    def close(self) -> None:
        """Wait for the device and free the workspace."""
        if self._handle is not None:
            handle, self._handle = self._handle, None
            _abi.call("mf_paged_attn_destroy", handle)

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        if getattr(self, "_handle", None) is not None:
            try:
                self.close()
            except Exception:
                pass  # interpreter shutdown, or the library is closed


class _Handle:
    """An object of the library that owns a workspace: created once, closed at the end."""

    _handle = None
    _destroy = ""

    def _create(self, name: str, *args) -> None:
        handle = ctypes.c_void_p()
        _abi.call(name, *args, ctypes.byref(handle))
        self._handle = handle.value

    def _open(self) -> int:
        if self._handle is None:
            raise TensorClosed(f"{type(self).__name__}: closed")
        return self._handle

    def close(self) -> None:
        """Wait for the device and free the workspace."""
        if self._handle is not None:
            handle, self._handle = self._handle, None
            _abi.call(self._destroy, handle)

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        if getattr(self, "_handle", None) is not None:
            try:
                self.close()
            except Exception:
                pass  # interpreter shutdown, or the library is closed


class PrefixAttention(_Handle):
    """``PagedAttention`` for groups of requests that share the pages of their first tokens (mf_prefix_attn_*).

    The shared tokens of a group are read once for all its requests: the beams of a prompt, or a batch that begins
    with the same instructions; groups for which that does not pay (small ones, few requests that see the tokens) only
    with ``always``.  Holds the workspace for up to ``max_requests``, so one object serves one stream at a time; it runs
    any number of requests, groups, steps and layers of its shape."""

    _destroy = "mf_prefix_attn_destroy"

    def __init__(self, cache: CacheLayout, q_heads: int, dtype: DType, max_pages: int, max_requests: int,
                 table_stride: int | None = None, scale: float | None = None, softcap: float = 0.0, window: int = 0,
                 slopes: int = 0, k_scale_inv: int = 0, v_scale_inv: int = 0, q_strides: tuple[int, int] | None = None,
                 out_strides: tuple[int, int] | None = None, always: bool = False):
        self.config = _attn_config(cache, q_heads, dtype, max_pages, table_stride, scale, softcap, window, slopes, k_scale_inv,
                                   v_scale_inv, q_strides, out_strides)
        self._create("mf_prefix_attn_create", ctypes.byref(self.config), int(max_requests))
        if always:
            _abi.call("mf_prefix_attn_share", self._handle, 1)
        self._attend = _abi.lib().mf_prefix_attn_run

    def run(self, q: int, k_cache: int, v_cache: int, table: int, lens: int, n_requests: int, starts: int, shared: int,
            n_groups: int, out: int, lse: int = 0, stream=None) -> None:
        """Requests starts[g] .. starts[g + 1] - 1 have their first shared[g] tokens in the same pages."""
        rc = self._attend(self._open(), q, k_cache, v_cache, table, lens, n_requests, starts, shared, n_groups, out, lse,
                          stream if stream is None else stream_handle(stream))
        if rc:
            _raise("mf_prefix_attn_run", rc)


class PageBook(_Handle):
    """Page tables whose rows share pages: rows continued by parents, or ended (``fork``), and the pages in use
    moved together (``compact``); mf_page_book_*.  Both list the pages to copy: run ``PageCopy`` next.

    Holds the workspace for up to ``max_requests`` rows, so one object serves one stream at a time."""

    _destroy = "mf_page_book_destroy"

    def __init__(self, page_size: int, max_pages: int, n_pages: int, max_requests: int, table_stride: int | None = None):
        self.config = _abi.PageBookConfig(int(page_size), int(max_pages), int(max_pages if table_stride is None else table_stride),
                                          int(n_pages), int(max_requests))
        self._create("mf_page_book_create", ctypes.byref(self.config))
        self._fork, self._compact = _abi.lib().mf_page_book_fork, _abi.lib().mf_page_book_compact

    def fork(self, table: int, lens: int, n_before: int, parents: int, n_after: int, shares: int, free_pages: int, pool: int,
             table_after: int, lens_after: int, shares_after: int, free_after: int, pool_after: int, moves: int,
             stream=None) -> None:
        """Row r of n_after continues row parents[r] of n_before; ``moves`` has room for n_after entries of 16 bytes."""
        rc = self._fork(self._open(), table, lens, n_before, parents, n_after, shares, free_pages, pool, table_after, lens_after,
                        shares_after, free_after, pool_after, moves, stream if stream is None else stream_handle(stream))
        if rc:
            _raise("mf_page_book_fork", rc)

    def compact(self, table: int, lens: int, n_requests: int, shares: int, free_pages: int, pool: int, limit: int,
                table_after: int, shares_after: int, free_after: int, pool_after: int, numbers: int, moves: int,
                stream=None) -> None:
        """Pages in use from ``limit`` on (0: from their count on) moved below it; ``moves`` has room for n_pages / 2."""
        rc = self._compact(self._open(), table, lens, n_requests, shares, free_pages, pool, limit, table_after, shares_after,
                           free_after, pool_after, numbers, moves, stream if stream is None else stream_handle(stream))
        if rc:
            _raise("mf_page_book_compact", rc)


class PageCopy:
    """The moves of ``PageBook`` carried out in every cache of a layout: keys and values of all layers (mf_page_copy)."""

    def __init__(self, cache: CacheLayout, caches: list[int]):
        self._layout = ctypes.byref(cache.struct)
        self._caches = (ctypes.c_void_p * len(caches))(*caches)
        self._n = len(caches)
        self._copy = _abi.lib().mf_page_copy

    def run(self, moves: int, n_moves: int, count: int = 0, stream=None) -> None:
        """The first n_moves moves, or as many as ``count`` says on the device (``pool_after`` + 8 bytes)."""
        rc = self._copy(self._layout, self._caches, self._n, moves, n_moves, count or None,
                        stream if stream is None else stream_handle(stream))
        if rc:
            _raise("mf_page_copy", rc)
