"""The operators for several continuations without a device: descriptions, the closed library, and the plain forms themselves."""
import ctypes
import math

import numpy as np
import pytest

from manifesto_b200 import _abi, beams, paged
from manifesto_b200.dtype import DType

from . import beams_ref as plain


def test_struct_sizes_match_the_header():
    assert [ctypes.sizeof(t) for t in (_abi.BeamSelectConfig, _abi.PageBookConfig)] == [32, 24]


def test_entry_points_refuse_before_init():
    count = ctypes.c_int(0)
    _abi.lib().mf_device_count(ctypes.byref(count))
    if count.value:
        pytest.skip("a GPU is visible; this checks the closed path")
    from manifesto_b200.errors import BackendClosed
    layout = paged.CacheLayout(4, 16, 2, 64, DType.BFLOAT16)
    for make in (lambda: beams.BeamSelect(DType.FLOAT32, 10, 2, 2, 1), lambda: paged.PageBook(16, 4, 10, 2),
                 lambda: paged.PrefixAttention(layout, 4, DType.BFLOAT16, 4, 2), lambda: paged.PageCopy(layout, [16]).run(16, 1)):
        with pytest.raises(BackendClosed):
            make()
    for name in ("mf_beam_select_run", "mf_page_book_fork", "mf_page_book_compact", "mf_prefix_attn_run"):
        args = [t(0) if t is not ctypes.c_void_p else None for t in _abi.SIGNATURES[name]]
        with pytest.raises(BackendClosed):
            _abi.call(name, *args)
    for name in ("mf_beam_select_destroy", "mf_page_book_destroy", "mf_prefix_attn_destroy"):
        _abi.call(name, None)  # nothing to destroy


def test_plain_selection():
    x = np.log(np.array([[0.5, 0.25, 0.25], [0.1, 0.2, 0.7]]))
    s, t, p, e = plain.select(x, np.array([0.0, -1.0], np.float32), None, 2, 4, 1)
    # log 0.7 - 1 = -1.357 lies between log 0.5 = -0.693 and log 0.25 = -1.386
    assert t[0].tolist() == [0, 2, 1, 2] and p[0].tolist() == [0, 1, 0, 0] and e[0].tolist() == [0, 0, 1, 0]
    assert np.allclose(s[0], [math.log(0.5), math.log(0.7) - 1, math.log(0.25), math.log(0.25)])
    # a beam at its end goes on by the end's token; one that is not in use not at all
    s, t, p, e = plain.select(x, np.array([-0.1, -np.inf], np.float32), [1, 0], 2, 2, 1)
    assert t[0].tolist() == [1, -1] and p[0].tolist() == [0, -1] and e[0].tolist() == [1, 0] and s[0, 1] == -np.inf


def books(seed, n=12, page=4, width=6, pages=90):
    """Rows of their own, then a few forks: every state keeps each page in one place."""
    rng = np.random.default_rng(seed)
    number = rng.permutation(pages).astype(np.int32)
    lens = rng.integers(0, page * width + 1, n)
    held = -(-lens // page)
    table = np.full((n, width), -1, np.int32)
    at = 0
    for r in range(n):
        table[r, :held[r]] = number[at:at + held[r]]
        at += held[r]
    free = np.zeros(pages, np.int32)
    free[:pages - at] = number[at:]
    return lens.astype(np.int32), table, np.zeros(pages, np.int32), free, np.array([0, pages - at], np.int32)


def check_books(lens, table, shares, free, pool, page):
    pages = len(shares)
    held = [row[:-(-int(n) // page)] for row, n in zip(table, lens)]
    holders = np.bincount(np.concatenate(held) if held else np.zeros(0, int), minlength=pages)
    listed = free[pool[0]:pool[0] + pool[1]]
    assert len(set(listed.tolist())) == len(listed)
    assert np.array_equal(np.sort(np.concatenate([listed, np.where(holders > 0)[0]])), np.arange(pages))
    assert np.array_equal(shares, np.maximum(holders - 1, 0))
    for row, n in zip(held, lens):  # the page that a row writes next is its own
        if n % page:
            assert holders[row[-1]] == 1


@pytest.mark.parametrize("seed", range(6))
def test_plain_forks_keep_every_page(seed):
    rng = np.random.default_rng(100 + seed)
    lens, table, shares, free, pool = books(seed)
    check_books(lens, table, shares, free, pool, 4)
    none = np.full(len(shares), -1, np.int32)
    for _ in range(5):
        parents = rng.integers(-1, len(lens), 12)
        table, lens, shares, free, after, moves = plain.fork(table, lens, parents, shares, free, pool, 4, 6, np.full((12, 4), -1, np.int32), none)
        pool = after[:2]
        assert after[2] == (moves[:, 0] >= 0).sum()
        check_books(lens, table, shares, free, pool, 4)
        numbers_of = table.copy()
        table, shares, free, after, numbers, _ = plain.compact(table, lens, shares, free, pool, 0, 4, 6, np.zeros((45, 4), np.int32), none)
        pool = after[:2]
        check_books(lens, table, shares, free, pool, 4)
        held = numbers_of >= 0
        assert np.array_equal(table[held], numbers[numbers_of[held]]) and table.max() < len(shares) - pool[1]


def test_plain_copies():
    a = np.arange(3 * 2 * 4 * 1).reshape(3, 2, 4, 1)
    b = plain.copy(a.copy(), np.array([[0, 2, 3, 0], [9, 1, 4, 0]]), 4, "HND")
    assert np.array_equal(b[2, :, :3], a[0, :, :3]) and np.array_equal(b[2, :, 3], a[2, :, 3]) and np.array_equal(b[:2], a[:2])


def test_sources_of_the_tensor_core_kernel():
    """No load of the attention over a shared prefix is a multicast one, and every wait of it has a limit."""
    from manifesto_b200.build import CSRC
    text = (CSRC / "prefix_attn.cu").read_text()
    assert "multicast" not in text and "mbar_wait(" not in text and "while (!mbar_try_wait(bar, parity))" in text
