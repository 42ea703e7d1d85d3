"""Outputs of the append and the attention that share memory with the arrays that the same launch reads beside the
rows (positions, windows' rows, masks) are refused; arrays in the gaps of the outputs' rows are not.  No GPU: a
good call is TIE_HIP_ENOINIT there."""
import ctypes
import os

import numpy as np
import pytest

import tie_amd
from test_kv_host import A, W, cache, seqs

pytestmark = pytest.mark.skipif(not os.path.exists(tie_amd.LIB_PATH), reason="libtie_hip.so not built")
T, Q, OUT, ROW = 5, A, A + 32768, W * 4  # five tokens of 4 heads of 64
PAIRS = bytes([0, 1, 2, 3] * 8)


def append(out, pos, so=W):
    return tie_amd.lib().tie_hip_kv_append(ctypes.byref(cache()), 0, ctypes.byref(seqs()), Q, W, A + 8192, 128, A + 16384, 128, 4, None,
                                           None, 1e-6, 1e6, pos, out, so, None)


def axes(out, pos, so=W, n=3):
    return tie_amd.lib().tie_hip_kv_append_axes(ctypes.byref(cache()), 0, ctypes.byref(seqs()), Q, W, A + 8192, 128, A + 16384, 128, 4,
                                                None, None, 1e-6, 1e6, pos, n, bytes(32) if n < 4 else PAIRS, out, so, None)


def tree(out, mask, words=2, so=W):
    return tie_amd.lib().tie_hip_tree_attention(ctypes.byref(cache()), 0, ctypes.byref(seqs()), Q, W, 4, 0.1, mask, words, out, so, None,
                                                0, None)


def window(out, at, mask=None, words=0, so=W):
    return tie_amd.lib().tie_hip_window_attention(ctypes.byref(cache()), 0, ctypes.byref(seqs()), Q, W, 4, 0.1, 7, 1, at, mask, words, out,
                                                  so, None, 0, None)


# what the call reads, and how long that is
CALLS = {"append": (append, T * 4), "axes": (axes, 3 * T * 4), "axes4": (lambda *a, **kw: axes(*a, n=4, **kw), 4 * T * 4),
         "tree": (tree, T * 16), "window at": (window, T * 4),
         "window mask": (lambda out, m, **kw: window(out, A + 24576, m, 2, **kw), T * 16)}


@pytest.mark.parametrize("name", CALLS)
def test_what_is_read_while_outputs_are_written(name):
    call, size = CALLS[name]
    end = OUT + T * ROW
    for p in (OUT - size, end, A + 24576 + 64):
        assert call(OUT, p) == tie_amd.ENOINIT, p - OUT
    for p in (OUT - size + 8, OUT - 8, OUT, OUT + ROW, OUT + 2 * ROW + 40, end - 8):
        assert call(OUT, p) == tie_amd.EINVAL, p - OUT
        assert "overlaps" in tie_amd.last_error()
    assert call(OUT, None) == (tie_amd.EINVAL if name.startswith("axes") else tie_amd.ENOINIT)


@pytest.mark.parametrize("name", CALLS)
def test_gaps_between_the_outputs_rows(name):
    """Rows of W + 64 floats' stride: 256 bytes of each are no output's."""
    call, size = CALLS[name]
    row = ROW + 256
    for gap in (0, 3):
        begin = OUT + gap * row + ROW
        for p in (begin, begin + 256 - size):
            assert call(OUT, p, so=W + 64) == tie_amd.ENOINIT, (gap, p - begin)
        for p in (begin - 8, begin + 256 - size + 8):
            assert call(OUT, p, so=W + 64) == tie_amd.EINVAL, (gap, p - begin)
    assert call(OUT, OUT + 4 * row + ROW, so=W + 64) == tie_amd.ENOINIT  # (behind the last row)


def test_no_tokens_no_memory():
    s = seqs(n_seqs=0, n_tokens=0)
    got = tie_amd.lib().tie_hip_window_attention(ctypes.byref(cache()), 0, ctypes.byref(s), Q, W, 4, 0.1, 7, 1, OUT, OUT, 1, OUT, W, None,
                                                 0, None)
    assert got == tie_amd.ENOINIT


def test_against_rows_written_out():
    """The same question answered byte by byte, for small rows anywhere."""
    rng = np.random.default_rng(0)
    met = 0
    for _ in range(400):
        so, p = W + 4 * int(rng.integers(0, 40)), OUT + 8 * int(rng.integers(-60, 900))
        used = np.zeros(16384, bool)
        for t in range(T):
            used[2048 + t * so * 4: 2048 + t * so * 4 + ROW] = True
        meets = bool(used[2048 + p - OUT: 2048 + p - OUT + T * 16].any())
        assert tree(OUT, p, so=so) == (tie_amd.EINVAL if meets else tie_amd.ENOINIT), (so, p - OUT)
        met += meets
    assert 40 < met < 390
