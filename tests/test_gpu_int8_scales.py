"""Attention over int8 rows whose V scales lie many binades apart: a row that a
query does not see, or that weighs nothing for it, leaves no trace in its
result, whatever its scale; one that weighs little but is large counts.
Against the plain 64-bit form; tolerances: kv_ref.tolerance (derived there)."""
import numpy as np
import pytest

import kv_ref
from test_gpu_tree_attention import check, device, run, words  # noqa: F401 (device: the module's fixture)

pytestmark = pytest.mark.gpu

# (H, kvh, hd, committed rows, tokens): tiles of 16 rows whole and in parts, of 64, of 128
SIZES = [(8, 1, 128, 90, 3), (8, 1, 128, 2500, 1), (8, 1, 128, 900, 30), (8, 2, 64, 700, 90), (64, 4, 128, 45, 515)]


def case(rng, H, kvh, hd, length, n, far):
    """Queries whose first column is 8, keys that are 0 there, so that a row of
    key (x, 0, ..) has the score 8 x / sqrt(hd) for every query; V of 0.5 / 50.
    far: {row: (score, size of V)}, in all kv heads."""
    c = kv_ref.Cache(rng, "i8", kvh, hd, [length], [n], fill=False)
    k, v = rng.standard_normal((length + n, kvh, hd)), 0.01 * rng.standard_normal((length + n, kvh, hd))
    k[:, :, 0] = 0
    for row, (score, size) in far.items():
        k[row] = 0
        k[row, :, 0] = score * hd ** 0.5 / 8
        v[row] = size * rng.standard_normal((kvh, hd))
    c.set_rows(0, 0, 0, k, v)
    q = rng.standard_normal((n, H, hd)).astype(np.float32)
    q[:, :, 0] = 8
    return c, q


def attention(c, q, scale, sees):
    """kv_ref.attention with what a sum over rows of other sizes leaves in a
    column where the large ones' codes are 0.  The second product's weights y_j =
    w_j vs_j are held in two f16 parts, to 2^-22 of each (in kv_ref.tolerance), but
    not below half of f16's least step, 2^-25, where a query's largest is 2^12 or
    more: each y_j is off by 2^-37 max_i y_i at most, times a code of up to 127 in
    every column.  That is n 2^-37 max_i (w_i max_column |v_i|) beside the
    column's own tolerance."""
    want, tol = kv_ref.attention(c, 0, q, scale, sees)
    group, n = q.shape[1] // c.kvh, c.lens[0]
    k, v = c.rows(0, 0, 0, n + c.counts[0])
    for i in range(c.counts[0]):
        on = np.concatenate([np.ones(n, bool), np.array([sees(0, i, j) for j in range(c.counts[0])], bool)])
        for h in range(q.shape[1]):
            s = k[on, h // group] @ q[i, h].astype(np.float64) * scale
            w = np.exp(s - s.max())
            tol[i, h] += on.sum() * 2.0 ** -37 * (w / w.sum() * np.abs(v[on, h // group]).max(1)).max()
    return want, tol


def trees(rng, n, unseen=()):
    sees = np.tril(rng.random((n, n)) < 0.6) | np.eye(n, dtype=bool)
    sees[:, list(unseen)] = False
    return sees


@pytest.mark.parametrize("H,kvh,hd,length,n", [s for s in SIZES if s[4] > 1])
@pytest.mark.parametrize("size", [1e4, 1e6, 1e30])
def test_rows_that_no_token_sees(H, kvh, hd, length, n, size):
    """A drafted token of a branch that nobody looks at, a million times the others' size."""
    rng = np.random.default_rng(n)
    c, q = case(rng, H, kvh, hd, length, n, {length + 1: (0.0, size)})
    sees = trees(rng, n, [1])
    want, tol = attention(c, q, hd ** -0.5, lambda b, i, j: sees[i, j])
    check(run(c, q, hd ** -0.5, words([sees])), want, tol)


@pytest.mark.parametrize("H,kvh,hd,length,n", SIZES)
@pytest.mark.parametrize("score,size", [(-20.0, 1e4), (-40.0, 1e6), (-300.0, 1e30)])
def test_rows_that_weigh_nothing(H, kvh, hd, length, n, score, size):
    """Committed rows far below the others' scores (the last is 0 in F32), with
    large values, in the first page and in the last."""
    rng = np.random.default_rng(n + 1)
    c, q = case(rng, H, kvh, hd, length, n, {3: (score, size), length - 2: (score, size)})
    want, tol = attention(c, q, hd ** -0.5, lambda b, i, j: j <= i)
    check(run(c, q, hd ** -0.5), want, tol)


@pytest.mark.parametrize("H,kvh,hd,length,n", SIZES)
@pytest.mark.parametrize("score,size", [(-30.0, 1e13), (-60.0, 1e26), (30.0, 1e-15)])
def test_small_weights_of_large_values(H, kvh, hd, length, n, score, size):
    """A weight of e^-30 times values of 1e13 is what the other rows give
    together; and the other way round."""
    rng = np.random.default_rng(n + 2)
    c, q = case(rng, H, kvh, hd, length, n, {length // 2: (score, size)})
    want, tol = attention(c, q, hd ** -0.5, lambda b, i, j: j <= i)
    check(run(c, q, hd ** -0.5), want, tol)


@pytest.mark.parametrize("H,kvh,hd,length,n", SIZES)
def test_tokens_that_see_a_large_row_beside_tokens_that_do_not(H, kvh, hd, length, n):
    """In one tile: each query's result has its own size."""
    if n == 1:
        pytest.skip("one token")
    rng = np.random.default_rng(n + 3)
    c, q = case(rng, H, kvh, hd, length, n, {length: (0.0, 1e8)})
    sees = trees(rng, n)
    sees[:, 0] = False
    sees[::2, 0] = True
    want, tol = attention(c, q, hd ** -0.5, lambda b, i, j: sees[i, j])
    assert np.abs(want[0]).min() < np.abs(want[1]).max() * 1e9 and np.abs(want[::2]).max() > 1e4 * np.abs(want[1::2]).max()
    check(run(c, q, hd ** -0.5, words([sees])), want, tol)


@pytest.mark.parametrize("H,kvh,hd,length,n", SIZES)
@pytest.mark.parametrize("size", [0.0, 1e-25, 1e-12, 1e12, 1e28])
def test_values_of_any_size(H, kvh, hd, length, n, size):
    """All of one size, and zeros with scores that grow by 80 before the first
    row that has values."""
    rng = np.random.default_rng(n + 4)
    if size:
        c, q = case(rng, H, kvh, hd, length, n, {})
        c.vs *= np.float32(size)
    else:
        far = {j: (80.0 * j / length - 80.0, 0.0) for j in range(length * 3 // 4)}
        c, q = case(rng, H, kvh, hd, length, n, far)
    want, tol = attention(c, q, hd ** -0.5, lambda b, i, j: j <= i)
    assert np.abs(want).max() > 1e-4 * (size or 1.0)
    # (the tolerance's own 1e-30 is below all of these)
    check(run(c, q, hd ** -0.5), want, tol)
