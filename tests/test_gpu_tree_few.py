"""Trees and masks by the kernel of few rows over f16 caches (up to 128 query
rows a sequence): against the plain 64-bit form; tolerances: kv_ref.tolerance."""
import numpy as np
import pytest

import kv_ref
from test_gpu_tree_attention import ancestors, check, device, run, words  # noqa: F401 (device: the module's fixture)

pytestmark = pytest.mark.gpu

# (H, kvh, hd, committed rows, tokens) of each sequence: one tile, some, parts
# over a long cache, rows that fill tiles and rows that do not, group of one
SIZES = [(8, 1, 128, [900], [16]), (32, 4, 128, [300], [15]), (16, 8, 64, [70], [60]), (8, 1, 128, [2500], [9]), (4, 4, 64, [40], [128]),
         (8, 2, 64, [129, 0], [13, 6]), (16, 1, 64, [3100], [7]), (6, 2, 128, [0], [40])]
BY = pytest.mark.parametrize("H,kvh,hd,lens,counts", SIZES)


@pytest.fixture(autouse=True)
def sizes_are_the_kernels(request):
    p = request.node.callspec.params
    rows = sum(p["counts"]) * (p["H"] // p["kvh"])
    assert rows <= 128 * len(p["counts"]) and rows * p["kvh"] <= 1024 and max(p["lens"]) + 64 < 10240


def masks(rng, counts):
    """Random masks; every third row sees no token of the tree."""
    sees = [rng.random((n, n)) < 0.4 for n in counts]
    for m in sees:
        m[::3] = False
    return sees


@BY
@pytest.mark.parametrize("columns", [None, 200])
def test_any_mask(H, kvh, hd, lens, counts, columns):
    """(columns: a page table wider than the sequences need, past 10240 rows,
    where trees of more than 64 rows go to the other kernel)"""
    rng = np.random.default_rng(sum(counts))
    c = kv_ref.Cache(rng, "f16", kvh, hd, lens, counts)
    if columns:
        wide = np.full((len(lens), columns), -1, np.int32)
        wide[:, :c.table.shape[1]] = c.table
        c.table = wide
    q = rng.standard_normal((sum(counts), H, hd)).astype(np.float32)
    sees = masks(rng, counts)
    want, tol = kv_ref.attention(c, 0, q, hd ** -0.5, lambda b, i, j: sees[b][i, j])
    o, t = run(c, q, hd ** -0.5, words(sees)), 0
    check(o, want, tol)
    for n, m in zip(lens, counts):
        if n == 0:
            assert (o[t:t + m:3] == 0).all()
        t += m


@BY
@pytest.mark.parametrize("branch", [1, 2, 5])
def test_branching_trees(H, kvh, hd, lens, counts, branch):
    rng = np.random.default_rng(sum(counts) + branch)
    c = kv_ref.Cache(rng, "f16", kvh, hd, lens, counts)
    q = rng.standard_normal((sum(counts), H, hd)).astype(np.float32)
    sees = [ancestors(n, branch) for n in counts]
    want, tol = kv_ref.attention(c, 0, q, hd ** -0.5, lambda b, i, j: sees[b][i, j])
    check(run(c, q, hd ** -0.5, words(sees)), want, tol)


@BY
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_values_that_are_not_finite_and_one_token_sees(H, kvh, hd, lens, counts, value):
    """In a V element of a node in each page half, and in a key: the token that
    sees it gets what is not finite in that column (for a key: in all), the
    others are as if the row were not there."""
    rng = np.random.default_rng(sum(counts) + 7)
    c = kv_ref.Cache(rng, "f16", kvh, hd, lens, counts)
    T, n, group = sum(counts), counts[0], H // kvh
    q = rng.standard_normal((T, H, hd)).astype(np.float32)
    sees = masks(rng, counts)
    nodes = sorted({1, n // 2, n - 1})
    who = [2, 4, 5]  # (token who[i] alone sees node nodes[i])
    sees[0][:, nodes] = False
    clean, tol = kv_ref.attention(c, 0, q, hd ** -0.5, lambda b, i, j: sees[b][i, j])
    for i, j in zip(who, nodes):
        sees[0][i, j] = True
    want, tol1 = kv_ref.attention(c, 0, q, hd ** -0.5, lambda b, i, j: sees[b][i, j])  # (before the values are put)
    tol, bad = np.maximum(tol, tol1), np.zeros((T, H, hd), bool)
    for x, (i, j) in enumerate(zip(who, nodes)):
        p, r = c.place(0, lens[0] + j)
        if x < 2:
            column, kv = (3, 0) if x == 0 else (hd - 4, kvh - 1)
            c.v[0, p, kv, column, r] = value
            bad[i, kv * group:(kv + 1) * group, column] = True
        else:
            c.k[0, p, 0, r, 9] = np.nan
            bad[i, :group] = True
    o = run(c, q, hd ** -0.5, words(sees))
    assert not np.isfinite(o[bad]).any()
    # (a value of infinity is that, of its sign, whatever the weight; NaN is NaN)
    first = o[who[0], :group, 3]
    assert np.isnan(first).all() if np.isnan(value) else (first == value).all()
    ok = ~bad
    assert np.isfinite(o[ok]).all() and (np.abs(o - want)[ok] <= tol[ok]).all()
    untouched = np.ones(T, bool)
    untouched[who] = False
    assert (np.abs(o - clean)[untouched] <= tol[untouched]).all()


@BY
def test_rows_behind_the_last_are_not_read(H, kvh, hd, lens, counts):
    """Whatever lies behind a sequence's rows in its last page (here infinity
    and NaN in turn) has no part in it, causal or masked."""
    rng = np.random.default_rng(sum(counts) + 9)
    c = kv_ref.Cache(rng, "f16", kvh, hd, lens, counts)
    for b, (n, m) in enumerate(zip(lens, counts)):
        p, r = c.place(b, n + m - 1)
        c.k[0, p, :, r + 1:], c.v[0, p, :, :, r + 1:] = np.inf, np.inf
        c.v[0, p, :, ::2, r + 1:] = np.nan
    q = rng.standard_normal((sum(counts), H, hd)).astype(np.float32)
    want, tol = kv_ref.attention(c, 0, q, hd ** -0.5, lambda b, i, j: j <= i)
    check(run(c, q, hd ** -0.5), want, tol)
    check(run(c, q, hd ** -0.5, words([np.tril(np.ones((n, n), bool)) for n in counts])), want, tol)
