"""Log-probabilities of rows whose mass lies in many equal or near logits, where the exponentials' errors do not average
out: against the 64-bit form, to an ulp of each exponential whatever its argument."""
import numpy as np
import pytest

import tie_amd
from test_gpu_logprobs import call, expect

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    import torch
    assert torch.cuda.is_available(), "GPU test without a GPU"
    tie_amd.init(0)
    yield
    tie_amd.shutdown()


def bounds(l, T):
    """What log Z and the entropy may be off by.

    Arguments are 64 bits wide; their rest beside a whole power of two is rounded to 23 bits (off by 2^-24, log 2 times
    that of p: 0.35 2^-23), and v_exp_f32 is good to an ulp (2^-23 of a result from 1 on): p is off by at most
    e = 1.4 2^-23 of itself, and that of the largest logit is exactly 1.  So log Z by e times the mass of the others,
    the entropy log Z + sum p a (a: the argument's size) by that, by e sum p a for the exponentials and by as much of the
    sum as Z is off by."""
    e = 1.4 * 2.0 ** -23
    x = l.astype(np.float64)
    a = (x.max(1, keepdims=True) - x) / np.float64(np.float32(T))
    p = np.exp(-a)
    p /= p.sum(1, keepdims=True)
    with np.errstate(invalid="ignore"):
        off = e * np.where(a > 0, p, 0.0).sum(1)
        mean = np.where(p > 0, p * a, 0.0).sum(1)
    return off, off + e * mean + off * mean


def check(l, tokens, T, n=3, times=1):
    """times: so many copies of the rows in the call, with equal results."""
    N = len(l)
    got = call(np.tile(l, (times, 1)), np.tile(tokens, times), T, n)
    for g in got:
        assert np.array_equal(g, np.tile(g[:N], (times,) + (1,) * (g.ndim - 1)), equal_nan=g.dtype == np.float32)
    lp, rank, ent, tops, top = (g[:N] for g in got)
    w = expect(l, tokens, T, n)
    off, off_e = bounds(l, T)
    assert np.array_equal(rank, w[1]) and np.array_equal(tops, w[3])
    for g, want, o in ((lp, w[0], off), (ent, w[2], off_e), (top, w[4], off[:, None])):
        with np.errstate(invalid="ignore"):
            wrong = np.where(g == want, -1.0, np.abs(g - want) - (o + 2.0 ** -24 * np.abs(want)))
        assert (wrong <= 0).all(), (T, float(wrong.max()), g[wrong > 0][:4], want[wrong > 0][:4], np.broadcast_to(o, g.shape)[wrong > 0][:4])


def rows(V, T):
    """Equal logits below four largest ones, which each of a workgroup's waves meets first, at distances where they weigh
    as much as those (and where an argument's half unit in the last place is 5e-7 of an exponential)."""
    d = (np.linspace(11.1, 12.9, 24) * T).astype(np.float32)
    l = np.repeat(-d[:, None], V, 1)
    l[:, :1024:256] = 0.0
    return l


@pytest.mark.parametrize("T", [1.0, 0.7, 1.3])
@pytest.mark.parametrize("up", [0.0, 3.7, -20.3, 300.2])  # (where the difference of two F32 logits is no F32)
@pytest.mark.parametrize("V", [151936, 65001])
def test_flat_tails(V, up, T):
    l = rows(V, T) + np.float32(up)
    check(l, np.arange(len(l)) % 4 * 256, T, times=17)  # (408 rows: a workgroup each)
    check(l[:2], np.array([0, 77]), T)  # (in parts)


@pytest.mark.parametrize("T", [1.0, 0.7, 3.0])
def test_tails_of_near_logits_and_masks(T):
    """Tails that spread over a few units in the last place, over a whole unit, and with half of them masked."""
    rng = np.random.default_rng(1)
    l = rows(100000, T)
    l[:8] = np.nextafter(l[:8], np.where(rng.random(l[:8].shape) < 0.5, -1e9, 1e9).astype(np.float32))
    l[8:12] += rng.random(l[8:12].shape).astype(np.float32)
    l[12:18][rng.random(l[12:18].shape) < 0.5] = -np.inf
    l[18:][rng.random(l[18:].shape) < 0.5] = -3.4028234663852886e38
    l[:, :1024:256] = 0.25
    check(l, np.arange(len(l)) % 4 * 256, T, 1, times=17)


@pytest.mark.parametrize("N,V", [(2, 40001), (600, 9000)])
def test_rows_without_a_distribution_between_others(N, V):
    """NaN anywhere in a row (the first, a middle, the last chunk; alone in a chunk of masked ones), +infinity, nothing: NaN, and
    the rows beside them as they are."""
    rng = np.random.default_rng(V)
    good = (2.5 * rng.standard_normal((N, V))).astype(np.float32)
    tokens = rng.integers(0, V, N)
    beside = call(good, tokens, 1.0, 5)
    keep = np.arange(N) != 1
    for where in (0, 4095, 4096, V // 2, V - 1):
        for what in ("nan", "masked", "inf", "both", "none"):
            l = good.copy()
            if what in ("masked", "none"):
                l[1] = -np.inf
            if what != "none":
                l[1, where] = np.inf if what == "inf" else np.nan
            if what == "both":
                l[1, (where + 5000) % V] = np.inf
            got = call(l, tokens, 1.0, 5)
            lp, rank, ent, tops, top = got
            assert np.isnan(lp[1]) and np.isnan(ent[1]) and np.isnan(top[1]).all() and rank[1] == -1 and (tops[1] == -1).all(), (where, what)
            assert all(np.array_equal(g[keep], b[keep]) for g, b in zip(got, beside)), (where, what)


def test_the_lowest_values_as_the_largest():
    """Rows whose largest logit is F32's lowest, beside masked ones, and rows of large magnitudes at both temperatures' ends."""
    low = np.float32(-3.4028234663852886e38)
    l = np.full((4, 5000), -np.inf, np.float32)
    l[0, 7:4000:3], l[1, 4999], l[2, :100] = low, low, np.float32(3e38)
    l[3, :200], l[3, 200:300] = np.float32(1e30), low
    for T in (1.0, 1e-6, 1e6):
        check(l, np.array([7, 4999, 3, 0]), T, 4)
