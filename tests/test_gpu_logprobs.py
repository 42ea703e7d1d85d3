"""Log-probabilities, ranks, entropies and alternatives against a 64-bit form."""
import numpy as np
import pytest

import kv_ref
import tie_amd

pytestmark = pytest.mark.gpu
F32_LOW = -3.4028234663852886e38


@pytest.fixture(scope="module", autouse=True)
def device():
    import torch
    assert torch.cuda.is_available(), "GPU test without a GPU"
    tie_amd.init(0)
    yield
    tie_amd.shutdown()


def expect(l, tokens, T, n):
    """logprob, rank, entropy, top tokens, top logprobs, and what logprobs and entropies may be off by.

    An exponential's argument y / T has three F32 roundings (the difference, two of the product) and v_exp_f32 is good to
    an ulp: p is off by at most (1 + 2 |y| / T) 2^-23 of itself, log Z by the mean of that under p, and sum y p by the mean of it
    times |y| / T; the 64-bit rest is exact beside them.  Then one rounding to F32."""
    N, V = l.shape
    T = np.float64(np.float32(T))
    x = l.astype(np.float64)
    m = x.max(1, keepdims=True)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        y = (x - m) / T
        p = np.exp(y)
        z = p.sum(1, keepdims=True)
        p, logz = p / z, np.log(z)
        lp = y - logz
        entropy = -np.where(p > 0, p * lp, 0.0).sum(1)
        a = np.where(p > 0, -y, 0.0)
        off = (p * (1 + 2 * a)).sum(1) * 2.0 ** -23
        off_e = off + (p * a * (1 + 2 * a)).sum(1) * 2.0 ** -23 + off * (p * a).sum(1)
    order = np.lexsort((np.arange(V)[None].repeat(N, 0), -x), axis=1)[:, :n] if n else np.zeros((N, 0), np.int64)
    top = np.take_along_axis(lp, order, 1)
    tops = np.where(np.take_along_axis(x, order, 1) > -np.inf, order, -1)
    if n > V:
        tops = np.concatenate([tops, np.full((N, n - V), -1)], 1)
        top = np.concatenate([top, np.full((N, n - V), -np.inf)], 1)
    t = np.clip(tokens, 0, V - 1)
    mine = np.take_along_axis(x, t[:, None], 1)
    rank = ((x > mine) | ((x == mine) & (np.arange(V) < t[:, None]))).sum(1)
    of = np.take_along_axis(lp, t[:, None], 1)[:, 0]
    out = (tokens < 0) | (tokens >= V)
    rank, of = np.where(out, -1, rank), np.where(out, np.nan, of)
    bad = ~np.isfinite(z[:, 0]) | ~np.isfinite(m[:, 0])
    rank[bad], of[bad], entropy[bad], tops[bad], top[bad] = -1, np.nan, np.nan, -1, np.nan
    return of, rank, entropy, tops, top, off, off_e


def call(l, tokens, T, n, work=None, wide=0):
    import torch
    N, V = l.shape
    ld = torch.full((N, V + wide), 1e30, device="cuda")[:, wide // 2: wide // 2 + V]
    ld.copy_(torch.from_numpy(l))
    td = torch.from_numpy(tokens.astype(np.int32)).cuda()
    f = lambda *s: torch.full(s, -7.0, device="cuda")  # noqa: E731
    i = lambda *s: torch.full(s, -7, dtype=torch.int32, device="cuda")  # noqa: E731
    lp, rank, ent, tt, tl = f(N), i(N), f(N), i(N, n), f(N, n)
    if work is not None:
        work = torch.zeros(tie_amd.token_logprobs_work_bytes(V, N, n), dtype=torch.uint8, device="cuda")
    for _ in range(2):
        tie_amd.token_logprobs(ld, td, lp, rank=rank, entropy=ent, top_tokens=tt if n else None, top_logprobs=tl if n else None,
                               temperature=T, work=work)
    torch.cuda.synchronize()
    return [x.cpu().numpy() for x in (lp, rank, ent, tt, tl)]


def check(l, tokens, T=1.0, n=20, **kw):
    got = call(l, tokens, T, n, **kw)
    of, rank, ent, tops, top, off, off_e = expect(l, tokens, T, n)
    assert np.array_equal(got[1], rank), (np.argwhere(got[1] != rank)[:5], got[1][got[1] != rank][:5], rank[got[1] != rank][:5])
    assert np.array_equal(got[3], tops), np.argwhere(got[3] != tops)[:5]
    for g, w, o in ((got[0], of, off), (got[2], ent, off_e), (got[4], top, off[:, None])):
        # (what lies past F32's range, from 2^128 - 2^103 on, rounds to infinity: a logit of the lowest value at half the temperature)
        w = np.where(np.abs(w) >= 2.0 ** 128 - 2.0 ** 103, np.copysign(np.inf, w), w)
        with np.errstate(invalid="ignore"):
            fine = (np.isnan(g) & np.isnan(w)) | (g == w) | (np.abs(g - w) <= o + 2.0 ** -24 * np.abs(w) + 1e-45)
        assert fine.all(), (np.argwhere(~fine)[:5], g[~fine][:5], w[~fine][:5])


def some(rng, N, V, size=2.5):
    return (size * rng.standard_normal((N, V))).astype(np.float32)


@pytest.mark.parametrize("N", [1, 3, 61])
@pytest.mark.parametrize("V", [1, 2, 63, 64, 65, 1000, 4095, 4096, 4097, 8195, 40001])
@pytest.mark.parametrize("n,T", [(0, 1.0), (1, 1.0), (20, 0.7), (64, 3.0)])
def test_sizes(N, V, n, T):
    rng = np.random.default_rng(V + N)
    check(some(rng, N, V), rng.integers(0, V, N), T, n)


@pytest.mark.parametrize("N,V,n", [(1, 151936, 20), (7, 151936, 5), (1030, 5000, 20), (1023, 9000, 3), (2000, 300, 64)])
def test_rows_in_parts_and_whole(N, V, n):
    rng = np.random.default_rng(V)
    check(some(rng, N, V), rng.integers(0, V, N), 1.0, n, work=True)


def test_a_row_of_more_parts_than_a_workgroup_has_threads():
    rng = np.random.default_rng(2)
    l = some(rng, 1, 9000001)
    check(l, np.array([8999999]), 1.0, 20, work=True)
    l[0, rng.integers(0, 9000001, 5)] = 30.0
    check(l, np.array([77]), 0.5, 3)


@pytest.mark.parametrize("V", [100, 5000, 30000])
def test_equal_logits(V):
    """The lowest index first among equals: rows of one value, of few values, of -0 and 0, with the token anywhere."""
    rng = np.random.default_rng(V)
    l = np.zeros((9, V), np.float32)
    l[1] = rng.integers(0, 3, V)
    l[2] = rng.integers(0, 2, V) * 1e-40
    l[3] = np.where(rng.random(V) < 0.5, -0.0, 0.0)
    l[4] = rng.integers(0, V // 20, V)
    l[5, rng.integers(0, V, 5)] = -1.0
    l[6] = -3.25
    l[7, -1] = 1.0
    l[8, 0] = 1.0
    for tokens in (rng.integers(0, V, 9), np.zeros(9, int), np.full(9, V - 1)):
        for n in (1, 20, 64):
            check(l, tokens, 1.0, n)


@pytest.mark.parametrize("V", [50, 6000])
def test_rows_in_order(V):
    """Ascending and descending rows: every logit, or none behind the first, is a candidate."""
    l = np.stack([np.arange(V), -np.arange(V), np.arange(V) % 777, np.arange(V) // 64]).astype(np.float32) * 0.01
    check(l, np.array([0, V - 1, V // 2, V // 3]), 1.0, 64)


@pytest.mark.parametrize("V", [70, 5000, 20001])
def test_masked_logits(V):
    """-infinity, the lowest finite value and -1e9 in masked places; rows that leave one token, or fewer than asked for."""
    rng = np.random.default_rng(V)
    l = some(rng, 12, V)
    for r, fill in enumerate([-np.inf, F32_LOW, -1e9]):
        l[4 * r][rng.random(V) < 0.5] = fill
        l[4 * r + 1][rng.permutation(V)[: V - 7]] = fill
        l[4 * r + 2][np.arange(V) != V // 2] = fill
        l[4 * r + 3][np.arange(V) != V - 1] = fill
    for tokens in (rng.integers(0, V, 12), np.full(12, V // 2)):
        check(l, tokens, 1.0, 20)
        check(l, tokens, 0.5, 64)


@pytest.mark.parametrize("V", [64, 9000])
def test_rows_that_are_no_distribution_and_tokens_that_are_none(V):
    rng = np.random.default_rng(V)
    l = some(rng, 8, V)
    l[0] = -np.inf
    l[1, 5] = np.nan
    l[2, V - 1] = np.inf
    l[3] = np.nan
    l[4] = np.where(np.arange(V) % 2, np.nan, -np.inf)
    check(l, np.array([0, 5, 3, 0, 0, -1, V, 0x7fffffff]), 1.0, 20)
    check(l, np.array([0, 5, 3, 0, 0, -1, V, -0x80000000]), 1.0, 0)


@pytest.mark.parametrize("size,T", [(1e-6, 1.0), (100.0, 1.0), (1e30, 1.0), (2.5, 1e-6), (2.5, 1e6), (1e-30, 1e-6), (F32_LOW / 10, 1e6)])
def test_extremes(size, T):
    rng = np.random.default_rng(3)
    check(some(rng, 3, 5000, size), rng.integers(0, 5000, 3), T, 20)


def test_sure_tokens_keep_their_small_logarithms():
    """Where one token has nearly all, log p is -(the rest): the sums in 64 bits hold it."""
    l = np.full((4, 5000), -20.0, np.float32)
    l[:, 17] = [0.0, 5.0, 8.0, 12.0]
    got = call(l, np.full(4, 17), 1.0, 5)
    of = expect(l, np.full(4, 17), 1.0, 5)[0]
    # the rest is 4999 equal exponentials, off by (1 + 2 |y|) 2^-23 each; 1 + rest is rounded at 2^-53
    rest = -of
    assert (np.abs(got[0] - of) <= rest * (1 + 2 * 32) * 2.0 ** -23 + 2.0 ** -52).all()


@pytest.mark.parametrize("wide", [4, 7, 64])
def test_strides_and_alignment(wide):
    rng = np.random.default_rng(wide)
    check(some(rng, 5, 9001), rng.integers(0, 9001, 5), 1.0, 20, wide=wide)
    check(some(rng, 5, 8192), rng.integers(0, 8192, 5), 1.0, 20, wide=wide)


def test_outputs_left_out():
    import torch
    l = torch.randn(3, 700, device="cuda")
    ent, lp = torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda")
    tie_amd.token_logprobs(l, entropy=ent)
    tie_amd.token_logprobs(l, torch.zeros(3, dtype=torch.int32, device="cuda"), lp)
    want = torch.log_softmax(l.double(), 1)
    torch.cuda.synchronize()
    assert ((ent - -(want.exp() * want).sum(1)).abs() < 1e-5).all()
    assert ((lp - want[:, 0]).abs() < 1e-5).all()


def test_replayed_graph():
    import torch
    rng = np.random.default_rng(6)
    N, V, n = 5, 30000, 8
    l, tok = torch.zeros(N, V, device="cuda"), torch.zeros(N, dtype=torch.int32, device="cuda")
    lp, ent, rank = torch.zeros(N, device="cuda"), torch.zeros(N, device="cuda"), torch.zeros(N, dtype=torch.int32, device="cuda")
    tt, tl = torch.zeros(N, n, dtype=torch.int32, device="cuda"), torch.zeros(N, n, device="cuda")
    work = torch.zeros(tie_amd.token_logprobs_work_bytes(V, N, n), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with kv_ref.capture(graph):
        tie_amd.token_logprobs(l, tok, lp, rank=rank, entropy=ent, top_tokens=tt, top_logprobs=tl, work=work)
    for step in range(4):
        x, t = some(rng, N, V), rng.integers(0, V, N)
        l.copy_(torch.from_numpy(x))
        tok.copy_(torch.from_numpy(t.astype(np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        got = [a.cpu().numpy() for a in (lp, rank, ent, tt, tl)]
        eager = call(x, t, 1.0, n)
        for a, b in zip(got, eager):
            assert np.array_equal(a.view(np.uint32), b.view(np.uint32)), step
