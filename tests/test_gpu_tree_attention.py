"""Attention of single tokens, causal chunks and drafted trees over the paged
cache, against a plain 64-bit form.  Every row of the cache that belongs to no
sequence holds NaN.  Tolerances: kv_ref.tolerance (derived there)."""
import gc

import numpy as np
import pytest

import kv_ref
import tie_amd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    import torch
    assert torch.cuda.is_available(), "GPU test without a GPU"
    tie_amd.init(0)
    yield
    tie_amd.shutdown()


def cuda(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def parents(n, branch):
    return [(j - 1) // branch for j in range(n)]


def ancestors(n, branch):
    """sees[i][j]: node i's path from the root holds j."""
    sees = np.zeros((n, n), bool)
    for i, p in enumerate(parents(n, branch)):
        if p >= 0:
            sees[i] = sees[p]
        sees[i, i] = True
    return sees


def words(sees, n_words=None):
    """[T][words] of int64 bit patterns of a list of boolean matrices."""
    w = n_words or max(-(-m.shape[1] // 64) for m in sees)
    out = np.zeros((sum(len(m) for m in sees), w), np.uint64)
    t = 0
    for m in sees:
        for row in m:
            for j in np.nonzero(row)[0]:
                if j < 64 * w:
                    out[t, j // 64] |= np.uint64(1) << np.uint64(j % 64)
            t += 1
    return out.view(np.int64)


def run(c, q, scale, mask=None, stride=0, layer=0, **kw):
    """The kernel's result, its rows `stride` floats apart (0: dense), with two
    rows more than there are tokens, which must stay."""
    import torch
    T, H, hd = q.shape
    kv, seqs = c.gpu(), c.seqs()
    w = H * hd
    qb = torch.full((T + 2, max(stride, w)), 3.0, device="cuda")
    ob = torch.full((T + 2, max(stride, w)), -7.0, device="cuda")
    qb[:T, :w] = cuda(q.reshape(T, w))
    m = cuda(mask) if mask is not None else None
    torch.cuda.synchronize()
    kv.attention(layer, seqs, qb[:, :w], ob[:, :w], scale, mask=m, **kw)
    torch.cuda.synchronize()
    o = ob.cpu().numpy()
    assert (o[T:] == -7.0).all() and (o[:, w:] == -7.0).all()
    return o[:T, :w].reshape(T, H, hd)


def check(o, want, tol, what=""):
    assert np.isfinite(o).all(), what
    err = np.abs(o - want)
    assert (err <= tol).all(), (what, float((err / tol).max()), float(np.linalg.norm(o - want) / np.linalg.norm(want)))


HEADS = [(8, 1, 128), (32, 4, 128), (16, 1, 128), (6, 2, 64), (5, 5, 64), (12, 4, 128)]


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("H,kvh,hd", HEADS)
@pytest.mark.parametrize("lens", [[0], [1], [63, 64, 65], [0, 500, 127], [1500]])
def test_single_tokens(kind, H, kvh, hd, lens):
    rng = np.random.default_rng(len(lens) * 7 + H)
    c = kv_ref.Cache(rng, kind, kvh, hd, lens, [1] * len(lens))
    q = rng.standard_normal((len(lens), H, hd)).astype(np.float32) * 2
    want, tol = kv_ref.attention(c, 0, q, hd ** -0.5, lambda b, i, j: True)
    check(run(c, q, hd ** -0.5), want, tol)


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("H,kvh,hd,lens,counts", [(8, 1, 128, [0], [2]), (8, 2, 128, [5], [70]), (4, 4, 64, [63, 0, 200], [33, 130, 1]),
                                                  (32, 4, 128, [61], [40]), (6, 2, 64, [0], [259]), (16, 1, 128, [100], [37])])
def test_causal_chunks(kind, H, kvh, hd, lens, counts):
    rng = np.random.default_rng(sum(counts))
    c = kv_ref.Cache(rng, kind, kvh, hd, lens, counts, layers=2)
    q = rng.standard_normal((sum(counts), H, hd)).astype(np.float32)
    want, tol = kv_ref.attention(c, 1, q, hd ** -0.5, lambda b, i, j: j <= i)
    check(run(c, q, hd ** -0.5, layer=1, stride=H * hd + 8), want, tol)
    check(run(c, q, hd ** -0.5, layer=1, stride=H * hd + 3), want, tol)


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("H,kvh,hd,lens,counts,branch", [(8, 1, 128, [700], [26], 3), (32, 4, 128, [0, 63, 129], [5, 64, 17], 2),
                                                         (6, 2, 64, [40], [150], 4), (16, 1, 128, [62, 1], [2, 3], 1),
                                                         (8, 8, 64, [64, 10], [64, 100], 3)])
def test_trees(kind, H, kvh, hd, lens, counts, branch):
    rng = np.random.default_rng(sum(counts) + branch)
    c = kv_ref.Cache(rng, kind, kvh, hd, lens, counts)
    q = rng.standard_normal((sum(counts), H, hd)).astype(np.float32)
    sees = [ancestors(n, branch) for n in counts]
    want, tol = kv_ref.attention(c, 0, q, hd ** -0.5, lambda b, i, j: sees[b][i, j])
    check(run(c, q, hd ** -0.5, words(sees)), want, tol)
    # a word more than needed, and bits that name no token
    w = words(sees, max(-(-n // 64) for n in counts) + 1)
    w[:, -1] = -1
    check(run(c, q, hd ** -0.5, w), want, tol)


@pytest.mark.parametrize("kind", ["f16", "i8"])
def test_any_mask(kind):
    """Random masks, rows that see nothing (0, exactly) or only committed rows."""
    rng = np.random.default_rng(77)
    lens, counts, H, kvh, hd = [0, 30, 0], [70, 90, 3], 8, 2, 64
    c = kv_ref.Cache(rng, kind, kvh, hd, lens, counts)
    q = rng.standard_normal((sum(counts), H, hd)).astype(np.float32)
    sees = [rng.random((n, n)) < 0.3 for n in counts]
    for m in sees:
        m[::3] = False
    want, tol = kv_ref.attention(c, 0, q, 0.2, lambda b, i, j: sees[b][i, j])
    o = run(c, q, 0.2, words(sees))
    check(o, want, tol)
    assert (o[0:70:3] == 0).all() and (o[160:163:3] == 0).all() and (o[70:160] != 0).any(-1).all()


def test_narrow_masks():
    """Fewer words than tokens: the tokens past them are not seen."""
    rng = np.random.default_rng(78)
    c = kv_ref.Cache(rng, "i8", 1, 64, [10], [140])
    q = rng.standard_normal((140, 2, 64)).astype(np.float32)
    sees = np.tril(np.ones((140, 140), bool))
    want, tol = kv_ref.attention(c, 0, q, 0.125, lambda b, i, j: sees[i, j] and j < 64)
    check(run(c, q, 0.125, words([sees], 1)), want, tol)


@pytest.mark.parametrize("kind", ["f16", "i8"])
def test_masked_values_that_are_not_finite(kind):
    """NaN and infinity in rows that some tokens see and others do not: those
    that do not are as if the rows were not there, those that do get what is
    not finite in the columns it is in (all, for a key)."""
    rng = np.random.default_rng(79)
    H, kvh, hd, n = 8, 2, 64, 40
    c = kv_ref.Cache(rng, kind, kvh, hd, [50], [n])
    q = rng.standard_normal((n, H, hd)).astype(np.float32)
    sees = ancestors(n, 2)
    sees[:, 5] = sees[:, 20] = sees[:, 33] = False
    sees[7, 5] = sees[9, 20] = sees[11, 33] = True
    want, tol = kv_ref.attention(c, 0, q, hd ** -0.5, lambda b, i, j: sees[i, j])

    def at(j):
        return c.place(0, 50 + j)

    (p5, r5), (p20, r20), (p33, r33) = at(5), at(20), at(33)
    if kind == "f16":
        c.v[0, p5, 0, 3, r5] = np.nan
        c.v[0, p20, 1, 60, r20] = np.inf
        c.k[0, p33, 0, r33, 9] = np.nan
    else:
        c.vs[0, p5, 0, r5] = np.nan
        c.vs[0, p20, 1, r20] = np.nan
        c.ks[0, p33, 0, r33] = np.nan
    o = run(c, q, hd ** -0.5, words([sees]))
    half = H // kvh
    bad = np.zeros_like(o, bool)
    if kind == "f16":
        bad[7, :half, 3] = True
        bad[9, half:, 60] = True
    else:
        bad[7, :half] = True
        bad[9, half:] = True
    bad[11, :half] = True
    assert not np.isfinite(o[bad]).any()
    ok = ~bad
    assert np.isfinite(o[ok]).all()
    assert (np.abs(o - want)[ok] <= tol[ok]).all()


# sizes that take each kernel: tiles of 16 rows, of 64 (cut into parts or
# whole) and of 128
@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("H,kvh,hd,length,n", [(8, 1, 128, 900, 30), (16, 1, 128, 900, 41), (8, 2, 64, 700, 90), (64, 8, 64, 70, 300),
                                               (64, 4, 128, 45, 515), (64, 2, 64, 100, 515)])
def test_any_mask_at_every_size(kind, H, kvh, hd, length, n):
    """Random masks, rows that see nothing, and rows of the cache with values
    that are not finite, which one token sees and the others do not."""
    rng = np.random.default_rng(n)
    lens, counts = [length, 0], [n, 6]
    c = kv_ref.Cache(rng, kind, kvh, hd, lens, counts)
    q = rng.standard_normal((n + 6, H, hd)).astype(np.float32)
    sees = [rng.random((m, m)) < 0.3 for m in counts]
    sees[0][::3] = sees[1][::2] = False
    sees[0][:, [5, 20, 29]] = False
    want, tol = kv_ref.attention(c, 0, q, hd ** -0.5, lambda b, i, j: sees[b][i, j])
    sees[0][[7, 9, 11], [5, 20, 29]] = True
    (p5, r5), (p20, r20), (p29, r29) = (c.place(0, length + j) for j in (5, 20, 29))
    bad, half = np.zeros((n + 6, H, hd), bool), H // kvh
    if kind == "f16":
        c.v[0, p5, 0, 3, r5] = np.nan
        c.v[0, p20, kvh - 1, hd - 4, r20] = np.inf
        c.k[0, p29, 0, r29, 9] = np.nan
        bad[7, :half, 3] = bad[9, -half:, hd - 4] = bad[11, :half] = True
    else:
        c.vs[0, p5, 0, r5] = np.nan
        c.vs[0, p20, kvh - 1, r20] = np.nan
        c.ks[0, p29, 0, r29] = np.nan
        bad[7, :half] = bad[9, -half:] = bad[11, :half] = True
    o = run(c, q, hd ** -0.5, words(sees))
    assert not np.isfinite(o[bad]).any()
    # (tokens 7, 9 and 11 see a row more than `want` knows in their other heads)
    ok = ~bad
    ok[[7, 9, 11]] = False
    assert np.isfinite(o[ok]).all() and (np.abs(o - want)[ok] <= tol[ok]).all()
    assert (o[n:n + 6:2] == 0).all() and (o[:n] != 0).any(-1).all()


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("H,kvh,hd,lens,counts", [(64, 4, 128, [70, 3], [300, 230]), (64, 2, 64, [10], [520]), (8, 1, 128, [2500], [33]),
                                                  (8, 1, 128, [2500], [7]), (16, 4, 64, [700, 0, 65], [20, 64, 130])])
def test_causal_at_every_size(kind, H, kvh, hd, lens, counts):
    rng = np.random.default_rng(sum(counts) + H)
    c = kv_ref.Cache(rng, kind, kvh, hd, lens, counts)
    q = rng.standard_normal((sum(counts), H, hd)).astype(np.float32)
    want, tol = kv_ref.attention(c, 0, q, hd ** -0.5, lambda b, i, j: j <= i)
    check(run(c, q, hd ** -0.5), want, tol)


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("most", [2, 5, 40])
def test_many_sequences(kind, most):
    """More than a wave has lanes, of 0 to `most` - 1 tokens, one of them long."""
    rng = np.random.default_rng(90 + most)
    lens, counts = [int(x) for x in rng.integers(0, 100, 140)], [int(x) for x in rng.integers(0, most, 140)]
    lens[100], counts[63:66], counts[100] = 1500, [0, 0, 0], 1
    c = kv_ref.Cache(rng, kind, 2, 64, lens, counts)
    q = rng.standard_normal((sum(counts), 8, 64)).astype(np.float32)
    want, tol = kv_ref.attention(c, 0, q, 0.125, lambda b, i, j: j <= i)
    check(run(c, q, 0.125), want, tol)


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("H,kvh,hd,lens,counts", [(8, 1, 128, [700], [3]), (16, 1, 128, [900, 4], [41, 2]), (64, 4, 128, [45], [515])])
def test_rows_behind_the_last_sequence(kind, H, kvh, hd, lens, counts):
    """A batch padded to more token rows than its sequences have, and a replay
    of it with other ranges: rows of no sequence stay."""
    import torch
    rng = np.random.default_rng(95)
    c = kv_ref.Cache(rng, kind, kvh, hd, lens, counts)
    kv, T = c.gpu(), sum(counts)
    q = rng.standard_normal((T + 9, H, hd)).astype(np.float32)
    first = cuda(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
    seqs = tie_amd.KVSeqs(cuda(c.table), cuda(np.array(lens, np.int32)), first, T + 9)
    qd, out = cuda(q), torch.full((T + 9, H, hd), -7.0, device="cuda")
    work = torch.zeros(kv.attention_work_bytes(seqs, H), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    g, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with kv_ref.capture(g, stream):
        kv.attention(0, seqs, qd, out, hd ** -0.5, work=work, stream=torch.cuda.current_stream().cuda_stream)
    for last in (counts[-1], 1, counts[-1]):
        c.counts[-1] = last
        n = sum(c.counts)
        first[-1] = n
        out.fill_(-7.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want, tol = kv_ref.attention(c, 0, q[:n], hd ** -0.5, lambda b, i, j: j <= i)
        o = out.cpu().numpy()
        check(o[:n], want, tol)
        assert (o[n:] == -7.0).all()
    del g
    gc.collect()


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("size", [1e-4, 1.0, 3e3])
def test_sizes_of_queries_and_values(kind, size):
    """Values and queries of other sizes than a trained layer's, and rows a
    thousandth of their neighbours: both parts of a split stay in range."""
    rng = np.random.default_rng(80)
    lens, n, H, kvh, hd = [300], 5, 8, 1, 128
    c = kv_ref.Cache(rng, kind, kvh, hd, lens, [n], fill=False)
    mag = np.where(rng.random((305, 1, 1)) < 0.5, 1e-3, 1.0)
    c.set_rows(0, 0, 0, rng.standard_normal((305, kvh, hd)), size * mag * rng.standard_normal((305, kvh, hd)))
    q = rng.standard_normal((n, H, hd)).astype(np.float32) / np.float32(size)
    q[3] = 0.0
    scale = size * hd ** -0.5
    want, tol = kv_ref.attention(c, 0, q, scale, lambda b, i, j: j <= i)
    check(run(c, q, scale), want, tol)


@pytest.mark.parametrize("kind", ["f16", "i8"])
def test_large_scores(kind):
    """Scores of several hundred, one row far above the rest, and the running
    maximum growing to the last page."""
    rng = np.random.default_rng(81)
    H, kvh, hd, L = 8, 1, 64, 700
    c = kv_ref.Cache(rng, kind, kvh, hd, [L - 1], [1], fill=False)
    k = rng.standard_normal((L, kvh, hd)) * np.linspace(0.1, 12.0, L)[:, None, None]
    c.set_rows(0, 0, 0, k, rng.standard_normal((L, kvh, hd)))
    q = (rng.standard_normal((1, H, hd)) * 8).astype(np.float32)
    want, tol = kv_ref.attention(c, 0, q, 1.0, lambda b, i, j: True)
    check(run(c, q, 1.0), want, tol)


def test_bad_sequences_give_nan():
    """A page that is none, a negative length, a length past the table: NaN for
    that sequence's rows alone."""
    import torch
    rng = np.random.default_rng(82)
    lens, counts, H, kvh, hd = [100, 100, 100, 100, 100], [3, 3, 3, 3, 3], 8, 2, 64
    c = kv_ref.Cache(rng, "i8", kvh, hd, lens, counts)
    q = rng.standard_normal((15, H, hd)).astype(np.float32)
    want, tol = kv_ref.attention(c, 0, q, 0.125, lambda b, i, j: j <= i)
    c.table[0, 1], c.table[3, 0] = -1, c.n_pages
    c.lens[1], c.lens[4] = -1, 126
    kv, seqs = c.gpu(), c.seqs()
    out, qd = torch.zeros(15, H, hd, device="cuda"), cuda(q)
    torch.cuda.synchronize()
    kv.attention(0, seqs, qd, out, 0.125)
    torch.cuda.synchronize()
    o = out.cpu().numpy()
    for b in (0, 1, 3, 4):
        assert np.isnan(o[3 * b: 3 * b + 3]).all(), b
    assert (np.abs(o - want)[6:9] <= tol[6:9]).all()


def test_query_that_is_not_finite():
    rng = np.random.default_rng(83)
    c = kv_ref.Cache(rng, "f16", 1, 64, [70], [4])
    q = rng.standard_normal((4, 4, 64)).astype(np.float32)
    want, tol = kv_ref.attention(c, 0, q, 0.125, lambda b, i, j: j <= i)
    q[1, 2, 5], q[2, 0, 0] = np.nan, np.inf
    o = run(c, q, 0.125)
    bad = np.zeros((4, 4), bool)
    bad[1, 2] = bad[2, 0] = True
    assert np.isnan(o[bad]).all() and (np.abs(o - want)[~bad] <= tol[~bad]).all()


@pytest.mark.parametrize("kind,lens,counts", [("i8", [3000, 10, 777], [1, 1, 1]), ("f16", [200], [150]), ("f16", [2000], [9])])
def test_in_place_streams_work_and_graphs(kind, lens, counts):
    """out over q; the caller's memory and the stream's give equal bits; so do
    two streams at once, and replays of a captured call between eager ones."""
    import torch
    rng = np.random.default_rng(84)
    H, kvh, hd, T = 32, 4, 128, sum(counts)
    c = kv_ref.Cache(rng, kind, kvh, hd, lens, counts)
    kv, seqs = c.gpu(), c.seqs()
    q = cuda(rng.standard_normal((T, H, hd)).astype(np.float32))
    outs = [torch.zeros_like(q) for _ in range(4)]
    torch.cuda.synchronize()
    kv.attention(0, seqs, q, outs[0], 0.09)
    torch.cuda.synchronize()
    want = outs[0].clone()
    both = q.clone()
    need = kv.attention_work_bytes(seqs, H)
    work = torch.zeros(need, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    kv.attention(0, seqs, both, both, 0.09)
    kv.attention(0, seqs, q, outs[1], 0.09, work=work)
    torch.cuda.synchronize()
    assert torch.equal(both, want) and torch.equal(outs[1], want)
    with pytest.raises(tie_amd.TieError):
        kv.attention(0, seqs, q, outs[1], 0.09, work=work[: need - 16])
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(8):
        kv.attention(0, seqs, q, outs[i % 2], 0.09, stream=streams[i % 2].cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        mine = torch.zeros(need, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        with kv_ref.capture(g, streams[i]):
            kv.attention(0, seqs, q, outs[2 + i], 0.09, work=mine, stream=torch.cuda.current_stream().cuda_stream)
        graphs.append((g, mine))
    for rep in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i][0].replay()
        kv.attention(0, seqs, q, outs[0], 0.09, stream=streams[0].cuda_stream)
        torch.cuda.synchronize()
        for i in (0, 2, 3):
            assert torch.equal(outs[i], want), (rep, i)
    # a stream whose workspace would have to grow: refused, and the capture goes on
    fresh, said = torch.cuda.Stream(), ""
    g = torch.cuda.CUDAGraph()
    with kv_ref.capture(g, fresh):
        outs[3].fill_(5.0)
        try:
            kv.attention(0, seqs, q, outs[1], 0.09, stream=torch.cuda.current_stream().cuda_stream)
        except tie_amd.TieError as e:
            said = str(e)
    assert "capture" in said
    g.replay()
    torch.cuda.synchronize()
    assert (outs[3] == 5.0).all()
    for s in streams:
        tie_amd.stream_release(s.cuda_stream)
    del g, graphs
    gc.collect()
