"""Attention through a sliding window, with first rows that stay visible, against
a 64-bit form; the bound of each element's error is kv_ref.tolerance()."""
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


def visible(lens, counts, window, sinks, at=None, mask=None):
    """[token] -> the rows it sees, by the header's words."""
    out, t = [], 0
    for n, m in zip(lens, counts):
        for j in range(m):
            stand = n + j if at is None else int(at[t])
            rows = [r for r in range(n) if r < sinks or r > stand - window]
            if mask is None:
                rows += [n + i for i in range(j + 1) if n + i < sinks or n + i > stand - window]
            else:
                rows += [n + i for i in range(m) if i // 64 < mask.shape[1] and int(mask[t, i // 64]) >> (i % 64) & 1]
            out.append(rows)
            t += 1
    return out


def expect(c, q, scale, rows):
    T, H, hd = q.shape
    out, tol, t, group = np.zeros((T, H, hd)), np.zeros((T, H, hd)), 0, H // c.kvh
    for b, (n, m) in enumerate(zip(c.lens, c.counts)):
        if m:
            k, v = c.rows(0, b, 0, n + m)
        for _ in range(m):
            for h in range(H if rows[t] else 0):
                kk, vv = k[rows[t], h // group], v[rows[t], h // group]
                s = kk @ q[t, h].astype(np.float64) * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                out[t, h], tol[t, h] = w @ vv, kv_ref.tolerance(q[t, h].astype(np.float64), kk, vv, w, scale)
            t += 1
    return out, tol


def run(c, q, window, sinks, at=None, mask=None, work=None, scale=0.09):
    import torch
    kv, seqs = c.gpu(), c.seqs()
    cuda = lambda a: torch.from_numpy(a).cuda() if a is not None else None  # noqa: E731
    out = torch.full((len(q) + 1,) + q.shape[1:], -7.0, device="cuda")
    m = None if mask is None else cuda(mask.view(np.int64))
    args = (0, seqs, cuda(np.concatenate([q, q[:1]]) if len(q) else q), out, scale, window)
    if work is not None:
        work = torch.zeros(kv.window_attention_work_bytes(seqs, q.shape[1]), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    kv.window_attention(*args, sinks=sinks, at=cuda(at), mask=m, work=work)
    first = out.clone()
    kv.window_attention(*args, sinks=sinks, at=cuda(at), mask=m, work=work)
    torch.cuda.synchronize()
    assert torch.equal(first.view(torch.int32), out.view(torch.int32))  # two equal calls, equal bits
    got = out.cpu().numpy()
    assert (got[len(q):] == -7.0).all()
    return got[: len(q)]


def check(c, q, window, sinks, at=None, mask=None, work=None):
    got = run(c, q, window, sinks, at, mask, work)
    want, tol = expect(c, q, 0.09, visible(c.lens, c.counts, window, sinks, at, mask))
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])


HEADS = [(8, 2, 128), (10, 2, 64), (3, 3, 64), (20, 1, 128)]
WINDOWS = [(1, 0), (1, 1), (5, 64), (64, 0), (65, 70), (100, 3), (130, 300), (1 << 20, 0), (0x7fffffff, 0x7fffffff)]


def queries(rng, c, H):
    return (2 * rng.standard_normal((sum(c.counts), H, c.hd))).astype(np.float32)


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("H,kvh,hd", HEADS)
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_single_tokens(kind, H, kvh, hd, window, sinks):
    rng = np.random.default_rng(hd + window % 1000)
    lens = [0, 1, 63, 64, 200, 413, 128]
    c = kv_ref.Cache(rng, kind, kvh, hd, lens, [1] * len(lens))
    check(c, queries(rng, c, H), window, sinks)


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("H,kvh,hd", HEADS)
@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_chunks(kind, H, kvh, hd, window, sinks):
    rng = np.random.default_rng(hd + window % 999)
    c = kv_ref.Cache(rng, kind, kvh, hd, [0, 130, 64, 3, 300], [70, 0, 33, 9, 1])
    check(c, queries(rng, c, H), window, sinks, work=True)


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("H,kvh,hd,n,lens", [(16, 2, 128, 300, 129), (10, 2, 64, 517, 0), (32, 4, 64, 1100, 65), (32, 4, 128, 700, 1000)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (64, 64), (100, 5), (500, 200)])
def test_long_chunks(kind, H, kvh, hd, n, lens, window, sinks):
    """The kernels of many rows, by 64 and by 128; a few heads and rows are looked at."""
    rng = np.random.default_rng(n)
    c = kv_ref.Cache(rng, kind, kvh, hd, [lens], [n])
    q = queries(rng, c, H)
    got = run(c, q, window, sinks)
    rows = visible(c.lens, c.counts, window, sinks)
    pick = sorted(set(rng.integers(0, n, 40).tolist() + [0, 1, n - 1, min(n - 1, 63), min(n - 1, 64)]))
    k, v = c.rows(0, 0, 0, lens + n)
    for t in pick:
        for h in {0, H - 1, int(rng.integers(H))}:
            kk, vv = k[rows[t], h // (H // kvh)], v[rows[t], h // (H // kvh)]
            s = kk @ q[t, h].astype(np.float64) * 0.09
            w = np.exp(s - s.max())
            w /= w.sum()
            tol = kv_ref.tolerance(q[t, h].astype(np.float64), kk, vv, w, 0.09)
            assert (np.abs(got[t, h] - w @ vv) <= tol).all(), (t, h)


def tree(rng, counts):
    """Random trees: masks of ancestors, and depths."""
    words = max(1, -(-max(counts) // 64))
    mask, deep = np.zeros((sum(counts), words), np.uint64), []
    t = 0
    for m in counts:
        for j in range(m):
            if j:
                up = int(rng.integers(max(0, j - 4), j))
                mask[t + j] = mask[t + up]
            mask[t + j, j // 64] |= np.uint64(1) << np.uint64(j % 64)
            deep.append(deep[t + up] + 1 if j else 0)
        t += m
    return mask, np.array(deep, np.int32)


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("H,kvh,hd,counts", [(8, 2, 128, [7, 0, 26, 1]), (10, 2, 64, [70, 3]), (64, 4, 128, [26]), (32, 4, 64, [130, 100])])
@pytest.mark.parametrize("window,sinks", [(1, 0), (3, 3), (100, 64), (200, 0), (5000, 0)])
def test_trees(kind, H, kvh, hd, counts, window, sinks):
    rng = np.random.default_rng(window + H)
    lens = [300, 64, 129, 0][: len(counts)]
    c = kv_ref.Cache(rng, kind, kvh, hd, lens, counts)
    mask, deep = tree(rng, counts)
    at = (np.repeat(lens, counts) + deep).astype(np.int32)
    if sum(counts) * H > 2000:  # the reference takes its time: fewer heads are looked at
        got = run(c, queries(rng, c, H), window, sinks, at, mask)
        rng = np.random.default_rng(window + H)
        c = kv_ref.Cache(rng, kind, kvh, hd, lens, counts)
        tree(rng, counts)
        q, group = queries(rng, c, H), H // kvh
        heads = [group * (h + 1) - 1 for h in range(kvh)]
        want, tol = expect(c, q[:, heads], 0.09, visible(lens, counts, window, sinks, at, mask))
        assert (np.abs(got[:, heads] - want) <= tol).all()
    else:
        check(c, queries(rng, c, H), window, sinks, at, mask)


@pytest.mark.parametrize("kind", ["f16", "i8"])
def test_rows_that_see_nothing_and_places_of_their_own(kind):
    """A token that stands past its window sees its mask alone; with no bits: 0.  Places below the committed rows
    show all above; a causal token whose window lies ahead of its own row sees nothing."""
    rng = np.random.default_rng(4)
    counts, lens = [6, 5], [200, 90]
    c = kv_ref.Cache(rng, kind, 2, 128, lens, counts)
    at = np.array([200, 999, 205, 260, 1 << 30, 0x7fffffff, 0, -5, 90, 91, 40], np.int32)
    mask = np.array([1, 0, 4, 0, 16, 0, 1, 2, 0, 9, 16], np.uint64).reshape(-1, 1)
    q = queries(rng, c, 8)
    check(c, q, 50, 0, at, mask)
    got = run(c, q, 50, 0, at, mask)
    assert (got[1] == 0).all() and (got[5] == 0).all()
    check(c, q, 50, 7, at, mask)
    check(c, q, 50, 0, at)
    check(c, q, 50, 70, at)


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("H,n", [(8, 1), (8, 9), (16, 400)])
def test_pages_behind_the_window_and_what_lies_in_unseen_rows(kind, H, n):
    """Entries of pages that no token sees may be none or wrong; rows that none sees may hold anything."""
    rng = np.random.default_rng(n)
    window, sinks, kvh = 150, 5, 2
    lens, counts = [700, 64, 3], [n, 1, 2]
    c = kv_ref.Cache(rng, kind, kvh, 128, lens, counts)
    q = queries(rng, c, H)
    want = run(c, q, window, sinks)
    low = lens[0] - window + 1
    for r in range(sinks, low):
        p, i = c.place(0, r)
        if kind == "f16":
            c.k[0, p, :, i], c.v[0, p, :, :, i] = np.nan, np.inf if r % 2 else np.nan
        else:
            c.ks[0, p, :, i], c.vs[0, p, :, i] = np.inf, np.nan
    for p in range(1, low // 64):
        c.table[0, p] = [-1, 1 << 30, c.n_pages][p % 3]
    got = run(c, q, window, sinks)
    assert np.array_equal(got.view(np.uint32), want.view(np.uint32))


@pytest.mark.parametrize("kind", ["f16", "i8"])
def test_a_page_that_is_none_and_lengths_that_do_not_fit(kind):
    rng = np.random.default_rng(8)
    lens, counts = [700, 300, 100, 100], [1, 1, 1, 1]
    c = kv_ref.Cache(rng, kind, 2, 64, lens, counts)
    q = queries(rng, c, 8)
    want = run(c, q, 150, 5)
    c.table[0, 700 // 64] = -1
    c.table[1, 0] = -1  # the first rows' page
    c.lens[2] = 64 * c.table.shape[1]
    got = run(c, q, 150, 5)
    assert np.isnan(got[:3]).all()
    assert np.array_equal(got[3], want[3])
    c.lens[2] = -3
    got = run(c, q, 150, 5)
    assert np.isnan(got[2]).all() and np.array_equal(got[3], want[3])


@pytest.mark.parametrize("kind,H,kvh,hd", [("f16", 40, 8, 64), ("i8", 32, 4, 128), ("f16", 8, 8, 128)])
@pytest.mark.parametrize("lens,window", [([3000], 2500), ([5000, 2000, 100], 1500), ([400] * 70, 300), ([9000], 9000)])
def test_rows_in_parts_and_many_sequences(kind, H, kvh, hd, lens, window):
    rng = np.random.default_rng(len(lens))
    c = kv_ref.Cache(rng, kind, kvh, hd, lens, [1] * len(lens))
    check(c, queries(rng, c, H), window, 4, work=True)


def test_first_none_strides_and_in_place():
    """One token to a sequence without ranges; q and out are columns of a wider matrix, the same ones."""
    import torch
    rng = np.random.default_rng(3)
    lens = [500, 20, 64]
    c = kv_ref.Cache(rng, "f16", 2, 64, lens, [1] * 3)
    q = queries(rng, c, 6)
    want, tol = expect(c, q, 0.09, visible(lens, [1] * 3, 70, 2))
    kv = c.gpu()
    seqs = tie_amd.KVSeqs(torch.from_numpy(c.table).cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    wide = torch.full((3, 1001), -7.0, device="cuda")
    wide[:, 9: 9 + 384] = torch.from_numpy(q.reshape(3, -1)).cuda()
    kv.window_attention(0, seqs, wide[:, 9: 9 + 384], wide[:, 9: 9 + 384], 0.09, 70, sinks=2)
    got = wide.cpu().numpy()
    assert (np.abs(got[:, 9: 393].reshape(3, 6, 64) - want) <= tol).all()
    assert (got[:, :9] == -7.0).all() and (got[:, 393:] == -7.0).all()


def test_replayed_graph_follows_the_lengths():
    import torch
    rng = np.random.default_rng(5)
    lens, window, sinks = [650, 70, 300], 200, 3
    c = kv_ref.Cache(rng, "i8", 2, 128, [n + 40 for n in lens], [1] * 3)
    kv = c.gpu()
    n_dev = torch.tensor(lens, dtype=torch.int32).cuda()
    seqs = tie_amd.KVSeqs(torch.from_numpy(c.table).cuda(), n_dev)
    q = queries(rng, c, 8)
    qd, out = torch.from_numpy(q).cuda(), torch.zeros(3, 8, 128, device="cuda")
    work = torch.zeros(kv.window_attention_work_bytes(seqs, 8), dtype=torch.uint8, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with kv_ref.capture(graph, side):
        kv.window_attention(0, seqs, qd, out, 0.09, window, sinks=sinks, work=work)
    for step in range(4):
        now = [n + 13 * step for n in lens]
        n_dev.copy_(torch.tensor(now, dtype=torch.int32))
        out.fill_(-7.0)
        graph.replay()
        torch.cuda.synchronize()
        c.lens = now
        want, tol = expect(c, q, 0.09, visible(now, [1] * 3, window, sinks))
        assert (np.abs(out.cpu().numpy() - want) <= tol).all()
        _ = torch.randn(1000, device="cuda").sum().item()


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("H,n", [(8, 5), (16, 500)])
def test_whole_tiles_that_see_nothing(kind, H, n):
    """Every token stands past its window and the mask names none, or (causal) all stand ahead of their rows: zeros."""
    rng = np.random.default_rng(n)
    c = kv_ref.Cache(rng, kind, 2, 128, [400], [n])
    q, at = queries(rng, c, H), np.full(n, 100000, np.int32)
    assert (run(c, q, 70, 0, at, np.zeros((n, 1), np.uint64)) == 0).all()
    assert (run(c, q, 70, 0, at) == 0).all()
    rows = visible(c.lens, c.counts, 70, 3, at)
    got = run(c, q, 70, 3, at)
    k, v = c.rows(0, 0, 0, 3)
    for t in (0, n // 2, n - 1):
        assert rows[t] == [0, 1, 2]
        for h in range(H):
            kk, vv = k[:, h // (H // 2)], v[:, h // (H // 2)]
            s = kk @ q[t, h].astype(np.float64) * 0.09
            w = np.exp(s - s.max())
            w /= w.sum()
            assert (np.abs(got[t, h] - w @ vv) <= kv_ref.tolerance(q[t, h].astype(np.float64), kk, vv, w, 0.09)).all()


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("H,n", [(8, 30), (16, 400)])
def test_ranges_that_are_none(kind, H, n):
    """Ranges that fall, overlap, begin below 0 or end past the rows: rows of no sequence stay as they are, and sequences
    whose ranges lie apart from the others' keep their results."""
    import torch
    rng = np.random.default_rng(n)
    lens, counts = [200, 70, 300, 90], [n, 6, 4, 9]
    c = kv_ref.Cache(rng, kind, 2, 64, lens, counts)
    q, T = queries(rng, c, H), sum(counts)
    want = run(c, q, 100, 4)
    kv = c.gpu()
    qd = torch.from_numpy(q).cuda()
    for first in ([0, n, n + 6, n + 10, T + 1], [0, n, n + 6, n + 10, 0x7fffffff], [0, n, n + 6, n + 4, T], [0, n, -0x80000000, n + 10, T],
                  [5, 0, 3, -2, 7], [T, T, T, T, T], [-5, n, n + 6, n + 10, T]):
        seqs = tie_amd.KVSeqs(torch.from_numpy(c.table).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                              torch.tensor(first, dtype=torch.int32).cuda(), T)
        out = torch.full((T + 3, H, 64), -7.0, device="cuda")
        kv.window_attention(0, seqs, qd, out[:T], 0.09, 100, sinks=4)
        torch.cuda.synchronize()
        got = out.cpu().numpy()
        assert (got[T:] == -7.0).all()
        if first[0] == 0 and first[1] == n:
            tol = 1e-5 * (1 + np.abs(want[:n]).max())
            assert (np.abs(got[:n] - want[:n]) <= tol).all(), first
        if first[4] > T:
            assert (got[n + 10: T] == -7.0).all()


def test_the_streams_own_memory_is_for_calls_it_has_seen():
    """Without work memory a capture is refused where the stream's has to grow, and taken once the call has run there."""
    import torch
    rng = np.random.default_rng(2)
    c = kv_ref.Cache(rng, "f16", 2, 64, [700, 100], [40, 3])
    kv, seqs = c.gpu(), c.seqs()
    q = queries(rng, c, 8)
    qd, out = torch.from_numpy(q).cuda(), torch.zeros(43, 8, 64, device="cuda")
    l, lp = torch.randn(3, 9000, device="cuda"), torch.zeros(3, device="cuda")
    tok = torch.zeros(3, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()

    def calls():
        kv.window_attention(0, seqs, qd, out, 0.09, 100, sinks=4)
        tie_amd.token_logprobs(l, tok, lp)

    torch.cuda.synchronize()
    tie_amd.stream_release(side.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(tie_amd.TieError) as e:
        with kv_ref.capture(graph, side):
            calls()
    assert e.value.code == tie_amd.EINVAL
    with torch.cuda.stream(side):
        calls()
    torch.cuda.synchronize()
    want, want_lp = out.clone(), lp.clone()
    graph = torch.cuda.CUDAGraph()
    with kv_ref.capture(graph, side):
        calls()
    for _ in range(3):
        out.zero_(), lp.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lp, want_lp)


def test_two_streams_at_once():
    """Calls of one size on two streams, each with its stream's memory: the results of calls one behind another."""
    import torch
    rng = np.random.default_rng(7)
    cs = [kv_ref.Cache(rng, "i8", 2, 128, [5000], [1]) for _ in range(2)]
    qs = [queries(rng, c, 8) for c in cs]
    want = [run(c, q, 4500, 4) for c, q in zip(cs, qs)]
    kvs, seqs = [c.gpu() for c in cs], [c.seqs() for c in cs]
    qd, outs = [torch.from_numpy(q).cuda() for q in qs], [torch.zeros(1, 8, 128, device="cuda") for _ in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in (0, 1):
            kvs[i].window_attention(0, seqs[i], qd[i], outs[i], 0.09, 4500, sinks=4, stream=streams[i].cuda_stream)
    torch.cuda.synchronize()
    for i in (0, 1):
        assert np.array_equal(outs[i].cpu().numpy(), want[i])
