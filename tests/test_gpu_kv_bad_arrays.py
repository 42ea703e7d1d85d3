"""What the device arrays say wrong (lengths, ranges of rows, pages, paths): the
cache's every byte, and each row of the outputs."""
import numpy as np
import pytest

import kv_ref
import tie_amd
from test_gpu_kv import EPS, cuda, device, done, same  # noqa: F401 (device: the module's fixture)

pytestmark = pytest.mark.gpu

H, KVH, HD = 4, 2, 64
KINDS = pytest.mark.parametrize("kind", ["f16", "i8"])


class Call:
    """Four sequences of two tokens behind ten rows each, and the call's buffers."""

    def __init__(self, kind, seed, lens=(10, 10, 10, 10), counts=(2, 2, 2, 2), rows=8):
        self.rng = np.random.default_rng(seed)
        self.c = kv_ref.Cache(self.rng, kind, KVH, HD, lens, counts, layers=2)
        self.kind, self.rows, self.table, self.lens = kind, rows, self.c.table.copy(), np.array(lens, np.int32)
        self.first = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.x = self.rng.standard_normal((rows, (H + 2 * KVH) * HD)).astype(np.float32)
        self.kv = self.c.gpu()

    def seqs(self):
        return tie_amd.KVSeqs(cuda(self.table), cuda(self.lens), cuda(self.first), self.rows)

    def append(self, pos=None):
        """The queries; layer 1."""
        import torch
        xd = cuda(self.x)
        out = torch.full((self.rows, H, HD), -7.0, device="cuda")
        self.kv.append(1, self.seqs(), xd[:, :H * HD], xd[:, H * HD:(H + KVH) * HD], xd[:, (H + KVH) * HD:], out,
                       None if pos is None else cuda(pos))
        return done(out)[0]

    def read(self):
        import torch
        k, v = (torch.full((2, self.rows, KVH, HD), -7.0, device="cuda") for _ in range(2))
        self.kv.read(self.seqs(), k, v, n_layers=2)
        return done(k, v)

    def written(self, b, t0, t1, first_row, pos):
        """Rows t0 .. t1 - 1 go to sequence b's cache rows from `first_row` on."""
        k = kv_ref.norm_rotate(self.x[t0:t1].reshape(t1 - t0, -1, HD)[:, H:H + KVH], None, pos, EPS, 1e6).astype(np.float32)
        self.c.set_rows(1, b, first_row, k, self.x[t0:t1, (H + KVH) * HD:].reshape(t1 - t0, KVH, HD))

    def query(self, t0, t1, pos):
        return kv_ref.norm_rotate(self.x[t0:t1, :H * HD].reshape(t1 - t0, H, HD), None, pos, EPS, 1e6)

    def check_cache(self, what=""):
        for name, got, want in zip(("k", "v", "k_scale", "v_scale"), self.c.back(), (self.c.k, self.c.v, self.c.ks, self.c.vs)):
            if want is not None:
                same(got.view(np.uint8) if got.dtype != np.float32 else got, want.view(np.uint8) if got.dtype != np.float32 else want,
                     (name, what))


def near(got, want):
    np.testing.assert_allclose(got, want, rtol=2.0 ** -23, atol=1e-8)


@KINDS
@pytest.mark.parametrize("bad", [-5, -2 ** 31, 63, 64, 2 ** 31 - 1])
def test_append_of_a_length_that_is_none(kind, bad):
    """Without positions the queries' rotation goes by the length: NaN, for that
    sequence.  With positions they are what they are.  Nothing is written for
    it either way, and the other sequences are served."""
    for pos in (None, np.array([3, 9, 4, 4, 1000, 0, 77, 8], np.int32)):
        m = Call(kind, 5)
        m.lens[1] = bad
        q = m.append(pos)
        for b in range(4):
            t = slice(2 * b, 2 * b + 2)
            if b == 1:
                if pos is None:
                    assert np.isnan(q[t]).all()
                else:
                    near(q[t], m.query(2, 4, pos[t]))
                continue
            at = np.array([10, 11]) if pos is None else pos[t]
            near(q[t], m.query(2 * b, 2 * b + 2, at))
            m.written(b, 2 * b, 2 * b + 2, 10, at)
        m.check_cache((bad, pos is None))


@KINDS
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("long", [False, True])
def test_keep_over_pages_that_are_none(kind, in_place, long):
    """A path ends at the first entry whose row has no page, or goes to a row
    that has none: the length counts the rows before it, which are moved, and
    nothing else is.  (long: entries past the first 64 as well)"""
    import torch
    m = Call(kind, 7, lens=(60, 60, 60, 60, 5), counts=(200, 200, 200, 200, 200), rows=1000)
    c = m.c
    # sequence 0: rows of page 2 (nodes 68 .. 131) have none; 1: page 0 (the first 4 targets); 2: page 1; 3: a page past the last; 4: all good
    m.table[0, 2], m.table[1, 0], m.table[2, 1], m.table[3, 3] = -1, -7, c.n_pages, 2 ** 31 - 1
    step = 1 if long else 9
    path = list(range(1, 200, step))
    pad = np.full((5, 220), -1, np.int32)
    pad[:, :len(path)] = path
    want = []
    for b in range(5):
        def there(node):
            return 0 <= m.table[b, (m.lens[b] + node) // 64] < c.n_pages
        kept = next((j for j, p in enumerate(path) if not (there(p) and there(j))), len(path))
        want.append(m.lens[b] + kept)
        for j in range(kept):
            (fp, fr), (tp, tr) = c.place(b, m.lens[b] + path[j]), c.place(b, m.lens[b] + j)
            c.k[:, tp, :, tr], c.v[:, tp, :, :, tr] = c.k[:, fp, :, fr].copy(), c.v[:, fp, :, :, fr].copy()
            if kind == "i8":
                c.ks[:, tp, :, tr], c.vs[:, tp, :, tr] = c.ks[:, fp, :, fr].copy(), c.vs[:, fp, :, fr].copy()
    assert len(set(want)) == 5 and want[1] == 60 and want[4] == 5 + len(path)
    seqs = m.seqs()
    lens = seqs.keep[1] if in_place else torch.full((5,), -7, dtype=torch.int32, device="cuda")
    m.kv.keep(seqs, cuda(pad), cuda(np.full(5, len(path), np.int32)), lens)
    same(done(lens)[0], np.array(want, np.int32))
    m.check_cache()


RANGES = pytest.mark.parametrize("first", [[0, 2, 1, 6, 8], [0, 2, 1, 6, 9], [-4, 2, 4, 900, 901], [0, 2, 4, 4, 4], [5, 2, 2, 8, 3],
                                           [8, 8, 9, 2, 4], [2 ** 31 - 1, -2 ** 31, 0, 3, 8]])


def good_rows(m):
    """For each token row the (sequence, token) that a good range makes of it."""
    rows = [[] for _ in range(m.rows)]
    for b in range(4):
        t0, t1 = int(m.first[b]), int(m.first[b + 1])
        if 0 <= t0 <= t1 <= m.rows:
            for t in range(t0, t1):
                rows[t].append((b, t - t0))
    return rows


@KINDS
@RANGES
def test_append_of_ranges_that_do_not_ascend(kind, first):
    """A row goes to the last sequence that begins at or before it, if that one's
    range is good and holds it; the others' queries stay, and so does every
    byte of the cache that is no such row."""
    m = Call(kind, 9)
    m.first = np.array(first, np.int32)
    q = m.append()
    for t in range(m.rows):
        begun = [b for b in range(4) if first[b] <= t]
        b = begun[-1] if begun else -1
        if b < 0 or not (0 <= first[b] <= t < first[b + 1] <= m.rows):
            assert (q[t] == -7.0).all(), t
            continue
        j = t - first[b]
        near(q[t:t + 1], m.query(t, t + 1, np.array([10 + j])))
        m.written(b, t, t + 1, 10 + j, np.array([10 + j]))
    m.check_cache(first)


@KINDS
@RANGES
def test_read_of_ranges_that_do_not_ascend(kind, first):
    """Rows of a good range are read (of either sequence where two have it), the others stay."""
    m = Call(kind, 10, counts=(8, 8, 8, 8))
    m.first = np.array(first, np.int32)
    k, v = m.read()
    for t, of in enumerate(good_rows(m)):
        for layer in range(2):
            want = [[x[0].astype(np.float32) for x in m.c.rows(layer, b, 10 + j, 11 + j)] for b, j in of] or [[np.full((KVH, HD), -7.0)] * 2]
            assert any((k[layer, t] == w[0]).all() for w in want) and any((v[layer, t] == w[1]).all() for w in want), (t, of)
    m.check_cache(first)


@KINDS
@RANGES
def test_attention_of_ranges_that_do_not_ascend(kind, first):
    import torch
    m = Call(kind, 11, counts=(8, 8, 8, 8))
    m.first = np.array(first, np.int32)
    q = m.rng.standard_normal((m.rows, H, HD)).astype(np.float32)
    out = torch.full((m.rows, H, HD), -7.0, device="cuda")
    m.kv.attention(1, m.seqs(), cuda(q), out, 0.125)
    o, = done(out)
    for t, of in enumerate(good_rows(m)):
        if not of:
            assert (o[t] == -7.0).all(), t
            continue
        held = np.zeros((len(of), H), bool)
        for i, (b, j) in enumerate(of):
            k, v = m.c.rows(1, b, 0, 11 + j)
            for h in range(H):
                qq, kk, vv = q[t, h].astype(np.float64), k[:, h // (H // KVH)], v[:, h // (H // KVH)]
                w = np.exp(kk @ qq * 0.125 - (kk @ qq * 0.125).max())
                w /= w.sum()
                held[i, h] = (np.abs(o[t, h] - w @ vv) <= kv_ref.tolerance(qq, kk, vv, w, 0.125)).all()
        assert held.any(0).all(), (t, of)


@KINDS
@RANGES
def test_keep_of_ranges_that_do_not_ascend(kind, first):
    """A path of nodes 1, 3, 7: those that are nodes of a good range."""
    import torch
    m = Call(kind, 12, counts=(8, 8, 8, 8))
    m.first = np.array(first, np.int32)
    c, want = m.c, []
    for b in range(4):
        n = first[b + 1] - first[b] if 0 <= first[b] <= first[b + 1] <= m.rows else 0
        kept = [p for p in (1, 3, 7) if p < n]
        want.append(10 + len(kept))
        for j, p in enumerate(kept):
            (fp, fr), (tp, tr) = c.place(b, 10 + p), c.place(b, 10 + j)
            c.k[:, tp, :, tr], c.v[:, tp, :, :, tr] = c.k[:, fp, :, fr].copy(), c.v[:, fp, :, :, fr].copy()
            if kind == "i8":
                c.ks[:, tp, :, tr], c.vs[:, tp, :, tr] = c.ks[:, fp, :, fr].copy(), c.vs[:, fp, :, fr].copy()
    lens = torch.full((4,), -7, dtype=torch.int32, device="cuda")
    m.kv.keep(m.seqs(), cuda(np.array([[1, 3, 7]] * 4, np.int32)), cuda(np.array([3, 3, 3, 3], np.int32)), lens)
    same(done(lens)[0], np.array(want, np.int32))
    m.check_cache(first)


@KINDS
def test_pages_that_are_none(kind):
    """Below 0, past the last: nothing is written there, reads give NaN, the
    attention of that sequence too; queries need no page; the others are served."""
    import torch
    m = Call(kind, 13)
    m.table[0, 0], m.table[2, 0] = -3, m.c.n_pages
    q = m.append()
    near(q, m.query(0, 8, np.array([10, 11] * 4)))
    for b in (1, 3):
        m.written(b, 2 * b, 2 * b + 2, 10, np.array([10, 11]))
    m.check_cache("append")
    k, v = m.read()
    for b in range(4):
        t = slice(2 * b, 2 * b + 2)
        if b in (0, 2):
            assert np.isnan(k[:, t]).all() and np.isnan(v[:, t]).all()
            continue
        for layer in range(2):
            wk, wv = m.c.rows(layer, b, 10, 12)
            same(k[layer, t], wk.astype(np.float32))
            same(v[layer, t], wv.astype(np.float32))
    out = torch.full((8, H, HD), -7.0, device="cuda")
    m.kv.attention(1, m.seqs(), cuda(q), out, 0.125)
    o, = done(out)
    want, tol = kv_ref.attention(m.c, 1, q, 0.125, lambda b, i, j: j <= i)
    for b in range(4):
        t = slice(2 * b, 2 * b + 2)
        assert np.isnan(o[t]).all() if b in (0, 2) else (np.abs(o[t] - want[t]) <= tol[t]).all(), b


@KINDS
@pytest.mark.parametrize("bad", [-1, -2 ** 31, 63, 2 ** 31 - 1])
def test_lengths_that_are_none(kind, bad):
    """Reads and attention give NaN, keep moves nothing and leaves the length."""
    import torch
    m = Call(kind, 14)
    m.lens[2] = bad
    k, v = m.read()
    out, q = torch.full((8, H, HD), -7.0, device="cuda"), m.rng.standard_normal((8, H, HD)).astype(np.float32)
    m.kv.attention(1, m.seqs(), cuda(q), out, 0.125)
    o, = done(out)
    want, tol = kv_ref.attention(m.c, 1, q, 0.125, lambda b, i, j: j <= i)
    for b in range(4):
        t = slice(2 * b, 2 * b + 2)
        if b == 2:
            assert np.isnan(k[:, t]).all() and np.isnan(v[:, t]).all() and np.isnan(o[t]).all()
            continue
        for layer in range(2):
            wk, wv = m.c.rows(layer, b, 10, 12)
            same(k[layer, t], wk.astype(np.float32))
            same(v[layer, t], wv.astype(np.float32))
        assert (np.abs(o[t] - want[t]) <= tol[t]).all()
    lens = torch.full((4,), -7, dtype=torch.int32, device="cuda")
    m.kv.keep(m.seqs(), cuda(np.array([[0, 1]] * 4, np.int32)), cuda(np.array([2, 1, 2, -3], np.int32)), lens)
    same(done(lens)[0], np.array([12, 11, bad, 10], np.int32))
    m.check_cache(bad)
