"""The paged cache on the GPU: norm, rotation and quantised write, reading
back, and the rows of an accepted path, against 64-bit forms."""
import numpy as np
import pytest

import kv_ref
import tie_amd
from conftest import bits

pytestmark = pytest.mark.gpu
EPS = 1e-6


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


def done(*tensors):
    import torch
    torch.cuda.synchronize()
    return [t.cpu().numpy() for t in tensors]


def same(a, b, what=""):
    """Equal bit patterns, any NaN equal to any other."""
    a, b = np.asarray(a), np.asarray(b)
    assert a.dtype == b.dtype and a.shape == b.shape
    np.testing.assert_array_equal(a, b, what)


# (kind, H, kvh, hd, lens, counts): one token, tokens that cross pages, a
# sequence of none, groups of one, odd ones, more heads than a wave takes
APPEND = [("f16", 8, 2, 128, [0], [1]), ("i8", 32, 4, 128, [1003], [1]), ("i8", 6, 2, 64, [63, 0, 130], [2, 0, 70]),
          ("f16", 5, 5, 64, [10, 64], [130, 1]), ("i8", 32, 4, 128, [5], [300]), ("f16", 64, 4, 128, [61, 1], [7, 3])]


def append_case(case, seed, theta, norms=True, far=0):
    kind, H, kvh, hd, lens, counts = case
    rng = np.random.default_rng(seed)
    c = kv_ref.Cache(rng, kind, kvh, hd, lens, counts, layers=2, fill=False)
    T = sum(counts)
    x = rng.standard_normal((T + 2, (H + 2 * kvh) * hd)).astype(np.float32) * 3
    w = [(1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) if norms else None for _ in range(2)]
    pos = np.concatenate([np.arange(n, n + m) // 2 for n, m in zip(lens, counts)] + [[0] * 0]).astype(np.int32) + far
    return c, x, w, pos


def expect(c, case, x, w, pos, theta):
    kind, H, kvh, hd, lens, counts = case
    T = sum(counts)
    x = x[:T].reshape(T, H + 2 * kvh, hd)
    q = kv_ref.norm_rotate(x[:, :H], w[0], pos, EPS, theta)
    k = kv_ref.norm_rotate(x[:, H: H + kvh], w[1], pos, EPS, theta).astype(np.float32)
    t = 0
    for b, (n, m) in enumerate(zip(lens, counts)):
        c.set_rows(1, b, n, k[t: t + m], x[t: t + m, H + kvh:])
        t += m
    return q


@pytest.mark.parametrize("case", APPEND)
@pytest.mark.parametrize("theta,far,norms", [(1e6, 0, True), (1e4, 1 << 20, True), (1e4, 7, False)])
def test_append(case, theta, far, norms):
    """Queries to one F32 rounding of the 64-bit form (2^-24 relative, and the
    form's own 64-bit rounding of large angles, below 1e-9); the cache's bytes
    equal, and every byte that the call does not own as it was."""
    import torch
    kind, H, kvh, hd, lens, counts = case
    c, x, w, pos = append_case(case, 5, theta, norms, far)
    T = sum(counts)
    kv, seqs = c.gpu(), c.seqs()
    xd = cuda(x)
    q_out = torch.full((T + 2, H, hd), -7.0, device="cuda")
    nd = [cuda(a) if a is not None else None for a in w]
    kv.append(1, seqs, xd[:, : H * hd], xd[:, H * hd: (H + kvh) * hd], xd[:, (H + kvh) * hd:], q_out, cuda(pos),
              q_norm=nd[0], k_norm=nd[1], eps=EPS, theta=theta)
    got, = done(q_out)
    q = expect(c, case, x, w, pos, theta)
    assert (got[T:] == -7.0).all()
    np.testing.assert_allclose(got[:T], q, rtol=2.0 ** -23, atol=1e-8)
    k, v, ks, vs = c.back()
    if far > 1000:
        # an angle of 1e6 has 64-bit forms 1e-9 apart, and a value that near to
        # a border between two codes may fall on either side: half a step each
        for b, (n, m) in enumerate(zip(lens, counts)):
            for j in range(n, n + m):
                p, r = c.place(b, j)
                t = sum(counts[:b]) + j - n
                want = kv_ref.norm_rotate(x[t: t + 1].reshape(1, -1, hd)[:, H: H + kvh], w[1], pos[t: t + 1], EPS, theta)[0]
                if kind == "i8":
                    np.testing.assert_allclose(ks[1, p, :, r], np.abs(want).max(-1) / 127, rtol=2.0 ** -22)
                    held, half = k[1, p, :, r] * ks[1, p, :, r, None].astype(np.float64), ks[1, p, :, r, None] * 0.5
                else:
                    held, half = k[1, p, :, r].astype(np.float64), np.abs(want) * 2.0 ** -11 + 2.0 ** -25
                assert (np.abs(held - want) <= half * (1 + 1e-5) + 1e-7).all()
                c.k[1, p, :, r] = k[1, p, :, r]
                if kind == "i8":
                    c.ks[1, p, :, r] = ks[1, p, :, r]
    # (a 64-bit value within 1e-12 of a border may fall on either side: no
    # such value is among these inputs)
    same(k.view(np.uint8), c.k.view(np.uint8), "k")
    same(v.view(np.uint8), c.v.view(np.uint8), "v")
    if kind == "i8":
        same(ks, c.ks, "k_scale")
        same(vs, c.vs, "v_scale")


def test_append_in_place_and_default_positions():
    import torch
    case = ("i8", 8, 2, 128, [70, 3], [3, 66])
    c, x, w, _ = append_case(case, 9, 1e6)
    pos = np.concatenate([np.arange(n, n + m) for n, m in zip([70, 3], [3, 66])]).astype(np.int32)
    kv, seqs, T = c.gpu(), c.seqs(), 69
    xd = cuda(x)
    q = xd[:, : 8 * 128]
    kv.append(1, seqs, q, xd[:, 8 * 128: 10 * 128], xd[:, 10 * 128:], q, q_norm=cuda(w[0]), k_norm=cuda(w[1]), eps=EPS)
    got, = done(xd)
    want = expect(c, case, x, w, pos, 1e6)
    np.testing.assert_allclose(got[:T, : 8 * 128].reshape(T, 8, 128), want, rtol=2.0 ** -23, atol=1e-8)
    same(got[:, 8 * 128:], x[:, 8 * 128:])
    same(got[T:], x[T:])
    same(c.back()[0], c.k)


@pytest.mark.parametrize("kind", ["f16", "i8"])
def test_append_odd_values(kind):
    """Zeros, values beyond f16, subnormals, and rows with NaN or infinity: an
    int8 row then has scale NaN and codes of 0, and no other row changes."""
    import torch
    H, kvh, hd = 2, 2, 64
    rng = np.random.default_rng(3)
    c = kv_ref.Cache(rng, kind, kvh, hd, [62], [6], fill=False)
    k, v = rng.standard_normal((6, kvh, hd)).astype(np.float32), rng.standard_normal((6, kvh, hd)).astype(np.float32)
    v[0] = 0.0
    v[1, 0, 3], v[1, 1, 5] = 1e6, -3e38
    v[2] *= np.float32(1e-41)
    v[3, 0, 7], v[3, 1, 9] = np.nan, np.inf
    v[4, 0, 1] = -np.inf
    kv, seqs = c.gpu(), c.seqs()
    q = torch.zeros(6, H, hd, device="cuda")
    kv.append(0, seqs, q, cuda(k.reshape(6, -1)), cuda(v.reshape(6, -1)), q, pos=torch.zeros(6, dtype=torch.int32, device="cuda"))
    done(q)
    bad = ~np.isfinite(v).all(-1)  # [6][kvh]
    vv = np.where(bad[..., None], 0.0, v) if kind == "i8" else v
    c.set_rows(0, 0, 62, k, vv)
    if kind == "i8":
        for j, h in zip(*np.nonzero(bad)):
            p, r = c.place(0, 62 + j)
            c.vs[0, p, h, r] = np.nan
    gk, gv, gks, gvs = c.back()
    same(gk, c.k)
    same(gv, c.v)
    if kind == "i8":
        same(gvs, c.vs)
        same(gks, c.ks)


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("H,kvh,hd,lens,counts", [(4, 2, 64, [0], [1]), (4, 4, 128, [129, 0, 7], [37, 0, 60]),
                                                  (3, 3, 64, [0, 63], [200, 2]), (4, 1, 128, [40], [25])])
def test_read(kind, H, kvh, hd, lens, counts):
    import torch
    rng = np.random.default_rng(11)
    c = kv_ref.Cache(rng, kind, kvh, hd, lens, counts, layers=3)
    kv, seqs, T = c.gpu(), c.seqs(), sum(counts)
    for layer, n in ((0, 3), (1, 2), (2, 1)):
        k, v = (torch.full((n, T, kvh, hd), -7.0, device="cuda") for _ in range(2))
        kv.read(seqs, k, v, layer=layer, n_layers=n)
        k, v = done(k, v)
        t = 0
        for b, (a, m) in enumerate(zip(lens, counts)):
            for i in range(n):
                wk, wv = c.rows(layer + i, b, a, a + m)
                same(k[i, t: t + m], wk.astype(np.float32))
                same(v[i, t: t + m], wv.astype(np.float32))
            t += m


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("kvh,hd", [(4, 128), (3, 64)])
@pytest.mark.parametrize("in_place", [False, True])
def test_keep(kind, kvh, hd, in_place):
    """Paths that move nothing, everything, over a page's end, of no nodes, and
    such that end early (not ascending, no node); other rows stay."""
    import torch
    rng = np.random.default_rng(21)
    lens, counts = [0, 60, 127, 5, 9, 64], [4, 26, 30, 3, 40, 12]
    paths = [[0, 1, 2], [0, 3, 9, 25], list(range(1, 30, 2)), [], [0, 5, 5, 7], [2, 11, 12]]
    valid = [3, 4, 15, 0, 2, 2]
    c = kv_ref.Cache(rng, kind, kvh, hd, lens, counts, layers=3)
    kv, seqs = c.gpu(), c.seqs()
    most = 16
    pad = np.full((6, most), -1, np.int32)
    for b, p in enumerate(paths):
        pad[b, : len(p)] = p
    n_keep = np.array([len(p) for p in paths], np.int32)
    n_keep[2] = 99  # more than max_path: the path's own entries end it
    len_out = seqs.keep[1] if in_place else torch.zeros(6, dtype=torch.int32, device="cuda")
    kv.keep(seqs, cuda(pad), cuda(n_keep), len_out)
    got, = done(len_out)
    same(got, (np.array(lens) + valid).astype(np.int32))
    for b, (n, p) in enumerate(zip(lens, paths)):
        for layer in range(3):
            for j in range(valid[b]):
                (fp, fr), (tp, tr) = c.place(b, n + p[j]), c.place(b, n + j)
                c.k[layer, tp, :, tr], c.v[layer, tp, :, :, tr] = c.k[layer, fp, :, fr].copy(), c.v[layer, fp, :, :, fr].copy()
                if kind == "i8":
                    c.ks[layer, tp, :, tr], c.vs[layer, tp, :, tr] = c.ks[layer, fp, :, fr].copy(), c.vs[layer, fp, :, fr].copy()
    for a, w in zip(c.back(), (c.k, c.v, c.ks, c.vs)):
        if w is not None:
            same(a, w)


@pytest.mark.parametrize("kind", ["f16", "i8"])
def test_many_sequences(kind):
    """More than a wave has lanes, some of no tokens."""
    rng = np.random.default_rng(22)
    lens, counts = [int(x) for x in rng.integers(0, 100, 150)], [int(x) for x in rng.integers(0, 4, 150)]
    counts[63:66] = [0, 0, 0]
    test_append((kind, 4, 2, 64, lens, counts), 1e6, 0, True)
    test_read(kind, 4, 2, 64, lens, counts)


@pytest.mark.parametrize("kind", ["f16", "i8"])
def test_keep_long_paths(kind):
    """Paths of more entries than a wave has lanes, one that stops ascending
    behind them."""
    import torch
    rng = np.random.default_rng(23)
    kvh, hd, lens, counts = 1, 64, [30, 64, 0], [300, 200, 140]
    paths = [sorted(rng.choice(300, 150, replace=False).tolist()), list(range(200)), list(range(1, 131)) + [130, 131]]
    valid = [150, 200, 130]
    c = kv_ref.Cache(rng, kind, kvh, hd, lens, counts, layers=2)
    kv, seqs = c.gpu(), c.seqs()
    pad = np.full((3, 203), -1, np.int32)
    for b, p in enumerate(paths):
        pad[b, : len(p)] = p
    len_out = torch.zeros(3, dtype=torch.int32, device="cuda")
    kv.keep(seqs, cuda(pad), cuda(np.array([len(p) for p in paths], np.int32)), len_out)
    got, = done(len_out)
    same(got, (np.array(lens) + valid).astype(np.int32))
    for b, (n, p) in enumerate(zip(lens, paths)):
        for layer in range(2):
            for j in range(valid[b]):
                (fp, fr), (tp, tr) = c.place(b, n + p[j]), c.place(b, n + j)
                c.k[layer, tp, :, tr], c.v[layer, tp, :, :, tr] = c.k[layer, fp, :, fr].copy(), c.v[layer, fp, :, :, fr].copy()
                if kind == "i8":
                    c.ks[layer, tp, :, tr], c.vs[layer, tp, :, tr] = c.ks[layer, fp, :, fr].copy(), c.vs[layer, fp, :, fr].copy()
    for a, w in zip(c.back(), (c.k, c.v, c.ks, c.vs)):
        if w is not None:
            same(a, w)


@pytest.mark.parametrize("kind", ["f16", "i8"])
def test_what_the_device_arrays_may_not_say(kind):
    """Lengths, row ranges and pages outside the call's sizes: nothing is
    written to the cache, reads give NaN, and good sequences are served."""
    import torch
    rng = np.random.default_rng(31)
    kvh, hd, H = 2, 64, 4
    c = kv_ref.Cache(rng, kind, kvh, hd, [10, 10, 10, 10], [2, 2, 2, 2])
    kv = c.gpu()
    table, first = c.table.copy(), np.array([0, 2, 4, 6, 8], np.int32)
    lens = np.array([10, 10, -5, 10], np.int32)
    table[0, 0], table[1, 0] = -3, c.n_pages  # no pages
    seqs = tie_amd.KVSeqs(cuda(table), cuda(lens), cuda(first), 8)
    x = rng.standard_normal((8, (H + 2 * kvh) * hd)).astype(np.float32)
    xd = cuda(x)
    q_out = torch.zeros(8, H, hd, device="cuda")
    kv.append(0, seqs, xd[:, : H * hd], xd[:, H * hd: (H + kvh) * hd], xd[:, (H + kvh) * hd:], q_out)
    k, v = (torch.zeros(1, 8, kvh, hd, device="cuda") for _ in range(2))
    kv.read(seqs, k, v)
    k, v, q = done(k, v, q_out)
    assert np.isnan(k[0, :6]).all() and np.isnan(v[0, :6]).all()
    assert np.isfinite(k[0, 6:]).all() and np.isfinite(v[0, 6:]).all() and np.isfinite(q[6:]).all()
    gk = c.back()[0]
    for b in range(3):
        p = c.table[b, 0]
        same(gk[0, p].view(np.uint8), c.k[0, p].view(np.uint8))
    # a length beyond the table, ranges that fall or pass n_tokens
    for lens, first in (([64, 10, 10, 10], [0, 2, 4, 6, 8]), ([10, 10, 10, 2147483647], [0, 2, 4, 6, 8]),
                        ([10] * 4, [0, 2, 1, 6, 9]), ([10] * 4, [-4, 2, 4, 900, 901])):
        seqs = tie_amd.KVSeqs(cuda(c.table), cuda(np.array(lens, np.int32)), cuda(np.array(first, np.int32)), 8)
        kv.append(0, seqs, xd[:, : H * hd], xd[:, H * hd: (H + kvh) * hd], xd[:, (H + kvh) * hd:], q_out)
        kd, vd = (torch.zeros(1, 8, kvh, hd, device="cuda") for _ in range(2))
        kv.read(seqs, kd, vd)
        kv.keep(seqs, cuda(np.array([[0, 1]] * 4, np.int32)), cuda(np.array([2, 2, -1, 2], np.int32)),
                torch.zeros(4, dtype=torch.int32, device="cuda"))
        done(kd)


def test_nothing_to_do():
    import torch
    c = kv_ref.Cache(np.random.default_rng(1), "f16", 2, 64, [3], [1])
    kv = c.gpu()
    e = torch.zeros(0, dtype=torch.int32, device="cuda")
    seqs = tie_amd.KVSeqs(torch.zeros(0, 1, dtype=torch.int32, device="cuda"), e, None, 0)
    z = torch.zeros(0, 4, 64, device="cuda")
    k = torch.zeros(1, 0, 2, 64, device="cuda")
    kv.append(0, seqs, z, z[:, :2], z[:, :2], z)
    kv.read(seqs, k, k.clone())
    kv.keep(seqs, torch.zeros(0, 1, dtype=torch.int32, device="cuda"), e, e)
    kv.attention(0, seqs, z, z, 1.0)
    done(z)


@pytest.mark.parametrize("kind", ["f16", "i8"])
def test_offsets_past_32_bits(kind):
    """Pages whose bytes lie beyond 4 GiB from the layer's start."""
    import torch
    kvh, hd, H = 8, 128, 8
    per = kvh * 64 * hd * (2 if kind == "f16" else 1)
    pages = (5 << 30) // per
    dt = torch.float16 if kind == "f16" else torch.int8
    k = torch.empty(1, pages, kvh, 64, hd, dtype=dt, device="cuda")
    v = torch.empty(1, pages, kvh, hd, 64, dtype=dt, device="cuda")
    sc = [torch.empty(1, pages, kvh, 64, device="cuda") for _ in range(2)] if kind == "i8" else [None, None]
    kv = kv_ref.after_torch(k, v, *sc)
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device="cuda")
    lens, first = torch.zeros(1, dtype=torch.int32, device="cuda"), torch.tensor([0, 150], dtype=torch.int32, device="cuda")
    seqs = tie_amd.KVSeqs(table, lens, first, 150)
    rng = np.random.default_rng(41)
    x = rng.standard_normal((150, 3 * 8 * hd)).astype(np.float32)
    xd = cuda(x)
    q = torch.empty(150, H, hd, device="cuda")
    kv.append(0, seqs, xd[:, : 8 * hd], xd[:, 8 * hd: 16 * hd], xd[:, 16 * hd:], q, pos=torch.zeros(150, dtype=torch.int32, device="cuda"))
    ko, vo = (torch.empty(1, 150, kvh, hd, device="cuda") for _ in range(2))
    kv.read(seqs, ko, vo)
    out = torch.empty_like(q)
    kv.attention(0, seqs, q, out, hd ** -0.5)  # (the library's stream, behind the append)
    ko, vo, o, qq = done(ko, vo, out, q)
    c = kv_ref.Cache(rng, kind, kvh, hd, [0], [150], fill=False, order=range(5))
    c.set_rows(0, 0, 0, x[:, 8 * hd: 16 * hd].reshape(150, 8, hd), x[:, 16 * hd:].reshape(150, 8, hd))
    wk, wv = c.rows(0, 0, 0, 150)
    same(ko[0], wk.astype(np.float32))
    same(vo[0], wv.astype(np.float32))
    want, tol = kv_ref.attention(c, 0, qq, hd ** -0.5, lambda b, i, j: j <= i)
    assert (np.abs(o - want) <= tol).all()
