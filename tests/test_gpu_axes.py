"""Append with positions on several axes against a 64-bit form; the cache's bytes equal."""
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


def rotate(x, w, pos, axes, eps, theta):
    """x [T][heads][hd]: pair i turned by its own axis' position."""
    x = np.asarray(x, np.float64)
    T, _, hd = x.shape
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    out = np.empty_like(x)
    for i in range(hd // 2):
        ang = pos[axes[i]].astype(np.float64) * float(theta) ** (-2.0 * i / hd)
        c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
        a, b = x[:, :, i], x[:, :, i + hd // 2]
        out[:, :, i], out[:, :, i + hd // 2] = a * c - b * s, b * c + a * s
    return out


@pytest.mark.parametrize("kind,H,kvh,hd", [("i8", 8, 2, 128), ("f16", 10, 2, 64), ("i8", 5, 5, 64), ("f16", 4, 1, 128)])
@pytest.mark.parametrize("lens,counts", [([63], [1]), ([70, 3, 0], [3, 0, 66]), ([5], [700]), ([77, 0], [1300, 1250])])
@pytest.mark.parametrize("n_axes,norms", [(1, True), (3, True), (4, False)])
def test_append_axes(kind, H, kvh, hd, lens, counts, n_axes, norms):
    """Queries to one F32 rounding of the 64-bit form (2^-24 relative, and 1e-9 for angles up to 2000); keys and values
    to the byte (no value among these lies within 1e-12 of a border between two codes); nothing else written."""
    import torch
    rng = np.random.default_rng(hd + n_axes)
    c = kv_ref.Cache(rng, kind, kvh, hd, lens, counts, layers=2, fill=False)
    T, theta, eps = sum(counts), 1e4, 1e-6
    x = rng.standard_normal((T, (H + 2 * kvh) * hd)).astype(np.float32)
    w = [(1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) if norms else None for _ in range(2)]
    pos, axes = rng.integers(0, 2000, (n_axes, T)).astype(np.int32), rng.integers(0, n_axes, hd // 2).tolist()
    kv, seqs = c.gpu(), c.seqs()
    cuda = lambda a: torch.from_numpy(a).cuda() if a is not None else None  # noqa: E731
    xd, q_out = cuda(x), torch.full((T + 1, H, hd), -7.0, device="cuda")
    kv.append_axes(1, seqs, xd[:, : H * hd], xd[:, H * hd: (H + kvh) * hd], xd[:, (H + kvh) * hd:], q_out, cuda(pos), axes,
                   q_norm=cuda(w[0]), k_norm=cuda(w[1]), eps=eps, theta=theta)
    torch.cuda.synchronize()
    x = x.reshape(T, H + 2 * kvh, hd)
    got = q_out.cpu().numpy()
    assert (got[T:] == -7.0).all()
    np.testing.assert_allclose(got[:T], rotate(x[:, :H], w[0], pos, axes, eps, theta), rtol=2.0 ** -23, atol=1e-8)
    k = rotate(x[:, H: H + kvh], w[1], pos, axes, eps, theta).astype(np.float32)
    t = 0
    for b, (n, m) in enumerate(zip(lens, counts)):
        c.set_rows(1, b, n, k[t: t + m], x[t: t + m, H + kvh:])
        t += m
    for mine, theirs in zip(c.back(), (c.k, c.v, c.ks, c.vs)):
        if theirs is not None:
            assert np.array_equal(mine.view(np.uint8), theirs.view(np.uint8))


def test_one_position_on_all_axes_is_append():
    """Bit for bit, whatever axis a pair names."""
    import torch
    rng = np.random.default_rng(1)
    lens, counts, H, kvh, hd, T = [100, 7], [5, 60], 8, 2, 128, 65
    x = torch.from_numpy(rng.standard_normal((T, (H + 2 * kvh) * hd)).astype(np.float32)).cuda()
    pos = torch.from_numpy(rng.integers(0, 1 << 20, T).astype(np.int32)).cuda()
    q, k, v = x[:, : H * hd], x[:, H * hd: (H + kvh) * hd], x[:, (H + kvh) * hd:]
    got = []
    for how in (0, 1):
        c = kv_ref.Cache(np.random.default_rng(2), "i8", kvh, hd, lens, counts, fill=False)
        kv, seqs, out = c.gpu(), c.seqs(), torch.zeros(T, H, hd, device="cuda")
        if how:
            kv.append_axes(0, seqs, q, k, v, out, pos.repeat(3, 1), [0, 1, 2, 1] * 16)
        else:
            kv.append(0, seqs, q, k, v, out, pos)
        torch.cuda.synchronize()
        got.append([out.cpu().numpy()] + c.back())
    for a, b in zip(*got):
        assert np.array_equal(a.view(np.uint8), b.view(np.uint8))


@pytest.mark.parametrize("kind,H,kvh,hd", [("i8", 4, 2, 128), ("f16", 4, 2, 64), ("i8", 3, 3, 64), ("f16", 2, 1, 128)])
@pytest.mark.parametrize("n_seqs,most", [(3, 500), (40, 60), (150, 11), (700, 3), (33, 150)])
@pytest.mark.parametrize("plain", [False, True])
def test_many_tokens_of_many_sequences(kind, H, kvh, hd, n_seqs, most, plain):
    """Rows that begin anywhere in a page, sequences without tokens, rows of no sequence, a page that is none, lengths that do
    not fit, values that are not finite: the cache to the byte, and the queries of all sequences whose rows fit."""
    import torch
    rng = np.random.default_rng(n_seqs + hd)
    lens, counts = rng.integers(0, 200, n_seqs).tolist(), rng.integers(0, most + 1, n_seqs).tolist()
    counts[-1] += max(0, (2600 if n_seqs == 33 else 600) - sum(counts))  # (heads of 64 have a kernel from 2500 on)
    c = kv_ref.Cache(rng, kind, kvh, hd, lens, counts, fill=False)
    T, pad = sum(counts), 21
    x = rng.standard_normal((T + pad, (H + 2 * kvh) * hd)).astype(np.float32)
    x[rng.integers(0, T, 5), -3] = [np.inf, np.nan, -np.inf, 1e6, -7e4]
    pos = rng.integers(0, 3000, (2, T + pad)).astype(np.int32)
    axes = rng.integers(0, 2, hd // 2).tolist()
    first = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    b_len, b_page = (int(np.argsort(counts)[-1 - i]) for i in (1, 2))
    lens[b_len] = 64 * c.table.shape[1] if n_seqs % 2 else -1
    gone = -(-(lens[b_page] + counts[b_page]) // 64) - 1
    c.table[b_page, gone] = -5
    kv = c.gpu()
    seqs = tie_amd.KVSeqs(torch.from_numpy(c.table).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), torch.from_numpy(first).cuda(),
                          T + pad)
    xd, pd = torch.from_numpy(x).cuda(), torch.from_numpy(pos).cuda()
    q_out = torch.full((T + pad, H, hd), -7.0, device="cuda")
    parts = (xd[:, : H * hd], xd[:, H * hd: (H + kvh) * hd], xd[:, (H + kvh) * hd:], q_out)
    if plain:  # (and rows that are not 16-byte aligned)
        shifted = torch.zeros(T + pad, x.shape[1] + 3, device="cuda")
        shifted[:, 1: 1 + x.shape[1]] = xd
        xd = shifted[:, 1: 1 + x.shape[1]]
        parts = (xd[:, : H * hd], xd[:, H * hd: (H + kvh) * hd], xd[:, (H + kvh) * hd:], q_out)
        kv.append(0, seqs, *parts, pd[0].contiguous())
        pos, axes = pos[:1], [0] * (hd // 2)
    else:
        kv.append_axes(0, seqs, *parts, pd, axes)
    torch.cuda.synchronize()
    x = x.reshape(T + pad, H + 2 * kvh, hd)
    got = q_out.cpu().numpy()
    assert (got[T:] == -7.0).all()
    np.testing.assert_allclose(got[:T], rotate(x[:T, :H], None, pos[:, :T], axes, 1e-6, 1e6), rtol=2.0 ** -23, atol=1e-8)
    k, v = rotate(x[:T, H: H + kvh], None, pos[:, :T], axes, 1e-6, 1e6).astype(np.float32), x[:T, H + kvh:]
    for b, (n, m) in enumerate(zip(lens, counts)):
        if b == b_len:
            continue
        t = first[b]
        m = min(m, gone * 64 - n) if b == b_page else m
        if m <= 0:
            continue
        for j in range(m):
            p, r = c.place(b, n + j)
            if kind == "f16":
                c.k[0, p, :, r] = kv_ref.held_f16(k[t + j])
                c.v[0, p, :, :, r] = np.where(np.isnan(v[t + j]), np.float16(np.nan), kv_ref.held_f16(v[t + j]))
            else:
                bad = ~np.isfinite(v[t + j]).all(-1)
                kc, ks = kv_ref.codes(k[t + j])
                vc, vs = kv_ref.codes(np.where(bad[:, None], np.float32(0), v[t + j]))
                c.k[0, p, :, r], c.ks[0, p, :, r], c.v[0, p, :, :, r], c.vs[0, p, :, r] = kc, ks, vc, np.where(bad, np.nan, vs)
    for mine, theirs in zip(c.back(), (c.k, c.v, c.ks, c.vs)):
        if theirs is not None:
            assert np.array_equal(mine, theirs, equal_nan=mine.dtype != np.int8)
