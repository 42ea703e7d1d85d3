"""The scratch memory of the attention and verification calls: what is enough
for a call is enough for every smaller one."""
import ctypes
import os

import numpy as np
import pytest

import tie_amd

needs_lib = pytest.mark.skipif(not os.path.exists(tie_amd.LIB_PATH), reason="libtie_hip.so not built")


def need(kind, H, kvh, hd, tokens, seqs, pages):
    c = tie_amd.KVCacheDesc(type=kind, n_layers=1, n_pages=4, kv_heads=kvh, head_dim=hd, k=256, v=256, k_scale=256, v_scale=256)
    s = tie_amd.KVSeqsDesc(n_seqs=seqs, max_pages=pages, n_tokens=tokens, pages=256, len=256, first=256)
    got = tie_amd.lib().tie_hip_tree_attention_work_bytes(ctypes.byref(c), ctypes.byref(s), H)
    assert got > 0
    return got


def call_needs(kind, H, kvh, hd, tokens, seqs, pages):
    """What one call writes, by the rules that cut it: which kernel, tiles of 16,
    64 or 128 query rows, none cut where they fill the card, else so many units
    of a tile's rows; an F32 row for each, of hd + 4."""
    rows, i8 = tokens * (H // kvh), kind == tie_amd.I8
    most, units = (256, 448) if i8 else (128 if pages * 64 <= 10240 else 64, 64)
    few = rows <= 16 * seqs or (rows <= most * seqs and rows * kvh <= units * 16)
    tile = 16 if few else 64 if rows * kvh < 256 * 128 else 128
    n = ((256 if few else 512) + kvh) + (rows + min(seqs, tokens) * (tile - 1)) // tile * kvh
    cut = rows // tile * kvh < 256 and not (few and n > 8192)
    return 8192 * 4 + (n * tile * (hd + 4) * 4 if cut else 0)


HEADS = [(32, 4, 128), (64, 4, 128), (32, 8, 64), (8, 8, 64), (5, 5, 128), (1, 1, 64), (96, 1, 128), (1024, 1024, 64)]


@needs_lib
@pytest.mark.parametrize("kind", [tie_amd.F16, tie_amd.I8])
@pytest.mark.parametrize("H,kvh,hd", HEADS)
def test_attention_memory_for_a_call_is_memory_for_every_smaller_one(kind, H, kvh, hd):
    rng = np.random.default_rng(H + kvh + kind)

    def some(most):
        return int(np.exp(rng.random() * np.log(most + 0.99)))

    grid = [(t, s, p) for t in (1, 2, 5, 26, 64, 128, 511, 2048, 5000) for s in (1, 4, 16, 128) if s <= t for p in (1, 160, 161, 5000)]
    grid += [(t, min(some(t), 65535), some(20000)) for t in (some(8192) for _ in range(400))]
    got = {g: need(kind, H, kvh, hd, *g) for g in grid}
    for g in grid:
        assert got[g] >= call_needs(kind, H, kvh, hd, *g), g
    for _ in range(20000):
        a, b = (grid[i] for i in rng.integers(0, len(grid), 2))
        if all(x <= y for x, y in zip(a, b)):
            assert got[a] <= got[b], (a, b)
    for g in grid[:60]:  # against its parts: sequences and columns fewer, tokens fewer
        for h in ((max(1, g[0] // 2), min(g[1], max(1, g[0] // 2)), g[2]), (g[0], 1, g[2]), (g[0], g[1], 1), (1, 1, 1)):
            assert need(kind, H, kvh, hd, *h) <= got[g], (h, g)


@needs_lib
def test_verification_memory_grows_with_each_size():
    sizes = [(v, n, k, d) for v in (1, 4096, 4097, 151936) for n in (1, 5, 200) for k in (1, 16) for d in (False, True)]
    got = {s: tie_amd.verify_tree_work_bytes(*s) for s in sizes}
    for a in sizes:
        for b in sizes:
            if all(x <= y for x, y in zip(a, b)):
                assert got[a] <= got[b], (a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "i8"])
def test_small_calls_behind_a_large_one(kind):
    """A stream that has run a prompt's chunk captures the calls of trees and
    tokens behind it, and takes them with the memory asked for the chunk."""
    import gc

    import torch

    import kv_ref
    assert torch.cuda.is_available(), "GPU test without a GPU"
    tie_amd.init(0)
    rng = np.random.default_rng(3)
    H, kvh, hd, length, chunk = 32, 4, 128, 300, 2048
    c = kv_ref.Cache(rng, kind, kvh, hd, [length], [40])
    kv = c.gpu()
    lens, pages = torch.tensor([length], dtype=torch.int32, device="cuda"), torch.from_numpy(c.table).cuda()

    def seqs(n):
        return tie_amd.KVSeqs(pages, lens, torch.tensor([0, n], dtype=torch.int32, device="cuda"), n)

    # (the chunk's own rows would lie past this table: NaN, but the memory is its size's)
    big, q = seqs(chunk), torch.randn(chunk, H, hd, device="cuda")
    out = torch.zeros_like(q)
    work = torch.zeros(kv.attention_work_bytes(big, H), dtype=torch.uint8, device="cuda")
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    kv.attention(0, big, q, out, 0.1, stream=stream.cuda_stream)
    torch.cuda.synchronize()
    assert bool(torch.isnan(out).all())
    for n in (40, 26, 7, 1):
        small, o = seqs(n), [torch.zeros(n, H, hd, device="cuda") for _ in range(2)]
        assert kv.attention_work_bytes(small, H) <= work.numel()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with kv_ref.capture(g, stream):
            kv.attention(0, small, q[:n], o[0], 0.1)
        kv.attention(0, small, q[:n], o[1], 0.1, work=work)
        c.counts = [n]
        want, tol = kv_ref.attention(c, 0, q[:n].cpu().numpy(), 0.1, lambda b, i, j: j <= i)
        for _ in range(3):
            o[0].zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o[0], o[1])
        assert (np.abs(o[0].cpu().numpy() - want) <= tol).all()
        del g
        gc.collect()
    tie_amd.stream_release(stream.cuda_stream)
    tie_amd.shutdown()


@needs_lib
def test_pages_whose_rows_pass_32_bits_are_refused():
    """(keep forms page * 64 + row in 32 bits: the last page of 2^25 is the last that fits)"""
    assert (2 ** 25 - 1) * 64 + 63 == 2 ** 31 - 1
    mem = np.zeros(1 << 17, np.uint8)
    a = (mem.ctypes.data + 255) & ~255
    s = tie_amd.KVSeqsDesc(n_seqs=2, max_pages=3, n_tokens=5, pages=a, len=a, first=a)
    L, r = tie_amd.lib(), ctypes.byref
    for kind in (tie_amd.F16, tie_amd.I8):
        for n, want in ((2 ** 25, tie_amd.ENOINIT), (2 ** 25 + 1, tie_amd.EINVAL), (2 ** 31 - 1, tie_amd.EINVAL)):
            c = tie_amd.KVCacheDesc(type=kind, n_layers=1, n_pages=n, kv_heads=1, head_dim=64, k=a, v=a, k_scale=a, v_scale=a)
            assert L.tie_hip_kv_keep(r(c), r(s), a, 4, a + 4096, None, None) == want
            assert L.tie_hip_kv_read(r(c), 0, 1, r(s), a, a + 32768, None) == want
            assert L.tie_hip_tree_attention(r(c), 0, r(s), a, 256, 4, 0.1, None, 0, a + 32768, 256, None, 0, None) == want
            assert L.tie_hip_kv_append(r(c), 0, r(s), a, 256, a + 8192, 64, a + 16384, 64, 4, a, a, 1e-6, 1e6, None, a + 32768, 256,
                                       None) == want
            assert (L.tie_hip_tree_attention_work_bytes(r(c), r(s), 4) > 0) == (want == tie_amd.ENOINIT)
