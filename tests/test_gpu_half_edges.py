"""Calls of the attention half at the ends of what the header allows: head
groups, scales, thousands of sequences, pages that sequences share, batches of
nothing, vocabularies of many blocks."""
import gc

import numpy as np
import pytest

import kv_ref
import tie_amd
from test_gpu_int8_scales import attention
from test_gpu_tree_attention import check, cuda, device, run, words  # noqa: F401 (device: the module's fixture)
from test_gpu_verify import Case

pytestmark = pytest.mark.gpu

KINDS = pytest.mark.parametrize("kind", ["f16", "i8"])


@KINDS
@pytest.mark.parametrize("H,kvh,hd,lens,counts", [(96, 1, 64, [130], [1]), (96, 1, 128, [70], [5]), (200, 1, 64, [300, 3], [2, 1]),
                                                  (130, 130, 64, [700], [1]), (300, 300, 64, [70], [2]), (129, 3, 64, [200], [9])])
def test_head_groups(kind, H, kvh, hd, lens, counts):
    """A token's heads of one kv head fill several tiles; more kv heads than units fill the card."""
    rng = np.random.default_rng(H)
    c = kv_ref.Cache(rng, kind, kvh, hd, lens, counts)
    q = rng.standard_normal((sum(counts), H, hd)).astype(np.float32)
    want, tol = kv_ref.attention(c, 0, q, hd ** -0.5, lambda b, i, j: j <= i)
    check(run(c, q, hd ** -0.5), want, tol)


@KINDS
@pytest.mark.parametrize("scale", [0.0, -0.0, -0.125, 1e-20, 3.0])
@pytest.mark.parametrize("H,kvh,hd,length,n", [(8, 2, 64, 200, 3), (8, 2, 64, 300, 90)])
def test_scales(kind, scale, H, kvh, hd, length, n):
    """0: the mean of what a token sees; negative ones turn the scores round.
    (At 3 one row has nearly all the weight, and in a column where it is 0 the
    others' weights of e^-20 are all there is: the tolerance has the weights'
    least step, derived in attention().)"""
    rng = np.random.default_rng(n)
    c = kv_ref.Cache(rng, kind, kvh, hd, [length], [n])
    q = rng.standard_normal((n, H, hd)).astype(np.float32)
    want, tol = attention(c, q, scale, lambda b, i, j: j <= i)
    check(run(c, q, scale), want, tol)


@KINDS
def test_thousands_of_sequences(kind):
    """Single tokens, some sequences of none, without and with `first`; their
    rows appended, attended to, kept."""
    import torch
    n, kvh, hd, H = 3000, 1, 64, 2
    rng = np.random.default_rng(7)
    lens, counts = rng.integers(0, 60, n).tolist(), [1] * n
    lens[2000] = 700
    for holes in (False, True):
        if holes:
            counts = (rng.random(n) < 0.7).astype(int).tolist()
        T = sum(counts)
        c = kv_ref.Cache(rng, kind, kvh, hd, lens, counts, fill=True)
        kv, seqs = c.gpu(), c.seqs()
        if not holes:
            seqs = tie_amd.KVSeqs(*seqs.keep[:2])
        x = rng.standard_normal((T, (H + 2 * kvh) * hd)).astype(np.float32)
        xd, pos = cuda(x), torch.zeros(T, dtype=torch.int32, device="cuda")
        q = torch.empty(T, H, hd, device="cuda")
        kv.append(0, seqs, xd[:, :H * hd], xd[:, H * hd:(H + kvh) * hd], xd[:, (H + kvh) * hd:], q, pos)
        t = 0
        for b in range(n):
            if counts[b]:
                c.set_rows(0, b, lens[b], x[t:t + 1, H * hd:(H + kvh) * hd].reshape(1, kvh, hd),
                           x[t:t + 1, (H + kvh) * hd:].reshape(1, kvh, hd))
                t += 1
        out = torch.full((T, H, hd), -7.0, device="cuda")
        kv.attention(0, seqs, q, out, 0.125)
        torch.cuda.synchronize()
        for a, w in zip(c.back(), (c.k, c.v, c.ks, c.vs)):
            if w is not None:
                np.testing.assert_array_equal(a, w)
        want, tol = kv_ref.attention(c, 0, q.cpu().numpy(), 0.125, lambda b, i, j: True)
        check(out.cpu().numpy(), want, tol)
        path = torch.zeros(n, 1, dtype=torch.int32, device="cuda")
        kv.keep(seqs, path, torch.ones(n, dtype=torch.int32, device="cuda"), seqs.keep[1])
        torch.cuda.synchronize()
        assert seqs.keep[1].cpu().tolist() == [a + m for a, m in zip(lens, counts)]


@KINDS
def test_pages_that_sequences_share(kind):
    """A prompt's full pages named by three sequences, each with pages of its own behind them."""
    rng = np.random.default_rng(8)
    H, kvh, hd = 8, 2, 64
    c = kv_ref.Cache(rng, kind, kvh, hd, [128, 150, 190], [4, 30, 1])
    c.table[1, :2] = c.table[2, :2] = c.table[0, :2]
    q = rng.standard_normal((35, H, hd)).astype(np.float32)
    want, tol = kv_ref.attention(c, 0, q, 0.125, lambda b, i, j: j <= i)
    check(run(c, q, 0.125), want, tol)
    # one page three times in a table: the rows count three times
    c = kv_ref.Cache(rng, kind, kvh, hd, [192], [1])
    c.table[0, 1] = c.table[0, 2] = c.table[0, 0]
    q = rng.standard_normal((1, H, hd)).astype(np.float32)
    want, tol = kv_ref.attention(c, 0, q, 0.125, lambda b, i, j: True)
    check(run(c, q, 0.125), want, tol)


@KINDS
@pytest.mark.parametrize("n_seqs", [1, 3, 200])
def test_sequences_of_nothing(kind, n_seqs):
    """Token rows that belong to nobody: every output stays, and the next call is served."""
    import torch
    rng = np.random.default_rng(9)
    c = kv_ref.Cache(rng, kind, 2, 64, [10] * n_seqs, [1] * n_seqs)
    kv, seqs = c.gpu(), c.seqs()
    first = seqs.keep[2]
    first.zero_()
    T = n_seqs
    x, out = torch.randn(T, 4, 64, device="cuda"), torch.full((T, 4, 64), -7.0, device="cuda")
    rows = [torch.full((1, T, 2, 64), -7.0, device="cuda") for _ in range(2)]
    lens = torch.full((n_seqs,), -7, dtype=torch.int32, device="cuda")
    kv.append(0, seqs, x, x[:, :2].contiguous(), x[:, 2:].contiguous(), out)
    kv.attention(0, seqs, x, out, 0.125)
    kv.read(seqs, *rows)
    kv.keep(seqs, torch.zeros(n_seqs, 2, dtype=torch.int32, device="cuda"), torch.full((n_seqs,), 2, dtype=torch.int32, device="cuda"), lens)
    torch.cuda.synchronize()
    assert bool((out == -7).all()) and all(bool((r == -7).all()) for r in rows) and lens.tolist() == [10] * n_seqs
    for a, w in zip(c.back(), (c.k, c.v, c.ks, c.vs)):
        if w is not None:
            np.testing.assert_array_equal(a, w)
    q = rng.standard_normal((T, 4, 64)).astype(np.float32)
    want, tol = kv_ref.attention(c, 0, q, 0.125, lambda b, i, j: True)
    check(run(c, q, 0.125), want, tol)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("V", [64 * 4096, 64 * 4096 + 1, 300001, 130 * 4096 - 5])
def test_vocabularies_of_many_blocks(draft, V):
    """More blocks of 4096 logits than a wave has lanes."""
    c = Case(31, [4, 2], V, draft, branch=2)
    for temperature in (0.0, 0.8):
        c.check(temperature, 2, 4)
    c.us[:] = 1 - 2.0 ** -24  # the last tokens
    c.check(0.8, 2, 4)
    c.logits[:, : V - 70] = -np.inf  # all of it behind the first 64 blocks
    c.tokens[:] = V - 1 - np.arange(6)
    c.us[:] = np.random.default_rng(3).random(6).astype(np.float32)
    for temperature in (0.0, 0.8):
        c.check(temperature, 2, 4)


@pytest.mark.parametrize("temperature", [1e-6, 1e-3, 1e4, 1e30])
def test_temperatures(temperature):
    Case(32, [7, 7], 4000, False, branch=2).check(temperature, 2, 7)
    Case(33, [7, 7], 4000, True, branch=2).check(temperature, 2, 7)


def test_work_memory_of_both_kinds_of_calls():
    """One block of memory for attention and verification in turn, eagerly and in
    one replayed graph, beside a second graph with memory of its own."""
    import torch
    rng = np.random.default_rng(10)
    c = kv_ref.Cache(rng, "i8", 2, 64, [900], [7])
    kv, seqs = c.gpu(), c.seqs()
    q0 = rng.standard_normal((7, 8, 64)).astype(np.float32)
    want, tol = kv_ref.attention(c, 0, q0, 0.125, lambda b, i, j: j <= i)
    v = Case(34, [7], 9000, True, branch=2)
    path0, n0, next0 = v.want(0.8, 2, 7)
    q, args = cuda(q0), [cuda(x) for x in (v.logits, v.first, v.tokens, v.parent, v.ua, v.us)]
    draft = cuda(v.draft)
    need = max(kv.attention_work_bytes(seqs, 8), tie_amd.verify_tree_work_bytes(9000, 7, 2, True))
    graphs = []
    for _ in range(2):
        work = torch.zeros(need, dtype=torch.uint8, device="cuda")
        outs = [torch.zeros(7, 8, 64, device="cuda"), torch.zeros(1, 7, dtype=torch.int32, device="cuda"),
                *(torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2))]

        def step():
            for _ in range(2):
                kv.attention(0, seqs, q, outs[0], 0.125, work=work)
                tie_amd.verify_tree(*args, *outs[1:], temperature=0.8, draft=draft, max_children=2, work=work)

        step()
        torch.cuda.synchronize()
        g, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with kv_ref.capture(g, stream):
            step()
        graphs.append((g, stream, work, outs, step))
    for rep in range(3):
        for g, stream, work, outs, step in graphs:
            for o in outs:
                o.fill_(-7)
        torch.cuda.synchronize()
        for g, stream, work, outs, step in graphs:
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for g, stream, work, outs, step in graphs:
            check(outs[0].cpu().numpy(), want, tol)
            for got, w in zip(outs[1:], (path0, n0, next0)):
                np.testing.assert_array_equal(got.cpu().numpy(), w)
        graphs[0][4]()  # (eagerly between, with the first graph's memory)
        torch.cuda.synchronize()
    del g, graphs
    gc.collect()


def test_times_of_calls_on_the_default_stream():
    """(the library's own event timing)"""
    rng = np.random.default_rng(11)
    c = kv_ref.Cache(rng, "f16", 2, 64, [100], [3])
    q = rng.standard_normal((3, 4, 64)).astype(np.float32)
    tie_amd.profile_enable(True)
    try:
        run(c, q, 0.125)
        ms, calls = tie_amd.profile_read()["attention"]
    finally:
        tie_amd.profile_enable(False)
    assert calls == 1 and 0 < ms < 100
