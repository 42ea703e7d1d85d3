"""What the page plan, the append of several axes, the attention through a window
and the log-probabilities refuse, without a GPU (a good call is TIE_HIP_ENOINIT
there), the memory that they ask for, and the streams that the binding names."""
import ctypes
import os

import numpy as np
import pytest

import tie_amd
from test_kv_host import A, BAD_CACHE, BAD_SEQS, W, cache, seqs

pytestmark = pytest.mark.skipif(not os.path.exists(tie_amd.LIB_PATH), reason="libtie_hip.so not built")
NAN, INF = float("nan"), float("inf")
PAIRS = bytes([0, 1, 2, 0] * 8)  # a head of 64


def axes(c=None, s=None, layer=0, heads=4, eps=1e-6, theta=1e6, q=A, k=A + 8192, v=A + 16384, out=A + 32768, sq=W, sk=128, sv=128,
         so=W, pos=A, n=3, axis=PAIRS):
    return tie_amd.lib().tie_hip_kv_append_axes(ctypes.byref(c or cache()), layer, ctypes.byref(s or seqs()), q, sq, k, sk, v, sv,
                                                heads, A, A, eps, theta, pos, n, axis, out, so, None)


def window(c=None, s=None, layer=0, heads=4, scale=0.1, win=5, sinks=0, at=None, mask=None, words=0, q=A, out=A + 32768, sq=W, so=W,
           work=None, nw=0):
    return tie_amd.lib().tie_hip_window_attention(ctypes.byref(c or cache()), layer, ctypes.byref(s or seqs()), q, sq, heads, scale,
                                                  win, sinks, at, mask, words, out, so, work, nw, None)


# (the arrays apart: the table of 3 x 5 at A, out at A + 4096, the ring of 100 at A + 8192, ...)
def plan(n_pages=100, free=A + 8192, state=A + 12288, state_out=A + 12288, n_seqs=3, cols=5, n=7, pages=A, lens=A + 1024,
         new=A + 2048, win=0, sinks=0, out=A + 4096, first=A + 16384, pos=A + 20480, slot=A + 24576):
    pool = tie_amd.KVPoolDesc(n_pages, free, state, state_out)
    return tie_amd.lib().tie_hip_kv_plan(ctypes.byref(pool), n_seqs, cols, n, pages, lens, new, win, sinks, out, first, pos, slot, None, 0,
                                         None)


def logprobs(logits=A, stride=100, vocab=100, n=5, tokens=A + 4096, temp=1.0, top=3, lp=A + 8192, rank=A + 12288, ent=A + 16384,
             tt=A + 20480, tl=A + 24576):
    return tie_amd.lib().tie_hip_token_logprobs(logits, stride, vocab, n, tokens, temp, top, lp, rank, ent, tt, tl, None, 0, None)


@pytest.mark.parametrize("call", [axes, window])
def test_caches_and_sequences(call):
    assert call() == tie_amd.ENOINIT
    for kw in BAD_CACHE:
        assert call(c=cache(**kw)) == tie_amd.EINVAL, kw
        assert tie_amd.last_error()
    for kw in BAD_SEQS:
        assert call(s=seqs(**kw)) == tie_amd.EINVAL, kw
    assert call(c=cache(type=tie_amd.F16, k_scale=None, v_scale=None)) == tie_amd.ENOINIT


@pytest.mark.parametrize("call,bad", [
    (axes, [dict(n=0), dict(n=5), dict(n=2), dict(axis=None), dict(pos=None), dict(axis=bytes(31) + b"\3"), dict(layer=2), dict(heads=3),
            dict(theta=0.0), dict(eps=NAN), dict(q=None), dict(out=None), dict(sq=W - 1), dict(so=W - 1), dict(out=A + 4)]),
    (window, [dict(win=0), dict(win=-1), dict(sinks=-1), dict(layer=2), dict(heads=3), dict(scale=NAN), dict(mask=A, words=0),
              dict(mask=A + 4, words=1), dict(q=None), dict(out=None), dict(sq=W - 1), dict(out=A + 16)]),
    (plan, [dict(n_pages=0), dict(n_pages=(1 << 25) + 1), dict(free=None), dict(state=None), dict(state_out=None), dict(n_seqs=-1),
            dict(n_seqs=65536), dict(cols=0), dict(cols=1 << 26), dict(n=-1), dict(win=-1), dict(sinks=-1), dict(pages=None),
            dict(lens=None), dict(new=None), dict(out=None), dict(first=None), dict(out=A + 4), dict(out=A + 1024 - 4),
            dict(first=A + 4096), dict(pos=A + 20480, slot=A + 20484), dict(first=A + 1024 - 12), dict(pos=A + 2048 + 8),
            dict(state_out=A + 12292), dict(free=A + 4096 + 56), dict(state_out=A + 2048), dict(slot=A)]),
    (logprobs, [dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(n=-1), dict(n=(1 << 23) + 1), dict(stride=99), dict(temp=0.0),
                dict(temp=-1.0), dict(temp=NAN), dict(temp=INF), dict(temp=1e7), dict(top=-1), dict(top=65), dict(logits=None),
                dict(tt=None), dict(tl=None), dict(tokens=None), dict(tokens=None, rank=None), dict(lp=A + 1996), dict(rank=A + 4096),
                dict(ent=A + 8192 + 16), dict(tl=A + 20480 + 56)]),
])
def test_arguments(call, bad):
    assert call() == tie_amd.ENOINIT
    for kw in bad:
        assert call(**kw) == tie_amd.EINVAL, kw
        assert tie_amd.last_error()


def test_what_may_be_left_out_or_shared():
    assert plan(out=A, state_out=A + 12288) == tie_amd.ENOINIT  # in place
    assert plan(state_out=A + 14000, pos=None, slot=None) == tie_amd.ENOINIT
    assert plan(n_seqs=0, pages=None, lens=None, new=None, out=None) == tie_amd.ENOINIT
    assert logprobs(tokens=None, lp=None, rank=None) == tie_amd.ENOINIT
    assert logprobs(top=0, tt=None, tl=None, ent=None, rank=None) == tie_amd.ENOINIT
    assert logprobs(top=64) == tie_amd.ENOINIT
    assert logprobs(n=0, logits=None) == tie_amd.ENOINIT
    assert axes(n=4, axis=bytes([3] * 32)) == tie_amd.ENOINIT
    assert axes(out=A) == tie_amd.ENOINIT
    assert window(win=0x7fffffff, sinks=0x7fffffff, at=A) == tie_amd.ENOINIT
    assert tie_amd.lib().tie_hip_kv_plan(None, 0, 1, 0, None, None, None, 0, 0, None, A, None, None, None, 0, None) == tie_amd.EINVAL
    assert tie_amd.kv_plan_work_bytes(-1) == tie_amd.kv_plan_work_bytes(65536) == 0
    assert tie_amd.token_logprobs_work_bytes(0, 1, 1) == tie_amd.token_logprobs_work_bytes(10, 1, 65) == 0


def need(kind, H, kvh, hd, tokens, n_seqs, pages):
    c = tie_amd.KVCacheDesc(type=kind, n_layers=1, n_pages=4, kv_heads=kvh, head_dim=hd, k=256, v=256, k_scale=256, v_scale=256)
    s = tie_amd.KVSeqsDesc(n_seqs=n_seqs, max_pages=pages, n_tokens=tokens, pages=256, len=256, first=256)
    return tie_amd.lib().tie_hip_window_attention_work_bytes(ctypes.byref(c), ctypes.byref(s), H)


@pytest.mark.parametrize("kind", [tie_amd.F16, tie_amd.I8])
@pytest.mark.parametrize("H,kvh,hd", [(32, 4, 128), (40, 8, 64), (5, 5, 128), (96, 1, 128), (1024, 1024, 64)])
def test_window_memory_for_a_call_is_memory_for_every_smaller_one(kind, H, kvh, hd):
    rng = np.random.default_rng(H)
    some = lambda most: int(np.exp(rng.random() * np.log(most + 0.99)))  # noqa: E731
    grid = [(t, min(some(t), 65535), some(20000)) for t in (some(8192) for _ in range(300))]
    got = {g: need(kind, H, kvh, hd, *g) for g in grid}
    for t, s, p in grid:
        # whichever of the kernels takes the rows (that follows the window too), by the
        # rules that cut them: units of 16, 64 or 128 rows, none cut where tiles fill the card
        rows = t * (H // kvh)
        for tile in (16, 64 if rows * kvh < 256 * 128 else 128):
            n = ((256 if tile == 16 else 512) + kvh) + (rows + min(s, t) * (tile - 1)) // tile * kvh
            few_only = tile > 16 and rows <= 16 * s
            if rows // tile * kvh < 256 and not (tile == 16 and n > 8192) and not few_only:
                assert got[t, s, p] >= 8192 * 4 + n * tile * (hd + 4) * 4, (t, s, p, tile)
    for _ in range(10000):
        a, b = (grid[i] for i in rng.integers(0, len(grid), 2))
        if all(x <= y for x, y in zip(a, b)):
            assert got[a] <= got[b], (a, b)


def test_plan_and_logprobs_memory_grows_with_each_size():
    sizes = [(v, n, k) for v in (1, 4096, 4097, 151936) for n in (1, 5, 200, 1023, 1024, 5000) for k in (0, 1, 64)]
    got = {s: tie_amd.token_logprobs_work_bytes(*s) for s in sizes}
    for a in sizes:
        for b in sizes:
            if all(x <= y for x, y in zip(a, b)):
                assert got[a] <= got[b], (a, b)
    plans = [tie_amd.kv_plan_work_bytes(n) for n in range(1, 3000, 7)]
    assert plans == sorted(plans)


def test_the_binding_names_the_stream(monkeypatch):
    import torch
    from test_kv_streams import Recorder
    i32 = dict(dtype=torch.int32)
    k = torch.zeros(1, 2, 2, 64, 64, dtype=torch.float16)
    c, s = tie_amd.KVCache(k, k.clone()), tie_amd.KVSeqs(torch.zeros(2, 3, **i32), torch.zeros(2, **i32))
    q, kv, two = torch.zeros(2, 256), torch.zeros(2, 128), torch.zeros(2, **i32)
    pool = tie_amd.KVPool(torch.zeros(9, **i32), torch.zeros(2, **i32))
    calls = (lambda **kw: c.append_axes(0, s, q, kv, kv, q, torch.zeros(3, 2, **i32), PAIRS, **kw),
             lambda **kw: c.window_attention(0, s, q, q, 1.0, 7, sinks=1, at=two, **kw),
             lambda **kw: pool.plan(torch.zeros(2, 3, **i32), two, two, torch.zeros(2, 3, **i32), torch.zeros(3, **i32), pos=two, **kw),
             lambda **kw: tie_amd.token_logprobs(torch.zeros(2, 50), two, torch.zeros(2), **kw))
    lib, now = Recorder(), [0]
    monkeypatch.setattr(tie_amd, "lib", lambda: lib)
    real = tie_amd._current
    monkeypatch.setattr(tie_amd, "_current", lambda stream, device: real(stream, 0))  # (the tensors' device is the CPU here)
    monkeypatch.setattr(tie_amd, "_raw_stream", lambda device: now[0])
    for call in calls:
        for torchs, given, want in ((0, None, 1), (77, None, 77), (77, 0, 1), (77, 88, 88)):
            now[0] = torchs
            call(**({} if given is None else dict(stream=given)))
            assert lib.streams.pop() == want, (torchs, given)
    i64 = torch.zeros(2, dtype=torch.int64)
    for bad in (lambda: c.append_axes(0, s, q, kv, kv, q, torch.zeros(3, 2, **i32), PAIRS[1:]),
                lambda: c.append_axes(0, s, q, kv, kv, q, torch.zeros(3, 3, **i32), PAIRS),
                lambda: c.window_attention(0, s, q, q, 1.0, 7, at=i64),
                lambda: pool.plan(torch.zeros(2, 3, **i32), i64, two, torch.zeros(2, 3, **i32), torch.zeros(3, **i32), n_tokens=2),
                lambda: pool.plan(torch.zeros(2, 3, **i32), two, two, torch.zeros(2, 3, **i32), torch.zeros(3, **i32)),
                lambda: pool.plan(torch.zeros(2, 3, **i32), two, two, torch.zeros(2, 4, **i32), torch.zeros(3, **i32), n_tokens=2),
                lambda: tie_amd.token_logprobs(torch.zeros(2, 50), i64, torch.zeros(2)),
                lambda: tie_amd.token_logprobs(torch.zeros(2, 50), top_tokens=torch.zeros(2, 3, **i32)),
                lambda: tie_amd.token_logprobs(torch.zeros(2, 50, dtype=torch.float16), two, torch.zeros(2))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("bad", [32, np.zeros(4, np.int64), np.zeros(16, np.int16), [0] * 31 + [256], [0] * 31 + [-1], [0.0] * 32])
def test_axes_that_are_not_one_small_number_for_each_pair(bad):
    """(32 is not 32 zeros, and an array's numbers are looked at, not its memory)"""
    import torch
    k = torch.zeros(1, 2, 2, 64, 64, dtype=torch.float16)
    c, s = tie_amd.KVCache(k, k.clone()), tie_amd.KVSeqs(torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    q, kv = torch.zeros(2, 256), torch.zeros(2, 128)
    with pytest.raises((ValueError, TypeError)):
        c.append_axes(0, s, q, kv, kv, q, torch.zeros(3, 2, dtype=torch.int32), bad)
    with pytest.raises(tie_amd.TieError):
        c.append_axes(0, s, q, kv, kv, q, None, PAIRS)
    assert "n_axes" in tie_amd.last_error()
