"""What the calls of the attention half refuse, without a GPU: arguments are
checked before anything else, so a bad one is TIE_HIP_EINVAL (and names what is
wrong) even where the library is not initialised, and a good call then is
TIE_HIP_ENOINIT."""
import ctypes
import os

import numpy as np
import pytest

import tie_amd

pytestmark = pytest.mark.skipif(not os.path.exists(tie_amd.LIB_PATH), reason="libtie_hip.so not built")

# addresses that no call follows here
MEM = np.zeros(1 << 16, np.uint8)
A = (MEM.ctypes.data + 255) & ~255


def cache(**kw):
    d = dict(type=tie_amd.I8, n_layers=2, n_pages=4, kv_heads=2, head_dim=64, k=A, v=A, k_scale=A, v_scale=A)
    d.update(kw)
    return tie_amd.KVCacheDesc(**d)


def seqs(**kw):
    d = dict(n_seqs=2, max_pages=3, n_tokens=5, pages=A, len=A, first=A)
    d.update(kw)
    return tie_amd.KVSeqsDesc(**d)


W = 4 * 64  # a query row


def append(c=None, s=None, layer=0, heads=4, eps=1e-6, theta=1e6, q=A, k=A + 8192, v=A + 16384, out=A + 32768, sq=W, sk=128, sv=128,
           so=W):
    return tie_amd.lib().tie_hip_kv_append(ctypes.byref(c or cache()), layer, ctypes.byref(s or seqs()), q, sq, k, sk, v, sv, heads,
                                           A, A, eps, theta, None, out, so, None)


def read(c=None, s=None, layer=0, n=1, k=A, v=A + 32768):
    return tie_amd.lib().tie_hip_kv_read(ctypes.byref(c or cache()), layer, n, ctypes.byref(s or seqs()), k, v, None)


def keep(c=None, s=None, path=A, most=4, n=A + 4096, out=None):
    return tie_amd.lib().tie_hip_kv_keep(ctypes.byref(c or cache()), ctypes.byref(s or seqs()), path, most, n, out, None)


def attention(c=None, s=None, layer=0, heads=4, scale=0.1, mask=None, words=0, q=A, out=A + 32768, sq=W, so=W):
    return tie_amd.lib().tie_hip_tree_attention(ctypes.byref(c or cache()), layer, ctypes.byref(s or seqs()), q, sq, heads, scale,
                                                mask, words, out, so, None, 0, None)


def verify(logits=A, ls=100, draft=None, ds=0, vocab=100, n_seqs=2, n=5, first=A, tokens=A, parent=A, ua=A, us=A, temp=1.0, kids=2,
           most=3, path=A + 4096, nk=A + 8192, nxt=A + 8448):
    return tie_amd.lib().tie_hip_verify_tree(logits, ls, draft, ds, vocab, n_seqs, n, first, tokens, parent, ua, us, temp, kids, most,
                                             path, nk, nxt, None, 0, None)


BAD_CACHE = [dict(type=tie_amd.BF16), dict(type=8), dict(n_layers=0), dict(n_pages=0), dict(kv_heads=0), dict(head_dim=96),
             dict(head_dim=256), dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=A + 8), dict(v_scale=A + 4)]
BAD_SEQS = [dict(n_seqs=-1), dict(n_seqs=65536), dict(n_tokens=-1), dict(max_pages=0), dict(max_pages=1 << 30), dict(pages=None),
            dict(len=None), dict(first=None)]


@pytest.mark.parametrize("call", [append, read, keep, attention])
def test_caches_and_sequences(call):
    assert call() == tie_amd.ENOINIT
    for kw in BAD_CACHE:
        assert call(c=cache(**kw)) == tie_amd.EINVAL, kw
        assert tie_amd.last_error()
    for kw in BAD_SEQS:
        assert call(s=seqs(**kw)) == tie_amd.EINVAL, kw
    assert call(c=cache(type=tie_amd.F16, k_scale=None, v_scale=None)) == tie_amd.ENOINIT
    assert call(s=seqs(first=None, n_tokens=2)) == tie_amd.ENOINIT


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("call,bad", [
    (append, [dict(layer=2), dict(layer=-1), dict(heads=3), dict(heads=0), dict(theta=0.0), dict(theta=NAN), dict(theta=INF),
              dict(eps=-1.0), dict(eps=NAN), dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(sq=W - 1), dict(sk=127),
              dict(sv=127), dict(so=W - 1), dict(out=A + 4), dict(out=A, so=W + 4), dict(out=A + 8192 + 256)]),
    (read, [dict(layer=2), dict(n=0), dict(n=3), dict(layer=1, n=2), dict(k=None), dict(v=None), dict(v=A + 16)]),
    (keep, [dict(path=None), dict(most=0), dict(n=None), dict(out=A + 4096 + 4), dict(out=A + 4)]),
    (attention, [dict(layer=2), dict(heads=3), dict(scale=NAN), dict(scale=INF), dict(mask=A, words=0), dict(mask=A + 4, words=1),
                 dict(q=None), dict(out=None), dict(sq=W - 1), dict(so=W - 1), dict(out=A + 16), dict(out=A, so=W + 4)]),
    (verify, [dict(vocab=0), dict(vocab=(1 << 24) + 1), dict(n=-1), dict(n=65536), dict(n_seqs=-1), dict(ls=99), dict(draft=A, ds=99),
              dict(temp=-1.0), dict(temp=NAN), dict(temp=INF), dict(kids=0), dict(kids=17), dict(most=0), dict(first=None),
              dict(logits=None), dict(tokens=None), dict(parent=None), dict(ua=None), dict(us=None), dict(path=None), dict(nk=None),
              dict(nxt=None), dict(path=A + 16), dict(nk=A + 4096 + 20), dict(nxt=A + 8196), dict(nxt=A),
              dict(draft=A + 8192, ds=100)]),
])
def test_arguments(call, bad):
    assert call() == tie_amd.ENOINIT
    for kw in bad:
        assert call(**kw) == tie_amd.EINVAL, kw
        assert tie_amd.last_error()


def test_in_place_is_no_overlap():
    assert append(out=A) == tie_amd.ENOINIT
    assert attention(out=A) == tie_amd.ENOINIT
    # rows side by side in one matrix are none either; rows that share columns are
    one = dict(sq=1024, sk=1024, sv=1024, so=1024)
    beside = dict(one, k=A + W * 4, v=A + W * 4 + 512, out=A)
    assert append(**beside) == tie_amd.ENOINIT
    assert append(**dict(beside, out=A + W * 4 + 1024)) == tie_amd.ENOINIT
    for bad in (dict(k=A), dict(v=A + W * 4 - 4), dict(k=A + 4096 + 256), dict(out=A + W * 4 + 1020), dict(out=A + 4096 - 4)):
        assert append(**dict(beside, **bad)) == tie_amd.EINVAL, bad
    assert attention(out=A + 4 * W, sq=2 * W, so=2 * W) == tie_amd.ENOINIT
    assert attention(out=A + 4 * W - 4, sq=2 * W, so=2 * W) == tie_amd.EINVAL


def test_null_structures():
    lib = tie_amd.lib()
    c, s = ctypes.byref(cache()), ctypes.byref(seqs())
    for a, b in ((None, s), (c, None)):
        assert lib.tie_hip_kv_read(a, 0, 1, b, A, A + 32768, None) == tie_amd.EINVAL
        assert lib.tie_hip_kv_keep(a, b, A, 1, A, None, None) == tie_amd.EINVAL
        assert lib.tie_hip_tree_attention(a, 0, b, A, W, 4, 0.1, None, 0, A + 32768, W, None, 0, None) == tie_amd.EINVAL
        assert lib.tie_hip_tree_attention_work_bytes(a, b, 4) == 0


def test_work_bytes():
    """Asked for without a GPU; 0 for what the call would refuse."""
    lib = tie_amd.lib()
    assert lib.tie_hip_tree_attention_work_bytes(ctypes.byref(cache()), ctypes.byref(seqs()), 4) > 0
    assert lib.tie_hip_tree_attention_work_bytes(ctypes.byref(cache(head_dim=96)), ctypes.byref(seqs()), 4) == 0
    assert lib.tie_hip_tree_attention_work_bytes(ctypes.byref(cache()), ctypes.byref(seqs()), 5) == 0
    assert tie_amd.verify_tree_work_bytes(1000, 5, 2, True) > tie_amd.verify_tree_work_bytes(1000, 5, 2, False) > 0
    assert tie_amd.verify_tree_work_bytes(1000, 5, 17, False) == 0


def test_the_binding_checks_tensors():
    import torch
    k, v = torch.zeros(1, 2, 2, 64, 64, dtype=torch.float16), torch.zeros(1, 2, 2, 64, 64, dtype=torch.float16)
    c = tie_amd.KVCache(k, v)
    i32 = dict(dtype=torch.int32)
    s = tie_amd.KVSeqs(torch.zeros(2, 3, **i32), torch.zeros(2, **i32), torch.tensor([0, 2, 5], **i32))
    assert s.n_tokens == 5
    for bad in (lambda: tie_amd.KVCache(k.float(), v), lambda: tie_amd.KVCache(k, v[:, :1]), lambda: tie_amd.KVCache(k.to(torch.int8), v),
                lambda: tie_amd.KVCache(k.transpose(1, 2), v), lambda: tie_amd.KVSeqs(torch.zeros(2, 3), torch.zeros(2, **i32)),
                lambda: tie_amd.KVSeqs(torch.zeros(2, 3, **i32), torch.zeros(3, **i32))):
        with pytest.raises(ValueError):
            bad()
    q, kk = torch.zeros(5, 4, 64), torch.zeros(5, 2, 64)
    for bad in (dict(q=q[:4]), dict(q=q[:, :, :32]), dict(q=q.double()), dict(q_out=q.transpose(0, 1)), dict(k=q), dict(v=kk[:3]),
                dict(q_norm=torch.zeros(32)), dict(k=kk[:1].expand(5, 2, 64)), dict(pos=torch.zeros(4, **i32))):
        with pytest.raises(ValueError):
            c.append(0, s, **dict(dict(q=q, k=kk, v=kk, q_out=q.clone()), **bad))
    for bad in (dict(mask=torch.zeros(4, 1, dtype=torch.int64)), dict(mask=torch.zeros(5, 1, **i32)), dict(out=q[:, :3])):
        with pytest.raises(ValueError):
            c.attention(0, s, **dict(dict(q=q, out=q.clone(), scale=1.0), **bad))
    with pytest.raises(tie_amd.TieError) as e:
        c.attention(0, s, q, q.clone(), 1.0)
    assert e.value.code == tie_amd.ENOINIT


def test_the_binding_refuses_other_devices(monkeypatch):
    """(get_device of a tensor on the CPU is -1: the library is made to say that it has another GPU)"""
    import torch
    i32 = dict(dtype=torch.int32)
    k = torch.zeros(1, 2, 2, 64, 64, dtype=torch.float16)
    c, s = tie_amd.KVCache(k, k.clone()), tie_amd.KVSeqs(torch.zeros(2, 3, **i32), torch.zeros(2, **i32))
    q, kv, two = torch.zeros(2, 256), torch.zeros(2, 128), torch.zeros(2, **i32)
    calls = (lambda: c.append(0, s, q, kv, kv, q), lambda: c.read(s, kv.view(1, 2, 2, 64), kv.view(1, 2, 2, 64).clone()),
             lambda: c.attention(0, s, q, q, 1.0), lambda: c.keep(s, torch.zeros(2, 3, **i32), two),
             lambda: tie_amd.verify_tree(torch.zeros(2, 50), None, two, two, torch.zeros(2), torch.zeros(2), torch.zeros(2, 3, **i32),
                                         two, two))
    for call in calls:
        with pytest.raises(tie_amd.TieError):  # (not initialised)
            call()
    monkeypatch.setattr(tie_amd, "_device", 0)
    for call in calls:
        with pytest.raises(ValueError, match="device"):
            call()
    monkeypatch.setattr(tie_amd, "_device", None)
    monkeypatch.setattr(c, "device", 1)
    for call in calls[:4]:
        with pytest.raises(ValueError, match="device"):
            call()
