"""Which stream the attention half's calls go to, and that they stand in order
with the work before and behind them there."""
import os

import numpy as np
import pytest

import tie_amd

needs_lib = pytest.mark.skipif(not os.path.exists(tie_amd.LIB_PATH), reason="libtie_hip.so not built")


class Recorder:
    """A library whose calls succeed and leave their last argument, the stream."""

    def __init__(self):
        self.streams = []

    def __getattr__(self, name):
        def call(*args):
            self.streams.append(args[-1])
            return 0
        return call


def test_the_binding_names_the_stream(monkeypatch):
    """None: the one torch works on, for these calls, and the library's, for the
    others; 0, torch's handle of the default stream: HIP's default stream."""
    import torch
    i32 = dict(dtype=torch.int32)
    k = torch.zeros(1, 2, 2, 64, 64, dtype=torch.float16)
    c, s = tie_amd.KVCache(k, k.clone()), tie_amd.KVSeqs(torch.zeros(2, 3, **i32), torch.zeros(2, **i32))
    q, kv, two, rows = torch.zeros(2, 256), torch.zeros(2, 128), torch.zeros(2, **i32), torch.zeros(1, 2, 2, 64)
    calls = (lambda **kw: c.append(0, s, q, kv, kv, q, **kw), lambda **kw: c.read(s, rows, rows.clone(), **kw),
             lambda **kw: c.attention(0, s, q, q, 1.0, **kw), lambda **kw: c.keep(s, torch.zeros(2, 3, **i32), two, **kw),
             lambda **kw: tie_amd.verify_tree(torch.zeros(2, 50), None, two, two, torch.zeros(2), torch.zeros(2),
                                              torch.zeros(2, 3, **i32), two, two, **kw))
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
    for call in (tie_amd.stream_status, tie_amd.stream_release):
        for given, want in ((None, None), (0, 1), (88, 88)):
            call(given)
            assert lib.streams.pop() == want


@needs_lib
def test_the_header_names_the_default_stream():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with open(os.path.join(root, "include", "tie_hip.h")) as f:
        assert "#define TIE_HIP_STREAM_DEFAULT ((void *)%d)" % tie_amd.DEFAULT_STREAM in f.read()


@pytest.fixture(scope="module")
def device():
    import torch
    assert torch.cuda.is_available(), "GPU test without a GPU"
    tie_amd.init(0)
    yield
    tie_amd.shutdown()


def late(work, *pairs):
    """Fills each buffer behind some milliseconds of products on torch's stream."""
    for _ in range(6):
        work = work @ work * 1e-4
    for to, value in pairs:
        to.copy_(value)


@pytest.mark.gpu
@pytest.mark.parametrize("where", ["default", "side", "default by its handle"])
def test_in_order_without_synchronisation(device, where):
    """Inputs written on torch's stream right before a call, outputs read there
    right behind it and then overwritten; nothing waits for the GPU between.
    The results are a synchronised call's, bit for bit."""
    import torch
    rng = np.random.default_rng(5)
    H, kvh, hd, lens, counts, V = 8, 2, 64, [300, 40], [9, 3], 5000
    T = sum(counts)
    stream = torch.cuda.Stream() if where == "side" else torch.cuda.default_stream()
    kw = dict(stream=stream.cuda_stream) if where == "default by its handle" else {}

    def f32(*shape):
        return torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).cuda()

    def i32(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    k0, v0 = f32(2, 8, kvh, 64, hd).half(), f32(2, 8, kvh, hd, 64).half()
    pages, len0, first = i32([[5, 0, 3, 7, 1, -1], [2, 6, -1, -1, -1, -1]]), i32(lens), i32([0, 9, 12])
    x0, q0, logits0 = f32(T, (H + 2 * kvh) * hd), f32(T, H, hd), f32(T, V) * 3
    u, tokens = torch.rand(2, T, device="cuda"), i32(rng.integers(0, V, T).tolist())
    parent, path0, n0 = i32([-1, 0, 0, 1, 1, 2, 2, 3, 3, -1, 0, 1]), i32([[0, 2, 6, -1], [0, 1, -1, -1]]), i32([3, 2])
    work = f32(4096, 4096)

    def steps(go):
        """Every call, each between `go(inputs)` and a copy of its outputs."""
        got = []

        def out(*buffers):
            got.extend(b.clone() for b in buffers)
            for b in buffers:
                b.fill_(-7)

        k, v, ln = torch.zeros_like(k0), torch.zeros_like(v0), torch.zeros_like(len0)
        cache, seqs = tie_amd.KVCache(k, v), tie_amd.KVSeqs(pages, ln, first, T)
        x, q = torch.zeros_like(x0), torch.zeros_like(q0)
        rows = [torch.zeros(2, T, kvh, hd, device="cuda") for _ in range(2)]
        qo, o = torch.zeros_like(q0), torch.zeros_like(q0)
        go((k, k0), (v, v0), (ln, len0), (x, x0))
        cache.append(0, seqs, x[:, :H * hd], x[:, H * hd:(H + kvh) * hd], x[:, (H + kvh) * hd:], qo, **kw)
        out(qo)
        go((k[1], k0[0]), (v[1], v0[0]))
        cache.read(seqs, *rows, n_layers=2, **kw)
        out(*rows)
        go((q, q0))
        cache.attention(0, seqs, q, o, hd ** -0.5, **kw)
        out(o)
        path, n, nxt = torch.zeros_like(path0), torch.zeros_like(n0), torch.zeros_like(n0)
        go((path, path0), (n, n0))
        cache.keep(seqs, path, n, ln, **kw)
        got.extend((ln.clone(), k.clone(), v.clone()))
        logits = torch.zeros_like(logits0)
        go((logits, logits0))
        tie_amd.verify_tree(logits, first, tokens, parent, u[0], u[1], path, n, nxt, max_children=2, **kw)
        out(path, n, nxt)
        return got

    def at_once(*pairs):
        for to, value in pairs:
            to.copy_(value)
        torch.cuda.synchronize()

    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        steps(at_once)  # (the stream's workspace)
        torch.cuda.synchronize()
        want = steps(at_once)
        torch.cuda.synchronize()
        got = steps(lambda *pairs: late(work, *pairs))
    torch.cuda.synchronize()
    assert float(got[0].abs().max()) > 0
    for i, (a, b) in enumerate(zip(got, want)):
        assert torch.equal(a, b), i


@pytest.mark.gpu
def test_the_older_calls_take_the_default_stream(device):
    """A matrix product between torch's own, on the default stream by its handle."""
    import torch
    from tie_amd import synth
    rng = np.random.default_rng(6)
    m = tie_amd.Matrix(synth.expert_tensor(rng, synth.BF16, 1, 256, 256), synth.BF16, 256, 256)
    x0 = torch.from_numpy(rng.standard_normal((5, 256)).astype(np.float32)).cuda()
    x, out, work = torch.zeros_like(x0), torch.zeros(5, 256, device="cuda"), torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    m.mat_mat(x0, 5, out)
    torch.cuda.synchronize()
    want = out.clone()
    late(work, (x, x0))
    m.mat_mat(x, 5, out, stream=torch.cuda.default_stream().cuda_stream)
    got = out.clone()
    out.fill_(-7)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and float(want.abs().max()) > 0
    m.close()


@pytest.mark.gpu
def test_the_callers_device_stays(device):
    """Calls on the library's GPU from a program whose current device is another."""
    import torch
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    k = torch.zeros(1, 2, 2, 64, 64, dtype=torch.float16, device="cuda:0")
    i32 = dict(dtype=torch.int32, device="cuda:0")
    c, s = tie_amd.KVCache(k, k.clone()), tie_amd.KVSeqs(torch.zeros(2, 3, **i32), torch.zeros(2, **i32))
    q, kv, rows, two = (torch.zeros(n, device="cuda:0") for n in ((2, 256), (2, 128), (1, 2, 2, 64), 2))
    nodes = torch.zeros(2, **i32)
    with torch.cuda.device(1):
        for call in (lambda: c.append(0, s, q, kv, kv, q), lambda: c.read(s, rows, rows.clone()), lambda: c.attention(0, s, q, q, 1.0),
                     lambda: c.keep(s, torch.zeros(2, 3, **i32), nodes),
                     lambda: tie_amd.verify_tree(torch.zeros(2, 50, device="cuda:0"), None, nodes, nodes, two, two,
                                                 torch.zeros(2, 3, **i32), nodes.clone(), nodes.clone())):
            call()
            assert torch.cuda.current_device() == 1
