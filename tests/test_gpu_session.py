"""A long session as it is served: pages planned on the GPU, tokens appended with
positions on three axes, attention through a window whose pages go back to the
pool, and the log-probabilities of the tokens; eagerly and as a replayed graph."""
import numpy as np
import pytest

import kv_ref
import tie_amd
from test_gpu_axes import rotate

pytestmark = pytest.mark.gpu
H, KVH, HD, D, VOCAB = 8, 2, 64, 96, 500
WINDOW, SINKS, EPS, THETA, SCALE = 150, 4, 1e-6, 1e4, 0.125
AXES = [0, 1, 2, 0] * 8


@pytest.fixture(scope="module", autouse=True)
def device():
    import torch
    assert torch.cuda.is_available(), "GPU test without a GPU"
    tie_amd.init(0)
    yield
    tie_amd.shutdown()


class Model:
    """One layer whose queries, keys and values depend on the tokens alone, in the same bits whatever the batch."""

    def __init__(self, rng):
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.qkv = f(VOCAB, (H + 2 * KVH) * HD)  # (embedding and projections at once)
        self.norms, self.head = [1 + 0.1 * f(HD) for _ in range(2)], 0.2 * f(H * HD, VOCAB)

    def history(self, tokens, pos, kind):
        """Queries, and keys and values as the cache holds them, of a whole sequence, in 64 bits."""
        x = self.qkv[tokens].reshape(len(tokens), H + 2 * KVH, HD)
        q = rotate(x[:, :H], self.norms[0], pos, AXES, EPS, THETA).astype(np.float32)
        k = rotate(x[:, H: H + KVH], self.norms[1], pos, AXES, EPS, THETA).astype(np.float32)
        v = x[:, H + KVH:]
        if kind == "f16":
            return q, kv_ref.held_f16(k).astype(np.float64), kv_ref.held_f16(v).astype(np.float64)
        (kc, ks), (vc, vs) = kv_ref.codes(k), kv_ref.codes(v)
        return q, kc * ks[..., None].astype(np.float64), vc * vs[..., None].astype(np.float64)


def positions(n):
    """Text, an image of 6 x 7 patches, text, ...: each a third of the way or so."""
    out, at = [], 0
    while len(out) < n:
        out += [(at + i,) * 3 for i in range(29)]
        at += 29
        out += [(at, at + y, at + x) for y in range(6) for x in range(7)]
        at += 7
    return np.array(out[:n], np.int32).T


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("graph", [False, True])
def test_session(kind, graph):
    import torch
    rng = np.random.default_rng(12)
    model, B, M, N = Model(rng), 3, 12, 260
    total = [420, 300, 515]
    tokens = [rng.integers(0, VOCAB, n) for n in total]
    pos = [positions(n) for n in total]
    history = [model.history(t, p, kind) for t, p in zip(tokens, pos)]
    i32 = dict(dtype=torch.int32, device="cuda")
    cuda = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    P = 19  # fewer than the sequences fill in the end: 7 + 5 + 9
    if kind == "f16":
        k, v = torch.full((1, P, KVH, 64, HD), float("nan"), dtype=torch.float16, device="cuda"), None
        v = torch.full((1, P, KVH, HD, 64), float("nan"), dtype=torch.float16, device="cuda")
        kv = tie_amd.KVCache(k, v)
    else:
        k, v = (torch.zeros(s, dtype=torch.int8, device="cuda") for s in ((1, P, KVH, 64, HD), (1, P, KVH, HD, 64)))
        kv = tie_amd.KVCache(k, v, *(torch.full((1, P, KVH, 64), float("nan"), device="cuda") for _ in range(2)))
    table, lens, new, first = torch.full((B, M), -1, **i32), torch.zeros(B, **i32), torch.zeros(B, **i32), torch.zeros(B + 1, **i32)
    pool = tie_amd.KVPool(torch.arange(P, **i32), torch.tensor([0, P], **i32))
    row, slot, pos_d, of = torch.zeros(N, **i32), torch.zeros(N, **i32), torch.zeros(3, N, **i32), torch.zeros(N, **i32)
    x, q, out = torch.zeros(N, (H + 2 * KVH) * HD, device="cuda"), torch.zeros(N, H, HD, device="cuda"), torch.zeros(N, H, HD, device="cuda")
    logits, lp, ent = torch.zeros(N, VOCAB, device="cuda"), torch.zeros(N, device="cuda"), torch.zeros(N, device="cuda")
    head, norms = cuda(model.head), [cuda(w) for w in model.norms]
    seqs = tie_amd.KVSeqs(table, lens, first, N)
    work = torch.zeros(max(kv.window_attention_work_bytes(seqs, H), tie_amd.kv_plan_work_bytes(B),
                           tie_amd.token_logprobs_work_bytes(VOCAB, N, 0)), dtype=torch.uint8, device="cuda")

    def plan():
        pool.plan(table, lens, new, table, first, pos=row, slot=slot, window=WINDOW, sinks=SINKS, work=work)

    def layer():
        kv.append_axes(0, seqs, x[:, : H * HD], x[:, H * HD: (H + KVH) * HD], x[:, (H + KVH) * HD:], q, pos_d, AXES, q_norm=norms[0],
                       k_norm=norms[1], eps=EPS, theta=THETA)
        kv.window_attention(0, seqs, q, out, SCALE, WINDOW, sinks=SINKS, work=work)

    def score():
        tie_amd.token_logprobs(logits, of, lp, entropy=ent, work=work)

    steps = [plan, layer, score]
    if graph:
        for i, part in enumerate(steps):
            g = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with kv_ref.capture(g):
                part()
            steps[i] = g.replay
    n, seen_free, worst = np.zeros(B, np.int64), [], 0.0
    for step in range(400):
        # prompts in chunks first, then a token each (the second request begins later)
        ask = [0 if n[b] >= total[b] or (b == 1 and step < 3) else min(80 if n[b] < 240 else 1, total[b] - n[b]) for b in range(B)]
        if not any(ask):
            break
        lens.copy_(cuda(n.astype(np.int32)))
        new.copy_(cuda(np.array(ask, np.int32)))
        steps[0]()
        f = first.cpu().numpy()
        got = np.diff(f)
        assert (got == ask).all()  # the pool goes round: no request waits for pages
        x.fill_(float("nan"))
        out.fill_(-7.0)
        want = []
        for b in range(B):
            at = slice(f[b], f[b + 1])
            rows = slice(n[b], n[b] + got[b])
            x[at] = cuda(model.qkv[tokens[b][rows]])
            pos_d[:, at] = cuda(pos[b][:, rows])
            of[at] = cuda(tokens[b][rows].astype(np.int32))
            assert (row[at].cpu().numpy() == np.arange(n[b], n[b] + got[b])).all()
            for r in range(n[b], n[b] + got[b]):
                if got[b] > 5 and r % 7:
                    continue  # (of chunks every seventh)
                on = [i for i in range(r + 1) if i < SINKS or i > r - WINDOW]
                hq, hk, hv = history[b]
                for h in (0, H // KVH, H - 1):
                    kk, vv, qq = hk[on, h // (H // KVH)], hv[on, h // (H // KVH)], hq[r, h].astype(np.float64)
                    s = kk @ qq * SCALE
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    want.append((f[b] + r - n[b], h, w @ vv, kv_ref.tolerance(qq, kk, vv, w, SCALE)))
        steps[1]()
        o = out.cpu().numpy()
        assert (o[f[B]:] == -7.0).all()
        for t, h, value, tol in want:
            # (queries are rounded to F32 once more than the form's, and keys' codes follow)
            assert (np.abs(o[t, h] - value) <= tol + 2.0 ** -20 * np.abs(value).max()).all(), (step, t, h)
        torch.matmul(out.view(N, H * HD), head, out=logits)
        steps[2]()
        torch.cuda.synchronize()
        exact = torch.log_softmax(logits.double(), 1)[: f[B]]
        mine = exact.gather(1, of[: f[B]].long()[:, None])[:, 0]
        assert ((lp[: f[B]] - mine).abs() <= 2e-6 + 1e-7 * mine.abs()).all()
        assert ((ent[: f[B]] + (exact.exp() * exact).sum(1)).abs() <= 1e-5).all()
        n += got
        seen_free.append(int(pool.keep_alive[1][1]))
    assert (n == total).all()
    held = (table >= 0).sum().item()
    assert held + seen_free[-1] == P and sum(-(-t // 64) for t in total) > P
