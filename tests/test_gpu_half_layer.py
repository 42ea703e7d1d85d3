"""The operators of the attention half as a program runs them, beside the
products and the FFN block that were there before: a two-layer model (dense
projections, tree attention over the paged cache, the MoE block, an LM head)
decodes token by token, and again with trees of drafted tokens that are
verified and kept, eagerly and as one replayed graph.  The same tokens have to
come out, and the same cache."""
import gc

import numpy as np
import pytest

import kv_ref
import tie_amd
from conftest import synth_layer
from tie_amd import synth

pytestmark = pytest.mark.gpu

D, HEADS, KVH, HD, VOCAB, LAYERS, K, EPS = 256, 8, 2, 64, 512, 2, 2, 1e-6
PROMPTS, STEPS = (70, 5), 26


@pytest.fixture(scope="module", autouse=True)
def device():
    import torch
    assert torch.cuda.is_available(), "GPU test without a GPU"
    tie_amd.init(0)
    yield
    tie_amd.shutdown()


class Net:
    def __init__(self, stream):
        import torch
        rng = np.random.default_rng(5)
        self.stream, self.raw = stream, stream.cuda_stream

        def matrix(rows, inn):
            return tie_amd.Matrix(synth.expert_tensor(rng, synth.BF16, 1, rows, inn), synth.BF16, rows, inn)

        def vector(n):
            return torch.from_numpy((1 + 0.2 * rng.standard_normal(n)).astype(np.float32)).cuda()

        self.embed = torch.from_numpy(rng.standard_normal((VOCAB, D)).astype(np.float32)).cuda()
        self.qkv = [matrix((HEADS + 2 * KVH) * HD, D) for _ in range(LAYERS)]
        self.o = [matrix(D, HEADS * HD) for _ in range(LAYERS)]
        self.ffn = [tie_amd.Layer.from_synth(synth_layer(91 + i, D, 256, 8, synth.Q4_K, synth.Q6_K, None)) for i in range(LAYERS)]
        self.norms = [[vector(n) for n in (D, HD, HD, D)] for _ in range(LAYERS)]
        self.final, self.head = vector(D), matrix(VOCAB, D)

    def close(self):
        for m in self.qkv + self.o + self.ffn + [self.head]:
            m.close()

    def norm(self, x, w):
        import torch
        return x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * w

    def forward(self, cache, seqs, tokens, pos=None, mask=None):
        """Logits of the sequences' tokens (on the net's stream)."""
        import torch
        n = seqs.n_tokens
        x = self.embed[tokens]
        for i in range(LAYERS):
            w = self.norms[i]
            h, qkv = self.norm(x, w[0]), torch.empty((n, (HEADS + 2 * KVH) * HD), device="cuda")
            self.qkv[i].mat_mat(h, n, qkv, stream=self.raw)
            q, k, v = (qkv[:, a * HD:b * HD] for a, b in ((0, HEADS), (HEADS, HEADS + KVH), (HEADS + KVH, HEADS + 2 * KVH)))
            cache.append(i, seqs, q, k, v, q, pos=pos, q_norm=w[1], k_norm=w[2], eps=EPS, stream=self.raw)
            out = torch.empty((n, HEADS * HD), device="cuda")
            cache.attention(i, seqs, q, out, HD ** -0.5, mask=mask, stream=self.raw)
            o = torch.empty((n, D), device="cuda")
            self.o[i].mat_mat(out, n, o, stream=self.raw)
            x = x + o
            self.ffn[i].forward_residual(x, w[3], EPS, n, K, flags=tie_amd.PATH_EXACT, stream=self.raw)
        h, logits = self.norm(x, self.final), torch.empty((n, VOCAB), device="cuda")
        self.head.mat_mat(h, n, logits, stream=self.raw)
        return logits


def ints(x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def new_cache(kind):
    """An empty cache for both sequences, the pages in an order of their own."""
    import torch
    need = [-(-(p + 4 * STEPS) // 64) for p in PROMPTS]
    n, shape = sum(need) + 1, (LAYERS, sum(need) + 1, KVH)
    ids = list(np.random.default_rng(6).permutation(n))
    table = np.full((2, max(need)), -1, np.int32)
    for b, c in enumerate(need):
        table[b, :c] = [ids.pop() for _ in range(c)]
    t = torch.float16 if kind == "f16" else torch.int8
    k, v = torch.zeros(shape + (64, HD), dtype=t, device="cuda"), torch.zeros(shape + (HD, 64), dtype=t, device="cuda")
    scales = () if kind == "f16" else tuple(torch.zeros(shape + (64,), device="cuda") for _ in range(2))
    return tie_amd.KVCache(k, v, *scales), torch.from_numpy(table).cuda()


def prompt(net, cache, pages):
    """Both prompts in one call; the first token of each, and the lengths."""
    rng = np.random.default_rng(7)
    text = ints(rng.integers(0, VOCAB, sum(PROMPTS)))
    first = ints([0, PROMPTS[0], sum(PROMPTS)])
    logits = net.forward(cache, tie_amd.KVSeqs(pages, ints([0, 0]), first, sum(PROMPTS)), text)
    return logits[[PROMPTS[0] - 1, sum(PROMPTS) - 1]].argmax(1), ints(PROMPTS)


def token_by_token(net, kind):
    cache, pages = new_cache(kind)
    token, lens = prompt(net, cache, pages)
    out, gap = [token], np.inf
    for _ in range(STEPS):
        logits = net.forward(cache, tie_amd.KVSeqs(pages, lens), out[-1])
        best = logits.topk(2, 1).values
        gap = min(gap, float(((best[:, 0] - best[:, 1]) / logits.abs().amax(1)).min()))
        out.append(logits.argmax(1))
        lens = lens + 1
    return cache, pages, np.stack([t.cpu().numpy() for t in out], 1), gap


# Two trees: parents and depths of their nodes
PARENT = [[-1, 0, 0, 2, 2, 4, 1], [-1, 0, 1, 2]]
DEPTH = [[0, 1, 1, 2, 2, 3, 2], [0, 1, 2, 3]]
# the nodes that may hold the right token, by the round (the others hold a wrong one)
RIGHT = [[(2, 4, 5), (1, 6), (), (2, 3)], [(1,), (), (1, 2, 3), (1, 2)]]


def draft(tokens, at, b, turn):
    """Sequence b's tree behind token `at` of its text, and how many nodes are right."""
    right = RIGHT[b][turn % 4]
    out = [tokens[b][at]]
    for node in range(1, len(PARENT[b])):
        true = tokens[b][at + DEPTH[b][node]]
        out.append(true if node in right else (true + 1 + node) % VOCAB)
    return out, list(right)


@pytest.mark.parametrize("kind", ["f16", "i8"])
def test_tree_decoding_is_decoding(kind):
    import torch
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        net = Net(stream)
        cache0, pages0, want, gap = token_by_token(net, kind)
        # (the two runs' logits differ by F32 rounding, 1e-5 of the largest at most)
        assert gap > 1e-4, gap
        cache, pages = new_cache(kind)
        token, lens = prompt(net, cache, pages)
        assert token.tolist() == want[:, 0].tolist()

        n = sum(map(len, PARENT))
        first, parent = ints([0, len(PARENT[0]), n]), ints(sum(PARENT, []))
        depth, owner = ints(sum(DEPTH, [])), torch.tensor([0] * len(PARENT[0]) + [1] * len(PARENT[1]), device="cuda")
        sees = np.zeros((n, 1), np.int64)
        t = 0
        for p in PARENT:
            t0 = t
            for i, up in enumerate(p):
                sees[t, 0] = (sees[t0 + up, 0] if up >= 0 else 0) | 1 << i
                t += 1
        mask = torch.from_numpy(sees).cuda()
        tokens = torch.zeros(n, dtype=torch.int32, device="cuda")
        u = [torch.from_numpy(np.random.default_rng(8 + i).random(n, np.float32)).cuda() for i in range(2)]
        path, n_keep, following = torch.zeros((2, 5), dtype=torch.int32, device="cuda"), ints([0, 0]), ints([0, 0])
        seqs = tie_amd.KVSeqs(pages, lens, first, n)

        def step():
            logits = net.forward(cache, seqs, tokens, pos=lens[owner] + depth, mask=mask)
            tie_amd.verify_tree(logits, first, tokens, parent, u[0], u[1], path, n_keep, following, temperature=0.0,
                                max_children=2, stream=net.raw)
            cache.keep(seqs, path, n_keep, len_out=lens, stream=net.raw)
            return logits

        done, turn, graph = [0, 0], 0, None
        while max(done) + 4 < STEPS:
            trees = [draft(want, done[b], b, turn) for b in range(2)]
            tokens.copy_(ints(trees[0][0] + trees[1][0]))
            stream.synchronize()
            if turn == 3:
                graph = torch.cuda.CUDAGraph()
                with kv_ref.capture(graph, stream):
                    step()
            if turn < 3:
                logits = step()
                # the same logits, sampled: against the plain form
                p2, k2, f2 = torch.zeros_like(path), torch.zeros_like(n_keep), torch.zeros_like(following)
                tie_amd.verify_tree(logits, first, tokens, parent, u[0], u[1], p2, k2, f2, temperature=0.7, max_children=2,
                                    stream=net.raw)
                stream.synchronize()
                host = [x.cpu().numpy() for x in (logits, tokens, parent, u[0], u[1])]
                for b, (t0, t1) in enumerate(((0, len(PARENT[0])), (len(PARENT[0]), n))):
                    part = [x[t0:t1] for x in host]
                    ref_path, ref_next = kv_ref.verify(part[0], None, part[1], part[2], part[3], part[4], 0.7, 2, 5)[:2]
                    assert p2[b, :int(k2[b])].tolist() == list(ref_path)
                    assert int(f2[b]) == ref_next
            else:
                graph.replay()
                stream.synchronize()
            for b in range(2):
                right = [0] + trees[b][1]
                assert path[b].tolist() == right + [-1] * (5 - len(right)), (turn, b)
                assert int(n_keep[b]) == len(right)
                done[b] += len(right)
                assert int(following[b]) == want[b][done[b]], (turn, b)
            assert lens.tolist() == [PROMPTS[b] + done[b] for b in range(2)]
            turn += 1
        assert turn > 4  # (replayed more than once)

        # the caches: the first layer's rows are the same bits (they depend on
        # their token and position alone); the second's differ by what F32
        # rounding in the first layer's attention leaves (taken as 1e-4 of the
        # head's largest) and by a step of the type where that moves a rounding
        total = sum(PROMPTS) + sum(done)
        ends = ints([0, PROMPTS[0] + done[0], total])
        rows = []
        for c, p in ((cache0, pages0), (cache, pages)):
            r = [torch.empty((LAYERS, total, KVH, HD), device="cuda") for _ in range(2)]
            c.read(tie_amd.KVSeqs(p, ints([0, 0]), ends, total), r[0], r[1], 0, LAYERS, stream=net.raw)
            rows.append(r)
        stream.synchronize()
        for a, b in zip(*rows):
            assert torch.equal(a[0], b[0])
            top = a[1].abs().amax(-1, keepdim=True)
            step_of = a[1].abs() * 2.0 ** -10 if kind == "f16" else top / 127
            assert bool(((a[1] - b[1]).abs() <= step_of + 1e-4 * top).all())
        net.close()
        del graph
        gc.collect()
    torch.cuda.synchronize()
