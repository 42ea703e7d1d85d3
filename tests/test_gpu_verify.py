"""Acceptance of drafted tokens and the token after them, against a plain
64-bit form: whole numbers, so equal.  (The kernels' sums and the form's are
both in 64 bits; a random number within 1e-12 of a border would fall on either
side, and none of these does.)"""
import gc

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


def cuda(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


class Case:
    def __init__(self, seed, counts, V, draft, branch=2, peaked=2.5, parent=None, off=0.7):
        rng = np.random.default_rng(seed)
        self.counts, self.V = counts, V
        N = sum(counts)
        self.logits = (rng.standard_normal((N, V)) * peaked).astype(np.float32)
        d = self.logits + off * rng.standard_normal((N, V)).astype(np.float32)
        d = np.exp(d - d.max(1, keepdims=True))
        d = (d / d.sum(1, keepdims=True)).astype(np.float32)
        self.parent = np.concatenate([parent or [(j - 1) // branch for j in range(n)] for n in counts] + [[]]).astype(np.int32)
        self.first = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.tokens = np.zeros(N, np.int32)
        t0 = 0
        for n in counts:
            for j in range(n):
                row = d[t0 + max(0, self.parent[t0 + j])].astype(np.float64)
                self.tokens[t0 + j] = rng.choice(V, p=row / row.sum())
            t0 += n
        self.draft = d if draft else None
        self.ua, self.us = rng.random(N).astype(np.float32), rng.random(N).astype(np.float32)

    def want(self, temperature, kids, most):
        paths, n, nxt = np.full((len(self.counts), most), -1, np.int32), [], []
        for b in range(len(self.counts)):
            s = slice(self.first[b], self.first[b + 1])
            if s.stop == s.start:
                n.append(0)
                nxt.append(-1)
                continue
            p, x = kv_ref.verify(self.logits[s], self.draft[s] if self.draft is not None else None, self.tokens[s],
                                 self.parent[s], self.ua[s], self.us[s], temperature, kids, most)
            paths[b, : len(p)] = p
            n.append(len(p))
            nxt.append(x)
        return paths, np.array(n, np.int32), np.array(nxt, np.int32)

    def run(self, temperature, kids, most, stride=0, **kw):
        import torch
        N, V = self.logits.shape
        def rows(x):
            if x is None:
                return None
            b = torch.full((N, V + stride), float("nan"), device="cuda")
            b[:, :V] = cuda(x)
            return b[:, :V]
        B = len(self.counts)
        path = torch.full((B, most), 99, dtype=torch.int32, device="cuda")
        n, nxt = (torch.full((B,), 99, dtype=torch.int32, device="cuda") for _ in range(2))
        args = [rows(self.logits), cuda(self.first), cuda(self.tokens), cuda(self.parent), cuda(self.ua), cuda(self.us)]
        d = rows(self.draft)
        torch.cuda.synchronize()
        tie_amd.verify_tree(*args, path, n, nxt, temperature=temperature, draft=d, max_children=kids, **kw)
        torch.cuda.synchronize()
        return path.cpu().numpy(), n.cpu().numpy(), nxt.cpu().numpy()

    def check(self, temperature, kids, most, **kw):
        for g, w, what in zip(self.run(temperature, kids, most, **kw), self.want(temperature, kids, most), ("path", "n_keep", "next")):
            np.testing.assert_array_equal(g, w, what)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("temperature", [0.0, 0.3, 1.0, 5.0])
@pytest.mark.parametrize("V", [1, 2, 64, 4096, 4097, 32001])
def test_trees(draft, temperature, V):
    for seed in range(4):
        Case(seed, [5, 1, 13, 8], V, draft, branch=1 + seed % 3).check(temperature, 3, 13, stride=seed % 2 * 3)


@pytest.mark.parametrize("draft", [False, True])
def test_large_vocabulary(draft):
    Case(3, [9, 7], 151936, draft, branch=2).check(0.8, 2, 9)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("temperature", [0.0, 0.7])
def test_more_logits_than_run_at_once(draft, temperature):
    """(two blocks of 4096 logits to a workgroup; the last has one logit)"""
    Case(21, [13] * 14 + [1, 7], 5 * 4096 + 1, draft, branch=2).check(temperature, 2, 13)
    Case(22, [13] * 20, 4 * 4096, draft, branch=3).check(temperature, 3, 13, stride=1)


@pytest.mark.parametrize("draft", [False, True])
def test_more_rows_than_counters(draft):
    """(past 8192 rows and sequences the steps are launches of their own)"""
    c = Case(23, [9, 0, 8] * 520, 40, draft, branch=2, peaked=1.0)
    c.check(1.0, 2, 9)
    c.check(0.0, 2, 4)


@pytest.mark.parametrize("draft", [False, True])
def test_large_trees(draft):
    """(more nodes than the path's reader keeps in LDS)"""
    c = Case(24, [700, 511, 513], 64, draft, branch=3, peaked=1.0)
    for seed in range(3):
        c.ua[:] = np.random.default_rng(seed).random(len(c.ua)).astype(np.float32) ** 3
        c.check(1.0, 3, 12)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("first", [[0, 9, 5, 21], [0, 5, 9, 22], [-1, 5, 9, 21], [7, 3, 3, 3]])
def test_ranges_that_do_not_ascend(draft, first):
    """No paths, whatever the call before left in the workspace; rows behind
    the last sequence are nobody's.  Also where more sequences than a wave has
    lanes are searched."""
    import torch
    for more in (0, 70):
        c = Case(27, [5, 4, 12] + [1] * more, 3000, draft, branch=2, peaked=1.0)
        work = torch.full((tie_amd.verify_tree_work_bytes(3000, 21 + more, 2, draft),), 7, dtype=torch.uint8, device="cuda")
        work[:1 << 15] = 0
        good = c.first.copy()
        c.first[:4] = first
        if (np.diff(c.first) >= 0).all() and c.first[0] >= 0 and c.first[-1] <= 21 + more:
            continue  # (with the sequences behind them these ranges do ascend within the rows)
        path, n, nxt = c.run(1.0, 2, 6, work=work)
        assert (path == -1).all() and (n == 0).all() and (nxt == -1).all()
        c.first[:] = good
        c.check(1.0, 2, 6, work=work)
        c.first[3:] = 9
        if not more:
            c.counts = [5, 4, 0]
            c.check(1.0, 2, 6, work=work)


@pytest.mark.parametrize("kids", [1, 3])
def test_parents_that_are_no_nodes(kids):
    """A parent at or past its child, or below none, makes a node nobody's child."""
    c = Case(25, [6, 6], 50, True, branch=2, peaked=1.0)
    c.parent[3], c.parent[4], c.parent[8], c.parent[9] = 3, 5, -1, 100
    c.ua[:] = 0.0
    c.check(1.0, kids, 6)


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("temperature", [0.0, 1.0])
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
def test_rows_that_are_no_distribution(draft, temperature, value):
    """Logits of NaN or infinity alone: the sequence's outputs are tokens and
    nodes of it, and the other sequences' are what they were."""
    c = Case(26, [7, 7, 7], 9000, draft, branch=2)
    want = c.want(temperature, 2, 7)
    c.logits[7:14] = value
    path, n, nxt = c.run(temperature, 2, 7)
    for g, w in zip((path, n, nxt), want):
        np.testing.assert_array_equal(g[[0, 2]], w[[0, 2]])
    assert 1 <= n[1] <= 7 and 0 <= nxt[1] < 9000
    assert path[1, 0] == 0 and (np.diff(path[1, :n[1]]) > 0).all() and (path[1, n[1]:] == -1).all() and path[1].max() < 7


@pytest.mark.parametrize("draft", [False, True])
def test_many_children_and_cut_paths(draft):
    """16 children of one node, fewer tried than there are, paths cut at the
    outputs' depth, sequences of one node and of none, siblings of one token."""
    c = Case(11, [17, 0, 1, 40], 300, draft, branch=16)
    for kids in (1, 2, 16):
        for most in (1, 2, 5):
            c.check(0.9, kids, most)
    c = Case(12, [20, 20], 50, draft, branch=4, peaked=0.5)
    c.tokens[1:5] = c.tokens[1]
    c.tokens[21:25] = 7
    for s in range(6):
        c.ua[:] = np.random.default_rng(s).random(40).astype(np.float32)
        c.check(1.0, 4, 6)


@pytest.mark.parametrize("draft", [False, True])
def test_long_chains(draft):
    c = Case(13, [150, 70], 97, draft, branch=1, off=0.05)
    c.ua[:] *= 0.2  # most are taken
    c.check(1.0, 1, 200)
    c.ua[:] = 0.0  # all whose probability is not 0 are
    c.check(1.0, 1, 200)
    assert c.run(1.0, 1, 200)[1].tolist() == [150, 70]


@pytest.mark.parametrize("draft", [False, True])
def test_random_numbers_at_their_ends(draft):
    """0 and the largest below 1, logits of minus infinity, tokens that are
    none, equal largest logits."""
    c = Case(14, [7, 7, 7], 5000, draft, branch=2)
    c.logits[:, 100:4500] = -np.inf
    c.logits[3, :] = -np.inf
    c.logits[3, 4999] = 1.0
    c.logits[:, 7] = c.logits[:, 4700] = 20.0
    c.tokens[2], c.tokens[9] = -1, 5000
    for a in (0.0, 1 - 2.0 ** -24):
        for s in (0.0, 1 - 2.0 ** -24):
            c.ua[:], c.us[:] = a, s
            c.check(0.7, 2, 7)
            c.check(0.0, 2, 7)


def test_tokens_follow_the_target():
    """The first token after the root over many draws has the target's
    distribution, whatever the draft's: counts of 8 tokens in 20000 draws
    within 5 standard deviations."""
    V, n = 8, 20000
    rng = np.random.default_rng(15)
    logits = rng.standard_normal(V).astype(np.float32) * 1.5
    q = np.exp(rng.standard_normal(V) * 1.5)
    q = (q / q.sum()).astype(np.float32)
    c = Case(16, [3] * n, V, True, parent=[-1, 0, 0])
    c.logits[:], c.draft[:] = logits, q
    c.tokens[:] = rng.choice(V, size=3 * n, p=q.astype(np.float64) / q.astype(np.float64).sum())
    p = np.exp(logits.astype(np.float64))
    p /= p.sum()
    for draft in (c.draft, None):
        c.draft = draft
        path, kept, nxt = c.run(1.0, 2, 2)
        first = np.where(kept == 2, c.tokens[3 * np.arange(n) + np.clip(path[:, 1], 0, 2)], nxt)
        got = np.bincount(first, minlength=V)
        assert (np.abs(got - n * p) <= 5 * np.sqrt(n * p * (1 - p))).all(), (got, n * p)


@pytest.mark.parametrize("draft", [False, True])
def test_repeats_work_streams_and_graphs(draft):
    import torch
    c = Case(17, [9, 12], 20000, draft, branch=3)
    want = c.want(0.8, 3, 12)
    need = tie_amd.verify_tree_work_bytes(20000, 21, 3, draft)
    work = torch.zeros(need, dtype=torch.uint8, device="cuda")
    for kw in ({}, dict(work=work), dict(stream=torch.cuda.Stream().cuda_stream)):
        for g, w in zip(c.run(0.8, 3, 12, **kw), want):
            np.testing.assert_array_equal(g, w)
    with pytest.raises(tie_amd.TieError):
        c.run(0.8, 3, 12, work=work[: need - 16])
    args = [cuda(x) for x in (c.logits, c.first, c.tokens, c.parent, c.ua, c.us)]
    d = cuda(c.draft) if draft else None
    path, n, nxt = torch.zeros(2, 12, dtype=torch.int32, device="cuda"), *(torch.zeros(2, dtype=torch.int32, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with kv_ref.capture(g):
        tie_amd.verify_tree(*args, path, n, nxt, temperature=0.8, draft=d, max_children=3, work=work,
                            stream=torch.cuda.current_stream().cuda_stream)
    for rep in range(3):
        path.zero_()
        n.zero_()
        nxt.zero_()
        g.replay()
        torch.cuda.synchronize()
        for a, w in zip((path, n, nxt), want):
            np.testing.assert_array_equal(a.cpu().numpy(), w, str(rep))
    del g
    gc.collect()
