"""The attention half of a layer for drafted tokens, as cases that can be timed and checked.

Five operators over one paged key/value cache: `append` (norm and rotation of
queries and keys for each head, quantised write of keys and values), `read`
(rows of the cache as F32), `attention` (of a tree of drafted tokens, a causal
chunk or single tokens over the cache), `keep` (the accepted path's rows moved
down in every layer) and `verify` (the accepted path and the next token from the
target's logits and given random numbers).

The cache lies in pages of 64 rows: K [layer][page][kv head][64][head_dim], V
[layer][page][kv head][head_dim][64], f16, or int8 codes with an F32 scale for
each row and kv head.  A sequence has a row of the page table, `lens` committed
rows, and its tokens are rows first[b] .. first[b + 1] - 1 of the activations;
token j of a sequence is row lens[b] + j of its cache.

Head layouts are 32 query heads on 4 kv heads of 128, 64 on 4, and 32 on 8 of
64; the vocabulary of 151936 is that of the repository's LM head workload.
"""
import torch

own = False

HEADS = {"32x4x128": (32, 4, 128), "64x4x128": (64, 4, 128), "32x8x64": (32, 8, 64)}
EPS, THETA, ROWS = 1e-6, 1e6, 64
BYTES = {"f16": 2.0, "i8": 1.0}


def _case(op, **kw):
    return dict(dict(op=op), **kw)


def listed():
    return [
        # one decoded token enters the cache of a layer: the smallest call, latency counts
        _case("append", heads="32x4x128", type="i8", seqs=1, tokens=1, len=1003, name="append_decode"),
        # a prompt's chunk enters a 16-bit cache, starting inside a page
        _case("append", heads="32x4x128", type="f16", seqs=1, tokens=2048, len=37, name="append_prompt"),
        # a few rows of three sequences read back (a check, a moved session's tail)
        _case("read", heads="32x8x64", type="f16", seqs=3, tokens=37, len=129, name="read_tail"),
        # a long sequence read back
        _case("read", heads="32x4x128", type="i8", seqs=1, tokens=30001, len=0, name="read_long"),
        # one token of a short conversation
        _case("attention", heads="32x4x128", type="i8", seqs=1, tokens=1, len=500, branch=0, name="attn_decode_short"),
        # sixteen conversations of different lengths, a token each
        _case("attention", heads="32x4x128", type="i8", seqs=16, tokens=1, len=32000, branch=0, name="attn_decode_batch"),
        # a drafted tree of one sequence over a long cache, wide head groups
        _case("attention", heads="64x4x128", type="i8", seqs=1, tokens=26, len=8190, branch=3, name="attn_tree"),
        # a prompt's second chunk
        _case("attention", heads="32x4x128", type="f16", seqs=1, tokens=2048, len=1100, branch=0, name="attn_prompt"),
        # the accepted path of one sequence moved in all layers
        _case("keep", heads="32x4x128", type="i8", seqs=1, tokens=26, len=1021, branch=3, layers=48, name="keep_one"),
        # of sixteen
        _case("keep", heads="32x4x128", type="f16", seqs=16, tokens=24, len=250, branch=2, layers=48, name="keep_batch"),
        # a chain of five drafted tokens proposed without probabilities (looked up in the prompt)
        _case("verify", vocab=32000, seqs=1, tokens=5, branch=1, draft=False, greedy=False, name="verify_chain"),
        # trees of eight sequences against the draft's distributions
        _case("verify", vocab=151936, seqs=8, tokens=13, branch=2, draft=True, greedy=False, name="verify_trees"),
    ]


def _spread(rng, lo, hi):
    """A whole number spread over [lo, hi] in its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["append", "read", "attention", "attention", "attention", "keep", "verify"])
    heads, kind = rng.choice(sorted(HEADS)), rng.choice(["f16", "i8"])
    if op == "append":
        seqs = _spread(rng, 1, 16)
        return _case(op, heads=heads, type=kind, seqs=seqs, tokens=_spread(rng, 1, 2048 // seqs), len=_spread(rng, 1, 4000) - 1)
    if op == "read":
        seqs = _spread(rng, 1, 16)
        return _case(op, heads=heads, type=kind, seqs=seqs, tokens=_spread(rng, 1, 30001 // seqs), len=_spread(rng, 1, 1000) - 1)
    if op == "attention":
        how = rng.choice(["token", "tree", "chunk"])
        if how == "chunk":
            tokens = _spread(rng, 33, 1500)
            return _case(op, heads=heads, type=kind, seqs=1, tokens=tokens, len=_spread(rng, 1, 2500) - 1, branch=0)
        seqs = _spread(rng, 1, 16)
        tokens = 1 if how == "token" else _spread(rng, 2, 48)
        return _case(op, heads=heads, type=kind, seqs=seqs, tokens=tokens, len=_spread(rng, 1, 32000 // (seqs if tokens > 1 else 1)) - 1,
                     branch=0 if tokens == 1 else rng.randint(1, 4))
    if op == "keep":
        return _case(op, heads=heads, type=kind, seqs=_spread(rng, 1, 16), tokens=_spread(rng, 2, 64), len=_spread(rng, 1, 300) - 1,
                     branch=rng.randint(1, 4), layers=_spread(rng, 1, 48))
    draft = rng.random() < 0.5
    return _case(op, vocab=_spread(rng, 1000, 151936), seqs=_spread(rng, 1, 8), tokens=_spread(rng, 1, 13), branch=rng.randint(1, 3),
                 draft=draft, greedy=not draft and rng.random() < 0.3)


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _sizes(case):
    """The sequences' committed rows and tokens: the first has the case's own, the others spread below it."""
    at = [1.0 if b == 0 else (b * 0.6180339887) % 1.0 for b in range(case["seqs"])]
    lens = [int(case.get("len", 0) * f) for f in at]
    counts = [max(1, int(round(case["tokens"] * max(0.25, f)))) for f in at]
    return lens, counts


def _parents(n, branch):
    """A tree whose nodes have `branch` children each (0, 1: a chain), in breadth-first order."""
    return [(j - 1) // max(1, branch) for j in range(n)]  # the root: -1


def _tree(case):
    _, counts = _sizes(case)
    return [p for n in counts for p in _parents(n, case["branch"])]


def _table(g, lens, counts):
    need = [-(-(n + c) // ROWS) for n, c in zip(lens, counts)]
    pages = torch.randperm(sum(need) + 1, generator=g, device="cuda").int()
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = pages[at: at + n]
        at += n
    return table, sum(need) + 1


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _first(counts):
    first = [0]
    for n in counts:
        first.append(first[-1] + n)
    return first


def _cache(case, g, n_pages, layers):
    """A cache of normal rows: keys of about unit size after their norm, values below that."""
    _, kvh, hd = HEADS[case["heads"]]
    c = {}
    for name, shape, size in (("k", (ROWS, hd), 1.0), ("v", (hd, ROWS), 0.4)):
        if case["type"] == "f16":
            c[name] = torch.empty(layers, n_pages, kvh, *shape, dtype=torch.float16, device="cuda").normal_(0.0, size, generator=g)
        else:
            full = torch.empty(layers, n_pages, kvh, *shape, dtype=torch.float16, device="cuda").normal_(0.0, 38.0, generator=g)
            c[name] = full.round_().clamp_(-127.0, 127.0).to(torch.int8)
            del full
            c[name + "_scale"] = (torch.rand(layers, n_pages, kvh, ROWS, generator=g, device="cuda") + 0.5) * (size / 38.0)
    return c


def _cache_inputs(case, seed):
    g = _gen(seed)
    H, kvh, hd = HEADS[case["heads"]]
    lens, counts = _sizes(case)
    T = sum(counts)
    table, n_pages = _table(g, lens, counts)
    s = dict(case=case, table=table, lens=_int(lens), first=_int(_first(counts)), T=T, H=H, kvh=kvh, hd=hd)
    s["cache"] = _cache(case, g, n_pages, case.get("layers", 1))
    if case["op"] == "append":
        # the three projections' rows from one product
        s["qkv"] = _normal(g, T, (H + 2 * kvh) * hd)
        s["q_norm"], s["k_norm"] = 1.0 + 0.1 * _normal(g, hd), 1.0 + 0.1 * _normal(g, hd)
        s["pos"] = _int([n + j for n, c in zip(lens, counts) for j in range(c)])
        s["q_out"] = torch.zeros(T, H, hd, device="cuda")
    if case["op"] == "attention":
        s["q"], s["out"], s["mask"] = _normal(g, T, H, hd), torch.zeros(T, H, hd, device="cuda"), None
        if case["branch"]:
            rows = []
            for n in counts:
                up = _parents(n, case["branch"])
                bits = []
                for j in range(n):
                    bits.append((bits[up[j]] if up[j] >= 0 else 0) | 1 << j)
                rows += [b - (1 << 64) if b >> 63 else b for b in bits]
            s["mask"] = torch.tensor(rows, dtype=torch.int64, device="cuda").view(T, 1)
    if case["op"] == "keep":
        # each sequence accepts the path to one of its nodes
        pick = torch.rand(len(counts), generator=g, device="cuda").tolist()
        paths = []
        for n, u in zip(counts, pick):
            up, j, path = _parents(n, case["branch"]), int(u * n), []
            while j >= 0:
                path.append(j)
                j = up[j]
            paths.append(path[::-1])
        most = max(counts)
        s["path"] = _int([p + [-1] * (most - len(p)) for p in paths])
        s["n_keep"] = _int([len(p) for p in paths])
        s["len_out"] = torch.zeros_like(s["lens"])
    if case["op"] in ("append", "read", "keep"):
        shape = (case.get("layers", 1), T, kvh, hd)
        s["k_out"], s["v_out"] = torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda")
    return s


def _verify_inputs(case, seed):
    g = _gen(seed)
    _, counts = _sizes(case)
    N, V = sum(counts), case["vocab"]
    logits = _normal(g, N, V) * 2.5  # a few tokens hold most of the mass
    s = dict(case=case, logits=logits, first=_int(_first(counts)), parent=_int(_tree(case)), draft=None, N=N, V=V,
             temperature=0.0 if case["greedy"] else 0.8)
    draft = torch.softmax((logits + 0.7 * _normal(g, N, V)) / 0.8, 1)
    up = torch.tensor([f + max(p, 0) for f, n in zip(_first(counts), counts) for p in _parents(n, case["branch"])], device="cuda")
    cum = draft.double().cumsum(1)[up]
    u = torch.rand(N, 1, generator=g, device="cuda").double() * cum[:, -1:]
    s["tokens"] = torch.searchsorted(cum, u, right=True).clamp_(max=V - 1).view(N).int()
    if case["draft"]:
        s["draft"] = draft
    s["u_accept"], s["u_sample"] = torch.rand(N, generator=g, device="cuda"), torch.rand(N, generator=g, device="cuda")
    most = max(counts)
    s["path"] = torch.zeros(case["seqs"], most, dtype=torch.int32, device="cuda")
    s["n_keep"], s["next"] = (torch.zeros(case["seqs"], dtype=torch.int32, device="cuda") for _ in range(2))
    return s


def prepare(case, seed):
    s = _verify_inputs(case, seed) if case["op"] == "verify" else _cache_inputs(case, seed)
    if own:
        import tie_amd
        tie_amd.init(0)
        if case["op"] != "verify":  # the program's handles of the cache and of this step's sequences
            s["kv"] = tie_amd.KVCache(**s["cache"])
            s["seqs"] = tie_amd.KVSeqs(s["table"], s["lens"], s["first"], s["T"])
    return s


# ---------------------------------------------------------------- one pass
def run(state):
    case, op = state["case"], state["case"]["op"]
    if own:
        return _OWN[op](case, state)
    return _PLAIN[op](case, state)


def _own_append(case, s):
    H, kvh, hd, T = s["H"], s["kvh"], s["hd"], s["T"]
    q, k, v = s["qkv"][:, : H * hd], s["qkv"][:, H * hd: (H + kvh) * hd], s["qkv"][:, (H + kvh) * hd:]
    s["kv"].append(0, s["seqs"], q, k, v, s["q_out"], s["pos"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, theta=THETA)
    s["kv"].read(s["seqs"], s["k_out"], s["v_out"])
    return s["q_out"], s["k_out"], s["v_out"]


def _own_read(case, s):
    s["kv"].read(s["seqs"], s["k_out"], s["v_out"])
    return s["k_out"], s["v_out"]


def _own_attention(case, s):
    s["kv"].attention(0, s["seqs"], s["q"], s["out"], s["hd"] ** -0.5, mask=s["mask"])
    return s["out"]


def _own_keep(case, s):
    s["kv"].keep(s["seqs"], s["path"], s["n_keep"], s["len_out"])
    s["kv"].read(s["seqs"], s["k_out"], s["v_out"], n_layers=case["layers"])
    return s["len_out"], s["k_out"], s["v_out"]


def _own_verify(case, s):
    import tie_amd
    tie_amd.verify_tree(s["logits"], s["first"], s["tokens"], s["parent"], s["u_accept"], s["u_sample"], s["path"], s["n_keep"], s["next"],
                        temperature=s["temperature"], draft=s["draft"], max_children=max(1, case["branch"]))
    return s["path"], s["n_keep"], s["next"]


_OWN = dict(append=_own_append, read=_own_read, attention=_own_attention, keep=_own_keep, verify=_own_verify)


# ---------------------------------------------------------------- the plain forms
def _of_tokens(s):
    """(sequence, index in it) of each token row."""
    at = torch.arange(s["T"], device="cuda")
    b = torch.searchsorted(s["first"][1:].long(), at, right=True)
    return b, at - s["first"].long()[b]


def _places(s, row):
    """(page, row in it) of cache rows: row [T] of each token's sequence."""
    b, _ = _of_tokens(s)
    return s["table"].long()[b, row // ROWS], row % ROWS


def _read_rows(s, row):
    """K and V [layers][T][kvh][hd] F32 of a row for each token."""
    page, r = _places(s, row)
    c = s["cache"]
    k, v = c["k"][:, page, :, r], c["v"][:, page, :, :, r]  # [T][layers][kvh][hd]
    k, v = k.float(), v.float()
    if "k_scale" in c:
        k, v = k * c["k_scale"][:, page, :, r][..., None], v * c["v_scale"][:, page, :, r][..., None]
    return k.transpose(0, 1).contiguous(), v.transpose(0, 1).contiguous()


def _quantise(x):
    """int8 codes and the scale of the rows [..., hd]."""
    amax = x.abs().amax(-1, keepdim=True)
    scale = amax / torch.full_like(amax, 127.0)
    codes = torch.where(scale > 0, x / scale, torch.zeros_like(x))
    return codes.round().clamp(-127.0, 127.0).to(torch.int8), scale[..., 0]


def _write_rows(s, row, k, v):
    """k, v [T][kvh][hd] F32 into layer 0's rows."""
    page, r = _places(s, row)
    c = s["cache"]
    if "k_scale" in c:
        k, ks = _quantise(k)
        v, vs = _quantise(v)
        c["k_scale"][0, page, :, r], c["v_scale"][0, page, :, r] = ks, vs
    c["k"][0, page, :, r] = k.to(c["k"].dtype)
    c["v"][0, page, :, :, r] = v.to(c["v"].dtype)


def _norm_rotate(x, w, pos):
    """Norm of each head and rotation, in 64 bits: a quantised key next to a border falls on one side."""
    x, hd = x.double(), x.shape[-1]
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()
    freq = torch.pow(THETA, torch.arange(hd // 2, device="cuda", dtype=torch.float64) * (-2.0 / hd))
    angle = (pos.double()[:, None] * freq)[:, None]
    c, sn = torch.cos(angle), torch.sin(angle)
    a, b = x[..., : hd // 2], x[..., hd // 2:]
    return torch.cat([a * c - b * sn, b * c + a * sn], -1).float()


def _plain_append(case, s):
    T, H, kvh, hd = s["T"], s["H"], s["kvh"], s["hd"]
    x = s["qkv"].view(T, H + 2 * kvh, hd)
    _, j = _of_tokens(s)
    row = s["lens"].long()[_of_tokens(s)[0]] + j
    _write_rows(s, row, _norm_rotate(x[:, H: H + kvh], s["k_norm"], s["pos"]), x[:, H + kvh:])
    return (_norm_rotate(x[:, :H], s["q_norm"], s["pos"]), *_read_rows(s, row))


def _plain_read(case, s):
    b, j = _of_tokens(s)
    return _read_rows(s, s["lens"].long()[b] + j)


def _plain_attention(case, s):
    H, kvh, hd, B = s["H"], s["kvh"], s["hd"], case["seqs"]
    c, table = s["cache"], s["table"].long().clamp(min=0)
    L = table.shape[1] * ROWS
    b, j = _of_tokens(s)
    n = max(_sizes(case)[1])
    # every sequence padded to the longest: [B][kvh][...]
    k, v = c["k"][0][table].float(), c["v"][0][table].float()
    if "k_scale" in c:
        k, v = k * c["k_scale"][0][table][..., None], v * c["v_scale"][0][table][..., None, :]
    k = k.permute(0, 2, 1, 3, 4).reshape(B, kvh, L, hd)
    v = v.permute(0, 2, 1, 4, 3).reshape(B, kvh, L, hd)
    q = torch.zeros(B, n, H, hd, device="cuda")
    q[b, j] = s["q"]
    q = q.view(B, n, kvh, H // kvh, hd).transpose(1, 2).reshape(B, kvh, n * (H // kvh), hd)
    z = torch.matmul(q, k.transpose(2, 3)) * hd ** -0.5
    key, lens = torch.arange(L, device="cuda"), s["lens"].long()
    node = key - lens[:, None]  # [B][L]: the tree's node that a row holds
    if s["mask"] is None:
        sees = node[:, None] <= torch.arange(n, device="cuda")[:, None]
    else:
        bits = torch.zeros(B, n, dtype=torch.int64, device="cuda")
        bits[b, j] = s["mask"][:, 0]
        sees = (node < 0)[:, None] | ((bits[:, :, None] >> node.clamp(0, 63)[:, None] & 1) == 1) & (node < 64)[:, None]
    z = z.view(B, kvh, n, H // kvh, L).masked_fill_(~sees[:, None, :, None], float("-inf"))
    top = z.amax(-1, keepdim=True)
    e = torch.exp_(z.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(B, kvh, n * (H // kvh), L), v).view(B, kvh, n, H // kvh, hd)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.transpose(1, 2).reshape(B, n, H, hd)[b, j]


def _plain_keep(case, s):
    b, j = _of_tokens(s)
    lens, kept = s["lens"].long(), s["n_keep"].long()[b]
    from_row = lens[b] + torch.where(j < kept, s["path"].long()[b, j], j)
    page, r = _places(s, from_row)
    to_page, to_r = _places(s, lens[b] + j)
    c = s["cache"]
    for name in c:
        if name == "v":
            c[name][:, to_page, :, :, to_r] = c[name][:, page, :, :, r]
        else:
            c[name][:, to_page, :, to_r] = c[name][:, page, :, r]
    return ((lens + s["n_keep"]).int(), *_read_rows(s, lens[b] + j))


def _plain_verify(case, s):
    N, V, B = s["N"], s["V"], case["seqs"]
    first, parent, tokens = s["first"].long(), s["parent"].long(), s["tokens"].long()
    at, all_tokens = torch.arange(N, device="cuda"), torch.arange(V, device="cuda")
    base = first[torch.searchsorted(first[1:], at, right=True)]
    up = torch.where(parent >= 0, base + parent, torch.full_like(parent, -1))
    logits = s["logits"]
    if case["greedy"]:
        best = torch.where(logits == logits.amax(1, keepdim=True), all_tokens, V).amin(1, keepdim=True)
        p = (all_tokens == best).double()
    else:
        z = logits.double() / s["temperature"]
        p = torch.exp_(z.sub_(z.amax(1, keepdim=True)))
        p /= p.sum(1, keepdim=True)
    # a node's place among its siblings, and each node's children by place
    place = ((up[:, None] == up[None, :]) & (at[None, :] < at[:, None])).sum(1)
    C = max(1, case["branch"])
    child = torch.full((N + 1, C + 1), -1, dtype=torch.int64, device="cuda")
    child[torch.where(up >= 0, up, N), place.clamp(max=C)] = at
    child = child[:N, :C]
    taken = torch.full((N,), -1, dtype=torch.int64, device="cuda")
    c, M, w = torch.zeros(N, 1, device="cuda").double(), torch.ones(N, 1, device="cuda").double(), p
    q = s["draft"].double() if s["draft"] is not None else None
    for i in range(C):
        kid = child[:, i].clamp(min=0)
        x = tokens[kid][:, None]
        wx = w.gather(1, x)
        chance = s["u_accept"].double()[kid][:, None] * M
        yes = (chance * q.gather(1, x) < wx) if q is not None else chance < wx
        trying = (child[:, i: i + 1] >= 0) & (taken[:, None] < 0)
        taken = torch.where((trying & yes)[:, 0], kid, taken)
        no = trying & ~yes
        if q is not None:
            c = torch.where(no, c + M, c)
            w = torch.where(no, (p - c * q).clamp_(min=0.0), w)
        else:
            w = torch.where(no & (all_tokens == x), torch.zeros_like(w), w)
        M = torch.where(no, w.sum(1, keepdim=True), M)
    # the path, as deep as the outputs go; its last node's residual gives the next token
    cur, path, on = first[:-1].clone(), torch.full_like(s["path"], -1), torch.ones(B, dtype=torch.bool, device="cuda")
    last = cur
    for i in range(path.shape[1]):
        path[:, i] = torch.where(on, cur - first[:-1], torch.full_like(cur, -1)).int()
        last = torch.where(on, cur, last)
        step = taken[cur]
        on = on & (step >= 0)
        cur = torch.where(on, step, cur)
    cut = taken[last] >= 0  # the outputs' depth ended the path: the last node counts as a leaf
    w = torch.where((cut[:, None] | (M[last] <= 0)), p[last], w[last])
    cum = w.cumsum(1)
    over = cum > s["u_sample"].double()[last][:, None] * cum[:, -1:]
    nxt = torch.where(over, all_tokens, V).amin(1).clamp(max=V - 1)
    return path, (path >= 0).sum(1).int(), nxt.int()


_PLAIN = dict(append=_plain_append, read=_plain_read, attention=_plain_attention, keep=_plain_keep, verify=_plain_verify)


# ---------------------------------------------------------------- the least work
def work(case):
    lens, counts = _sizes(case)
    T = sum(counts)
    if case["op"] == "verify":
        return {"bytes": 4.0 * T * case["vocab"] * (2 if case["draft"] else 1), "flops": 3.0 * T * case["vocab"]}
    H, kvh, hd = HEADS[case["heads"]]
    row = 2.0 * kvh * (hd * BYTES[case["type"]] + (4.0 if case["type"] == "i8" else 0.0))  # one cache row, K and V
    full = 2.0 * kvh * hd * 4.0
    if case["op"] == "append":
        return {"bytes": T * (2 * 4.0 * H * hd + full + row + full), "flops": 10.0 * T * (H + kvh) * hd}
    if case["op"] == "read":
        return {"bytes": T * (row + full), "flops": 2.0 * T * kvh * hd}
    if case["op"] == "keep":
        return {"bytes": case["layers"] * T * (row + full), "flops": 2.0 * case["layers"] * T * kvh * hd}
    pairs = 0.0
    for n, c in zip(lens, counts):
        pairs += c * n + sum(_depths(c, case["branch"]))
    return {"bytes": sum(n + c for n, c in zip(lens, counts)) * row + 8.0 * T * H * hd, "flops": 4.0 * H * hd * pairs}


def _depths(n, branch):
    deep = []
    for p in _parents(n, branch):
        deep.append(1 + (deep[p] if p >= 0 else 0))
    return deep


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["op"]](case, s)


def _seq_rows(s, b, layer, start, stop):
    """Rows start .. stop - 1 of sequence b in float64, [rows][kvh][hd], page by page."""
    c, ids = s["cache"], s["table"][b, start // ROWS: -(-stop // ROWS)].tolist()
    k = torch.cat([c["k"][layer, i].double().transpose(0, 1) for i in ids])
    v = torch.cat([c["v"][layer, i].double().permute(2, 0, 1) for i in ids])
    if "k_scale" in c:
        k = k * torch.cat([c["k_scale"][layer, i].double().T for i in ids])[..., None]
        v = v * torch.cat([c["v_scale"][layer, i].double().T for i in ids])[..., None]
    cut = slice(start % ROWS, start % ROWS + stop - start)
    return k[cut], v[cut]


def _held(case, x):
    """What the cache holds for the rows x [..., hd] (F32 values)."""
    if case["type"] == "f16":
        return x.half().double()
    scale = (x.double().abs().amax(-1, keepdim=True) / 127.0).float()
    return (x.double() / scale.double()).float().double().round().clamp(-127, 127) * scale.double()


def _exact_append(case, s):
    T, H, kvh, hd = s["T"], s["H"], s["kvh"], s["hd"]
    q, k, v = s["qkv"].view(T, -1, hd).split([H, kvh, kvh], 1)
    turn = torch.exp(torch.arange(0, hd, 2, device="cuda").double() / -hd * torch.log(torch.tensor(THETA, device="cuda").double()))
    unit = torch.polar(torch.ones(T, 1, hd // 2, device="cuda").double(), s["pos"].double().view(T, 1, 1) * turn)

    def rotated(x, w):
        x = x.double()
        x = x / (x.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt() * w.double()
        z = torch.complex(x[..., : hd // 2].contiguous(), x[..., hd // 2:].contiguous()) * unit
        return torch.cat([z.real, z.imag], -1)

    return rotated(q, s["q_norm"]), _held(case, rotated(k, s["k_norm"]).float())[None], _held(case, v.contiguous())[None]


def _exact_read(case, s):
    lens, counts = _sizes(case)
    rows = [_seq_rows(s, b, 0, n, n + c) for b, (n, c) in enumerate(zip(lens, counts))]
    return torch.cat([r[0] for r in rows])[None], torch.cat([r[1] for r in rows])[None]


def _exact_attention(case, s):
    H, kvh, hd = s["H"], s["kvh"], s["hd"]
    lens, counts = _sizes(case)
    out, at = [], 0
    for b, (n, c) in enumerate(zip(lens, counts)):
        k, v = _seq_rows(s, b, 0, 0, n + c)
        up, sees = _parents(c, case["branch"]), torch.zeros(c, n + c, dtype=torch.bool)
        sees[:, :n] = True
        for i in range(c):
            if up[i] >= 0:
                sees[i, n:] = sees[up[i], n:]
            sees[i, n + i] = True
        sees = sees.cuda()
        heads = []
        for h in range(H):
            z = s["q"][at: at + c, h].double() @ k[:, h // (H // kvh)].T / hd ** 0.5
            heads.append(torch.softmax(torch.where(sees, z, -torch.inf), 1) @ v[:, h // (H // kvh)])
        out.append(torch.stack(heads, 1))
        at += c
    return torch.cat(out)


def _exact_keep(case, s):
    lens, counts = _sizes(case)
    path, kept = s["path"].tolist(), s["n_keep"].tolist()
    ks, vs = [], []
    for layer in range(case["layers"]):
        for b, (n, c) in enumerate(zip(lens, counts)):
            k, v = _seq_rows(s, b, layer, n, n + c)
            source = path[b][: kept[b]] + list(range(kept[b], c))
            ks.append(k[source])
            vs.append(v[source])
    shape = (case["layers"], s["T"], s["kvh"], s["hd"])
    return None, torch.cat(ks).view(shape), torch.cat(vs).view(shape)


def _exact_verify(case, s):
    return None  # whole numbers


_EXACT = dict(append=_exact_append, read=_exact_read, attention=_exact_attention, keep=_exact_keep, verify=_exact_verify)
