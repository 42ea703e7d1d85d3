"""Calls around a long-running session, as cases that can be timed and checked.

Four operators beside the paged key/value cache of 64-row pages: `plan` (pages
handed out and taken back from request lengths, ranges of rows, positions and
cache slots of a step's tokens), `append` (norm, rotation by positions on several
axes and cache write), `window` (attention over a sliding window of the cache and
its first rows) and `logprobs` (log-probabilities of given tokens with rank,
entropy and the likeliest alternatives).

The cache: K [layer][page][kv head][64][head_dim], V [layer][page][kv
head][head_dim][64], f16, or int8 codes with an F32 scale for each row and kv
head.  A sequence has a row of the page table, `lens` committed rows, and token
rows first[b] .. first[b + 1] - 1; its token j is row lens[b] + j of its cache.
Free pages lie in a ring: state [2] holds the place of the first one and how
many there are.

Head layouts are 32 query heads on 4 kv heads of 128, 64 on 4, and 40 on 8 of
64; the vocabulary of 151936 is that of the repository's LM head workload.
"""
import torch

own = False

HEADS = {"32x4x128": (32, 4, 128), "64x4x128": (64, 4, 128), "40x8x64": (40, 8, 64)}
EPS, THETA, ROWS = 1e-6, 1e6, 64
BYTES = {"f16": 2.0, "i8": 1.0}


def _case(op, **kw):
    return dict(dict(op=op), **kw)


def listed():
    return [
        # a few conversations decode on: the smallest call, latency counts
        _case("plan", seqs=5, columns=64, len=1500, mode="decode", window=0, sinks=0, rows=8, name="plan_decode"),
        # a server's step: tokens of many conversations behind a window, some that end, some prompts; the table is rebuilt
        _case("plan", seqs=257, columns=512, len=30000, mode="mixed", window=4096, sinks=4, rows=12000, name="plan_step"),
        # a large batch of prompts begins
        _case("plan", seqs=1024, columns=300, len=9000, mode="prompts", window=0, sinks=0, rows=65536, name="plan_prompts"),
        # one token behind an image enters an int8 cache: latency
        _case("append", heads="32x4x128", type="i8", seqs=1, tokens=1, len=1211, order="mixed", name="axes_decode"),
        # a prompt with images enters a 16-bit cache, starting inside a page
        _case("append", heads="40x8x64", type="f16", seqs=3, tokens=4001, len=45, order="blocks", name="axes_images"),
        # one token over a narrow window of a short conversation: latency
        _case("window", heads="32x4x128", type="i8", seqs=1, tokens=1, len=900, window=512, sinks=4, branch=0, name="window_decode"),
        # a decoding batch of long conversations
        _case("window", heads="40x8x64", type="f16", seqs=61, tokens=1, len=30000, window=4096, sinks=4, branch=0, name="window_batch"),
        # a drafted tree over a long cache
        _case("window", heads="64x4x128", type="i8", seqs=4, tokens=26, len=8190, window=1000, sinks=64, branch=3, name="window_tree"),
        # a long prompt's later chunk
        _case("window", heads="32x4x128", type="f16", seqs=1, tokens=4096, len=5003, window=1024, sinks=0, branch=0,
              name="window_chunk"),
        # one sampled token's log-probability with five alternatives
        _case("logprobs", vocab=32000, rows=1, top=5, allowed=1.0, name="logprobs_token"),
        # a decoding batch under a grammar that allows some tokens
        _case("logprobs", vocab=151936, rows=61, top=20, allowed=0.4, name="logprobs_batch"),
        # a prompt is scored
        _case("logprobs", vocab=151936, rows=2047, top=20, allowed=1.0, name="logprobs_prompt"),
    ]


def _spread(rng, lo, hi):
    """A whole number spread over [lo, hi] in its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["plan", "append", "window", "window", "window", "logprobs", "logprobs"])
    heads, kind = rng.choice(sorted(HEADS)), rng.choice(["f16", "i8"])
    if op == "plan":
        columns = _spread(rng, 8, 512)
        mode = rng.choice(["decode", "mixed", "prompts"])
        return _case(op, seqs=_spread(rng, 1, 1024), columns=columns, len=columns * ROWS // 2, mode=mode,
                     window=rng.choice([0, _spread(rng, 1, columns * 16)]), sinks=rng.choice([0, 4, 100]), rows=_spread(rng, 1, 65536))
    if op == "append":
        seqs = _spread(rng, 1, 16)
        return _case(op, heads=heads, type=kind, seqs=seqs, tokens=_spread(rng, 1, 8192 // seqs), len=_spread(rng, 1, 4000) - 1,
                     order=rng.choice(["blocks", "mixed"]))
    if op == "window":
        how, window = rng.choice(["token", "tree", "chunk"]), _spread(rng, 1, 4096)
        sinks = rng.choice([0, _spread(rng, 1, 200)])
        if how == "chunk":
            seqs = _spread(rng, 1, 4)
            most = min(3000, 1900000 // (window + sinks)) // seqs  # (wide windows: fewer tokens)
            return _case(op, heads=heads, type=kind, seqs=seqs, tokens=_spread(rng, 33, most), len=_spread(rng, 1, 8000) - 1,
                         window=window, sinks=sinks, branch=0)
        seqs = _spread(rng, 1, 64 if how == "token" else 8)
        tokens = 1 if how == "token" else _spread(rng, 2, 48)
        return _case(op, heads=heads, type=kind, seqs=seqs, tokens=tokens, len=_spread(rng, 1, 30000 if how == "token" else 8000) - 1,
                     window=window, sinks=sinks, branch=0 if tokens == 1 else rng.randint(1, 4))
    vocab = _spread(rng, 1000, 151936)
    return _case(op, vocab=vocab, rows=_spread(rng, 1, 2047), top=rng.randint(0, 32), allowed=rng.choice([1.0, 1.0, 0.3]))


# ---------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _sizes(case):
    """The sequences' committed rows and tokens: the first has the case's own, the others spread below it."""
    at = [1.0 if b == 0 else (b * 0.6180339887) % 1.0 for b in range(case["seqs"])]
    lens = [int(case["len"] * f) for f in at]
    counts = [max(1, int(round(case["tokens"] * max(0.25, f)))) for f in at]
    return lens, counts


def _parents(n, branch):
    """A tree whose nodes have `branch` children each, in breadth-first order (the root: -1)."""
    return [(j - 1) // max(1, branch) for j in range(n)]


def _depths(n, branch):
    deep = []
    for p in _parents(n, branch):
        deep.append(deep[p] + 1 if p >= 0 else 0)
    return deep


def _first(counts):
    first = [0]
    for n in counts:
        first.append(first[-1] + n)
    return first


def _table(g, lens, counts):
    need = [-(-(n + c) // ROWS) for n, c in zip(lens, counts)]
    pages = torch.randperm(sum(need) + 1, generator=g, device="cuda").int()
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = pages[at: at + n]
        at += n
    return table, sum(need) + 1


def _cache(case, g, n_pages):
    """One layer of normal rows: keys of about unit size after their norm, values below that."""
    _, kvh, hd = HEADS[case["heads"]]
    c = {}
    for name, shape, size in (("k", (ROWS, hd), 1.0), ("v", (hd, ROWS), 0.4)):
        if case["type"] == "f16":
            c[name] = torch.empty(1, n_pages, kvh, *shape, dtype=torch.float16, device="cuda").normal_(0.0, size, generator=g)
        else:
            full = torch.empty(1, n_pages, kvh, *shape, dtype=torch.float16, device="cuda").normal_(0.0, 38.0, generator=g)
            c[name] = full.round_().clamp_(-127.0, 127.0).to(torch.int8)
            c[name + "_scale"] = (torch.rand(1, n_pages, kvh, ROWS, generator=g, device="cuda") + 0.5) * (size / 38.0)
    return c


def _axes(case):
    """The axis (time, height, width) of each pair of a head: 3/8, 5/16 and 5/16 of them, in blocks or in turn."""
    half = HEADS[case["heads"]][2] // 2
    n = [half - 2 * (half * 5 // 16), half * 5 // 16, half * 5 // 16]
    if case["order"] == "blocks":
        return [0] * n[0] + [1] * n[1] + [2] * n[2]
    return [i % 3 if i < 3 * n[1] else 0 for i in range(half)]


def _grid_positions(count, start):
    """Positions on three axes of `count` tokens: texts of 37 between images of 24 x 36 patches."""
    out, at = [], start
    while len(out) < count:
        out += [(at + i,) * 3 for i in range(37)]
        at += 37
        out += [(at, at + y, at + x) for y in range(24) for x in range(36)]
        at += 36
    return out[:count]


def _cache_inputs(case, seed):
    g = _gen(seed)
    H, kvh, hd = HEADS[case["heads"]]
    lens, counts = _sizes(case)
    T = sum(counts)
    table, n_pages = _table(g, lens, counts)
    s = dict(case=case, table=table, lens=_int(lens), first=_int(_first(counts)), T=T, H=H, kvh=kvh, hd=hd)
    s["cache"] = _cache(case, g, n_pages)
    if case["op"] == "append":
        # the three projections' rows from one product
        s["qkv"] = _normal(g, T, (H + 2 * kvh) * hd)
        s["q_norm"], s["k_norm"] = 1.0 + 0.1 * _normal(g, hd), 1.0 + 0.1 * _normal(g, hd)
        if case["tokens"] == 1:  # text behind an image: one position on all axes, below the cache's row
            points = [(n // 2 + 3,) * 3 for n in lens]
        else:
            points = [p for n, c in zip(lens, counts) for p in _grid_positions(c, n)]
        s["pos"] = _int(points).T.contiguous()
        s["axes"] = _axes(case)
        s["q_out"] = torch.zeros(T, H, hd, device="cuda")
        s["k_out"], s["v_out"] = (torch.zeros(1, T, kvh, hd, device="cuda") for _ in range(2))
        return s
    s["q"], s["out"], s["mask"], s["at"] = _normal(g, T, H, hd), torch.zeros(T, H, hd, device="cuda"), None, None
    if case["branch"]:
        rows = []
        for n in counts:
            up, bits = _parents(n, case["branch"]), []
            for j in range(n):
                bits.append((bits[up[j]] if up[j] >= 0 else 0) | 1 << j)
            rows += [b - (1 << 64) if b >> 63 else b for b in bits]
        s["mask"] = torch.tensor(rows, dtype=torch.int64, device="cuda").view(T, 1)
        s["at"] = _int([n + d for n, c in zip(lens, counts) for d in _depths(c, case["branch"])])
    return s


def _plan_inputs(case, seed):
    """Requests in the middle of a service: pages held up to their lengths (some with one ahead, left by drafts), those
    behind the window given back up to the last step's length."""
    g = _gen(seed)
    B, M, W, S = case["seqs"], case["columns"], case["window"], case["sinks"]
    most = min(case["len"], (M - 1) * ROWS)
    u, v, w = (torch.rand(B, generator=g, device="cuda", dtype=torch.float64) for _ in range(3))
    lens = (u * (most + 1)).long()
    room = M * ROWS - lens
    if case["mode"] == "decode":
        new = torch.ones_like(lens)
    elif case["mode"] == "prompts":
        lens = torch.where(v < 0.5, torch.zeros_like(lens), lens)
        new = (w * w * 1000).long()
    else:  # nearly all decode with a few drafts, some end, some bring a prompt
        new = torch.where(v < 0.95, 1 + (w * 8).long(), torch.where(v < 0.97, torch.full_like(lens, -1), (w * 2000).long()))
    new = torch.minimum(new, M * ROWS - lens)
    held = (lens + ROWS - 1) // ROWS + ((u * 1000) % 1.0 < 0.2).long()
    col = torch.arange(M, device="cuda")
    gone = (col >= (S + ROWS - 1) // ROWS) & ((col + 1) * ROWS <= (lens[:, None] - 1 - W + 1)) if W else torch.zeros(B, M, device="cuda").bool()
    has = (col < held[:, None]) & ~gone
    n_held = M * B  # (an upper end that needs no copy to the host)
    free = int(B * 4 + case["rows"] // ROWS)
    n_pages = n_held + free
    ids = torch.randperm(n_pages, generator=g, device="cuda").int()
    table = torch.where(has, ids[: B * M].view(B, M), torch.full((), -1, dtype=torch.int32, device="cuda")).contiguous()
    ring = torch.full((n_pages,), -1, dtype=torch.int32, device="cuda")
    head = n_pages - free // 3  # the ring's first free page lies near its end
    at = (head + torch.arange(free, device="cuda")) % n_pages
    ring[at] = ids[B * M:]
    N = case["rows"]
    return dict(case=case, table=table, lens=lens.int(), new=new.int(), ring=ring, state=_int([head, free]), n_pages=n_pages, N=N,
                table_out=torch.empty_like(table), first=torch.empty(B + 1, dtype=torch.int32, device="cuda"), state_out=_int([0, 0]),
                pos=torch.empty(N, dtype=torch.int32, device="cuda"), slot=torch.empty(N, dtype=torch.int32, device="cuda"))


def _logprobs_inputs(case, seed):
    g = _gen(seed)
    N, V, n = case["rows"], case["vocab"], case["top"]
    logits = _normal(g, N, V).mul_(2.5)  # a few tokens hold most of the mass
    if case["allowed"] < 1.0:
        logits.masked_fill_(torch.rand(N, V, generator=g, device="cuda") > case["allowed"], float("-inf"))
    tokens = torch.empty(N, dtype=torch.int32, device="cuda")
    for i in range(0, N, 256):  # sampled ones
        noise = torch.empty_like(logits[i: i + 256]).exponential_(generator=g).log_()
        tokens[i: i + 256] = torch.argmax(logits[i: i + 256] - noise, 1).int()
    s = dict(case=case, logits=logits, tokens=tokens)
    s["logprob"], s["entropy"] = (torch.zeros(N, device="cuda") for _ in range(2))
    s["rank"] = torch.zeros(N, dtype=torch.int32, device="cuda")
    s["top_tokens"], s["top_logprobs"] = torch.zeros(N, n, dtype=torch.int32, device="cuda"), torch.zeros(N, n, device="cuda")
    return s


def prepare(case, seed):
    s = {"plan": _plan_inputs, "logprobs": _logprobs_inputs}.get(case["op"], _cache_inputs)(case, seed)
    if own:
        import tie_amd
        tie_amd.init(0)
        if case["op"] == "plan":
            s["pool"] = tie_amd.KVPool(s["ring"], s["state"])
        elif case["op"] != "logprobs":  # the program's handles of the cache and of this step's sequences
            s["kv"] = tie_amd.KVCache(**s["cache"])
            s["seqs"] = tie_amd.KVSeqs(s["table"], s["lens"], s["first"], s["T"])
    return s


# ---------------------------------------------------------------- one pass
def run(state):
    case, op = state["case"], state["case"]["op"]
    if own:
        return _OWN[op](case, state)
    return _PLAIN[op](case, state)


def _own_plan(case, s):
    s["pool"].plan(s["table"], s["lens"], s["new"], s["table_out"], s["first"], pos=s["pos"], slot=s["slot"], state_out=s["state_out"],
                   window=case["window"], sinks=case["sinks"])
    return s["table_out"], s["first"], s["pos"], s["slot"], s["ring"], s["state_out"]


def _own_append(case, s):
    H, kvh, hd = s["H"], s["kvh"], s["hd"]
    q, k, v = s["qkv"][:, : H * hd], s["qkv"][:, H * hd: (H + kvh) * hd], s["qkv"][:, (H + kvh) * hd:]
    s["kv"].append_axes(0, s["seqs"], q, k, v, s["q_out"], s["pos"], s["axes"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS,
                        theta=THETA)
    if case["type"] == "f16":
        return s["q_out"], s["cache"]["k"], s["cache"]["v"]
    s["kv"].read(s["seqs"], s["k_out"], s["v_out"])  # codes as the values they stand for
    return s["q_out"], s["k_out"], s["v_out"]


def _own_window(case, s):
    s["kv"].window_attention(0, s["seqs"], s["q"], s["out"], s["hd"] ** -0.5, case["window"], sinks=case["sinks"], at=s["at"],
                             mask=s["mask"])
    return s["out"]


def _own_logprobs(case, s):
    import tie_amd
    tie_amd.token_logprobs(s["logits"], s["tokens"], s["logprob"], rank=s["rank"], entropy=s["entropy"], top_tokens=s["top_tokens"],
                           top_logprobs=s["top_logprobs"])
    return s["logprob"], s["rank"], s["entropy"], s["top_tokens"], s["top_logprobs"]


_OWN = dict(plan=_own_plan, append=_own_append, window=_own_window, logprobs=_own_logprobs)


# ---------------------------------------------------------------- the plain forms
def _plain_plan(case, s):
    M, N, P, W, S = case["columns"], s["N"], s["n_pages"], case["window"], case["sinks"]
    table, lens, new, head, free = s["table"].long(), s["lens"].long(), s["new"].long(), s["state"][0].long(), s["state"][1].long()
    col = torch.arange(M, device="cuda")
    there = (table >= 0) & (table < P)
    good = (lens >= 0) & (new >= 0) & (lens + new <= M * ROWS)
    want = torch.where(good, new, torch.zeros_like(new))
    # pages that the new rows lie on and that the table does not name
    fresh = (col >= (lens[:, None] + ROWS - 1) // ROWS) & (col < (lens[:, None] + want[:, None] + ROWS - 1) // ROWS) & ~there & (want > 0)[:, None]
    need = fresh.sum(1)
    served = (need.cumsum(0) <= free) & (want.cumsum(0) <= N)
    got = torch.where(served, want, torch.zeros_like(want))
    first = torch.cat([torch.zeros_like(got[:1]), got.cumsum(0)])
    fresh &= served[:, None]
    rank = fresh.view(-1).cumsum(0).view_as(fresh) - 1
    out = torch.where(fresh, s["ring"].long()[(head + rank.clamp(min=0)) % P], table)
    # pages of sequences that ended, and those that no later row sees
    away = there & (new < 0)[:, None]
    if W:
        away |= there & (col >= (S + ROWS - 1) // ROWS) & ((col + 1) * ROWS <= lens[:, None] - W + 1)
    place = away.view(-1).cumsum(0).view_as(away) - 1
    away &= place < P - free
    ring = torch.cat([s["ring"].long(), torch.zeros(1, dtype=torch.int64, device="cuda")])
    ring[torch.where(away, (head + free + place) % P, P).view(-1)] = table.view(-1)
    out = torch.where(away, torch.full_like(out, -1), out)
    state = torch.stack([(head + fresh.sum()) % P, free - fresh.sum() + away.sum()])
    t = torch.arange(N, device="cuda")
    b = torch.searchsorted(first[1:].contiguous(), t, right=True).clamp(max=len(got) - 1)
    row = lens[b] + t - first[b]
    on = t < first[-1]
    row = torch.where(on, row, torch.zeros_like(row))
    page = out[b, row // ROWS]
    slot = torch.where(on & (page >= 0) & (page < P), page * ROWS + row % ROWS, -1)
    pos = torch.where(on, row, torch.full_like(row, -1))
    return out.int(), first.int(), pos.int(), slot.int(), ring[:P].int(), state.int()


def _of_tokens(s):
    """(sequence, index in it) of each token row."""
    at = torch.arange(s["T"], device="cuda")
    b = torch.searchsorted(s["first"][1:].long(), at, right=True)
    return b, at - s["first"].long()[b]


def _norm_rotate(x, w, pos, axes):
    """Norm of each head and rotation, in 64 bits: a quantised key next to a border falls on one side."""
    x, hd = x.double(), x.shape[-1]
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()
    freq = torch.pow(THETA, torch.arange(hd // 2, device="cuda", dtype=torch.float64) * (-2.0 / hd))
    angle = (pos.double()[axes].T * freq)[:, None]
    c, sn = torch.cos(angle), torch.sin(angle)
    a, b = x[..., : hd // 2], x[..., hd // 2:]
    return torch.cat([a * c - b * sn, b * c + a * sn], -1).float()


def _quantise(x):
    """int8 codes and the scale of the rows [..., hd]."""
    amax = x.abs().amax(-1, keepdim=True)
    scale = amax / torch.full_like(amax, 127.0)
    codes = torch.where(scale > 0, x / scale, torch.zeros_like(x))
    return codes.round().clamp(-127.0, 127.0).to(torch.int8), scale[..., 0]


def _plain_append(case, s):
    T, H, kvh, hd, c = s["T"], s["H"], s["kvh"], s["hd"], s["cache"]
    x = s["qkv"].view(T, H + 2 * kvh, hd)
    b, j = _of_tokens(s)
    row = s["lens"].long()[b] + j
    page, r = s["table"].long()[b, row // ROWS], row % ROWS
    axes = torch.tensor(s["axes"], device="cuda")
    q, k, v = _norm_rotate(x[:, :H], s["q_norm"], s["pos"], axes), _norm_rotate(x[:, H: H + kvh], s["k_norm"], s["pos"], axes), x[:, H + kvh:]
    if case["type"] == "f16":
        c["k"][0, page, :, r], c["v"][0, page, :, :, r] = k.half(), v.half()
        return q, c["k"], c["v"]
    (kc, ks), (vc, vs) = _quantise(k), _quantise(v)
    c["k"][0, page, :, r], c["v"][0, page, :, :, r] = kc, vc
    c["k_scale"][0, page, :, r], c["v_scale"][0, page, :, r] = ks, vs
    return q, (kc.float() * ks[..., None])[None], (vc.float() * vs[..., None])[None]


def _plain_window(case, s):
    H, kvh, hd, B, W, S = s["H"], s["kvh"], s["hd"], case["seqs"], case["window"], case["sinks"]
    c, lens = s["cache"], s["lens"].long()
    sizes, counts = _sizes(case)
    n = max(counts)
    b, j = _of_tokens(s)
    stand = lens[b] + j if s["at"] is None else s["at"].long()  # the row that a token's window ends at
    # the rows that some token of the sequence sees: the first S, and from the root's window on
    low = (lens - W + 1).clamp(min=0)
    most = max(min(S, max(0, a - W + 1)) + a + c0 - max(0, a - W + 1) for a, c0 in zip(sizes, counts))
    i = torch.arange(most, device="cuda")
    heads = torch.minimum(low, torch.full_like(low, S))[:, None]
    row = torch.where(i < heads, i, low[:, None] + i - heads)  # [B][R]
    there = row < (lens + s["first"].long().diff())[:, None]
    row = row.clamp(max=s["table"].shape[1] * ROWS - 1)
    page, r = s["table"].long().gather(1, row // ROWS).clamp(min=0), row % ROWS
    k, v = c["k"][0][page, :, r].float(), c["v"][0][page, :, :, r].float()  # [B][R][kvh][hd]
    if "k_scale" in c:
        k, v = k * c["k_scale"][0][page, :, r][..., None], v * c["v_scale"][0][page, :, r][..., None]
    k, v = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
    q, at = torch.zeros(B, n, H, hd, device="cuda"), torch.zeros(B, n, dtype=torch.int64, device="cuda")
    q[b, j], at[b, j] = s["q"], stand
    q = q.view(B, n, kvh, H // kvh, hd).transpose(1, 2).reshape(B, kvh, n * (H // kvh), hd)
    node = row - lens[:, None]
    near = (row[:, None] < S) | (row[:, None] > at[:, :, None] - W)  # [B][n][R]
    if s["mask"] is None:
        sees = near & (node[:, None] <= torch.arange(n, device="cuda")[:, None])
    else:
        bits = torch.zeros(B, n, dtype=torch.int64, device="cuda")
        bits[b, j] = s["mask"][:, 0]
        sees = (near & (node < 0)[:, None]) | ((bits[:, :, None] >> node.clamp(0, 63)[:, None] & 1) == 1) & ((node >= 0) & (node < 64))[:, None]
    sees &= there[:, None]
    z = torch.matmul(q, k.transpose(2, 3).contiguous()) * hd ** -0.5
    z = z.view(B, kvh, n, H // kvh, most).masked_fill_(~sees[:, None, :, None], float("-inf"))
    top = z.amax(-1, keepdim=True)
    e = torch.exp_(z.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))))
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e.view(B, kvh, n * (H // kvh), most), v).view(B, kvh, n, H // kvh, hd)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.transpose(1, 2).reshape(B, n, H, hd)[b, j]


def _plain_logprobs(case, s):
    N, V, n = case["rows"], case["vocab"], case["top"]
    index, outs = torch.arange(V, device="cuda"), []
    for i in range(0, N, 256):
        l, tok = s["logits"][i: i + 256], s["tokens"][i: i + 256].long()[:, None]
        x = l - l.amax(1, keepdim=True)
        e = torch.exp(x)
        total = e.double().sum(1, keepdim=True)
        logz = torch.log(total)
        of = x.gather(1, tok).double() - logz
        entropy = logz - (torch.where(e > 0, x, torch.zeros_like(x)) * e).double().sum(1, keepdim=True) / total
        mine = l.gather(1, tok)
        rank = ((l > mine) | ((l == mine) & (index < tok))).sum(1)
        # larger values first, of equal ones the lowest index: as whole numbers
        bits = l.view(torch.int32).long()
        key = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * 2 ** 32 + (V - 1 - index)
        best = V - 1 - (torch.topk(key, n, 1).values & 0xffffffff) if n else key[:, :0]
        outs.append((of[:, 0].float(), rank.int(), entropy[:, 0].float(), best.int(), (x.gather(1, best).double() - logz).float()))
    return tuple(torch.cat(o) for o in zip(*outs))


_PLAIN = dict(plan=_plain_plan, append=_plain_append, window=_plain_window, logprobs=_plain_logprobs)


# ---------------------------------------------------------------- the least work
def work(case):
    if case["op"] == "plan":
        # the table read and written, lengths and counts read, ranges, positions and slots written
        return {"bytes": 8.0 * case["seqs"] * case["columns"] + 12.0 * case["seqs"] + 8.0 * case["rows"],
                "flops": 2.0 * case["seqs"] * case["columns"]}
    if case["op"] == "logprobs":
        return {"bytes": case["rows"] * (4.0 * case["vocab"] + 16.0 + 8.0 * case["top"]), "flops": 5.0 * case["rows"] * case["vocab"]}
    lens, counts = _sizes(case)
    T = sum(counts)
    H, kvh, hd = HEADS[case["heads"]]
    row = 2.0 * kvh * (hd * BYTES[case["type"]] + (4.0 if case["type"] == "i8" else 0.0))  # one cache row, K and V
    if case["op"] == "append":
        full = 2.0 * kvh * hd * 4.0
        return {"bytes": T * (8.0 * H * hd + full + row + 12.0 + (row + full if case["type"] == "i8" else 0.0)),
                "flops": 10.0 * T * (H + kvh) * hd}
    W, S, pairs, rows = case["window"], case["sinks"], 0.0, 0.0
    for n, c in zip(lens, counts):
        rows += c + n - max(0, n - W + 1) + min(S, max(0, n - W + 1))
        if case["branch"]:
            for d in _depths(c, case["branch"]):
                low = min(n, max(0, n + d - W + 1))
                pairs += n - low + min(S, low) + d + 1
        else:
            for i in range(c):
                low = max(0, n + i - W + 1)
                pairs += n + i + 1 - low + min(S, low)
    return {"bytes": rows * row + 8.0 * T * H * hd, "flops": 4.0 * H * hd * pairs}


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    return _EXACT[case["op"]](case, prepare(case, seed))


def _exact_plan(case, s):
    return None  # whole numbers


def _exact_append(case, s):
    T, H, kvh, hd, c = s["T"], s["H"], s["kvh"], s["hd"], s["cache"]
    q, k, v = s["qkv"].view(T, -1, hd).split([H, kvh, kvh], 1)
    turn = torch.exp(torch.arange(0, hd, 2, device="cuda").double() / -hd * torch.log(torch.tensor(THETA, device="cuda").double()))
    angle = torch.stack([s["pos"][a].double() * turn[i] for i, a in enumerate(s["axes"])], -1)[:, None]
    unit = torch.polar(torch.ones_like(angle), angle)

    def rotated(x, w):
        x = x.double()
        x = x / (x.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt() * w.double()
        z = torch.complex(x[..., : hd // 2].contiguous(), x[..., hd // 2:].contiguous()) * unit
        return torch.cat([z.real, z.imag], -1)

    def held(x):
        scale = (x.double().abs().amax(-1, keepdim=True) / 127.0).float()
        return (x.double() / scale.double()).float().double().round().clamp(-127, 127) * scale.double()

    q, k = rotated(q, s["q_norm"]), rotated(k, s["k_norm"]).float()
    if case["type"] == "i8":
        return q, held(k)[None], held(v.contiguous())[None]
    ck, cv = c["k"].double(), c["v"].double()
    lens, counts = _sizes(case)
    t = 0
    for b, (n, m) in enumerate(zip(lens, counts)):
        row = torch.arange(n, n + m, device="cuda")
        page = s["table"][b].long()[row // ROWS]
        ck[0, page, :, row % ROWS] = k[t: t + m].half().double()
        cv[0, page, :, :, row % ROWS] = v[t: t + m].half().double()
        t += m
    return q, ck, cv


def _exact_window(case, s):
    H, kvh, hd, W, S = s["H"], s["kvh"], s["hd"], case["window"], case["sinks"]
    lens, counts = _sizes(case)
    c, out, t = s["cache"], [], 0
    for b, (n, m) in enumerate(zip(lens, counts)):
        ids = s["table"][b, : -(-(n + m) // ROWS)].long()
        k = c["k"][0, ids].double().transpose(0, 1).reshape(kvh, -1, hd)
        v = c["v"][0, ids].double().permute(1, 0, 3, 2).reshape(kvh, -1, hd)
        if "k_scale" in c:
            k = k * c["k_scale"][0, ids].double().transpose(0, 1).reshape(kvh, -1, 1)
            v = v * c["v_scale"][0, ids].double().transpose(0, 1).reshape(kvh, -1, 1)
        k, v = k[:, : n + m], v[:, : n + m]
        rows = torch.arange(n + m)
        sees = torch.zeros(m, n + m, dtype=torch.bool)
        up, deep = _parents(m, case["branch"]), _depths(m, case["branch"])
        for i in range(m):
            if case["branch"]:
                sees[i] = (rows < n) & ((rows < S) | (n + deep[i] - rows < W))
                j = i
                while j >= 0:
                    sees[i, n + j] = True
                    j = up[j]
            else:
                sees[i] = (rows <= n + i) & ((rows < S) | (n + i - rows < W))
        sees = sees.cuda()
        heads = []
        for h in range(H):
            z = s["q"][t: t + m, h].double() @ k[h // (H // kvh)].T / hd ** 0.5
            heads.append(torch.softmax(torch.where(sees, z, -torch.inf), 1) @ v[h // (H // kvh)])
        out.append(torch.stack(heads, 1))
        t += m
    return torch.cat(out)


def _exact_logprobs(case, s):
    n, of, entropy, tops = case["top"], [], [], []
    for row, token in zip(s["logits"].split(64), s["tokens"].split(64)):
        lp = torch.log_softmax(row.double(), 1)
        of.append(lp.gather(1, token.long()[:, None])[:, 0])
        entropy.append(-(lp.exp() * lp.clamp(min=-1e300)).sum(1))
        tops.append(lp.topk(n, 1).values if n else lp[:, :0])
    return torch.cat(of), None, torch.cat(entropy), None, torch.cat(tops)


_EXACT = dict(plan=_exact_plan, append=_exact_append, window=_exact_window, logprobs=_exact_logprobs)
