"""Plain 64-bit forms of the cache, the attention and the verification, and
small caches to test them on."""
import contextlib
import gc

import numpy as np

ROWS = 64


@contextlib.contextmanager
def capture(graph, stream=None):
    """torch.cuda.graph with the garbage collected before and none during the
    capture: a collection that meets another test's graph there would destroy
    it inside the capture, which ends the process."""
    import torch
    gc.collect()
    gc.disable()
    try:
        with torch.cuda.graph(graph, stream=stream):
            yield
    finally:
        gc.enable()


class Cache:
    """A paged cache on the CPU (numpy) with a copy on the GPU: random page
    order, every byte that no test writes NaN (f16), or codes with NaN scales."""

    def __init__(self, rng, kind, kvh, hd, lens, counts, layers=1, spare=2, fill=True, order=None):
        self.kind, self.kvh, self.hd, self.lens, self.counts = kind, kvh, hd, list(lens), list(counts)
        need = [-(-(n + c) // ROWS) for n, c in zip(lens, counts)]
        self.n_pages = sum(need) + spare
        ids = list(rng.permutation(self.n_pages)) if order is None else list(order)
        self.table = np.full((len(need), max(need + [1])), -1, np.int32)
        for b, n in enumerate(need):
            self.table[b, :n] = [ids.pop() for _ in range(n)]
        shape = (layers, self.n_pages, kvh)
        if kind == "f16":
            self.k = np.full(shape + (ROWS, hd), np.nan, np.float16)
            self.v = np.full(shape + (hd, ROWS), np.nan, np.float16)
            self.ks = self.vs = None
        else:
            self.k = np.full(shape + (ROWS, hd), 77, np.int8)
            self.v = np.full(shape + (hd, ROWS), -77, np.int8)
            self.ks, self.vs = np.full(shape + (ROWS,), np.nan, np.float32), np.full(shape + (ROWS,), np.nan, np.float32)
        if fill:
            for b in range(len(need)):
                for layer in range(layers):
                    n = lens[b] + counts[b]
                    self.set_rows(layer, b, 0, rng.standard_normal((n, kvh, hd)), 0.5 * rng.standard_normal((n, kvh, hd)))

    def place(self, b, row):
        return int(self.table[b, row // ROWS]), row % ROWS

    def set_rows(self, layer, b, start, k, v):
        for j in range(len(k)):
            p, r = self.place(b, start + j)
            if self.kind == "f16":
                self.k[layer, p, :, r], self.v[layer, p, :, :, r] = held_f16(k[j]), held_f16(v[j])
            else:
                self.k[layer, p, :, r], self.ks[layer, p, :, r] = codes(k[j])
                self.v[layer, p, :, :, r], self.vs[layer, p, :, r] = codes(v[j])

    def rows(self, layer, b, start, stop):
        """K and V [rows][kvh][hd] in float64."""
        k, v = np.zeros((stop - start, self.kvh, self.hd)), np.zeros((stop - start, self.kvh, self.hd))
        for j in range(stop - start):
            p, r = self.place(b, start + j)
            k[j], v[j] = self.k[layer, p, :, r], self.v[layer, p, :, :, r]
            if self.kind == "i8":
                k[j] *= self.ks[layer, p, :, r, None]
                v[j] *= self.vs[layer, p, :, r, None]
        return k, v

    def gpu(self):
        import torch
        self.dev = [torch.from_numpy(x).cuda() if x is not None else None for x in (self.k, self.v, self.ks, self.vs)]
        return after_torch(*self.dev)

    def seqs(self):
        import torch
        import tie_amd
        first = np.concatenate([[0], np.cumsum(self.counts)]).astype(np.int32)
        return tie_amd.KVSeqs(torch.from_numpy(self.table).cuda(), torch.tensor(self.lens, dtype=torch.int32).cuda(),
                              torch.from_numpy(first).cuda(), int(first[-1]))

    def back(self):
        """The GPU's cache, as numpy arrays."""
        return [x.cpu().numpy() if x is not None else None for x in self.dev]


def after_torch(*tensors):
    """A KVCache whose calls wait for torch's own stream, which the library's
    does not: the tests fill their buffers there."""
    import torch
    import tie_amd

    def wait():
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.synchronize()

    class AfterTorch(tie_amd.KVCache):
        def append(self, *a, **kw):
            wait()
            super().append(*a, **kw)

        def read(self, *a, **kw):
            wait()
            super().read(*a, **kw)

        def keep(self, *a, **kw):
            wait()
            super().keep(*a, **kw)

    return AfterTorch(*tensors)


def held_f16(x):
    return np.clip(np.asarray(x, np.float32), -65504, 65504).astype(np.float16)


def codes(x):
    """int8 codes and F32 scales of rows [..., hd]."""
    x = np.asarray(x, np.float32)
    scale = (np.abs(x).max(-1) / np.float32(127)).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(scale[..., None] > 0, x / scale[..., None], np.float32(0))
    return np.clip(np.rint(q), -127, 127).astype(np.int8), scale


def norm_rotate(x, w, pos, eps, theta):
    """x [T][heads][hd] in float64."""
    x = np.asarray(x, np.float64)
    hd = x.shape[-1]
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    a, b = x[..., : hd // 2], x[..., hd // 2:]
    ang = np.asarray(pos, np.float64)[:, None, None] * float(theta) ** (-2.0 * np.arange(hd // 2) / hd)
    return np.concatenate([a * np.cos(ang) - b * np.sin(ang), b * np.cos(ang) + a * np.sin(ang)], -1)


def attention(cache, layer, q, scale, sees):
    """q [T][H][hd]; sees(b, i, j): whether token i of sequence b sees its token
    j.  Returns the result and, for each element, a bound of a kernel's error
    that holds scores and weights to 22 bits and sums in 32 (see tolerance())."""
    T, H, hd = q.shape
    out, tol, t = np.zeros((T, H, hd)), np.zeros((T, H, hd)), 0
    group = H // cache.kvh
    for b, (n, c) in enumerate(zip(cache.lens, cache.counts)):
        k, v = cache.rows(layer, b, 0, n + c)
        for i in range(c):
            on = np.concatenate([np.ones(n, bool), np.array([sees(b, i, j) for j in range(c)], bool)])
            for h in range(H):
                kk, vv = k[on, h // group], v[on, h // group]
                if len(kk):
                    qq = q[t, h].astype(np.float64)
                    s = kk @ qq * scale
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[t, h] = w @ vv
                    tol[t, h] = tolerance(qq, kk, vv, w, scale)
            t += 1
    return out, tol


def tolerance(q, k, v, w, scale):
    """A score is off by at most the rounding of the query's two parts (2^-22),
    of 2 hd / 32 matrix-core sums and the factors behind them (2^-23 each, hd /
    16 + 4 of them) times sum |q||k|; the weights then by twice that and by
    exp2's and their own two parts' 2^-21; the sums over the rows by 2^-23 for
    each 16 rows and each joined part (32)."""
    terms = np.abs(k) @ np.abs(q) * abs(scale)
    ds = terms * (2.0 ** -22 + (len(q) / 16 + 4) * 2.0 ** -23)
    rel = 2 * (ds.max() if len(ds) else 0.0) + 2.0 ** -21 + (len(k) / 16 + 32) * 2.0 ** -23
    return rel * (w @ np.abs(v)) + 1e-30


def verify(logits, draft, tokens, parent, u_accept, u_sample, temperature, max_children, max_path):
    """One sequence's path and next token."""
    n, V = logits.shape
    z = logits.astype(np.float64)

    def p_of(t):
        if temperature == 0:
            p = np.zeros(V)
            p[int(np.argmax(z[t]))] = 1.0
            return p
        e = np.exp((z[t] - z[t].max()) / np.float64(np.float32(temperature)))
        return e / e.sum()

    def pick(w, u):
        cum = np.cumsum(w)
        over = np.nonzero(cum > np.float64(u) * cum[-1])[0]
        return int(over[0]) if len(over) else int(np.nonzero(w > 0)[0][-1])

    t, path = 0, []
    while True:
        path.append(t)
        p = p_of(t)
        if len(path) >= max_path:
            return path, (int(np.argmax(z[t])) if temperature == 0 else pick(p, u_sample[t]))
        kids = [j for j in range(t + 1, n) if parent[j] == t][:max_children]
        w, c, M, to = p, 0.0, 1.0, None
        for j in kids:
            x = tokens[j]
            if not 0 <= x < V:
                continue
            if temperature == 0:
                if p[x] == 1.0:
                    to = j
                    break
                continue
            u = np.float64(u_accept[j])
            q = draft[t].astype(np.float64) if draft is not None else None
            if (u * M * q[x] if q is not None else u * M) < w[x]:
                to = j
                break
            if q is not None:
                c += M
                w = np.maximum(p - c * q, 0.0)
            else:
                w = w.copy()
                w[x] = 0.0
            M = w.sum()
        if to is None:
            return path, (int(np.argmax(z[t])) if temperature == 0 else pick(w if M > 0 else p, u_sample[t]))
        t = to
