"""Plain 64-bit forms of the paged-cache operators, for their tests."""
import math

import numpy as np

import goinfer_cuda as G

PART = 256  # alignment of a cache block's parts


class Cache:
    """A cache block on the host: K, V and (Q8_0) their scales as numpy views of one byte array."""

    def __init__(self, kind, n_pages, page, kv, dim):
        self.kind, self.n_pages, self.page, self.kv, self.dim = kind, n_pages, page, kv, dim
        n = n_pages * page * kv * dim
        up = lambda b: -(-b // PART) * PART  # noqa: E731
        val, sc = up(n * (2 if kind == G.TYPE_F16 else 1)), up(n // 32 * 2) if kind == G.TYPE_Q8_0 else 0
        self.data = np.zeros(2 * (val + sc), np.uint8)
        shape = (n_pages, kv, page, dim)
        t, w = (np.float16, 2) if kind == G.TYPE_F16 else (np.int8, 1)
        self.k, self.v = (self.data[a:a + n * w].view(t).reshape(shape) for a in (0, val))
        self.ks = self.vs = None
        if sc:
            self.ks, self.vs = (self.data[a:a + n // 16].view(np.float16).reshape(shape[:3] + (dim // 32,))
                                for a in (2 * val, 2 * val + sc))

    def fill(self, rng, poison=()):
        """Values of a normal model; the pages in `poison` hold what is not a number."""
        for x, s in ((self.k, self.ks), (self.v, self.vs)):
            if s is None:
                x[:] = rng.normal(size=x.shape)
                x[list(poison)] = np.nan
            else:
                x[:] = np.clip(rng.normal(size=x.shape) * 42, -127, 127)
                s[:] = rng.uniform(0.008, 0.04, s.shape)
                s[list(poison)] = np.nan
        return self

    def values(self):
        """(K, V) [n_pages, kv, page, dim] in float64."""
        if self.kind == G.TYPE_F16:
            return self.k.astype(np.float64), self.v.astype(np.float64)
        with np.errstate(invalid="ignore"):
            return tuple((x.reshape(s.shape + (32,)).astype(np.float32) * s.astype(np.float32)[..., None])
                         .astype(np.float16).astype(np.float64).reshape(x.shape)
                         for x, s in ((self.k, self.ks), (self.v, self.vs)))

    def rows(self, slots):
        k, v = (x.swapaxes(1, 2).reshape(-1, self.kv, self.dim) for x in self.values())
        return k[slots], v[slots]


def attention(cache, q, q_start, kv_len, pages, scale, prefix_pages=(), prefix_len=0, out=None):
    """(out, bound): softmax attention by its definition in float64; bound is how far float32 sums of
    operands held to 22 bits may be off.

    A score q.k of d products is off by at most (2^-22 + d 2^-24) |q||k| (the split of q, then the
    additions), so a weight by twice that (it and the sum below it), and by the exponent's rounding of the
    score itself (2^-23 of its size); P is split like q, and the P V sums and the merges of parts round
    at most ~64 times on the longest way: 2^-24 each."""
    K, V = cache.values()
    kv, page, dim = cache.kv, cache.page, cache.dim
    out = np.zeros(q.shape) if out is None else out.astype(np.float64)
    bound = np.zeros(q.shape[:2])
    group = q.shape[1] // kv

    def positions(table, n):
        got_k, got_v, ok = np.zeros((n, kv, dim)), np.zeros((n, kv, dim)), np.zeros(n, bool)
        for p in range(n):
            i = table[p // page]
            if 0 <= i < cache.n_pages:
                got_k[p], got_v[p], ok[p] = K[i, :, p % page], V[i, :, p % page], True
        return got_k, got_v, ok

    pk, pv, pok = positions(prefix_pages, prefix_len)
    for b, n in enumerate(kv_len):
        start, end = q_start[b], q_start[b + 1]
        own = positions(pages[b], n)
        k, v, ok = (np.concatenate(x) for x in zip((pk, pv, pok), own))
        for j in range(start, end):
            seen = ok & (np.arange(len(ok)) < prefix_len + n - (end - start) + (j - start) + 1)
            for h in range(q.shape[1]):
                x, y = k[seen, h // group], v[seen, h // group]
                if not len(x):
                    out[j, h] = 0
                    continue
                s = x @ q[j, h].astype(np.float64) * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                out[j, h] = w @ y
                norm = np.linalg.norm(q[j, h]) * np.linalg.norm(x, axis=1).max() * abs(scale)  # a size: whatever the scale's sign
                off = 2 * (norm * (2.0 ** -22 + dim * 2.0 ** -24) + (abs(s).max() + 1) * 2.0 ** -23)
                bound[j, h] = (off + 64 * 2.0 ** -24) * np.abs(y).max()
    return out, bound


def sample(x, u, t, k, p, least):
    """(id, share) of one row by the definition in include/goinfer_cuda.h."""
    x = np.asarray(x, np.float64)
    can = [i for i in range(len(x)) if x[i] > -math.inf]
    if not can:
        return -1, 0.0
    order = sorted(can, key=lambda i: (-x[i], i))
    if not t > 0:
        return order[0], 1.0
    top = x[order[0]]
    one = 1 << 42
    if top == math.inf:
        w = {i: one if x[i] == math.inf else 0 for i in can}
    else:
        w = {i: int(np.rint(np.exp((x[i] - top) / np.float64(t)) * one)) for i in can}
    if k > 0:
        order = order[:k]
    if p < 1:
        need = max(1, math.ceil(float(np.float32(p)) * float(sum(w[i] for i in order))))
        total, m = 0, 0
        while total < need:
            total += w[order[m]]
            m += 1
        order = order[:m]
    if least > 0:
        floor = math.ceil(min(float(np.float32(least)), 1.0) * one)
        order = [i for i in order if w[i] >= floor]
    total = sum(w[i] for i in order)
    want = min(math.floor(float(np.float32(min(max(u, 0.0), 1 - 2.0 ** -24))) * float(total)), total - 1)
    run = 0
    for i in sorted(order):
        run += w[i]
        if run > want:
            return i, w[i] / total
    raise AssertionError
