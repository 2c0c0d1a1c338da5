"""Cases and tolerance of the test that attention holds q and its weights to 22 bits.

The general bound of _serve.attention has to cover the worst order of every sum and would let operands of 11 bits
pass.  Here the error is taken relative to the output over all its values, where the errors of independent
roundings of the weights do not average out against the output itself (both are sums over the same positions)."""
import numpy as np

import goinfer_cuda as G
from _serve import Cache

# query heads, kv heads, head dim, positions, new tokens: units of up to 8, 16, 32 and (head dims 64, 128) 128 rows
SHAPES = [(4, 4, 64, 90, 1), (4, 4, 96, 90, 1), (8, 1, 128, 90, 1), (4, 2, 256, 90, 1),
          (16, 1, 64, 200, 1), (12, 1, 96, 200, 1), (16, 1, 128, 200, 1), (16, 1, 256, 200, 1),
          (32, 1, 64, 200, 1), (8, 2, 96, 200, 8), (8, 2, 128, 200, 8), (8, 2, 256, 200, 8),
          (8, 2, 64, 300, 40), (8, 2, 128, 300, 40), (8, 2, 128, 300, 70)]


class Case:
    """One sequence whose pages lie in order; the plain form in float64, its operands as given."""

    def __init__(self, kind, heads, kv, dim, n, new, page=16):
        rng = np.random.default_rng([kind, heads, dim, n, new])
        self.kind, self.heads, self.kv, self.dim, self.n, self.new, self.page = kind, heads, kv, dim, n, new, page
        self.cache = Cache(kind, -(-n // page), page, kv, dim).fill(rng)
        self.q = rng.normal(size=(new, heads, dim)).astype(np.float32)
        self.scale = dim ** -0.5
        self.k, self.v = self.cache.rows(np.arange(n))

    def out(self, q=lambda x: x, p=lambda x: x):
        """The output with q and the weights (as shares of the largest) rounded by q and p."""
        group = self.heads // self.kv
        r = np.zeros(self.q.shape)
        for j in range(self.new):
            m = self.n - self.new + j + 1
            for h in range(self.heads):
                s = self.k[:m, h // group] @ q(self.q[j, h].astype(np.float64)) * self.scale
                w = p(np.exp(s - s.max()))
                r[j, h] = w @ self.v[:m, h // group] / w.sum()
        return r

    def tolerance(self):
        """Of the error's norm over the output's: 2^-23 for each time a sum is cut or rounded on a score's way (two
        steps per 16 dimensions, each of a partial sum of at most `most`, then the factor and the exponent) and on
        the weighted sum's (at most 16 steps of a tile, 32 sums of a thread and 16 joins; exp2, splits)."""
        group = self.heads // self.kv
        most = max(np.abs(np.cumsum(self.k[:, h // group] * self.q[j, h].astype(np.float64), -1)).max() * self.scale
                   for j in range(self.new) for h in range(self.heads))
        return 2.0 ** -23 * ((self.dim / 8 + 2) * most + 64)


def half(x):
    """To 11 bits: what one half holds of an operand whose size is in its normal range."""
    m, e = np.frexp(x)
    return np.ldexp(np.rint(m * 2048), e - 11)


def off(got, want):
    return np.linalg.norm(got - want) / np.linalg.norm(want)


KINDS = [G.TYPE_F16, G.TYPE_Q8_0]
