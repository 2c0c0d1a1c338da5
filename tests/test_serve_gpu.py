"""The paged-cache operators on the GPU against plain 64-bit forms, through the C ABI."""
import math

import numpy as np
import pytest

import goinfer_cuda as G
import _precision
from _line import Line
from _serve import Cache, attention, sample

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

KINDS = [G.TYPE_F16, G.TYPE_Q8_0]


@pytest.fixture(scope="module", autouse=True)
def cuda():
    G.Init(0)
    assert G.IsAvailable()
    yield


def dev(a, t=None):
    return torch.from_numpy(np.ascontiguousarray(a if t is None else np.asarray(a, t))).to("cuda:0")


def on_gpu(cache):
    data = dev(cache.data)
    return data, G.KVCache(cache.kind, cache.n_pages, cache.page, cache.kv, cache.dim, data_ptr=data.data_ptr(),
                           nbytes=data.numel())


def back(cache, data):
    cache.data[:] = data.cpu().numpy()
    return cache


# ---- write and read ----------------------------------------------------------------

def write(cache, qkv, heads, slots, positions=None, freqs=None, rot=0, interleaved=False, mscale=1.0):
    """One kv_write_dev over rows of [q | k | v] as one projection leaves them: (q_out, cache)."""
    n, kv, dim = len(slots), cache.kv, cache.dim
    data, gc = on_gpu(cache)
    x, st = dev(qkv, np.float32), torch.cuda.Stream()
    out = torch.full((n, max(heads, 1), dim), 7.0, device="cuda:0")
    sl = dev(slots, np.int32)
    pos = dev(positions if positions is not None else np.zeros(n), np.int32)
    f = dev(freqs if freqs is not None else np.zeros(1), np.float64)
    rope = G.Rope(rot, f.data_ptr(), interleaved, mscale) if rot else None
    stride = qkv.shape[1]
    torch.cuda.synchronize()
    G.kv_write_dev(gc, x.data_ptr() + 4 * heads * dim, x.data_ptr() + 4 * (heads + kv) * dim, sl.data_ptr(), n,
                   k_stride=stride, v_stride=stride, q_ptr=x.data_ptr() if heads else 0,
                   q_out_ptr=out.data_ptr() if heads else 0, heads=heads, q_stride=stride if heads else 0,
                   positions_ptr=pos.data_ptr() if rot else 0, rope=rope, stream=st.cuda_stream)
    st.synchronize()
    return out.cpu().numpy(), back(cache, data)


def turned(x, positions, freqs, rot, interleaved, mscale):
    """x [n, heads, dim] rotated: in float32 with every operation rounded, and in float64."""
    a = np.asarray(positions, np.float64)[:, None, None] * freqs
    i = np.arange(rot // 2)
    lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    got = []
    for t in (np.float32, np.float64):
        c, s = (np.cos(a) * mscale).astype(t), (np.sin(a) * mscale).astype(t)
        y = x.astype(t).copy()
        y[..., lo] = x[..., lo] * c - x[..., hi] * s
        y[..., hi] = x[..., lo] * s + x[..., hi] * c
        got.append(y)
    return got


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,heads,kv,dim,page,rot,interleaved,scaling", [
    (1, 4, 4, 128, 16, 128, False, G.ROPE_NONE),
    (33, 8, 2, 128, 16, 128, True, G.ROPE_LLAMA3),
    (17, 6, 2, 64, 32, 32, False, G.ROPE_LINEAR),   # part of the head
    (9, 3, 1, 96, 16, 96, False, G.ROPE_YARN),
    (5, 2, 2, 256, 64, 256, True, G.ROPE_YARN),
    (7, 4, 1, 32, 16, 10, False, G.ROPE_NONE),      # pairs whose halves share no chunk of 4
    (7, 4, 1, 32, 16, 14, True, G.ROPE_NONE),
    (700, 5, 5, 64, 16, 64, False, G.ROPE_NONE),
    (6, 0, 3, 128, 16, 0, False, G.ROPE_NONE),      # no q, nothing turns
])
def test_write(kind, n, heads, kv, dim, page, rot, interleaved, scaling):
    rng = np.random.default_rng(1000 + n)
    n_pages = -(-n // page) + 2
    cache = Cache(kind, n_pages, page, kv, dim).fill(rng)
    before = cache.data.copy()
    slots = rng.permutation(n_pages * page)[:n].astype(np.int32)
    if n > 4:
        slots[[1, 3]] = -1, n_pages * page  # padding, and a slot past the end
    qkv = rng.normal(size=(n, (heads + 2 * kv) * dim)).astype(np.float32)
    positions = rng.integers(0, 120000, n)
    freqs, mscale = G.rope_freqs(max(rot, 2), 10000.0, scaling, factor=8.0, low=1.0, high=4.0, orig_ctx=4096.0)
    q_out, cache = write(cache, qkv, heads, slots, positions, freqs, rot, interleaved, mscale)
    q, k, v = np.split(qkv, [heads * dim, (heads + kv) * dim], axis=1)
    q, k, v = (x.reshape(n, -1, dim) for x in (q, k, v))
    if rot:
        (_, q64), (k32, _) = (turned(x, positions, freqs, rot, interleaved, mscale) for x in (q, k))
    else:
        q64, k32 = q.astype(np.float64), k
    if heads:
        # cos and sin, two products and a sum round by half a step each: 3 * 2^-24 of |x0| + |x1|
        size = 2 * np.abs(q).max(axis=(1, 2), keepdims=True) * mscale
        assert (np.abs(q_out - q64) <= 3 * 2.0 ** -24 * size + 1e-12).all()
    fresh = Cache(kind, n_pages, page, kv, dim)
    fresh.data[:] = before
    for t in range(n):
        if not 0 <= slots[t] < n_pages * page:
            continue
        p, o = divmod(int(slots[t]), page)
        for x, val, sc in ((k32, fresh.k, fresh.ks), (v, fresh.v, fresh.vs)):
            if kind == G.TYPE_F16:
                val[p, :, o] = x[t].astype(np.float16)
            else:  # the framework's own quantiser
                raw = G.quantize(G.TYPE_Q8_0, x[t].reshape(kv, dim)).reshape(kv, dim // 32, 34)
                sc[p, :, o] = raw[..., :2].copy().view(np.float16)[..., 0]
                val[p, :, o] = raw[..., 2:].copy().view(np.int8).reshape(kv, dim)
    # cos(double) here and there may differ in the last bit, which moves a float32 factor once in 2^29
    assert np.array_equal(fresh.data, cache.data)


@pytest.mark.parametrize("kind", KINDS)
def test_write_keeps_the_cache_finite(kind):
    dim, kv = 64, 1
    bad = np.zeros((4, 2 * dim), np.float32)
    bad[0, 3], bad[0, 40] = np.nan, 1.0
    bad[1, 5], bad[1, dim + 6] = np.inf, -np.inf
    bad[2, :] = 1e30
    bad[3, 8], bad[3, dim + 9] = 1e-30, 3e-7  # scales below half precision's range
    _, cache = write(Cache(kind, 1, 16, kv, dim), bad, 0, [0, 1, 2, 3])
    k, v = cache.rows([0, 1, 2, 3])
    assert np.isfinite(k).all() and np.isfinite(v).all()
    assert k[0, 0, 3] == 0 and abs(k[0, 0, 40] - 1) <= 2.0 ** -8
    top = 65504 * (1 - 2.0 ** -7)
    assert k[1, 0, 5] >= top and v[1, 0, 6] <= -top and (k[2] >= top).all()
    assert k[3, 0, 8] == 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,kv,dim,page", [(1, 1, 32, 16), (37, 8, 64, 16), (300, 3, 96, 32), (77, 2, 256, 64),
                                           (3000, 4, 128, 64)])
def test_read(kind, n, kv, dim, page):
    rng = np.random.default_rng(n)
    cache = Cache(kind, 9, page, kv, dim).fill(rng)
    data, gc = on_gpu(cache)
    slots = rng.integers(0, 9 * page, n).astype(np.int32)  # some more than once
    if n > 2:
        slots[[0, 2]] = -5, 9 * page
    k, v = (torch.full((n, kv, dim), 3.0, device="cuda:0") for _ in range(2))
    sl, st = dev(slots), torch.cuda.Stream()
    torch.cuda.synchronize()
    G.kv_read_dev(gc, k.data_ptr(), v.data_ptr(), sl.data_ptr(), n, stream=st.cuda_stream)
    st.synchronize()
    ok = (slots >= 0) & (slots < 9 * page)
    for got, want in zip((k, v), cache.rows(np.where(ok, slots, 0))):
        assert np.array_equal(got.cpu().numpy(), np.where(ok[:, None, None], want, 3.0))


# ---- attention ---------------------------------------------------------------------

class AttnCase:
    """A batch with its pages anywhere in the cache, and one poisoned page that no table entry in use names."""

    def __init__(self, seed, kind, heads, kv, dim, page, lens, new=None, prefix=0, pad=0, before=0, scale=None, hint=0):
        rng = np.random.default_rng(seed)
        self.new = new or [1] * len(lens)
        self.lens, self.prefix, self.page, self.kind = list(lens), prefix, page, kind
        need = [-(-n // page) for n in lens]
        shared = -(-prefix // page)
        n_pages = sum(need) + shared + 1
        self.cache = Cache(kind, n_pages, page, kv, dim).fill(rng, poison=[n_pages - 1])
        order = rng.permutation(n_pages - 1)
        self.width = max(1, max(need))
        self.table = np.full((len(lens), self.width), n_pages - 1, np.int32)
        self.prefix_pages = order[:shared].astype(np.int32)
        at = shared
        for b, m in enumerate(need):
            self.table[b, :m] = order[at:at + m]
            at += m
            if lens[b] % page:  # what lies behind a sequence in its last page is not read
                i, o = self.table[b, m - 1], lens[b] % page
                for x in ((self.cache.k, self.cache.v) if kind == G.TYPE_F16 else (self.cache.ks, self.cache.vs)):
                    x[i, :, o:] = np.nan
        if prefix % page:
            for x in ((self.cache.k, self.cache.v) if kind == G.TYPE_F16 else (self.cache.ks, self.cache.vs)):
                x[self.prefix_pages[-1], :, prefix % page:] = np.nan
        self.start = (before + np.concatenate(([0], np.cumsum(self.new)))).astype(np.int32)
        self.tokens = int(self.start[-1]) + pad
        self.q = rng.normal(size=(self.tokens, heads, dim)).astype(np.float32)
        self.scale = dim ** -0.5 if scale is None else scale
        self.data, self.gc = on_gpu(self.cache)
        self.d = {"q": dev(self.q), "start": dev(self.start), "len": dev(self.lens, np.int32), "table": dev(self.table),
                  "prefix": dev(self.prefix_pages) if prefix else None}
        self.out = torch.full((self.tokens, heads, dim), 5.0, device="cuda:0")
        self.att = G.Attention(self.gc, heads=heads, max_tokens=max(self.tokens, len(lens)), max_q_len=hint or max(self.new), scale=self.scale,
                               prefix_len=prefix)
        self.ws = torch.full((max(self.att.workspace_bytes, 1),), 255, dtype=torch.uint8, device="cuda:0")
        self.stream = torch.cuda.Stream()
        torch.cuda.synchronize()

    def call(self, stream=None, ragged=True):
        self.att(self.out.data_ptr(), self.d["q"].data_ptr(), len(self.lens), self.tokens, self.d["len"].data_ptr(),
                 self.d["table"].data_ptr(), self.width, self.ws.data_ptr(), self.ws.numel(),
                 q_start_ptr=self.d["start"].data_ptr() if ragged else 0,
                 prefix_pages_ptr=self.d["prefix"].data_ptr() if self.prefix else 0,
                 stream=(stream or self.stream).cuda_stream)

    def check(self, lens=None, table=None):
        got = self.out.cpu().numpy()
        want, bound = attention(self.cache, self.q, self.start, self.lens if lens is None else lens,
                                self.table if table is None else table, self.scale, self.prefix_pages, self.prefix,
                                out=np.full(got.shape, 5.0))
        err = np.abs(got - want).max(-1)
        assert (err <= bound).all(), (err.max(), float((err / np.maximum(bound, 1e-30)).max()), np.argwhere(err > bound)[:5])
        return got

    def run(self, **kw):
        self.call(**kw)
        self.stream.synchronize()
        return self.check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 64), (4, 4, 128), (8, 1, 128), (6, 2, 96), (10, 2, 64), (16, 1, 128),
                                          (4, 2, 256), (40, 1, 64)])
@pytest.mark.parametrize("page", [16, 64])
def test_attention_of_single_tokens(kind, heads, kv, dim, page):
    lens = [1, 0, 15, 16, 17, 33, 64, 65, 130, 257]
    AttnCase(heads * dim + page, kind, heads, kv, dim, page, lens).run()


@pytest.mark.parametrize("kind", KINDS)
def test_attention_without_q_start(kind):
    c = AttnCase(5, kind, 8, 2, 128, 32, [40, 7, 100])
    c.run(ragged=False)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens", [[1], [0], [31], [32], [3001], [2048, 1], [5, 4000, 9]])
def test_attention_of_long_and_short_sequences(kind, lens):
    AttnCase(sum(lens), kind, 8, 2, 128, 64, lens).run()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv", [(2, 2), (8, 2), (7, 1)])
@pytest.mark.parametrize("lens,new", [
    ([5], [5]), ([64], [33]), ([100, 3, 20], [1, 3, 7]), ([40, 40, 0], [40, 1, 2]), ([3], [9]), ([150, 70], [97, 2]), ([30, 50, 0, 9], [2, 0, 0, 1])])
def test_attention_of_chunks(kind, dim, heads, kv, lens, new):
    """Causal inside the chunk; [3] with 9 new tokens: the first 6 rows see nothing."""
    AttnCase(sum(lens) + heads, kind, heads, kv, dim, 16, lens, new, pad=2).run()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 128), (8, 1, 64), (6, 2, 128), (4, 2, 256)])
@pytest.mark.parametrize("prefix,lens,new", [
    (1, [0], None), (17, [0, 1, 40], None), (200, [5, 64, 0, 90], None), (333, [30, 12], [3, 5]),
    (64, list(range(40)), None), (130, [9, 9], [9, 4])])
def test_attention_with_a_shared_prefix(kind, heads, kv, dim, prefix, lens, new):
    AttnCase(prefix + dim, kind, heads, kv, dim, 16, lens, new, prefix=prefix, pad=1).run()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,dim,lens,new,prefix", [
    (4, 1, 128, [64], [64], 0), (4, 1, 64, [129], [33], 0), (2, 2, 128, [300, 1], [128, 1], 0),
    (8, 1, 128, [700, 1500, 0, 40], [300, 64, 1, 40], 0), (6, 2, 64, [1000], [257], 0),
    (4, 4, 128, [0] * 70, None, 1000), (8, 1, 64, list(range(60)), None, 513), (16, 2, 128, [30, 5], [30, 2], 2000),
    (5, 1, 128, [9] * 33, None, 128)])
def test_attention_of_many_rows(kind, heads, kv, dim, lens, new, prefix):
    """Units of 128 rows: one and several tiles of 128 positions, rows and positions that do not fill them."""
    AttnCase(sum(lens) + heads, kind, heads, kv, dim, 16, lens, new, prefix=prefix, pad=3).run()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_many_rows_that_see_nothing(kind, dim):
    """Unit after unit without a tile, with one that has tiles among them, in the run of every CTA."""
    n = 40
    lens = [300 if b % 7 == 3 else 0 for b in range(n)]
    AttnCase(35 + dim, kind, 8, 1, dim, 16, lens, [64] * n).run()


@pytest.mark.parametrize("kind", KINDS)
def test_attention_of_many_rows_skips_pages_outside_the_cache(kind):
    c = AttnCase(13, kind, 8, 2, 128, 16, [400, 133], [100, 20])
    c.table[0, [0, 9, 20]], c.table[1, 8] = [-1, c.cache.n_pages, 10 ** 9], -7
    c.d["table"].copy_(dev(c.table))
    torch.cuda.synchronize()
    c.run()


@pytest.mark.parametrize("kind", KINDS)
def test_attention_skips_pages_outside_the_cache(kind):
    """A page id outside the cache is never followed: its positions are not seen (also all of a sequence)."""
    c = AttnCase(3, kind, 4, 2, 128, 16, [60, 33, 16])
    c.table[0, 1], c.table[1, 2], c.table[2, 0] = -1, c.cache.n_pages, 2 ** 31 - 1
    c.d["table"].copy_(dev(c.table))
    torch.cuda.synchronize()
    c.run()


@pytest.mark.parametrize("kind", KINDS)
def test_attention_bounds_lengths(kind):
    """Lengths beyond the page table end at it; negative ones are empty."""
    c = AttnCase(4, kind, 4, 2, 64, 16, [64, 48, 20])
    c.d["len"].copy_(dev([10 ** 6, -3, 20], np.int32))
    torch.cuda.synchronize()
    c.call()
    c.stream.synchronize()
    c.check(lens=[64, 0, 20])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,hint", [([70, 3], 1), ([1, 1], 60), ([70, 3], 2)])
def test_attention_whatever_length_is_announced(kind, new, hint):
    """More new tokens than max_q_len, or far fewer: the other kernels, the same answer."""
    AttnCase(31, kind, 8, 2, 128, 16, [200, 130], new, prefix=40, pad=60 if hint > 2 else 0, hint=hint).run()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,prefix", [([1, 4], 0), ([40, 2], 33), ([1, 1], 200)])
def test_attention_leaves_rows_of_no_sequence(kind, new, prefix):
    """q_start may begin behind rows that belong to nobody."""
    AttnCase(32, kind, 8, 2, 128, 16, [50, 77], new, prefix=prefix, pad=2, before=5).run()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [0.0, -0.1])
@pytest.mark.parametrize("new", [[1, 2], [60, 2]])
def test_attention_scale_of_any_sign(kind, scale, new):
    AttnCase(33, kind, 8, 2, 128, 16, [90, 300], new, prefix=20, scale=scale).run()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [[1, 2], [60, 2]])
def test_attention_skips_prefix_pages_outside_the_cache(kind, new):
    c = AttnCase(34, kind, 8, 2, 128, 16, [70, 9], new, prefix=100)
    c.prefix_pages[[0, 3, 6]] = -1, c.cache.n_pages, 2 ** 31 - 1
    c.d["prefix"].copy_(dev(c.prefix_pages))
    torch.cuda.synchronize()
    c.run()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("start", [[500, 0, 600], [0, 600, 300], [-40, 700, 20], [600, 600, 0]])
def test_attention_with_a_q_start_that_does_not_ascend(kind, start):
    """What the rows hold is not defined, but nothing beside them is touched, and the next call is right."""
    c = AttnCase(36, kind, 4, 1, 128, 16, [540, 160], [500, 100], prefix=300)
    n, guard = c.ws.numel(), 1 << 16
    around = torch.full((n + 2 * guard,), 85, dtype=torch.uint8, device="cuda:0")
    out = torch.full((c.tokens + 64, 4, 128), 5.0, device="cuda:0")
    c.ws, c.out = around[guard:guard + n], out[32:32 + c.tokens]
    good = c.d["start"].clone()
    c.d["start"].copy_(dev(start, np.int32))
    torch.cuda.synchronize()
    c.call()
    c.stream.synchronize()
    assert (around[:guard] == 85).all() and (around[guard + n:] == 85).all()
    assert (out[:32] == 5).all() and (out[32 + c.tokens:] == 5).all()
    c.d["start"].copy_(good)
    torch.cuda.synchronize()
    c.run()


def test_attention_large_scores_and_flat_rows():
    """Scores of several hundred (one weight takes all) and a q of zeros (all weights equal)."""
    c = AttnCase(8, G.TYPE_F16, 4, 2, 128, 16, [70, 300])
    c.q[0] *= 300
    c.q[1] = 0
    c.d["q"].copy_(dev(c.q))
    torch.cuda.synchronize()
    c.run()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("lens,new,prefix", [
    ([30, 50, 9], [1, 1, 1], 0), ([5000, 40], [1, 1], 0), ([30, 3000], [1, 1], 70),         # whole units, cut ones, a prefix
    ([70, 300], [60, 64], 0), ([3000, 200], [64, 60], 0), ([900, 60], [64, 50], 500), ([3, 9] * 30, [1] * 60, 700)])
def test_attention_of_a_query_that_is_not_finite(kind, bad, lens, new, prefix):
    """Its row is not a number wherever the line of tiles is cut; every other row is as it would be without it."""
    c = AttnCase(37, kind, 8, 2, 128, 16, lens, new, prefix=prefix)
    rows = [(0, 1), (c.tokens - 1, 7), (c.tokens // 2, 4)]
    for t, h in rows:
        c.q[t, h, 5] = bad
        c.q[t, h, 6] = -c.q[t, h, 5]  # with an infinity no score is a number either
    c.d["q"].copy_(dev(c.q))
    torch.cuda.synchronize()
    c.call()
    c.stream.synchronize()
    got = c.out.cpu().numpy()
    for t, h in rows:
        assert np.isnan(got[t, h]).all()
    want, bound = attention(c.cache, np.nan_to_num(c.q, nan=0, posinf=0, neginf=0), c.start, c.lens, c.table, c.scale,
                            c.prefix_pages, prefix, out=np.full(got.shape, 5.0))
    ok = np.ones(got.shape[:2], bool)
    for t, h in rows:
        ok[t, h] = False
    assert (np.abs(got - want).max(-1)[ok] <= bound[ok]).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("seqs", [1, 40])
def test_attention_of_many_rows_keeps_far_scores_apart(kind, dim, seqs):
    """Scores near -757 * 60, exact in float32, whose maximum rises from tile to tile; V is 1 in even tiles and -1 in
    odd ones, so a weight's error that differs between tiles shows in full.  The maxima are just above -65536 in
    binades, where a sum with a few more binades would have coarser steps than they.

    With exact scores a weight is off by its exponent's factor (2^-23 of at most 4 binades of distance), the
    exponent's last rounding (2^-22 of a binade), exp2 (2^-22), the split (2^-22) and, in up to 11 tiles, the
    factors between maxima (2^-22 each); sums of 64 to 128 values round or cut at 2^-23 a step, once in the sums of
    weights and once in P V: below 2^-16 of max|V| in all, while half a step beyond 65536 is 2^-8."""
    n, new = 1400, 16
    c = AttnCase(38, kind, 8, 2, dim, 16, [n] * seqs, [new] * seqs, scale=1.0)
    rng = np.random.default_rng(39)
    k1 = np.array([rng.integers(-8, p // 128 + 1) for p in range(n)])
    sign = np.where(np.arange(n) // 128 % 2, -1.0, 1.0)
    c.cache.k[:], c.cache.v[:] = 0, 0
    for x in (c.cache.ks, c.cache.vs):
        if x is not None:
            x[:] = 1
    p = np.arange(n)
    for b in range(seqs):
        page, o = c.table[b, p // 16], p % 16
        c.cache.k[page, :, o, 0] = -60
        c.cache.k[page, :, o, 1] = k1[:, None]
        c.cache.v[page, :, o] = sign[:, None, None]
    c.q[:] = 0
    c.q[..., 0] = 757
    c.q[..., 1] = 0.125
    c.data.copy_(dev(c.cache.data)), c.d["q"].copy_(dev(c.q))
    torch.cuda.synchronize()
    c.call()
    c.stream.synchronize()
    w = np.exp(k1 / 8)
    want = (np.cumsum(w * sign) / np.cumsum(w))[n - new:]
    got = c.out.cpu().numpy().reshape(seqs, new, 8, dim)
    assert np.abs(got - want[:, None, None]).max() <= 2.0 ** -16


@pytest.mark.parametrize("size", [1e-30, 1e-3, 1e4])
@pytest.mark.parametrize("kind", KINDS)
def test_attention_of_any_magnitude_of_q_and_v(kind, size):
    c = AttnCase(9, kind, 8, 2, 128, 16, [90, 200])
    c.q *= size
    if kind == G.TYPE_F16:
        c.cache.v[:] = (c.cache.v.astype(np.float32) * min(size, 1e3)).astype(np.float16)
        c.data.copy_(dev(c.cache.data))
    c.d["q"].copy_(dev(c.q))
    torch.cuda.synchronize()
    c.run()


@pytest.mark.parametrize("kind", KINDS)
def test_attention_calls_repeat_bit_for_bit_and_side_by_side(kind):
    """Two streams at once, each call with a workspace of its own, then a captured call that follows new lengths."""
    a = AttnCase(20, kind, 8, 2, 128, 16, [500, 700, 3], prefix=100)
    b = AttnCase(21, kind, 8, 2, 128, 16, [90, 1100, 40], [4, 30, 1])
    first = (a.run(), b.run())
    for _ in range(3):
        a.out.fill_(5.0), b.out.fill_(5.0)
        torch.cuda.synchronize()
        for _ in range(4):
            a.call()
            b.call()
        a.stream.synchronize(), b.stream.synchronize()
        assert np.array_equal(a.out.cpu().numpy(), first[0]) and np.array_equal(b.out.cpu().numpy(), first[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=a.stream):
        a.call()
    a.d["len"].copy_(dev([10, 650, 3], np.int32))
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    a.check(lens=[10, 650, 3])


@pytest.mark.parametrize("kind", _precision.KINDS)
@pytest.mark.parametrize("shape", _precision.SHAPES)
def test_attention_holds_its_operands_to_22_bits(kind, shape):
    """The tolerance is one that a q or a weight in a single half fails (test_serve.py), in every kernel."""
    x = _precision.Case(kind, *shape)
    data, gc = on_gpu(x.cache)
    q, st = dev(x.q), torch.cuda.Stream()
    out = torch.zeros(x.new, x.heads, x.dim, device="cuda:0")
    att = G.Attention(gc, heads=x.heads, max_tokens=x.new, max_q_len=x.new, scale=x.scale)
    ws = torch.empty(max(att.workspace_bytes, 1), dtype=torch.uint8, device="cuda:0")
    lens, start = dev([x.n], np.int32), dev([0, x.new], np.int32)
    table = dev(np.arange(x.cache.n_pages), np.int32)
    torch.cuda.synchronize()
    att(out.data_ptr(), q.data_ptr(), 1, x.new, lens.data_ptr(), table.data_ptr(), x.cache.n_pages, ws.data_ptr(), ws.numel(),
        q_start_ptr=start.data_ptr(), stream=st.cuda_stream)
    st.synchronize()
    assert _precision.off(out.cpu().numpy(), x.out()) <= x.tolerance()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_of_many_rows_where_units_without_tiles_alternate(kind, dim):
    """Runs of ten and more units, those that see nothing between those that have tiles, in orders of every kind:
    the roles of a CTA skip the first and keep their phases through the others."""
    rng = np.random.default_rng(41)
    lens = [int(rng.choice([0, 0, 0, 40, 128, 129, 300])) for _ in range(1800)]
    c = AttnCase(42 + dim, kind, 4, 1, dim, 16, lens, [2] * len(lens), hint=16)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    line = Line(c.start.tolist(), lens, c.tokens, 4, 1, 128, 128, 4, sms, 1)
    runs = ["".join("T" if u[-1] else "E" for u in line.units(cta)) for cta in range(sms)]
    assert sum(len(r) >= 10 for r in runs) > sms // 2 and any("EEETE" in r for r in runs) and any("TETTE" in r for r in runs)
    c.run()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("size", [1e-30, 1e-3, 1e4])
def test_attention_of_many_rows_of_any_magnitude(kind, dim, size):
    c = AttnCase(43, kind, 8, 2, dim, 16, [400, 90], [70, 60], prefix=50)
    c.q *= size
    c.q[::5] = 0  # all weights equal
    c.q[1] *= 300  # scores of several hundred at size 1 and above: one weight takes all
    c.d["q"].copy_(dev(c.q))
    torch.cuda.synchronize()
    c.run()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dim,new", [(64, 1), (64, 40), (128, 1), (128, 40)])
@pytest.mark.parametrize("prefix", [0, 150])
@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 22, 2.0 ** 30, -2.0 ** 40, 2.0 ** 100])
def test_attention_of_scores_far_beyond_one_step(kind, dim, new, prefix, size):
    """One position's score is larger than every other's by far more than the exponent's range, and the scores
    themselves are so large that a step of them in float32 is: the row is that position's V."""
    n = 190
    c = AttnCase(49, kind, 8, 2, dim, 16, [n, n], [new] * 2, prefix=prefix)
    rng = np.random.default_rng(50)
    c.cache.k[:] = 0
    for x in (c.cache.ks, c.cache.vs):
        if x is not None:
            x[:] = 1
    v = rng.integers(-60, 60, c.cache.v.shape)
    c.cache.v[:] = v
    k0 = rng.permutation(201)[:n] - 100  # of the own positions; the prefix's lie below or among them
    p = np.arange(n)
    for b in range(2):
        c.cache.k[c.table[b, p // 16], :, p % 16, 0] = k0[:, None]
    if prefix:
        p = np.arange(prefix)
        kp = rng.integers(-120, 121, prefix) // 2 * 2 + 0.5 if kind == G.TYPE_F16 else rng.integers(-126, -100, prefix)
        c.cache.k[c.prefix_pages[p // 16], :, p % 16, 0] = kp[:, None]
    c.q[:] = 0
    c.q[..., 0] = size
    c.data.copy_(dev(c.cache.data)), c.d["q"].copy_(dev(c.q))
    torch.cuda.synchronize()
    c.call()
    c.stream.synchronize()
    got = c.out.cpu().numpy().reshape(2, new, 8, dim)
    sign = 1 if size > 0 else -1
    for b in range(2):
        for j in range(new):
            seen = n - new + j + 1
            score = sign * k0[:seen].astype(float)
            at = int(score.argmax())
            page, o = c.table[b, at // 16], at % 16
            if prefix and (sign * kp).max() > score[at]:
                best = np.flatnonzero(sign * kp == (sign * kp).max())
                want = np.mean([c.cache.v[c.prefix_pages[i // 16], :, i % 16].astype(float) for i in best], axis=0)
            else:
                want = c.cache.v[page, :, o].astype(float)
            # equal scores weigh the same to the exponent's 2^-22, the split and the sums round below 2^-18
            assert np.abs(got[b, j] - np.repeat(want, 4, axis=0)).max() <= 60 * 2.0 ** -18


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,lens,new,prefix", [
    (3, 1, [150, 70], [97, 2], 0), (6, 2, [40, 200, 9], [12, 1, 3], 0), (4, 4, [0, 30, 90], None, 170), (12, 1, [60, 33], [9, 4], 250)])
def test_attention_of_head_dim_96(kind, heads, kv, lens, new, prefix):
    AttnCase(44 + heads, kind, heads, kv, 96, 16, lens, new, prefix=prefix, pad=2).run()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens,new,prefix", [([20011, 9000], None, 0), ([30, 700], None, 12345), ([12007], [50], 0),
                                             ([40] * 50, None, 9001)])
def test_attention_over_long_contexts(kind, lens, new, prefix):
    AttnCase(45, kind, 4, 2, 64, 64, lens, new, prefix=prefix).run()


@pytest.mark.parametrize("kind", KINDS)
def test_cache_whose_offsets_pass_32_bits(kind):
    """The highest pages of a cache of 10 GB and more answer as a small cache's: what is written there, read back and
    attended over, by single tokens and by chunks."""
    kv, dim, page, n, heads = 8, 128, 64, 200, 16
    n_pages = (1 << 32) // (kv * dim * page) + 8  # values past 2^32
    rng = np.random.default_rng(46)
    kvs = dev(rng.normal(size=(2, n, kv, dim)), np.float32)
    q = dev(rng.normal(size=(64, heads, dim)), np.float32)
    st = torch.cuda.Stream()
    got = []
    for pages in (n_pages, 8):
        size = int(G.load_library().gi_kv_cache_bytes(kind, pages, page, kv, dim))
        data = torch.empty(size, dtype=torch.uint8, device="cuda:0")
        gc = G.KVCache(kind, pages, page, kv, dim, data_ptr=data.data_ptr(), nbytes=size)
        table = pages - 1 - np.array([0, 2, 5, 3])
        p = np.arange(n)
        slots = dev(table[p // page] * page + p % page, np.int32)
        back_k, back_v = torch.zeros(n, kv, dim, device="cuda:0"), torch.zeros(n, kv, dim, device="cuda:0")
        table, lens = dev(table, np.int32), dev([n], np.int32)
        torch.cuda.synchronize()
        G.kv_write_dev(gc, kvs[0].data_ptr(), kvs[1].data_ptr(), slots.data_ptr(), n, stream=st.cuda_stream)
        G.kv_read_dev(gc, back_k.data_ptr(), back_v.data_ptr(), slots.data_ptr(), n, stream=st.cuda_stream)
        outs = [back_k, back_v]
        for new in (1, 8, 64):
            att = G.Attention(gc, heads=heads, max_tokens=new, max_q_len=new, scale=dim ** -0.5)
            ws = torch.empty(att.workspace_bytes, dtype=torch.uint8, device="cuda:0")
            start, out = dev([0, new], np.int32), torch.zeros(new, heads, dim, device="cuda:0")
            torch.cuda.synchronize()
            att(out.data_ptr(), q.data_ptr(), 1, new, lens.data_ptr(), table.data_ptr(), 4, ws.data_ptr(), ws.numel(),
                q_start_ptr=start.data_ptr(), stream=st.cuda_stream)
            st.synchronize()
            outs.append(out)
        got.append([x.cpu().numpy() for x in outs])
        del data, gc, ws
        torch.cuda.empty_cache()
    for x, y in zip(*got):
        assert np.array_equal(x, y) and np.abs(x).max() > 0


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens,new,prefix,other", [
    ([30, 200, 90] * 17, [1] * 51, 700, [0, 17, 90] * 17),   # a prefix in units of 128 rows, single tokens beside it
    ([300, 90], [70, 40], 0, [280, 75]), ([300, 90], [70, 40], 400, [299, 40])])
def test_a_captured_call_of_many_rows_follows_its_lengths(kind, lens, new, prefix, other):
    c = AttnCase(47, kind, 8, 2, 128, 16, lens, new, prefix=prefix)
    first = c.run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=c.stream):
        c.call()
        c.call()
    for now in (other, lens):
        c.d["len"].copy_(dev(now, np.int32))
        c.out.fill_(5.0)
        torch.cuda.synchronize()
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        got = c.check(lens=now)
    assert np.array_equal(got, first)


def test_the_calls_allocate_nothing():
    """Free device memory is the same after a first and after many of the calls."""
    c = AttnCase(48, G.TYPE_Q8_0, 8, 2, 128, 16, [300, 90], [70, 1], prefix=100)
    n, vocab = 40, 5000
    k, v = torch.zeros(2, n, 2 * 128, device="cuda:0")
    slots = torch.arange(n, dtype=torch.int32, device="cuda:0")
    x, u = torch.zeros(3, vocab, device="cuda:0"), torch.zeros(3, device="cuda:0")
    ids = torch.zeros(3, dtype=torch.int32, device="cuda:0")

    def calls():
        s = c.stream.cuda_stream
        G.kv_read_dev(c.gc, k.data_ptr(), v.data_ptr(), slots.data_ptr(), n, stream=s)
        G.kv_write_dev(c.gc, k.data_ptr(), v.data_ptr(), slots.data_ptr(), n, stream=s)
        c.call()
        G.sample_dev(ids.data_ptr(), x.data_ptr(), 3, vocab, u.data_ptr(), stream=s)
        c.stream.synchronize()

    calls()
    free = torch.cuda.mem_get_info()[0]
    for _ in range(20):
        calls()
    assert torch.cuda.mem_get_info()[0] == free


# ---- sampling ----------------------------------------------------------------------

def draw_ids(x, u, t=None, k=None, p=None, least=None, stride=0):
    n, vocab = len(u), x.shape[1] if not stride else x.shape[1]
    st = torch.cuda.Stream()
    xs = x
    if stride:
        xs = np.full((n, stride), 1e9, np.float32)
        xs[:, :vocab] = x
    d = {"x": dev(xs, np.float32), "u": dev(u, np.float32)}
    for name, a, ty in (("t", t, np.float32), ("k", k, np.int32), ("p", p, np.float32), ("m", least, np.float32)):
        d[name] = dev(a, ty) if a is not None else None
    ptr = lambda name: d[name].data_ptr() if d[name] is not None else 0  # noqa: E731
    ids, prob = torch.full((n,), -7, dtype=torch.int32, device="cuda:0"), torch.full((n,), -7.0, device="cuda:0")
    torch.cuda.synchronize()
    G.sample_dev(ids.data_ptr(), d["x"].data_ptr(), n, vocab, d["u"].data_ptr(), temperature_ptr=ptr("t"),
                 top_k_ptr=ptr("k"), top_p_ptr=ptr("p"), min_p_ptr=ptr("m"), prob_ptr=prob.data_ptr(),
                 logits_stride=stride, stream=st.cuda_stream)
    st.synchronize()
    return ids.cpu().numpy(), prob.cpu().numpy()


def check_ids(x, u, t=None, k=None, p=None, least=None, stride=0):
    ids, prob = draw_ids(x, u, t, k, p, least, stride)
    n = len(u)
    full = lambda a, v: a if a is not None else [v] * n  # noqa: E731
    for r, row in enumerate(zip(x, u, full(t, 1.0), full(k, 0), full(p, 1.0), full(least, 0.0))):
        i, share = sample(*row)
        assert ids[r] == i, (r, ids[r], i, row[1:])
        assert abs(prob[r] - share) <= 2.0 ** -23 * share  # one rounding to float32, and double's
    return ids


@pytest.mark.parametrize("vocab", [1, 2, 31, 32, 33, 1000, 1024, 32000, 50257, 128256])
def test_sample_mixed_rows(vocab):
    rng = np.random.default_rng(vocab)
    n = 7
    x = (rng.normal(size=(n, vocab)) * 3).astype(np.float32)
    check_ids(x, rng.random(n, np.float32), [0.8, 1.0, 0.3, 1.7, 0.0, 5.0, 1.0], [40, 0, 1, 1000, 5, 7, vocab],
              [0.95, 1.0, 0.5, 0.9, 0.5, 1.0, 0.0], [0.05, 0.0, 0.2, 0.01, 0.0, 0.0, 0.0])


@pytest.mark.parametrize("rows,vocab", [(1, 1 << 20), (2, 400001), (40, 5000), (150, 3000), (300, 40), (70, 9001)])
def test_sample_row_counts_and_large_vocabularies(rows, vocab):
    """From a row spread over a cluster (and one too long for shared memory) to a CTA per row."""
    rng = np.random.default_rng(rows)
    x = (rng.normal(size=(rows, vocab)) * 2).astype(np.float32)
    u = rng.random(rows, np.float32)
    ks, ps = rng.choice([0, 3, 50, 600, 2000], rows), rng.choice([1.0, 0.97, 0.6], rows).astype(np.float32)
    check_ids(x, u, t=rng.uniform(0.2, 2, rows).astype(np.float32), k=ks, p=ps, least=rng.choice([0.0, 0.01], rows))


def test_sample_clustered_logits():
    """Nearly all logits in one narrow band below a far outlier: the first bins separate nothing."""
    rng = np.random.default_rng(6)
    x = (rng.normal(size=(12, 20000)) * 1e-3).astype(np.float32)
    x[:, 77] = rng.choice([1.0, 50.0], 12)
    x[6:] = np.round(x[6:], 3)  # and hundreds of equal ones
    x[:, 99] = -1e9
    u = rng.random(12, np.float32)
    check_ids(x, u, k=[1, 2, 600, 5000, 19999, 0] * 2)
    check_ids(x, u, t=[5.0] * 12, k=[0, 10000, 19998] * 4, p=[0.3, 0.7, 0.999, 0.5] * 3)


def test_sample_one_filter_at_a_time():
    rng = np.random.default_rng(1)
    x = (rng.normal(size=(64, 3001)) * 2).astype(np.float32)
    u = rng.random(64, np.float32)
    check_ids(x, u)
    check_ids(x, u, t=rng.uniform(0.1, 3, 64).astype(np.float32))
    check_ids(x, u, k=rng.integers(-1, 60, 64))
    check_ids(x, u, p=rng.uniform(0, 1.05, 64).astype(np.float32))
    check_ids(x, u, least=rng.uniform(0, 1.1, 64).astype(np.float32))
    check_ids(x, u, p=rng.uniform(0.2, 1, 64).astype(np.float32), stride=4000)


def test_sample_ties_go_to_the_lowest_index():
    """Few distinct logits: the borders of top-k and top-p fall inside runs of equal ones."""
    rng = np.random.default_rng(2)
    x = rng.integers(-3, 3, (48, 5000)).astype(np.float32)
    x[x == 0] *= rng.choice([-1.0, 1.0], int((x == 0).sum())).astype(np.float32)  # -0 and +0 are equal
    u = rng.random(48, np.float32)
    k = rng.integers(1, 3000, 48)
    check_ids(x, u, k=k)
    check_ids(x, u, k=k, p=rng.uniform(0.05, 1, 48).astype(np.float32))
    check_ids(x, u, p=rng.uniform(0.05, 1, 48).astype(np.float32), least=[0.1] * 48)
    check_ids(np.zeros((8, 777), np.float32), u[:8], k=[1, 2, 3, 500, 776, 777, 778, 0])


def test_sample_infinite_and_missing_logits():
    x = np.full((9, 300), -np.inf, np.float32)
    x[1, 7] = 1.0
    x[2, [3, 9]] = np.nan, -2.0
    x[3, [5, 6]] = np.inf, 3.0
    x[4, [10, 20, 30]] = np.inf
    x[5, :] = np.nan
    x[6, :] = 3.4e38
    x[7, [1, 2]] = 3e38, -3e38
    x[8, :] = -3.4e38
    for t in (0.0, 1.0, 1e-30, math.inf, math.nan, -1.0):
        check_ids(x, [0.5, 0.99, 0.0, 0.3, 0.7, 0.5, 0.999, 0.5, 0.25], t=[t] * 9, k=[2] * 9, p=[0.9] * 9)
        check_ids(x, [0.5, 0.99, 0.0, 0.3, 0.7, 0.5, 0.999, 0.5, 0.25], t=[t] * 9)


def test_sample_without_shares():
    x = np.random.default_rng(9).normal(size=(3, 500)).astype(np.float32)
    d, u, ids = dev(x), dev([0.1, 0.5, 0.9], np.float32), torch.zeros(3, dtype=torch.int32, device="cuda:0")
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    G.sample_dev(ids.data_ptr(), d.data_ptr(), 3, 500, u.data_ptr(), stream=st.cuda_stream)
    st.synchronize()
    assert ids.tolist() == [sample(x[r], u[r].item(), 1.0, 0, 1.0, 0.0)[0] for r in range(3)]


def test_nothing_to_do_is_no_error():
    cache = Cache(G.TYPE_F16, 2, 16, 1, 64)
    data, gc = on_gpu(cache)
    t = torch.zeros(64, device="cuda:0")
    p = t.data_ptr()
    G.kv_write_dev(gc, p, p, p, 0)
    G.kv_read_dev(gc, p, p, p, 0)
    G.sample_dev(p, p, 0, 10, p)
    a = G.Attention(gc, heads=1, max_tokens=4, scale=1.0)
    ws = torch.zeros(a.workspace_bytes, dtype=torch.uint8, device="cuda:0")
    a(p, p, 0, 0, p, p, 1, ws.data_ptr(), ws.numel(), q_start_ptr=p)
    with pytest.raises(G.GoInferCudaError) as e:
        a(p, p, 1, 1, p, p, 1, ws.data_ptr(), ws.numel() - 1)
    assert e.value.code == G.ERR_SHAPE and "workspace" in str(e.value)
    torch.cuda.synchronize()
    assert not data.any() and not t.any()


def test_sample_borders_of_u_and_parameters():
    rng = np.random.default_rng(3)
    x = rng.normal(size=(8, 1234)).astype(np.float32)
    u = [0.0, 1 - 2.0 ** -24, 1.0, 2.0, -1.0, 0.5, 0.5, 0.5]
    check_ids(x, u, p=[1.0, 1.0, 1.0, 0.9, 0.9, -1.0, 0.0, 1e-9], least=[0, 0, 0, 0, 0, 0, 5.0, -1.0])


def test_sample_shares_follow_the_distribution():
    """With u on a fine grid the picks' counts are the shares themselves (each within one step)."""
    x = np.tile(np.array([[0.0, 1.0, -1.0, 2.0, 0.5]], np.float32), (1000, 1))
    ids, _ = draw_ids(x, ((np.arange(1000) + 0.5) / 1000).astype(np.float32))
    w = np.exp(x[0].astype(np.float64))
    assert np.all(np.abs(np.bincount(ids, minlength=5) - 1000 * w / w.sum()) <= 1.0)


# ---- together -------------------------------------------------------------------------

@pytest.mark.parametrize("kind", KINDS)
def test_a_batch_is_served_step_by_step(kind):
    """Prompts of unequal lengths written and attended in one call, then single-token steps whose write, attention
    and pick are one captured graph: the cached rows, the attention and the ids follow the plain forms."""
    rng = np.random.default_rng(30)
    heads, kv, dim, page, vocab, seqs = 8, 2, 64, 16, 500, 3
    prompts, steps = [21, 1, 40], 4
    n_pages = 16
    cache = Cache(kind, n_pages, page, kv, dim)
    data, gc = on_gpu(cache)
    table = rng.permutation(n_pages)[:3 * 4].reshape(3, 4).astype(np.int32)
    freqs, m = G.rope_freqs(dim, 10000.0)
    fr = dev(freqs)
    rope = G.Rope(dim, fr.data_ptr(), mscale=m)
    st = torch.cuda.Stream()
    att = G.Attention(gc, heads=heads, max_tokens=sum(prompts), max_q_len=max(prompts), scale=dim ** -0.5)
    one = G.Attention(gc, heads=heads, max_tokens=seqs, scale=dim ** -0.5)
    ws = torch.empty(max(att.workspace_bytes, one.workspace_bytes, 1), dtype=torch.uint8, device="cuda:0")
    head = rng.normal(size=(heads * dim, vocab)).astype(np.float32)  # stands for the rest of the model
    table_d = dev(table)
    width = (heads + 2 * kv) * dim

    def slots_of(b, positions):
        return [int(table[b, p // page]) * page + p % page for p in positions]

    def step(new, lens, qkv, bufs, call):
        pos = [p for b in range(seqs) for p in range(lens[b] - new[b], lens[b])]
        slots = [x for b in range(seqs) for x in slots_of(b, range(lens[b] - new[b], lens[b]))]
        for name, a in (("qkv", qkv), ("pos", np.array(pos, np.int32)), ("slots", np.array(slots, np.int32)),
                        ("len", np.array(lens, np.int32)), ("start", np.concatenate(([0], np.cumsum(new))).astype(np.int32))):
            bufs[name].copy_(dev(a))
        torch.cuda.synchronize()
        call()
        torch.cuda.synchronize()
        back(cache, data)
        q, _ = turned(qkv[:, :heads * dim].reshape(-1, heads, dim), pos, freqs, dim, False, 1.0)
        assert np.abs(bufs["q"].cpu().numpy() - q).max() <= 2.0 ** -20
        want, bound = attention(cache, bufs["q"].cpu().numpy(), np.concatenate(([0], np.cumsum(new))), lens, table,
                                dim ** -0.5)
        assert (np.abs(bufs["out"].cpu().numpy() - want).max(-1) <= bound).all()

    def make(n):
        d = dict(qkv=torch.zeros(n, width, device="cuda:0"), pos=torch.zeros(n, dtype=torch.int32, device="cuda:0"),
                 slots=torch.zeros(n, dtype=torch.int32, device="cuda:0"),
                 len=torch.zeros(seqs, dtype=torch.int32, device="cuda:0"),
                 start=torch.zeros(seqs + 1, dtype=torch.int32, device="cuda:0"),
                 q=torch.zeros(n, heads, dim, device="cuda:0"), out=torch.zeros(n, heads, dim, device="cuda:0"))
        base = d["qkv"].data_ptr()

        def call(a):
            G.kv_write_dev(gc, base + 4 * heads * dim, base + 4 * (heads + kv) * dim, d["slots"].data_ptr(), n,
                           k_stride=width, v_stride=width, q_ptr=base, q_out_ptr=d["q"].data_ptr(), heads=heads,
                           q_stride=width, positions_ptr=d["pos"].data_ptr(), rope=rope, stream=st.cuda_stream)
            a(d["out"].data_ptr(), d["q"].data_ptr(), seqs, n, d["len"].data_ptr(), table_d.data_ptr(), 4, ws.data_ptr(),
              ws.numel(), q_start_ptr=d["start"].data_ptr(), stream=st.cuda_stream)
        return d, call

    lens = list(prompts)
    bufs, call = make(sum(prompts))
    step(prompts, lens, rng.normal(size=(sum(prompts), width)).astype(np.float32), bufs, lambda: call(att))
    bufs, call = make(seqs)
    w, u = dev(head), torch.zeros(seqs, device="cuda:0")
    logits = torch.zeros(seqs, vocab, device="cuda:0")
    ids = torch.zeros(seqs, dtype=torch.int32, device="cuda:0")
    temp, p = dev([0.7, 1.3, 0.0], np.float32), dev([0.9, 1.0, 1.0], np.float32)
    torch.mm(bufs["out"].view(seqs, -1), w, out=logits)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        call(one)
        torch.mm(bufs["out"].view(seqs, -1), w, out=logits)
        G.sample_dev(ids.data_ptr(), logits.data_ptr(), seqs, vocab, u.data_ptr(), temperature_ptr=temp.data_ptr(),
                     top_p_ptr=p.data_ptr(), stream=st.cuda_stream)
    for _ in range(steps):
        lens = [n + 1 for n in lens]
        u.copy_(torch.from_numpy(rng.random(seqs, np.float32)))
        step([1] * seqs, lens, rng.normal(size=(seqs, width)).astype(np.float32), bufs, graph.replay)
        x = logits.cpu().numpy()
        for r in range(seqs):
            assert ids[r].item() == sample(x[r], u[r].item(), [0.7, 1.3, 0.0][r] and float(np.float32([0.7, 1.3, 0.0][r])),
                                           0, [0.9, 1.0, 1.0][r], 0.0)[0]


# ---- the model's own paths ----------------------------------------------------------------

@pytest.fixture(scope="module")
def model_host():
    import synth
    cfg = synth.LlamaConfig(n_layers=2, dim=512, hidden=1024, n_heads=8, n_kv_heads=2, vocab=1000, max_seq=48)
    return synth.synth_model(cfg, seed=11)


@pytest.fixture()
def model(model_host):
    import synth
    dev = synth.DeviceModel(model_host)
    m = dev.model()
    yield m
    m.close()
    dev.close()


PROMPT = [3, 141, 59, 26, 535]


def test_model_samples_from_its_logits(model):
    """Step by step, each pick follows the rule from the logits the step returns; one call of all steps picks the same."""
    u = np.random.default_rng(5).random(12, np.float32)
    kw = dict(temperature=0.9, top_k=50, top_p=0.95, min_p=0.01)
    ids, _, _ = model.generate_sampled(PROMPT, u, **kw)
    model.reset()
    tokens, pos, got = list(PROMPT), 0, []
    for x in u:
        one, logits, _ = model.generate_sampled(tokens, [x], start_pos=pos, want_logits=True, **kw)
        assert one[0] == sample(logits, float(x), float(np.float32(0.9)), 50, 0.95, 0.01)[0]
        pos += len(tokens)
        tokens = [int(one[0])]
        got.append(int(one[0]))
    assert got == ids.tolist() and len(set(got)) > 3


def test_model_sampled_without_choice_is_greedy(model):
    greedy, logits, _ = model.generate(PROMPT, 20, want_logits=True)
    for kw in (dict(temperature=0.0), dict(top_k=1), dict(top_p=0.0), dict(min_p=1.0)):
        model.reset()
        ids, x, _ = model.generate_sampled(PROMPT, np.full(20, 0.999, np.float32), want_logits=True, **kw)
        assert np.array_equal(ids, greedy) and np.array_equal(x, logits)
    model.reset()
    assert np.array_equal(model.generate(PROMPT, 20)[0], greedy)


@pytest.mark.parametrize("kind,tol", [(G.TYPE_F16, 2.0 ** -8), (G.TYPE_Q8_0, 2.0 ** -4)])
def test_model_with_a_small_cache(model, kind, tol):
    """Logits of the F16 / Q8_0 cache near the float32 cache's, also past the cache's end (rolling).

    A cached value is off by 2^-11 of itself (F16) or by 1/254 of its block's largest, about 2^-6.5 of a
    typical value (Q8_0).  Through V that is the attention output's error; through K it moves a score by as
    much of its size (about 1 here) and so a weight by as much: twice 2^-11, or 2^-6.5 and less after
    averaging, per layer of 2, of an output that is then added to a residual of its size."""
    tokens = np.random.default_rng(7).integers(0, 1000, 70)
    for n in (1, 33, 70):
        model.set_kv_cache(G.TYPE_F32)
        _, want, _ = model.generate(tokens[:n], 1, want_logits=True)
        model.set_kv_cache(kind)
        first, got, _ = model.generate(tokens[:n], 1, want_logits=True)
        assert np.sqrt(np.mean((got - want) ** 2)) <= tol * np.sqrt(np.mean(want ** 2))
        model.reset()
        again, same, _ = model.generate(tokens[:n], 1, want_logits=True)
        assert np.array_equal(same, got) and first[0] == again[0] == np.argmax(got)


def test_model_cache_refusals(model, model_host):
    for kind in (2, G.TYPE_Q4_K):
        with pytest.raises(G.GoInferCudaError) as e:
            model.set_kv_cache(kind)
        assert e.value.code == G.ERR_UNSUPPORTED_TYPE
    model.set_kv_cache(G.TYPE_Q8_0)
    with pytest.raises(G.GoInferCudaError) as e:
        model.set_persistent(True)
    assert e.value.code == G.ERR_UNSUPPORTED_TYPE and "float32 cache" in str(e.value)
    model.set_kv_cache(G.TYPE_F32)
    model.set_persistent(True)
    with pytest.raises(G.GoInferCudaError) as e:
        model.set_kv_cache(G.TYPE_F16)
    assert e.value.code == G.ERR_UNSUPPORTED_TYPE
    greedy, _, _ = model.generate(PROMPT, 5)
    model.reset()
    assert np.array_equal(model.generate_sampled(PROMPT, np.zeros(5, np.float32), top_k=1)[0], greedy)
    model.set_persistent(False)
    with pytest.raises(G.GoInferCudaError):
        model.generate_sampled([], [0.5])
    import synth
    cfg = synth.LlamaConfig(n_layers=1, dim=256, hidden=512, n_heads=8, n_kv_heads=2, vocab=300, max_seq=16)
    dev = synth.DeviceModel(synth.synth_model(cfg, seed=3))  # heads of 32
    m = dev.model()
    with pytest.raises(G.GoInferCudaError) as e:
        m.set_kv_cache(G.TYPE_F16)
    assert e.value.code == G.ERR_SHAPE
    assert len(m.generate([1, 2], 3)[0]) == 3
    m.close()
    dev.close()
