"""The paged-cache operators without a GPU: refusals, sizes and frequencies, and the tests' own plain forms."""
import math

import numpy as np
import pytest

import goinfer_cuda as G
import _precision
from _serve import Cache, sample

CACHE = dict(type=G.TYPE_Q8_0, n_pages=4, page_size=16, n_kv_heads=2, head_dim=64)
A = 1 << 20  # addresses that no call may follow: every one of these calls is refused


def cache(**kw):
    d = {**CACHE, "data_ptr": A, **kw}
    size = G.load_library().gi_kv_cache_bytes(G.TYPE_F16, 4, 16, 2, 64) * 4
    c = G.KVCache.__new__(G.KVCache)
    c.desc = G.KVCacheDesc(d["type"], d["n_pages"], d["page_size"], d["n_kv_heads"], d["head_dim"], d["data_ptr"],
                           d.get("nbytes", size))
    c._p = G.ctypes.addressof(c.desc)
    c.n_kv_heads, c.head_dim, c.buf = d["n_kv_heads"], d["head_dim"], None
    return c


def refused(code, what, call, *a, **kw):
    with pytest.raises(G.GoInferCudaError) as e:
        call(*a, **kw)
    assert e.value.code == code and what in str(e.value), str(e.value)


@pytest.mark.parametrize("kind,pages,page,kv,dim", [(G.TYPE_F16, 3, 16, 2, 64), (G.TYPE_Q8_0, 5, 64, 3, 96),
                                                    (G.TYPE_Q8_0, 1, 16, 1, 32), (G.TYPE_F16, 7, 1024, 8, 256)])
def test_cache_bytes(kind, pages, page, kv, dim):
    assert G.load_library().gi_kv_cache_bytes(kind, pages, page, kv, dim) == Cache(kind, pages, page, kv, dim).data.size


@pytest.mark.parametrize("kw", [dict(type=0), dict(type=G.TYPE_Q4_K), dict(n_pages=0), dict(page_size=8), dict(page_size=48),
                                dict(page_size=1 << 17), dict(n_kv_heads=0), dict(n_kv_heads=1025), dict(head_dim=0),
                                dict(head_dim=48), dict(head_dim=288), dict(n_pages=1 << 28)])
def test_cache_shapes_that_are_refused(kw):
    d = {**CACHE, **kw}
    assert G.load_library().gi_kv_cache_bytes(*(d[k] for k in ("type", "n_pages", "page_size", "n_kv_heads", "head_dim"))) == -1
    with pytest.raises(G.GoInferCudaError):
        G.KVCache(**d)
    code = G.ERR_UNSUPPORTED_TYPE if "type" in kw else G.ERR_SHAPE
    refused(code, "cache", G.kv_read_dev, cache(**kw), A, A, A, 1)


def test_cache_data_that_is_refused():
    refused(G.ERR_BUFFER, "cache data", G.kv_read_dev, cache(data_ptr=None), A, A, A, 1)
    refused(G.ERR_BUFFER, "cache data", G.kv_read_dev, cache(nbytes=100), A, A, A, 1)
    refused(G.ERR_SHAPE, "256-byte", G.kv_read_dev, cache(data_ptr=A + 16), A, A, A, 1)


def test_a_closed_cache_is_refused():
    """Its buffer is gone: a call afterwards must not follow the address."""
    c = G.KVCache(G.TYPE_F16, 4, 16, 2, 64, data_ptr=A, nbytes=1 << 20)
    c.buf = G.Buffer(0, 1 << 20)  # as if the cache had made it
    c.close()
    refused(G.ERR_BUFFER, "cache data", G.kv_read_dev, c, A, A, A, 1)
    c.close()
    own = G.KVCache(G.TYPE_F16, 4, 16, 2, 64, data_ptr=A, nbytes=1 << 20)
    own.close()  # the caller's memory stays the caller's
    assert own.desc.data == A


def test_write_refusals():
    c, w = cache(), G.kv_write_dev
    rope = G.Rope(64, A)
    refused(G.ERR_SHAPE, "null", w, c, 0, A, A, 1)
    refused(G.ERR_SHAPE, "null", w, c, A, 0, A, 1)
    refused(G.ERR_SHAPE, "null", w, c, A, A, 0, 1)
    refused(G.ERR_SHAPE, "null", w, c, A, A, A, 1, q_ptr=A, heads=4)
    refused(G.ERR_SHAPE, "n_heads", w, c, A, A, A, 1, q_ptr=A, q_out_ptr=A)
    refused(G.ERR_SHAPE, "n_heads", w, c, A, A, A, 1, q_ptr=A, q_out_ptr=A, heads=1025)
    refused(G.ERR_SHAPE, "aligned", w, c, A + 4, A, A, 1)
    refused(G.ERR_SHAPE, "aligned", w, c, A, A, A, 1, k_stride=129)
    refused(G.ERR_SHAPE, "aligned", w, c, A, A, A, 1, q_ptr=A, q_out_ptr=A + 8, heads=2)
    refused(G.ERR_SHAPE, "shorter", w, c, A, A, A, 2, v_stride=64)
    refused(G.ERR_SHAPE, "freqs", w, c, A, A, A, 1, rope=rope)
    refused(G.ERR_SHAPE, "freqs", w, c, A, A, A, 1, positions_ptr=A, rope=G.Rope(64, 0))
    refused(G.ERR_SHAPE, "even", w, c, A, A, A, 1, positions_ptr=A, rope=G.Rope(66, A))
    refused(G.ERR_SHAPE, "even", w, c, A, A, A, 1, positions_ptr=A, rope=G.Rope(33, A))


def test_read_refusals():
    refused(G.ERR_SHAPE, "null", G.kv_read_dev, cache(), 0, A, A, 1)
    refused(G.ERR_SHAPE, "aligned", G.kv_read_dev, cache(), A, A + 4, A, 1)


def test_token_counts_that_are_refused():
    """Up to 2^30 tokens: a launch adds blocks to them in 32 bits, and near 2^31 it divided by zero."""
    c = cache()
    for n in ((1 << 30) + 1, (1 << 31) - 1, 1 << 31, (1 << 32) - 1):
        refused(G.ERR_SHAPE, "too many tokens", G.kv_write_dev, c, A, A, A, n)
        refused(G.ERR_SHAPE, "too many tokens", G.kv_read_dev, c, A, A, A, n)


def attention(c, **kw):
    d = {**dict(heads=4, max_tokens=8, max_q_len=4, scale=0.125, prefix_len=0), **kw}
    a = G.Attention.__new__(G.Attention)
    a.cache = c
    a.desc = G.AttnDesc(d["heads"], d["max_tokens"], d["max_q_len"], d["prefix_len"], d["scale"])
    a._p = G.ctypes.addressof(a.desc)
    G.load_library()
    return a


def test_attention_refusals():
    c = cache()
    args = (A, A, 2, 8, A, A, 3, A, 1 << 30)
    for kw, what in ((dict(heads=0), "n_heads"), (dict(heads=3), "n_heads"), (dict(heads=2048), "n_heads"),
                     (dict(max_tokens=0), "max_tokens"), (dict(max_q_len=0), "max_tokens"), (dict(max_q_len=9), "max_tokens"),
                     (dict(prefix_len=65), "prefix")):
        refused(G.ERR_SHAPE, what, attention(c, **kw), *args, q_start_ptr=A)
        refused(G.ERR_SHAPE, what, G.Attention, c, **{**dict(heads=4, max_tokens=8, max_q_len=4, scale=0.125), **kw})
    refused(G.ERR_SHAPE, "head dims", attention(cache(head_dim=32)), *args, q_start_ptr=A)
    a = attention(c)
    refused(G.ERR_SHAPE, "null", a, 0, *args[1:], q_start_ptr=A)
    refused(G.ERR_SHAPE, "null", attention(c, prefix_len=20), *args, q_start_ptr=A)
    refused(G.ERR_SHAPE, "more tokens", a, A, A, 2, 9, A, A, 3, A, 1 << 30, q_start_ptr=A)
    refused(G.ERR_SHAPE, "more sequences", a, A, A, 9, 8, A, A, 3, A, 1 << 30, q_start_ptr=A)
    refused(G.ERR_SHAPE, "without q_start", a, *args)
    refused(G.ERR_SHAPE, "pages_stride", a, A, A, 2, 8, A, A, 0, A, 1 << 30, q_start_ptr=A)
    refused(G.ERR_SHAPE, "pages_stride", a, A, A, 2, 8, A, A, 1 << 28, A, 1 << 30, q_start_ptr=A)
    refused(G.ERR_SHAPE, "aligned", a, A + 4, *args[1:], q_start_ptr=A)


def test_lengths_whose_last_tile_would_pass_32_bits_are_refused():
    """The kernels compare the end of a tile of up to 128 positions with the length in 32 bits."""
    c, args = cache(), (A, A, 2, 8, A, A)
    for stride in ((1 << 27) - 1, (1 << 27) - 15):  # pages of 16
        refused(G.ERR_SHAPE, "pages_stride", attention(c), *args, stride, A, 1 << 30, q_start_ptr=A)
    big = cache(n_pages=(1 << 27) - 1, nbytes=1 << 62)
    refused(G.ERR_SHAPE, "prefix", attention(big, prefix_len=(1 << 31) - 17), *args, 3, A, 1 << 30, q_start_ptr=A)


def test_sample_refusals():
    s = G.sample_dev
    refused(G.ERR_SHAPE, "vocab", s, A, A, 1, 0, A)
    refused(G.ERR_SHAPE, "vocab", s, A, A, 1, (1 << 20) + 1, A)
    refused(G.ERR_SHAPE, "null", s, 0, A, 1, 10, A)
    refused(G.ERR_SHAPE, "null", s, A, A, 1, 10, 0)
    refused(G.ERR_SHAPE, "stride", s, A, A, 2, 10, A, logits_stride=9)


def test_rope_frequency_refusals():
    for kw in (dict(dim=0), dict(dim=7), dict(theta=0.0), dict(theta=math.nan), dict(scaling=G.ROPE_LINEAR, factor=0.0),
               dict(scaling=G.ROPE_YARN, factor=2.0, low=4.0, high=4.0), dict(scaling=G.ROPE_LLAMA3, factor=2.0, orig_ctx=0.0)):
        refused(G.ERR_SHAPE, "rotary", G.rope_freqs, **{**dict(dim=8, theta=1e4), **kw})
    refused(G.ERR_UNSUPPORTED_TYPE, "scaling", G.rope_freqs, 8, 1e4, scaling=4)


def test_rope_frequencies():
    plain, m = G.rope_freqs(128, 10000.0)
    i = np.arange(64)
    assert m == 1.0 and np.allclose(plain, 10000.0 ** (-2 * i / 128), rtol=1e-15)
    assert np.allclose(G.rope_freqs(128, 10000.0, G.ROPE_LINEAR, 4.0)[0], plain / 4, rtol=1e-15)
    f, m = G.rope_freqs(128, 500000.0, G.ROPE_LLAMA3, 8.0, 1.0, 4.0, 8192.0)
    base, _ = G.rope_freqs(128, 500000.0)
    wave = 2 * math.pi / base
    assert m == 1.0 and np.array_equal(f[wave < 2048], base[wave < 2048])
    assert np.allclose(f[wave > 8192], base[wave > 8192] / 8, rtol=1e-15)
    mid = (wave > 2048) & (wave < 8192)
    assert mid.any() and ((f < base) & (f > base / 8))[mid].all() and (np.diff(f) < 0).all()
    f, m = G.rope_freqs(128, 10000.0, G.ROPE_YARN, 16.0, 1.0, 32.0, 4096.0)
    turns = 4096 * plain / (2 * math.pi)
    assert m == pytest.approx(0.1 * math.log(16) + 1, rel=1e-15)
    assert np.array_equal(f[turns > 40], plain[turns > 40]) and np.allclose(f[turns < 0.8], plain[turns < 0.8] / 16, rtol=1e-15)
    assert (np.diff(f) < 0).all()


def test_plain_sampler_draws_the_shares():
    """The tests' oracle: exact shares of a small row, each filter on its own."""
    x = [0.0, 1.0, -math.inf, 2.0, 1.0, math.nan]
    w = np.exp([0.0, 1.0, 2.0, 1.0])
    grid = [(i + 0.5) / 4000 for i in range(4000)]
    got = np.bincount([sample(x, u, 1.0, 0, 1.0, 0.0)[0] for u in grid], minlength=6)
    assert got[2] == got[5] == 0 and np.all(np.abs(got[[0, 1, 3, 4]] - 4000 * w / w.sum()) <= 1)
    assert {sample(x, u, 1.0, 2, 1.0, 0.0)[0] for u in grid} == {1, 3}  # of the equal ones the lower index
    assert {sample(x, u, 1.0, 0, 0.5, 0.0)[0] for u in grid} == {3}
    assert {sample(x, u, 1.0, 0, 1.0, 0.3)[0] for u in grid} == {1, 3, 4}
    assert sample(x, 0.9, 0.0, 0, 1.0, 0.0) == (3, 1.0) and sample([-math.inf] * 3, 0.5, 1.0, 0, 1.0, 0.0) == (-1, 0.0)


def test_model_refusals_without_a_model():
    lib = G.load_library()
    assert lib.gi_cuda_model_set_kv_cache(None, G.TYPE_F16) == G.ERR_SHAPE
    assert lib.gi_cuda_model_set_kv_cache(None, 2) == G.ERR_UNSUPPORTED_TYPE
    toks, out = (G.ctypes.c_int32 * 1)(1), (G.ctypes.c_uint32 * 1)()
    u = (G.ctypes.c_float * 1)(0.5)
    assert lib.gi_cuda_model_generate_sampled(None, toks, 1, 0, 1, 1.0, 0, 1.0, 0.0, u, out, None, None) == G.ERR_SHAPE


@pytest.mark.parametrize("kind", _precision.KINDS)
@pytest.mark.parametrize("shape", _precision.SHAPES)
def test_one_half_of_an_operand_misses_the_precision(kind, shape):
    """What the GPU's test of these cases would see if q, or the weights, were held in one half."""
    c = _precision.Case(kind, *shape)
    want, tol = c.out(), c.tolerance()
    assert _precision.off(c.out(q=_precision.half), want) > 2 * tol
    assert _precision.off(c.out(p=_precision.half), want) > 2 * tol
