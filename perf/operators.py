"""Cases and plain forms of the operators that serve tokens from a paged KV cache.

Four operators: ``write`` (rotary positions, then q out and k, v into the cache), ``read`` (cached rows
back to float32), ``attn`` (ragged attention over the cache, with a prefix that the batch shares) and
``sample`` (temperature, top-k, top-p, min-p from given uniforms).  Where ``own`` is false ``run``
computes them from elementary torch operations; where it is true it makes the calls of
go-infer_b200/goinfer_cuda.py.

The cache is one block of bytes: the K values [page][kv head][offset][head_dim], the V values likewise,
then for Q8_0 the K and the V scales [page][kv head][offset][head_dim / 32] (fp16); each of the parts
starts on a multiple of 256 bytes.  A Q8_0 value is code * scale rounded to half precision.
"""
import math
import os
import random
import sys

import torch

own = False

F16, Q8_0 = 1, 8
ONE = 2.0 ** 42  # a weight of 1 in the sampler's fixed point


# ---- cases ---------------------------------------------------------------------

def listed():
    return [
        # One decoded token of a 7B-shaped layer: 32 heads of 128, the latency of a step.
        dict(name="write_token", op="write", type=Q8_0, tokens=1, heads=32, kv_heads=32, dim=128, page=64, rot=128,
             interleaved=False, scaling="none", far=4096),
        # A ragged batch of prompt tokens, part of each head rotated, adjacent pairs, linear scaling.
        dict(name="write_batch_partial", op="write", type=Q8_0, tokens=1111, heads=32, kv_heads=8, dim=128, page=16,
             rot=64, interleaved=True, scaling="linear", far=16384),
        # Prefill of a 70B-shaped layer (64 query, 8 kv heads) into a half-precision cache, long-context frequencies.
        dict(name="write_prefill", op="write", type=F16, tokens=8191, heads=64, kv_heads=8, dim=128, page=64, rot=128,
             interleaved=False, scaling="llama3", far=131072),
        # Cached rows handed back: a short suffix, then a long context (moved to another place, or inspected).
        dict(name="read_few", op="read", type=F16, tokens=37, kv_heads=8, dim=64, page=16),
        dict(name="read_context", op="read", type=Q8_0, tokens=30011, kv_heads=8, dim=128, page=64),
        # One token against 4096 cached ones, every query head with a kv head of its own (7B shape).
        dict(name="attn_token", op="attn", type=Q8_0, seqs=1, heads=32, kv_heads=32, dim=128, page=64, q_max=1, lo=4096,
             hi=4096, prefix=0, pad=0),
        # A decoding batch of unequal requests, 70B shape; two padding rows behind the last one.
        dict(name="attn_decode_batch", op="attn", type=Q8_0, seqs=62, heads=64, kv_heads=8, dim=128, page=64, q_max=1,
             lo=1, hi=8192, prefix=0, pad=2),
        # Samples of one long prompt: 48 sequences share 6000 tokens, each has up to 700 of its own.
        dict(name="attn_shared_prefix", op="attn", type=F16, seqs=48, heads=32, kv_heads=8, dim=128, page=16, q_max=1,
             lo=0, hi=700, prefix=6000, pad=0),
        # Prompt chunks (and single tokens) of several requests in one call, causal inside each chunk.
        dict(name="attn_chunks", op="attn", type=Q8_0, seqs=7, heads=32, kv_heads=8, dim=128, page=64, q_max=512, lo=300,
             hi=4000, prefix=0, pad=0),
        # One row of a 32000-word head, and a decoding batch of a 128256-word head whose rows ask for different filters.
        dict(name="sample_row", op="sample", rows=1, vocab=32000, spread=3.0, mix=False),
        dict(name="sample_batch", op="sample", rows=64, vocab=128256, spread=3.0, mix=True),
        # An odd vocabulary, flat rows: nothing stands out, the filters cut deep inside.
        dict(name="sample_flat", op="sample", rows=17, vocab=50257, spread=0.5, mix=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = [work(c) for c in listed()]
    while True:
        case = _drawn(rng)
        w = work(case)
        if all(w[k] <= max(m[k] for m in most) for k in w):
            return case


def _drawn(rng):
    op = rng.choice(["write", "write", "read", "attn", "attn", "attn", "sample", "sample"])
    kind = rng.choice([F16, Q8_0])
    page = rng.choice([16, 32, 64, 128])
    if op == "write":
        dim = rng.choice([64, 96, 128, 256])
        kv = rng.choice([1, 2, 4, 8, 32])
        return dict(op=op, type=kind, tokens=_log(rng, 1, 8000), heads=kv * (1 if kv == 32 else rng.choice([1, 2, 4, 7, 8])),
                    kv_heads=kv, dim=dim, page=page, rot=rng.choice([dim, dim, dim // 2]), interleaved=rng.random() < 0.5,
                    scaling=rng.choice(["none", "linear", "llama3", "yarn"]), far=_log(rng, 5000, 1000000))
    if op == "read":
        return dict(op=op, type=kind, tokens=_log(rng, 1, 30000), kv_heads=rng.choice([1, 2, 8, 8]),
                    dim=rng.choice([64, 96, 128]), page=page)
    if op == "sample":
        return dict(op=op, rows=_log(rng, 1, 64), vocab=_log(rng, 200, 128256), spread=round(rng.uniform(0.3, 5.0), 3),
                    mix=rng.random() < 0.7)
    dim = rng.choice([64, 96, 128, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 5, 8])
    form = rng.choice(["decode", "decode", "prefix", "chunk"])
    seqs = _log(rng, 1, 64) if form != "chunk" else rng.randint(1, 7)
    hi = _log(rng, 20, max(40, min(16384, 300000 // seqs)))
    return dict(op=op, type=kind, seqs=seqs, heads=kv * group, kv_heads=kv, dim=dim, page=page,
                q_max={"decode": 1, "prefix": rng.choice([1, 1, 3]), "chunk": _log(rng, 2, 400)}[form],
                lo=rng.choice([0, 1, max(1, hi // 2)]), hi=hi, prefix=_log(rng, 17, 6000) if form == "prefix" else 0,
                pad=rng.choice([0, 0, 3]))


def _plan(case):
    """Lengths of the sequences of an attention case and how many new tokens each has: they follow from the case."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    lens = [r.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    lens[r.randrange(len(lens))] = case["hi"]
    new = [1 if case["q_max"] == 1 or r.random() < 0.2 else r.randint(1, case["q_max"]) for _ in lens]
    new[r.randrange(len(new))] = case["q_max"]
    return lens, new


# ---- inputs --------------------------------------------------------------------

def _parts(case, n_pages):
    """Byte offsets of the K and V values and scales in the cache block, and its size."""
    n = n_pages * case["kv_heads"] * case["page"] * case["dim"]
    up = lambda b: -(-b // 256) * 256  # noqa: E731
    val = up(n * (2 if case["type"] == F16 else 1))
    sc = up(n // 32 * 2) if case["type"] == Q8_0 else 0
    return [0, val, 2 * val, 2 * val + sc], 2 * (val + sc)


def _views(case, data, n_pages):
    """The cache block's parts as tensors."""
    at, _ = _parts(case, n_pages)
    shape = (n_pages, case["kv_heads"], case["page"], case["dim"])
    n = math.prod(shape)
    if case["type"] == F16:
        return [data[a:a + 2 * n].view(torch.float16).view(shape) for a in at[:2]] + [None, None]
    blocks = shape[:3] + (case["dim"] // 32,)
    return ([data[a:a + n].view(torch.int8).view(shape) for a in at[:2]]
            + [data[a:a + n // 16].view(torch.float16).view(blocks) for a in at[2:]])


def _cache(case, n_pages, gen, filled):
    """A cache of n_pages pages in use plus one that nothing may read: its values are not numbers."""
    data = torch.zeros(_parts(case, n_pages)[1], dtype=torch.uint8, device="cuda")
    parts = _views(case, data, n_pages)
    if filled:
        for x, s in zip(parts[:2], parts[2:]):
            if s is None:
                x.copy_(torch.randn(x.shape, generator=gen, device="cuda", dtype=torch.float32))
            else:
                x.copy_((torch.randn(x.shape, generator=gen, device="cuda") * 42).clamp(-127, 127))
                s.copy_(torch.rand(s.shape, generator=gen, device="cuda") * 0.03 + 0.008)
    for x in parts[2:] if case["type"] == Q8_0 else parts[:2]:
        x[n_pages - 1] = float("nan")
    return data


def _frequencies(case, dim, theta=500000.0):
    """Angle per position of each rotated pair (64 bits) and the factor on cos and sin."""
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    f = theta ** (-i / dim)
    if case["scaling"] == "linear":
        return f / 4.0, 1.0
    if case["scaling"] == "llama3":
        factor, low, high, old = 8.0, 1.0, 4.0, 8192.0
        wave = 2 * math.pi / f
        mid = (old / wave - low) / (high - low)
        g = torch.where(wave > old / low, f / factor, (1 - mid) * f / factor + mid * f)
        return torch.where(wave < old / high, f, g), 1.0
    if case["scaling"] == "yarn":
        factor, fast, slow, old = 16.0, 32.0, 1.0, 8192.0
        turn = lambda n: dim * math.log(old / (n * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        lo, hi = max(math.floor(turn(fast)), 0), min(math.ceil(turn(slow)), dim - 1)
        ramp = ((torch.arange(dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    s = {"case": case, "stream": torch.cuda.Stream()}
    if case["op"] == "sample":
        r = random.Random(seed)
        n = case["rows"]
        s["logits"] = rnd(n, case["vocab"]) * case["spread"]
        s["u"] = torch.rand(n, generator=gen, device="cuda")
        pick = lambda *v: [r.choice(v) if case["mix"] else v[0] for _ in range(n)]  # noqa: E731
        dev = lambda v, t: torch.tensor(v, dtype=t, device="cuda")  # noqa: E731
        s["temperature"] = dev(pick(0.8, 1.0, 0.3, 1.7, 0.0), torch.float32)
        s["top_k"] = dev(pick(40, 0, 1, 1000, 5), torch.int32)
        s["top_p"] = dev(pick(0.95, 1.0, 0.5, 0.9), torch.float32)
        s["min_p"] = dev(pick(0.05, 0.0, 0.0, 0.01), torch.float32)
        s["ids"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        s["prob"] = torch.zeros(n, device="cuda")
        return s
    kv, dim, page = case["kv_heads"], case["dim"], case["page"]
    if case["op"] in ("write", "read"):
        n = case["tokens"]
        n_pages = -(-n // page) + 3
        s["n_pages"], s["data"] = n_pages, _cache(case, n_pages, gen, case["op"] == "read")
        order = torch.randperm(n_pages - 1, generator=gen, device="cuda")  # a sequence's pages lie anywhere
        t = torch.arange(n, device="cuda")
        s["slots"] = (order[t // page] * page + t % page).to(torch.int32)
        if n > 8:
            s["slots"][torch.randint(0, n, (n // 9,), generator=gen, device="cuda")] = -1  # padding tokens
        s["k_out"], s["v_out"] = torch.zeros(n, kv, dim, device="cuda"), torch.zeros(n, kv, dim, device="cuda")
        if case["op"] == "read":
            return s
        qkv = rnd(n, (case["heads"] + 2 * kv) * dim)  # one projection's output: q, k and v are columns of it
        s["q"] = qkv[:, :case["heads"] * dim]
        s["k"], s["v"] = qkv[:, case["heads"] * dim:].split(kv * dim, dim=1)
        s["q_out"] = torch.zeros(n, case["heads"], dim, device="cuda")
        s["positions"] = torch.randint(0, case["far"], (n,), generator=gen, device="cuda", dtype=torch.int32)
        f, s["mscale"] = _frequencies(case, case["rot"])
        s["freqs"] = f.to("cuda")
        return s
    lens, new = _plan(case)
    shared = -(-case["prefix"] // page)
    n_pages = sum(-(-n // page) for n in lens) + shared + 3
    s["n_pages"], s["data"] = n_pages, _cache(case, n_pages, gen, True)
    order = torch.randperm(n_pages - 1, generator=gen, device="cuda").to(torch.int32).cpu().tolist()
    width = max(1, -(-max(lens) // page))
    table, at = [], shared
    for n in lens:
        need = -(-n // page)
        table.append(order[at:at + need] + [n_pages - 1] * (width - need))
        at += need
    dev = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    s["tokens"] = start[-1] + case["pad"]
    s["table"], s["kv_len"], s["q_start"] = dev(table), dev(lens), dev(start)
    s["prefix_pages"] = dev(order[:shared]) if shared else None
    s["q"] = rnd(s["tokens"], case["heads"], dim)
    s["out"] = torch.ones(s["tokens"], case["heads"], dim, device="cuda")
    return s


# ---- plain forms ---------------------------------------------------------------

def _values(x, scale):
    """What cached values stand for, in float32."""
    if scale is None:
        return x.float()
    return (x.float() * scale.float().repeat_interleave(32, dim=-1)).half().float()


def _turn(x, cos, sin, rot, interleaved):
    """x [n, heads, dim] with its first `rot` dimensions rotated."""
    part, rest = x[..., :rot], x[..., rot:]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :rot // 2], part[..., rot // 2:])
    r0, r1 = a * cos - b * sin, a * sin + b * cos
    r = torch.stack((r0, r1), dim=-1).flatten(-2) if interleaved else torch.cat((r0, r1), dim=-1)
    return torch.cat((r, rest), dim=-1)


def _q8(x):
    """Codes and fp16 scales of 32 values each: the largest over 127, its mantissa cut off, halves away from zero."""
    b = x.reshape(x.shape[:-1] + (-1, 32))
    d = b.abs().amax(-1) / torch.tensor(127.0, device=x.device)
    cut = (d.contiguous().view(torch.int32) & -8192).view(torch.float32)  # fp16's 10 bits of mantissa
    d = torch.where(d < 2.0 ** -14, torch.floor(d * 2.0 ** 24) * 2.0 ** -24, cut)
    inv = torch.where(d > 0, torch.ones_like(d) / d, torch.zeros_like(d))
    v = (b * inv[..., None]).clamp(-128, 127).double()
    return (torch.sign(v) * torch.floor(v.abs() + 0.5)).to(torch.int8).reshape(x.shape), d.half()


def _at(case, slots):
    page = case["page"]
    return torch.div(slots, page, rounding_mode="floor").long(), (slots % page).long()


def _plain_read(s, parts):
    case = s["case"]
    use = (s["slots"] >= 0).nonzero()[:, 0]
    p, o = _at(case, s["slots"][use])
    k, v = s["k_out"].clone(), s["v_out"].clone()
    for x, val, scale in ((k, parts[0], parts[2]), (v, parts[1], parts[3])):
        x[use] = _values(val[p, :, o], None if scale is None else scale[p, :, o])
    return k, v


def _plain_write(s):
    case = s["case"]
    n, dim = case["tokens"], case["dim"]
    angle = s["positions"].double()[:, None, None] * s["freqs"]
    cos, sin = (angle.cos() * s["mscale"]).float(), (angle.sin() * s["mscale"]).float()
    q, k = (_turn(x.reshape(n, -1, dim), cos, sin, case["rot"], case["interleaved"]) for x in (s["q"], s["k"]))
    v = s["v"].reshape(n, -1, dim)
    parts = _views(case, s["data"], s["n_pages"])
    use = (s["slots"] >= 0).nonzero()[:, 0]
    p, o = _at(case, s["slots"][use])
    for x, val, scale in ((k, parts[0], parts[2]), (v, parts[1], parts[3])):
        if scale is None:
            val[p, :, o] = x[use].clamp(-65504, 65504).half()
        else:
            val[p, :, o], scale[p, :, o] = _q8(x[use].clamp(-65504, 65504))
    if case["type"] == F16:
        return {"q": q, "k": parts[0][:-1], "v": parts[1][:-1]}
    k, v = _plain_read(s, parts)
    return {"q": q, "k": k, "v": v}


def _dense(case, s, table):
    """K and V values of the pages that `table` [..., pages] names: [..., kv_heads, tokens, dim]."""
    parts = _views(case, s["data"], s["n_pages"])
    got = []
    for x, scale in ((parts[0], parts[2]), (parts[1], parts[3])):
        t = table.long()
        y = _values(x[t], None if scale is None else scale[t])
        y = y.movedim(-3, -4)  # kv heads before pages
        got.append(y.flatten(-3, -2))
    return got


def _plain_attn(s):
    case = s["case"]
    kv, dim, page = case["kv_heads"], case["dim"], case["page"]
    n = case["seqs"]
    start, lens = s["q_start"].long(), s["kv_len"].long()
    new = start[1:] - start[:-1]
    j = torch.arange(case["q_max"], device="cuda")
    real = j < new[:, None]
    tok = torch.where(real, start[:-1, None] + j, 0)
    q = s["q"][tok].view(n, case["q_max"], kv, -1, dim).movedim(1, 3)  # [n, kv, group, q_max, dim]
    group = q.shape[2]
    q = q.reshape(n, kv, group * case["q_max"], dim)
    k, v = _dense(case, s, s["table"])
    width = k.shape[2]
    seen = torch.arange(width, device="cuda") < (lens - new)[:, None, None] + j[:, None] + 1  # [n, q_max, width]
    inside = torch.arange(width, device="cuda") < lens[:, None]
    k, v = (torch.where(inside[:, None, :, None], x, 0) for x in (k, v))
    score = (q @ k.transpose(-1, -2) * dim ** -0.5).view(n, kv, group, case["q_max"], width)
    score = score.masked_fill(~(seen & inside[:, None, :])[:, None, None], -math.inf)
    if case["prefix"]:
        pk, pv = (x[:, :case["prefix"]] for x in _dense(case, s, s["prefix_pages"]))
        first = (q @ pk.transpose(-1, -2) * dim ** -0.5).view(n, kv, group, case["q_max"], case["prefix"])
        score = torch.cat((first, score), dim=-1)
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = w.sum(-1, keepdim=True)
    w = (w / torch.where(total > 0, total, torch.ones_like(total))).view(n, kv, group * case["q_max"], -1)
    o = w[..., case["prefix"]:] @ v
    if case["prefix"]:
        o = o + w[..., :case["prefix"]] @ pv
    o = o.view(n, kv, group, case["q_max"], dim).movedim(3, 1).reshape(n, case["q_max"], kv * group, dim)
    out = s["out"].clone()
    out[tok[real]] = o[real]
    return out


def _plain_sample(s):
    x = s["logits"]
    n, vocab = x.shape
    at = torch.arange(vocab, device="cuda")
    can = x > -math.inf  # not a number: no candidate either
    x = torch.where(can, x, -math.inf)
    top = x.amax(1, keepdim=True)
    first = torch.where(can & (x == top), at, vocab).amin(1)
    t = s["temperature"].double()[:, None]
    w = torch.exp((x.double() - top.double()) / torch.where(t > 0, t, 1.0))
    w = torch.where(top == math.inf, (x == top).double(), w)
    w = torch.round(torch.where(can, w, 0.0) * ONE).long()
    order = torch.sort(x, dim=1, descending=True, stable=True)[1]
    ws = w.gather(1, order)
    k = s["top_k"].long()[:, None]
    ws = torch.where((at < k) | (k <= 0), ws, 0)
    p = s["top_p"].double()[:, None]
    need = torch.ceil(p * ws.sum(1, keepdim=True).double()).long().clamp(min=1)
    ws = torch.where((ws.cumsum(1) - ws < need) | (p >= 1), ws, 0)
    floor = torch.ceil(s["min_p"].double()[:, None].clamp(0, 1) * ONE).long()
    ws = torch.where(ws >= floor, ws, 0)
    w = torch.zeros_like(ws).scatter_(1, order, ws)
    cum = w.cumsum(1)
    total = cum[:, -1]
    u = s["u"].double().clamp(0, 1 - 2.0 ** -24)
    want = torch.floor(u * total.double()).long()
    pick = (cum <= want[:, None]).sum(1).clamp(max=vocab - 1)
    prob = w.gather(1, pick[:, None])[:, 0].double() / total.clamp(min=1).double()
    greedy = ~(s["temperature"] > 0)
    some = can.any(1)
    ids = torch.where(greedy, first, pick)
    prob = torch.where(greedy, 1.0, prob)
    return {"ids": torch.where(some, ids, -1).int(), "prob": torch.where(some, prob, 0.0).float()}


# ---- the framework's calls -----------------------------------------------------

def _own(s):
    at = os.path.join(os.getcwd(), "go-infer_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import goinfer_cuda as G

    case = s["case"]
    st = s["stream"].cuda_stream
    if case["op"] == "sample":
        if "bound" not in s:
            G.Init(torch.cuda.current_device())
            s["bound"] = True
        G.sample_dev(s["ids"].data_ptr(), s["logits"].data_ptr(), case["rows"], case["vocab"], s["u"].data_ptr(),
                     temperature_ptr=s["temperature"].data_ptr(), top_k_ptr=s["top_k"].data_ptr(),
                     top_p_ptr=s["top_p"].data_ptr(), min_p_ptr=s["min_p"].data_ptr(), prob_ptr=s["prob"].data_ptr(),
                     stream=st)
        return {"ids": s["ids"], "prob": s["prob"]}
    if "cache" not in s:  # handles that a program makes once
        G.Init(torch.cuda.current_device())
        s["cache"] = G.KVCache(case["type"], s["n_pages"], case["page"], case["kv_heads"], case["dim"],
                               data_ptr=s["data"].data_ptr(), nbytes=s["data"].numel())
        if case["op"] == "write":
            s["rope"] = G.Rope(case["rot"], s["freqs"].data_ptr(), interleaved=case["interleaved"], mscale=s["mscale"])
        if case["op"] == "attn":
            s["call"] = G.Attention(s["cache"], heads=case["heads"], max_tokens=s["tokens"], max_q_len=case["q_max"],
                                    scale=case["dim"] ** -0.5, prefix_len=case["prefix"])
            s["work"] = torch.empty(max(s["call"].workspace_bytes, 1), dtype=torch.uint8, device="cuda")
    cache = s["cache"]
    if case["op"] == "attn":
        s["call"](s["out"].data_ptr(), s["q"].data_ptr(), case["seqs"], s["tokens"], s["kv_len"].data_ptr(),
                  s["table"].data_ptr(), s["table"].shape[1], s["work"].data_ptr(), s["work"].numel(),
                  q_start_ptr=s["q_start"].data_ptr(),
                  prefix_pages_ptr=s["prefix_pages"].data_ptr() if case["prefix"] else 0, stream=st)
        return s["out"]
    if case["op"] == "write":
        stride = s["q"].stride(0)
        G.kv_write_dev(cache, s["k"].data_ptr(), s["v"].data_ptr(), s["slots"].data_ptr(), case["tokens"],
                       k_stride=stride, v_stride=stride, q_ptr=s["q"].data_ptr(), q_out_ptr=s["q_out"].data_ptr(),
                       heads=case["heads"], q_stride=stride, positions_ptr=s["positions"].data_ptr(), rope=s["rope"],
                       stream=st)
        if case["type"] == F16:
            k, v = _views(case, s["data"], s["n_pages"])[:2]
            return {"q": s["q_out"], "k": k[:-1], "v": v[:-1]}
    G.kv_read_dev(cache, s["k_out"].data_ptr(), s["v_out"].data_ptr(), s["slots"].data_ptr(), case["tokens"], stream=st)
    r = {"k": s["k_out"], "v": s["v_out"]}
    return {"q": s["q_out"], **r} if case["op"] == "write" else r


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "sample":
        return _plain_sample(state)
    if op == "attn":
        return _plain_attn(state)
    if op == "write":
        return _plain_write(state)
    k, v = _plain_read(state, _views(state["case"], state["data"], state["n_pages"]))
    return {"k": k, "v": v}


# ---- what a pass cannot do without -----------------------------------------------

def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 28 * case["rows"], "flops": 4 * n}
    row = case["kv_heads"] * case["dim"]  # values of a token's K
    held = row * (2 if case["type"] == F16 else 1 + 2 / 32)  # bytes they take in the cache
    if case["op"] == "read":
        return {"bytes": case["tokens"] * (2 * held + 8 * row + 4), "flops": 2 * case["tokens"] * row}
    if case["op"] == "write":
        n, q = case["tokens"], case["heads"] * case["dim"]
        back = 2 * held + 8 * row if case["type"] == Q8_0 else 0  # Q8_0 rows are read back
        return {"bytes": n * (8 * q + 8 * row + 2 * held + 8 + back), "flops": n * (3 * q + 8 * row)}
    lens, new = _plan(case)
    tokens = sum(new)
    seen = sum(max(0, n - m + i + 1) for n, m in zip(lens, new) for i in range(m)) + tokens * case["prefix"]
    return {"bytes": (sum(lens) + case["prefix"]) * 2 * held + 8 * tokens * case["heads"] * case["dim"],
            "flops": 4 * case["heads"] * case["dim"] * seen}


# ---- the operators in 64 bits, by their definitions --------------------------------

def _exact_values(case, s):
    parts = _views(case, s["data"], s["n_pages"])
    if case["type"] == F16:
        return [x.double() for x in parts[:2]]
    wide = lambda c, d: (c.double().unflatten(-1, (-1, 32)) * d.double()[..., None]).flatten(-2)  # noqa: E731
    return [wide(c, d).half().double() for c, d in ((parts[0], parts[2]), (parts[1], parts[3]))]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "sample":
        return _exact_sample(s)
    if op == "read":
        k, v = s["k_out"].double(), s["v_out"].double()
        for out, x in zip((k, v), _exact_values(case, s)):
            flat = x.movedim(1, 2).flatten(0, 1)  # by slot
            use = s["slots"] >= 0
            out[use] = flat[s["slots"][use].long()]
        return {"k": k, "v": v}
    if op == "write":  # what is rounded to a few bits in the cache has no 64-bit value
        q = s["q"].double().unflatten(1, (case["heads"], case["dim"])).clone()
        half = case["rot"] // 2
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
            e = torch.polar(torch.full_like(s["positions"], 1, dtype=torch.float64) * s["mscale"],
                            s["positions"].double() * s["freqs"][i])
            z = torch.complex(q[..., a], q[..., b]) * e[:, None]
            q[..., a], q[..., b] = z.real, z.imag
        return {"q": q, "k": None, "v": None}
    K, V = _exact_values(case, s)
    lens, new = _plan(case)
    out = s["out"].double()
    group = case["heads"] // case["kv_heads"]
    rows = lambda x, pages, n: x[pages.long()].movedim(0, 1).flatten(1, 2)[:, :n]  # noqa: E731
    at = 0
    for b, (n, m) in enumerate(zip(lens, new)):
        k, v = rows(K, s["table"][b], n), rows(V, s["table"][b], n)
        if case["prefix"]:
            k = torch.cat((rows(K, s["prefix_pages"], case["prefix"]), k), 1)
            v = torch.cat((rows(V, s["prefix_pages"], case["prefix"]), v), 1)
        for h in range(case["heads"]):
            x = s["q"][at:at + m, h].double() @ k[h // group].T / math.sqrt(case["dim"])
            last = case["prefix"] + n - m + torch.arange(m, device="cuda")
            hide = torch.arange(k.shape[1], device="cuda") > last[:, None]
            out[at:at + m, h] = torch.softmax(x.masked_fill(hide, -math.inf), -1).nan_to_num(0.0) @ v[h // group]
        at += m
    return out


def _exact_sample(s):
    ids, prob = [], []
    rows = [s[k].tolist() for k in ("temperature", "top_k", "top_p", "min_p", "u")]
    for x, t, k, p, least, u in zip(s["logits"].double(), *rows):
        x = x.nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        top, i = x.max(0)
        if top == -math.inf:
            ids.append(-1), prob.append(0.0)
            continue
        if not t > 0:
            ids.append(int((x == top).nonzero()[0, 0])), prob.append(1.0)
            continue
        y, order = torch.sort(x, descending=True, stable=True)
        w = torch.round(torch.exp((y - top) / t) * ONE).long()
        if k > 0:
            w, order = w[:k], order[:k]
        if p < 1:
            need = max(1, math.ceil(p * float(w.sum())))
            m = int((w.cumsum(0) < need).sum()) + 1
            w, order = w[:m], order[:m]
        m = max(1, int((w >= math.ceil(min(max(least, 0.0), 1.0) * ONE)).sum()))
        w, order = w[:m], order[:m]
        order, back = order.sort()
        w = w[back]
        c = w.cumsum(0)
        at = min(int((c <= math.floor(min(max(u, 0.0), 1 - 2.0 ** -24) * float(c[-1]))).sum()), len(c) - 1)
        ids.append(int(order[at])), prob.append(int(w[at]) / int(c[-1]))
    return {"ids": torch.tensor(ids, dtype=torch.int32), "prob": torch.tensor(prob, dtype=torch.float64)}
