"""The causal text model in 8 bits, as a caller of libhexanima_hip.so drives it: its operators in plain torch and through the
C-ABI, on the same inputs.

  quant   hxa_quantize_rows        activations (or weights) to int8 with a scale for each row
  linear  hxa_linear_i8            product of int8 activations and weights, scales for each token and each channel
  append  hxa_kv_append_q8         new keys (normed and rotated on the way) and values into a paged cache of int8 with a scale for each page and head
  cached  hxa_attention_cached_q8  new tokens over that cache, behind a prefix that the whole batch shares

What is held in 8 bits is returned as the values it stands for, in the type of the operator's 16-bit operands; quant and append form them with one
more elementwise pass over what they wrote, the same on both sides. Kernel calls go to torch's current stream.
"""
import ctypes as C
import math
import random

import torch

own = False  # True: run() makes the framework's calls; False: the operators' plain form

DEV = "cuda"
F64 = torch.float64
DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
TINY = 2.0 ** -64  # the least scale of a page that holds a value other than 0


# ----------------------------------------------------------------------------------------------------------------- cases
# quant: M rows of K. linear: M tokens, K -> N channels, bias or not. append, cached: query heads Hq, key / value heads Hk, head width hd, T new
# tokens of nseq sequences (their lengths follow from the salt); past: tokens already in the sequences' own pages, over the batch; prefix:
# tokens of the shared prefix; page: tokens a page; rot, layout: the rotated part of a head and its pairs.
def listed():
    return [
        # the hidden state of one new token
        dict(name="quant_step_1", op="quant", dtype="bf16", M=1, K=2048),
        # the MLP's activations of a batch of prompts, rows that fill no tile
        dict(name="quant_mlp_6500", op="quant", dtype="f16", M=6500, K=8192),
        # the fused qkv of one new token: 16 query heads and 8 key heads of 128
        dict(name="linear_step_1", op="linear", dtype="f16", M=1, K=2048, N=4096, bias=True),
        # a decoding step of 64 sequences through the MLP-down
        dict(name="linear_step_64", op="linear", dtype="bf16", M=64, K=8192, N=2048, bias=False),
        # one image prompt of an ordinary length behind its template, the MLP-down: long K, few tiles
        dict(name="linear_down_1000", op="linear", dtype="bf16", M=1000, K=8192, N=2048, bias=False),
        # a batch of prompts through the fused MLP up and gate
        dict(name="linear_up_6500", op="linear", dtype="f16", M=6500, K=2048, N=16384, bias=False),
        # a decoding step of 64 sequences: one new key and value each, most into pages that hold earlier tokens
        dict(name="append_step_64", op="append", dtype="bf16", Hq=32, Hk=8, hd=128, T=64, nseq=64, past=3000, prefix=1000,
             page=16, salt=1, rot=128, layout="half"),
        # 23 prompts of very different lengths go into the cache
        dict(name="append_prompts_9001", op="append", dtype="f16", Hq=16, Hk=8, hd=128, T=9001, nseq=23, past=1500, prefix=0,
             page=64, salt=2, rot=128, layout="half"),
        # one new token of one sequence
        dict(name="cached_step_1", op="cached", dtype="f16", Hq=16, Hk=8, hd=128, T=1, nseq=1, past=700, prefix=0, page=16,
             salt=1),
        # a decoding step of 64 sequences behind a 4096-token instruction
        dict(name="cached_step_64", op="cached", dtype="bf16", Hq=32, Hk=8, hd=128, T=64, nseq=64, past=30000, prefix=4096,
             page=64, salt=2),
        # 32 image prompts read behind one 1000-token template: the rest of each prompt attends to both
        dict(name="cached_prompts_32", op="cached", dtype="f16", Hq=16, Hk=8, hd=128, T=2400, nseq=32, past=0, prefix=1000,
             page=16, salt=3),
        # a decoding step of 16 long sequences behind a very long shared document
        dict(name="cached_long_16", op="cached", dtype="bf16", Hq=32, Hk=8, hd=128, T=16, nseq=16, past=90000, prefix=32768,
             page=64, salt=4),
    ]


HEADS = [(16, 8), (32, 8), (16, 16), (20, 4), (8, 1), (40, 8), (12, 12), (10, 2), (28, 4), (14, 2)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        m = most.setdefault(c["op"], dict(w))
        for k in w:
            m[k] = max(m[k], w[k])
    while True:
        op = rng.choice(["quant", "linear", "linear", "append", "cached", "cached"])
        c = dict(op=op, dtype=rng.choice(["f16", "bf16"]))
        if op == "quant":
            c |= dict(M=_log(rng, 1, 16384), K=_log(rng, 64, 16384))
        elif op == "linear":
            K = _log(rng, 128, 16384)
            c |= dict(M=_log(rng, 1, 8192), K=K if rng.random() < 0.3 else max(128, K // 128 * 128), N=8 * _log(rng, 16, 2048),
                      bias=rng.random() < 0.4)
        else:
            Hq, Hk = rng.choice(HEADS)
            hd = rng.choice([64, 128, 128, 256])
            step = rng.random() < 0.5  # one token a sequence, or pieces of prompts
            nseq = _log(rng, 1, 128)
            T = nseq if step else _log(rng, nseq, 8192)
            past = _log(rng, 1, 2000 if op == "cached" else 100) * nseq if step or rng.random() < 0.4 else 0
            c |= dict(Hq=Hq, Hk=Hk, hd=hd, T=T, nseq=nseq, past=past, prefix=rng.choice([0, _log(rng, 16, 16384)]) if op == "cached" else
                      rng.choice([0, 100]), page=rng.choice([1, 16, 16, 32, 64, 128]), salt=rng.randint(0, 999))
            if op == "append":
                c |= dict(rot=16 * rng.randint(1, hd // 16) if rng.random() < 0.5 else hd, layout=rng.choice(["half", "half", "pairs"]))
        w = work(c)
        if w["bytes"] <= most[op]["bytes"] and w["flops"] <= most[op]["flops"]:
            return c


def _split(total, n, salt, least=0):
    """total into n parts of very different sizes, each at least `least`"""
    r = random.Random(salt * 7919 + n)
    w = [r.expovariate(1.0) + 0.02 for _ in range(n)]
    free = total - least * n
    cut = [int(free * sum(w[:i]) / sum(w)) for i in range(n)] + [free]
    return [least + cut[i + 1] - cut[i] for i in range(n)]


def _lengths(c):
    """(new tokens, tokens already there) of each sequence"""
    new = [1] * c["nseq"] if c["T"] == c["nseq"] else _split(c["T"], c["nseq"], c["salt"], 1)
    past = _split(c["past"], c["nseq"], c["salt"] + 1) if c.get("past") else [0] * c["nseq"]
    return new, past


def work(case):
    c = dict(case)
    if c["op"] == "quant":
        return {"bytes": 3.0 * c["M"] * c["K"] + 4.0 * c["M"], "flops": 3.0 * c["M"] * c["K"]}
    if c["op"] == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        return {"bytes": float(M * K + N * K + 2 * M * N + 4 * (M + N)), "flops": 2.0 * M * N * K}
    T, Hq, Hk, hd = c["T"], c["Hq"], c["Hk"], c["hd"]
    if c["op"] == "append":
        return {"bytes": 6.0 * T * Hk * hd, "flops": 12.0 * T * Hk * hd}
    new, past = _lengths(c)
    pairs = sum(n * (p + (n + 1) / 2) for n, p in zip(new, past)) + T * c["prefix"]
    keys = sum(new) + sum(past) + c["prefix"]
    return {"bytes": hd * (4.0 * T * Hq + 2.0 * keys * Hk), "flops": 4.0 * pairs * Hq * hd}


# ---------------------------------------------------------------------------------------------------------------- inputs
class State:
    pass


def _gen(seed, salt=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1000003 + salt)
    return g


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * std).to(dtype)


def _freq(c):
    """radians a position of each pair, theta 10000 (heads of 256: 1000000)"""
    i = torch.arange(c["rot"] // 2, dtype=F64)
    return ((1e6 if c["hd"] == 256 else 1e4) ** (-2.0 * i / c["rot"])).float().to(DEV)


def _ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def _round128(n):
    return (n + 127) // 128 * 128


def _bytes_of(x):
    """rows of values as int8 rows, padded with zeros to a multiple of 128, and their scales"""
    s = x.abs().amax(-1) / 127
    q = torch.zeros(x.shape[0], _round128(x.shape[1]), dtype=torch.int8, device=DEV)
    q[:, :x.shape[1]] = torch.round(x / s[:, None]).to(torch.int8)
    return q, s


def _pool(g, *shape):
    """pages of earlier tokens: int8 whose largest value is about four times their spread, and the pages' scales"""
    q = torch.randn(*shape, generator=g, device=DEV).mul_(31).round_().clamp_(-127, 127).to(torch.int8)
    return q, torch.exp(torch.randn(*shape[:2], generator=g, device=DEV) * 0.2) / 31


def _inputs(c, seed):
    s = State()
    g = _gen(seed)
    dt = DTYPE[c["dtype"]]
    s.case = c
    if c["op"] == "quant":
        # activations: a few channels much wider than the others
        wide = torch.exp(torch.randn(c["K"], generator=g, device=DEV))
        s.x = (torch.randn(c["M"], c["K"], generator=g, device=DEV) * wide).to(dt)
        return s
    if c["op"] == "linear":
        s.a, s.sa = _bytes_of(_randn(g, c["M"], c["K"]))
        s.w, s.sw = _bytes_of(_randn(g, c["N"], c["K"], std=0.02))
        s.bias = _randn(g, c["N"], std=0.1) if c["bias"] else None
        return s
    T, Hq, Hk, hd = c["T"], c["Hq"], c["Hk"], c["hd"]
    s.scale = hd ** -0.5
    s.new, s.past = _lengths(c)
    cu = [0]
    for n in s.new:
        cu.append(cu[-1] + n)
    s.cu_host, s.cu = cu, _ints(cu)
    page, P = c["page"], c["prefix"]
    s.len_host = [n + p for n, p in zip(s.new, s.past)]
    own_pages = [(n + page - 1) // page for n in s.len_host]
    nprefix = (P + page - 1) // page
    s.npages = nprefix + sum(own_pages) + 3
    s.ldt = max(own_pages)
    order = list(range(s.npages))
    random.Random(int(seed) + 17).shuffle(order)  # pages in the order in which a pool hands them out
    s.prefix = _ints(order[:nprefix] or [0])
    table = torch.full((c["nseq"], s.ldt), -1, dtype=torch.int32)
    at = nprefix
    for i, n in enumerate(own_pages):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    s.table, s.len = table.to(DEV), _ints(s.len_host)
    s.kc, s.ks = _pool(g, s.npages, Hk, page, hd)
    s.vc, s.vs = _pool(g, s.npages, Hk, page, hd)
    if c["op"] == "cached":
        s.q = _randn(g, T, Hq * hd, std=1.5, dtype=dt)
    else:
        # columns of one projection's rows, q | k | v
        s.qkv = _randn(g, T, (Hq + 2 * Hk) * hd, dtype=dt)
        s.k, s.v = s.qkv[:, Hq * hd:(Hq + Hk) * hd], s.qkv[:, (Hq + Hk) * hd:]
        s.gk = 1.0 + _randn(g, hd, std=0.1)
        s.freq = _freq(c)
    return s


def prepare(case, seed):
    c = dict(case)
    s = _inputs(c, seed)
    dt = DTYPE[c["dtype"]]
    if c["op"] == "quant":
        s.q = torch.empty(c["M"], _round128(c["K"]), dtype=torch.int8, device=DEV)
        s.sc = torch.empty(c["M"], dtype=torch.float32, device=DEV)
        s.o = torch.empty(c["M"], c["K"], dtype=dt, device=DEV)
    elif c["op"] == "linear":
        s.o = torch.empty(c["M"], c["N"], dtype=dt, device=DEV)
    elif c["op"] == "cached":
        s.o = torch.empty(c["T"], c["Hq"] * c["hd"], dtype=dt, device=DEV)
    else:
        s.ko, s.vo = torch.empty(s.kc.shape, dtype=dt, device=DEV), torch.empty(s.vc.shape, dtype=dt, device=DEV)
    if own:
        from hexanima_amd import hip

        hip.init(0)
        s.dt = hip.DT_F16 if c["dtype"] == "f16" else hip.DT_BF16
        if c["op"] == "linear":
            s.ws_bytes = hip.lib().hxa_linear_i8_ws_bytes(c["M"], c["N"], c["K"])
        if c["op"] == "append":
            s.rope = hip.Rope(s.freq.data_ptr(), c["rot"], hip.ROPE_HALF if c["layout"] == "half" else hip.ROPE_PAIRS, 1.0)
        if c["op"] in ("append", "cached"):
            plan = hip.KvCache(s.dt, c["Hk"], c["hd"], c["page"], s.npages, s.kc.data_ptr(), s.vc.data_ptr(), s.prefix.data_ptr(),
                               c["prefix"], s.table.data_ptr(), s.ldt, s.len.data_ptr(), s.cu.data_ptr(), c["nseq"])
            s.cache = hip.KvCacheQ8(plan, s.ks.data_ptr(), s.vs.data_ptr())
        if c["op"] == "cached":
            s.ws_bytes = hip.lib().hxa_attention_cached_q8_ws_bytes(C.byref(s.cache), c["T"], c["Hq"])
        if c["op"] in ("linear", "cached"):
            s.ws = torch.empty(max(s.ws_bytes, 16), dtype=torch.uint8, device=DEV)
    return s


# ------------------------------------------------------------------------------------------------------------ plain form
def _norm_rope(x, H, gain, pos, freq, layout):
    """per-head RMSNorm * gain, then the rotation, in 32 bits; the angles of far positions in 64"""
    T, hd = x.shape[0], x.shape[1] // H
    u = x.float().reshape(T, H, hd)
    u = u * torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS) * gain
    r = freq.numel()
    th = pos.to(F64)[:, None] * freq.to(F64)
    cs, sn = torch.cos(th).float()[:, None], torch.sin(th).float()[:, None]
    a, b = (u[..., :r], u[..., r:2 * r]) if layout == "half" else (u[..., 0:2 * r:2], u[..., 1:2 * r:2])
    ra, rb = a * cs - b * sn, a * sn + b * cs
    rotated = torch.cat([ra, rb], -1) if layout == "half" else torch.stack([ra, rb], -1).view(T, H, 2 * r)
    return torch.cat([rotated, u[..., 2 * r:]], -1)


def _slots(s):
    """page, row and own position of each new token"""
    page = s.case["page"]
    seq = torch.repeat_interleave(torch.arange(s.case["nseq"], device=DEV), s.cu[1:] - s.cu[:-1], output_size=s.case["T"])
    t = torch.arange(s.case["T"], device=DEV)
    p = s.len[seq].long() - (s.cu[seq + 1] - t)
    return s.table[seq, p // page].long(), p % page, p


def _into_pages(pool, scale, x, pg, row):
    """rows x [T][H][hd] into rows `row` of pages `pg`: a page that held earlier rows keeps its scale or takes the least 2^j of it that the new
    rows fit, its values shifted by j bits; another page takes its largest value / 127"""
    n, H, page, _ = pool.shape
    first = torch.full((n,), page, device=DEV).index_reduce_(0, pg, row, "amin")  # rows of each page before the call's
    need = torch.zeros(n, H, device=DEV).index_reduce_(0, pg, x.abs().amax(-1), "amax") / 127
    need = torch.where(need > 0, need.clamp(min=TINY), need)
    old = torch.where((first > 0)[:, None], scale, 0.0)
    m, e = torch.frexp(need / old.clamp(min=TINY))
    j = torch.where((old > 0) & (need > old), e - (m == 0.5).int(), 0)
    new = torch.where(old > 0, torch.ldexp(old, j), need)
    touched = first < page
    scale.copy_(torch.where(touched[:, None], new, scale))
    held = touched[:, None] & (torch.arange(page, device=DEV) < first[:, None])  # rows behind the call's stay as they are
    pool.copy_(torch.where(held[:, None, :, None], torch.round(torch.ldexp(pool.float(), -j[:, :, None, None])), pool).to(torch.int8))
    inv = torch.where(new > 0, 1.0 / new, 0.0)[pg]
    pool[pg, :, row] = torch.round(x * inv[..., None]).clamp(-127, 127).to(torch.int8)


def _soft(sc):
    e = sc.sub_(sc.amax(-1, keepdim=True)).exp_()
    return e.div_(e.sum(-1, keepdim=True))


def _attend(q, keys, vals, G, scale, first, o):
    """rows of q at key positions first, first + 1, ... over keys [n][Hk][hd]; o gets the rounded rows"""
    n, Hk, hd = keys.shape
    kt = keys.permute(1, 2, 0).contiguous()
    v = vals.transpose(0, 1).contiguous()
    for t in range(0, q.shape[0], 1024):
        m = min(1024, q.shape[0] - t)
        e = min(n, first + t + m)
        x = q[t:t + m].reshape(m, Hk, G, hd).permute(1, 2, 0, 3).float().reshape(Hk, G * m, hd)
        sc = (torch.matmul(x, kt[:, :, :e]) * scale).view(Hk, G, m, e)
        late = torch.arange(e, device=DEV) > torch.arange(first + t, first + t + m, device=DEV)[:, None]
        pr = _soft(sc.masked_fill_(late, -math.inf)).view(Hk, G * m, e)
        o[t:t + m] = torch.matmul(pr, v[:, :e]).view(Hk, G, m, hd).permute(2, 0, 1, 3).reshape(m, Hk * G, hd).to(o.dtype)


def _gather(pool, scale, pages, n):
    """tokens 0 .. n - 1 of the given pages as rows [n][H][hd] of values"""
    x = pool[pages.long()].float() * scale[pages.long()][:, :, None, None]
    return x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])[:n]


def _plain(s):
    c = s.case
    dt = DTYPE[c["dtype"]]
    if c["op"] == "quant":
        x = s.x.float()
        top = x.abs().amax(-1)
        sc = top / 127
        q = torch.round(x * torch.where(top > 0, 127 / top, 0.0)[:, None]).clamp(-127, 127).to(torch.int8)
        return [(q * sc[:, None]).to(dt), sc]
    if c["op"] == "linear":
        o = torch.matmul(s.a.float(), s.w.float().t()) * s.sa[:, None] * s.sw
        return (o if s.bias is None else o + s.bias).to(dt)
    T, Hq, Hk, hd = c["T"], c["Hq"], c["Hk"], c["hd"]
    if c["op"] == "append":
        pg, row, p = _slots(s)
        _into_pages(s.kc, s.ks, _norm_rope(s.k, Hk, s.gk, p + c["prefix"], s.freq, c["layout"]), pg, row)
        _into_pages(s.vc, s.vs, s.v.float().reshape(T, Hk, hd), pg, row)
        return _cache(s)
    o, q = s.o.view(T, Hq, hd), s.q.view(T, Hq, hd)
    pk, pv = _gather(s.kc, s.ks, s.prefix, c["prefix"]), _gather(s.vc, s.vs, s.prefix, c["prefix"])
    for i, (b, e) in enumerate(zip(s.cu_host, s.cu_host[1:])):
        n = s.len_host[i]
        pages = s.table[i, :(n + c["page"] - 1) // c["page"]]
        keys, vals = torch.cat([pk, _gather(s.kc, s.ks, pages, n)]), torch.cat([pv, _gather(s.vc, s.vs, pages, n)])
        _attend(q[b:e], keys, vals, Hq // Hk, s.scale, c["prefix"] + s.past[i], o[b:e])
    return s.o


def _cache(s):
    """the cache's values, and its scales"""
    torch.mul(s.kc, s.ks[:, :, None, None], out=s.ko)
    torch.mul(s.vc, s.vs[:, :, None, None], out=s.vo)
    return [s.ko, s.vo, s.ks, s.vs]


# ------------------------------------------------------------------------------------------------------------------- run
def run(s):
    if not own:
        return _plain(s)
    from hexanima_amd import hip

    L, c = hip.lib(), s.case
    st = torch.cuda.current_stream().cuda_stream
    if c["op"] == "quant":
        hip.check(L.hxa_quantize_rows(s.dt, s.x.data_ptr(), s.x.stride(0), c["M"], c["K"], s.q.data_ptr(), s.q.stride(0), s.sc.data_ptr(),
                                      st), "quantize_rows")
        torch.mul(s.q[:, :c["K"]], s.sc[:, None], out=s.o)
        return [s.o, s.sc]
    if c["op"] == "linear":
        hip.check(L.hxa_linear_i8(s.dt, s.a.data_ptr(), s.a.stride(0), s.sa.data_ptr(), c["M"], s.w.data_ptr(), s.w.stride(0),
                                  s.sw.data_ptr(), c["N"], c["K"], s.bias.data_ptr() if c["bias"] else None, s.o.data_ptr(), c["N"],
                                  s.ws.data_ptr(), s.ws_bytes, st), "linear_i8")
        return s.o
    T, Hq, hd = c["T"], c["Hq"], c["hd"]
    if c["op"] == "append":
        hip.check(L.hxa_kv_append_q8(C.byref(s.cache), s.k.data_ptr(), s.k.stride(0), s.v.data_ptr(), s.v.stride(0), T, s.gk.data_ptr(), EPS,
                                     C.byref(s.rope), st), "kv_append_q8")
        return _cache(s)
    hip.check(L.hxa_attention_cached_q8(C.byref(s.cache), s.q.data_ptr(), Hq * hd, s.o.data_ptr(), Hq * hd, T, Hq, s.scale, s.ws.data_ptr(),
                                        s.ws_bytes, st), "attention_cached_q8")
    return s.o


# ----------------------------------------------------------------------------------------------------------------- exact
def _turn(x, H, gain, pos, freq, layout):
    """the norm and the rotation in 64 bits, pairs as complex numbers"""
    T, hd, r = x.shape[0], x.shape[1] // H, freq.numel()
    u = x.to(F64).reshape(T, H, hd)
    u = u / torch.sqrt(torch.sum(u ** 2, -1, keepdim=True) / hd + EPS) * gain.to(F64)
    w = torch.polar(torch.ones(T, r, dtype=F64, device=DEV), torch.outer(pos.to(F64), freq.to(F64)))[:, None]
    re, im = (slice(0, r), slice(r, 2 * r)) if layout == "half" else (slice(0, 2 * r, 2), slice(1, 2 * r, 2))
    z = torch.complex(u[..., re], u[..., im]) * w
    u = u.clone()
    u[..., re], u[..., im] = z.real, z.imag
    return u


def _page_in(q, s, r, x):
    """rows x [n][H][hd] behind the r rows that a page holds: the page's values [H][r + n][hd] and its scales, by the definition"""
    x = x.transpose(0, 1)
    need = x.abs().amax((1, 2)) / 127
    if r == 0:
        new = need
    else:
        s = s.to(F64)
        new = s.clone()
        while bool((new < need).any()):
            new = torch.where(new < need, new * 2, new)
    held = torch.round(q[:, :r].to(F64) * (s / new)[:, None, None]) if r else q[:, :0].to(F64)
    return torch.cat([held, torch.round(x / new[:, None, None])], 1) * new[:, None, None], new


def exact(case, seed):
    c = dict(case)
    s = _inputs(c, seed)
    if c["op"] == "quant":
        x = s.x.to(F64)
        sc = x.abs().max(1, keepdim=True).values / 127
        return [torch.round(x / sc) * sc, sc[:, 0]]
    if c["op"] == "linear":
        o = torch.empty(c["M"], c["N"], dtype=F64, device=DEV)
        w = (s.w.to(F64) * s.sw.to(F64)[:, None]).t().contiguous()
        for m in range(0, c["M"], 1024):
            o[m:m + 1024] = (s.a[m:m + 1024].to(F64) * s.sa[m:m + 1024].to(F64)[:, None]) @ w
        return o if s.bias is None else o + s.bias.to(F64)
    T, Hq, Hk, hd, G, page = c["T"], c["Hq"], c["Hk"], c["hd"], c["Hq"] // c["Hk"], c["page"]
    if c["op"] == "append":
        out = [s.kc.to(F64) * s.ks.to(F64)[:, :, None, None], s.vc.to(F64) * s.vs.to(F64)[:, :, None, None], s.ks.to(F64), s.vs.to(F64)]
        if sum(s.new) // page + 2 * c["nseq"] > 4000:
            return None
        table = s.table.tolist()
        for i, b in enumerate(s.cu_host[:-1]):
            p = torch.arange(s.past[i], s.len_host[i], device=DEV)
            k = _turn(s.k[b:b + s.new[i]], Hk, s.gk, p + c["prefix"], s.freq, c["layout"])
            v = s.v[b:b + s.new[i]].to(F64).reshape(-1, Hk, hd)
            at = s.past[i]
            while at < s.len_host[i]:
                end = min(s.len_host[i], (at // page + 1) * page)
                pg, r, j = table[i][at // page], at % page, slice(at - s.past[i], end - s.past[i])
                for n, (pool, sc, x) in enumerate(((s.kc, s.ks, k), (s.vc, s.vs, v))):
                    rows, out[2 + n][pg] = _page_in(pool[pg], sc[pg], r, x[j])
                    out[n][pg, :, :r + end - at] = rows
                    out[n][pg, :, r + end - at:] = pool[pg, :, r + end - at:].to(F64) * out[2 + n][pg][:, None, None]
                at = end
        return out
    o = torch.empty(T, Hq * hd, dtype=F64, device=DEV)
    for i, (b, e) in enumerate(zip(s.cu_host, s.cu_host[1:])):
        x = torch.arange(s.len_host[i], device=DEV)
        y = torch.arange(c["prefix"], device=DEV)
        pages = torch.cat([s.prefix[y // page].long(), s.table[i][x // page].long()])
        rows = torch.cat([y % page, x % page])
        first = c["prefix"] + s.past[i]
        for h in range(Hk):
            k = s.kc[pages, h, rows].to(F64) * s.ks[pages, h].to(F64)[:, None]
            v = s.vc[pages, h, rows].to(F64) * s.vs[pages, h].to(F64)[:, None]
            kt = k.t().contiguous()
            for u in range(h * G, h * G + G):
                sc = s.q[b:e, u * hd:(u + 1) * hd].to(F64) @ kt * s.scale
                seen = torch.ones_like(sc).tril_(first)
                o[b:e, u * hd:(u + 1) * hd] = torch.softmax(torch.where(seen > 0, sc, torch.full_like(sc, -math.inf)), -1) @ v
    return o
