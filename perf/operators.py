"""The attention path of a causal text model, as a caller of libhexanima_hip.so drives it: its operators in plain torch and
through the C-ABI, on the same inputs.

  qk      hxa_qk_norm_rope       queries and keys: per-head RMSNorm and rotary positions in one pass
  append  hxa_kv_append          new keys (normed and rotated on the way) and values into a paged cache
  causal  hxa_attention_causal   whole prompts: causal, grouped heads, packed sequences of different lengths
  cached  hxa_attention_cached   new tokens over the paged cache, behind a prefix that the whole batch shares

q, k and v are columns of one projection's rows, as a fused qkv linear leaves them. Kernel calls go to torch's current stream.
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


# ----------------------------------------------------------------------------------------------------------------- cases
# Every case: type, query heads Hq, key / value heads Hk, head width hd, new tokens T of nseq sequences (their lengths follow
# from the salt). rot, layout: the rotated part of a head and its pairs. past: tokens already in the sequences' own pages,
# over the batch; prefix: tokens of the shared prefix; page: tokens a page.
def listed():
    return [
        # one token of one sequence, far into a long context: nothing but latency
        dict(name="qk_step_1", op="qk", dtype="f16", Hq=16, Hk=8, hd=128, T=1, first=70000, rot=128, layout="half"),
        # heads of 256 that rotate a quarter of their width, the rows of a ragged batch
        dict(name="qk_part_1031", op="qk", dtype="f16", Hq=10, Hk=2, hd=256, T=1031, first=0, rot=64, layout="pairs"),
        # a long prompt, heads of 128
        dict(name="qk_prompt_8192", op="qk", dtype="bf16", Hq=32, Hk=8, hd=128, T=8192, first=0, rot=128, layout="half"),
        # a decoding step of 64 sequences: one new key and value each
        dict(name="append_step_64", op="append", dtype="bf16", Hq=32, Hk=8, hd=128, T=64, nseq=64, past=30000, prefix=1000,
             page=16, salt=1, rot=128, layout="half"),
        # 23 prompts of very different lengths go into the cache
        dict(name="append_prompts_9001", op="append", dtype="f16", Hq=16, Hk=8, hd=128, T=9001, nseq=23, past=1500, prefix=0,
             page=64, salt=2, rot=128, layout="half"),
        # one image prompt of an ordinary length
        dict(name="causal_prompt_77", op="causal", dtype="f16", Hq=16, Hk=8, hd=128, T=77, nseq=1, salt=1),
        # a batch of prompts of different lengths packed into 6500 rows
        dict(name="causal_packed_6500", op="causal", dtype="f16", Hq=16, Hk=8, hd=128, T=6500, nseq=9, salt=3),
        # a long document
        dict(name="causal_long_16384", op="causal", dtype="bf16", Hq=32, Hk=8, hd=128, T=16384, nseq=1, salt=1),
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
        op = rng.choice(["qk", "append", "causal", "causal", "cached", "cached"])
        Hq, Hk = rng.choice(HEADS)
        hd = rng.choice([64, 128, 128, 256])
        c = dict(op=op, dtype=rng.choice(["f16", "bf16"]), Hq=Hq, Hk=Hk, hd=hd)
        if op == "qk":
            c |= dict(T=_log(rng, 1, 16384), first=rng.choice([0, 0, _log(rng, 100, 1000000)]))
        elif op == "causal":
            T = _log(rng, 1, 16384)
            c |= dict(T=T, nseq=min(T, _log(rng, 1, 64)), salt=rng.randint(0, 999))
        else:
            step = rng.random() < 0.5  # one token a sequence, or pieces of prompts
            nseq = _log(rng, 1, 128)
            T = nseq if step else _log(rng, nseq, 8192)
            c |= dict(T=T, nseq=nseq, past=_log(rng, 1, 2000) * nseq if step or rng.random() < 0.4 else 0,
                      prefix=rng.choice([0, _log(rng, 16, 16384)]), page=rng.choice([1, 16, 16, 32, 64, 128]), salt=rng.randint(0, 999))
        if op in ("qk", "append"):
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
    T, Hq, Hk, hd = c["T"], c["Hq"], c["Hk"], c["hd"]
    if c["op"] == "qk":
        return {"bytes": 4.0 * T * (Hq + Hk) * hd, "flops": 8.0 * T * (Hq + Hk) * hd}
    if c["op"] == "append":
        return {"bytes": 8.0 * T * Hk * hd, "flops": 8.0 * T * Hk * hd}
    new, past = _lengths(c)
    pairs = sum(n * (p + (n + 1) / 2) for n, p in zip(new, past)) + T * c.get("prefix", 0)
    keys = sum(new) + sum(past) + c.get("prefix", 0)
    return {"bytes": 4.0 * hd * (T * Hq + keys * Hk), "flops": 4.0 * pairs * Hq * hd}


# ---------------------------------------------------------------------------------------------------------------- inputs
class State:
    pass


def _gen(seed, salt=0):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1000003 + salt)
    return g


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * std).to(dtype)


def _gain(g, hd):
    return 1.0 + _randn(g, hd, std=0.1)


def _freq(c):
    """radians a position of each pair, theta 10000 (heads of 256: 1000000)"""
    i = torch.arange(c["rot"] // 2, dtype=F64)
    return ((1e6 if c["hd"] == 256 else 1e4) ** (-2.0 * i / c["rot"])).float().to(DEV)


def _ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def _inputs(c, seed):
    s = State()
    g = _gen(seed)
    dt = DTYPE[c["dtype"]]
    T, Hq, Hk, hd = c["T"], c["Hq"], c["Hk"], c["hd"]
    s.case = c
    # one projection's rows, q | k | v
    s.qkv = _randn(g, T, (Hq + 2 * Hk) * hd, dtype=dt)
    s.q, s.k, s.v = s.qkv[:, :Hq * hd], s.qkv[:, Hq * hd:(Hq + Hk) * hd], s.qkv[:, (Hq + Hk) * hd:]
    s.gq, s.gk = _gain(g, hd), _gain(g, hd)
    s.scale = hd ** -0.5
    if "rot" in c:
        s.freq = _freq(c)
    if c["op"] == "qk":
        s.pos = torch.arange(c["first"], c["first"] + T, dtype=torch.int32, device=DEV)
        return s
    s.new, s.past = _lengths(c)
    cu = [0]
    for n in s.new:
        cu.append(cu[-1] + n)
    s.cu_host, s.cu = cu, _ints(cu)
    if c["op"] == "causal":
        # queries and keys come from the norm in tensors of their own; its gains make the scores about this wide
        s.q, s.k = _randn(g, T, Hq * hd, std=1.5, dtype=dt), _randn(g, T, Hk * hd, dtype=dt)
        return s
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
    s.kc = _randn(g, s.npages, Hk, page, hd, dtype=dt)
    s.vc = _randn(g, s.npages, Hk, page, hd, dtype=dt)
    if c["op"] == "cached":
        s.q = _randn(g, T, Hq * hd, std=1.5, dtype=dt)
    return s


def prepare(case, seed):
    c = dict(case)
    s = _inputs(c, seed)
    dt = DTYPE[c["dtype"]]
    if c["op"] == "qk":
        s.qo = torch.empty(c["T"], c["Hq"] * c["hd"], dtype=dt, device=DEV)
        s.ko = torch.empty(c["T"], c["Hk"] * c["hd"], dtype=dt, device=DEV)
    elif c["op"] != "append":
        s.o = torch.empty(c["T"], c["Hq"] * c["hd"], dtype=dt, device=DEV)
    if own:
        from hexanima_amd import hip

        hip.init(0)
        s.dt = hip.DT_F16 if c["dtype"] == "f16" else hip.DT_BF16
        if "rot" in c:
            s.rope = hip.Rope(s.freq.data_ptr(), c["rot"], hip.ROPE_HALF if c["layout"] == "half" else hip.ROPE_PAIRS, 1.0)
        if c["op"] in ("append", "cached"):
            s.cache = hip.KvCache(s.dt, c["Hk"], c["hd"], c["page"], s.npages, s.kc.data_ptr(), s.vc.data_ptr(), s.prefix.data_ptr(),
                                  c["prefix"], s.table.data_ptr(), s.ldt, s.len.data_ptr(), s.cu.data_ptr(), c["nseq"])
        if c["op"] == "cached":
            s.ws_bytes = hip.lib().hxa_attention_cached_ws_bytes(C.byref(s.cache), c["T"], c["Hq"])
            s.ws = torch.empty(max(s.ws_bytes, 16), dtype=torch.uint8, device=DEV)
    return s


# ------------------------------------------------------------------------------------------------------------ plain form
def _norm_rope(x, H, gain, pos, freq, layout):
    """per-head RMSNorm * gain, then the rotation, in 32 bits; the angles of far positions in 64"""
    T, hd = x.shape[0], x.shape[1] // H
    u = x.float().view(T, H, hd)
    u = u * torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS) * gain
    r = freq.numel()
    th = pos.to(F64)[:, None] * freq.to(F64)
    cs, sn = torch.cos(th).float()[:, None], torch.sin(th).float()[:, None]
    a, b = (u[..., :r], u[..., r:2 * r]) if layout == "half" else (u[..., 0:2 * r:2], u[..., 1:2 * r:2])
    ra, rb = a * cs - b * sn, a * sn + b * cs
    rotated = torch.cat([ra, rb], -1) if layout == "half" else torch.stack([ra, rb], -1).view(T, H, 2 * r)
    return torch.cat([rotated, u[..., 2 * r:]], -1).view(T, H * hd).to(x.dtype)


def _slots(s):
    """page, row and own position of each new token"""
    page = s.case["page"]
    seq = torch.repeat_interleave(torch.arange(s.case["nseq"], device=DEV), s.cu[1:] - s.cu[:-1])
    t = torch.arange(s.case["T"], device=DEV)
    p = s.len[seq].long() - (s.cu[seq + 1] - t)
    return s.table[seq, p // page].long(), p % page, p


def _soft(sc):
    e = sc.sub_(sc.amax(-1, keepdim=True)).exp_()
    return e.div_(e.sum(-1, keepdim=True))


def _attend(q, keys, vals, G, scale, first, o):
    """rows of q at key positions first, first + 1, ... over keys [n][Hk hd]; o gets the rounded rows"""
    n, Hk = keys.shape[0], q.shape[1] // G
    hd = keys.shape[1] // Hk
    kt = keys.reshape(n, Hk, hd).permute(1, 2, 0).float().contiguous()
    v = vals.reshape(n, Hk, hd).transpose(0, 1).float().contiguous()
    for t in range(0, q.shape[0], 1024):
        m = min(1024, q.shape[0] - t)
        e = min(n, first + t + m)
        x = q[t:t + m].reshape(m, Hk, G, hd).permute(1, 2, 0, 3).float().reshape(Hk, G * m, hd)
        sc = (torch.matmul(x, kt[:, :, :e]) * scale).view(Hk, G, m, e)
        late = torch.arange(e, device=DEV) > torch.arange(first + t, first + t + m, device=DEV)[:, None]
        pr = _soft(sc.masked_fill_(late, -math.inf)).view(Hk, G * m, e)
        o[t:t + m] = torch.matmul(pr, v[:, :e]).view(Hk, G, m, hd).permute(2, 0, 1, 3).reshape(m, Hk * G, hd).to(o.dtype)


def _gather(pool, pages, n):
    """tokens 0 .. n - 1 of the given pages as rows"""
    x = pool[pages.long()]
    return x.transpose(1, 2).reshape(-1, x.shape[1] * x.shape[3])[:n]


def _plain(s):
    c = s.case
    T, Hq, Hk, hd = c["T"], c["Hq"], c["Hk"], c["hd"]
    if c["op"] == "qk":
        return [_norm_rope(s.q, Hq, s.gq, s.pos, s.freq, c["layout"]), _norm_rope(s.k, Hk, s.gk, s.pos, s.freq, c["layout"])]
    if c["op"] == "append":
        pg, row, p = _slots(s)
        s.kc[pg, :, row] = _norm_rope(s.k, Hk, s.gk, p + c["prefix"], s.freq, c["layout"]).view(T, Hk, hd)
        s.vc[pg, :, row] = s.v.reshape(T, Hk, hd)
        return [s.kc, s.vc]
    o, q = s.o.view(T, Hq, hd), s.q.view(T, Hq, hd)
    if c["op"] == "causal":
        for b, e in zip(s.cu_host, s.cu_host[1:]):
            _attend(q[b:e], s.k[b:e], s.v[b:e], Hq // Hk, s.scale, 0, o[b:e])
        return s.o
    pk, pv = _gather(s.kc, s.prefix, c["prefix"]), _gather(s.vc, s.prefix, c["prefix"])
    for i, (b, e) in enumerate(zip(s.cu_host, s.cu_host[1:])):
        n = s.len_host[i]
        pages = s.table[i, :(n + c["page"] - 1) // c["page"]]
        keys, vals = torch.cat([pk, _gather(s.kc, pages, n)]), torch.cat([pv, _gather(s.vc, pages, n)])
        _attend(q[b:e], keys, vals, Hq // Hk, s.scale, c["prefix"] + s.past[i], o[b:e])
    return s.o


# ------------------------------------------------------------------------------------------------------------------- run
def run(s):
    if not own:
        return _plain(s)
    from hexanima_amd import hip

    L, c = hip.lib(), s.case
    T, Hq, Hk, hd = c["T"], c["Hq"], c["Hk"], c["hd"]
    st = torch.cuda.current_stream().cuda_stream
    if c["op"] == "qk":
        hip.check(L.hxa_qk_norm_rope(s.dt, s.q.data_ptr(), s.q.stride(0), Hq, s.k.data_ptr(), s.k.stride(0), Hk, T, hd, s.gq.data_ptr(),
                                     s.gk.data_ptr(), EPS, s.pos.data_ptr(), C.byref(s.rope), s.qo.data_ptr(), Hq * hd, s.ko.data_ptr(),
                                     Hk * hd, st), "qk_norm_rope")
        return [s.qo, s.ko]
    if c["op"] == "append":
        hip.check(L.hxa_kv_append(C.byref(s.cache), s.k.data_ptr(), s.k.stride(0), s.v.data_ptr(), s.v.stride(0), T, s.gk.data_ptr(), EPS,
                                  C.byref(s.rope), st), "kv_append")
        return [s.kc, s.vc]
    if c["op"] == "causal":
        hip.check(L.hxa_attention_causal(s.dt, s.q.data_ptr(), Hq * hd, s.k.data_ptr(), Hk * hd, s.v.data_ptr(), s.v.stride(0),
                                         s.o.data_ptr(), Hq * hd, T, s.cu.data_ptr(), c["nseq"], Hq, Hk, hd, s.scale, st),
                  "attention_causal")
        return s.o
    hip.check(L.hxa_attention_cached(C.byref(s.cache), s.q.data_ptr(), Hq * hd, s.o.data_ptr(), Hq * hd, T, Hq, s.scale, s.ws.data_ptr(),
                                     s.ws_bytes, st), "attention_cached")
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
    return u.reshape(T, H * hd)


def _head(q, k, v, scale, first):
    """one query head: its rows stand at key positions first, first + 1, ..."""
    o = torch.empty_like(q)
    for t in range(0, len(q), 1024):
        x = q[t:t + 1024] @ k.t().contiguous() * scale
        seen = torch.ones_like(x).tril_(first + t)
        o[t:t + 1024] = torch.softmax(torch.where(seen > 0, x, torch.full_like(x, -math.inf)), -1) @ v
    return o


def exact(case, seed):
    c = dict(case)
    s = _inputs(c, seed)
    T, Hq, Hk, hd, G = c["T"], c["Hq"], c["Hk"], c["hd"], c["Hq"] // c["Hk"]
    if c["op"] == "qk":
        return [_turn(s.q, Hq, s.gq, s.pos, s.freq, c["layout"]), _turn(s.k, Hk, s.gk, s.pos, s.freq, c["layout"])]
    if c["op"] == "append":
        kc, vc = s.kc.to(F64), s.vc.to(F64)
        for i, b in enumerate(s.cu_host[:-1]):
            n = s.new[i]
            p = torch.arange(s.past[i], s.past[i] + n, device=DEV)
            k = _turn(s.k[b:b + n], Hk, s.gk, p + c["prefix"], s.freq, c["layout"]).view(n, Hk, hd)
            v = s.v[b:b + n].to(F64).reshape(n, Hk, hd)
            at = s.table[i][torch.div(p, c["page"], rounding_mode="floor")].long()
            for h in range(Hk):
                kc[at, h, p % c["page"]] = k[:, h]
                vc[at, h, p % c["page"]] = v[:, h]
        return [kc, vc]
    o = torch.empty(T, Hq * hd, dtype=F64, device=DEV)
    for i, (b, e) in enumerate(zip(s.cu_host, s.cu_host[1:])):
        for hk in range(Hk):
            j = slice(hk * hd, (hk + 1) * hd)
            if c["op"] == "causal":
                k, v, first = s.k[b:e, j].to(F64), s.v[b:e, j].to(F64), 0
            else:
                x = torch.arange(s.len_host[i], device=DEV)
                y = torch.arange(c["prefix"], device=DEV)
                own_at, pre_at = s.table[i][x // c["page"]].long(), s.prefix[y // c["page"]].long()
                k = torch.cat([s.kc[pre_at, hk, y % c["page"]], s.kc[own_at, hk, x % c["page"]]]).to(F64)
                v = torch.cat([s.vc[pre_at, hk, y % c["page"]], s.vc[own_at, hk, x % c["page"]]]).to(F64)
                first = c["prefix"] + s.past[i]
            for h in range(hk * G, hk * G + G):
                o[b:e, h * hd:(h + 1) * hd] = _head(s.q[b:e, h * hd:(h + 1) * hd].to(F64), k, v, s.scale, first)
    return o
