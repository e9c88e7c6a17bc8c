"""Helpers of the 8-bit text model's tests: the operators' definitions in 64 bits (32 where a definition names a 32-bit step), and caches of int8."""
import numpy as np

from tests._causal import BF16, HALF_STEP, TINY, U24, Cache, narrow, norm_rope, widen

LEAST = np.float32(2.0 ** -64)


def round128(k):
    return -(-k // 128) * 128


def quantize(x):
    """rows of float64 (16-bit values) -> (int8 values as float64, fp32 scales), by the definition's 32-bit steps"""
    with np.errstate(all="ignore"):
        x = x.astype(np.float32)
        top = np.where(np.isfinite(x), np.abs(x), 0).max(-1).astype(np.float32)
        t = np.maximum(top, np.float32(127) * LEAST)
        scale = page_scale(top)
        inv = np.where(top > 0, np.float32(1) / t * np.float32(127), np.float32(0)).astype(np.float32)
        r = x * inv[..., None]
    return to_byte(r), scale


def to_byte(r):
    return np.clip(np.rint(np.where(np.isnan(r), 0, r)), -127, 127)


def page_scale(top):
    """the scale of values whose largest finite magnitude is top (fp32)"""
    top = np.asarray(top, np.float32)
    return np.where(top > 0, np.maximum(top * np.float32(1 / 127), LEAST), np.float32(0)).astype(np.float32)


def grow(old, need):
    """(scale, doublings) of a page that had `old` and needs `need`"""
    if not old > 0:
        return need, 0
    j = 0
    while np.float64(old) * 2.0 ** j < need and j < 300:
        j += 1
    return old * 2.0 ** j, j


def linear_bound(dot, want, dtype):
    """the fp32 steps of a sum's scaling (the sum to fp32, the row's scale, the column's with the bias) and the output's rounding"""
    return HALF_STEP[dtype] * np.abs(want) + 3 * U24 * (np.abs(dot) + np.abs(want)) + TINY[dtype]


def attend_q8_bound(o, a, vtop, n, hd, smax, lmax, kmax, dtype):
    """As attend_bound: the output's own rounding; the weights' rounding to fp16 (relative 2^-11 of the mean of |v|; 2^-25 where they are subnormal, of
    weights of which the largest is at least 1 before its byte, so n 2^-25 127 of the largest scale); the fp32 sums; the exponent's terms, the score
    (smax) and the logarithm of the value's scale (lmax), each with a few half steps of its own; of bf16 queries what fp16 loses beside a largest value of 1 or more, 2^-25 a
    dim, times the largest key (kmax, scaled)."""
    return HALF_STEP[dtype] * np.abs(o) + (2.0 ** -11 + (n + (hd + 8) * smax + 8 * lmax + 256) * U24 + hd * 2.0 ** -25 * kmax) * a + n * 2.0 ** -25 * vtop + TINY[dtype]


class CacheQ8(Cache):
    """a paged cache of int8. Scales of pages that no token owns are NaN, bytes of rows that none owns -128. spread: how widely the pages' scales differ."""

    def __init__(self, hip, rng, new, past, prefix, page, H, hd, dtype, bad=None, spread=0.5, empty=False):
        super().__init__(hip, rng, new, past, prefix, page, H, hd, dtype, bad=bad, empty=True)
        shape = (self.npages, H, page, hd)
        self.k, self.v = np.full(shape, -128, np.int8), np.full(shape, -128, np.int8)
        self.ks, self.vs = np.full(shape[:2], np.nan, np.float32), np.full(shape[:2], np.nan, np.float32)
        if empty:
            return
        prefix_pages, table = self.good
        for i in range(-1, len(self.lens)):
            n, pages = (prefix, prefix_pages) if i < 0 else (self.lens[i], table[i])
            for s in range(-(-n // page)):
                m = min(page, n - s * page)
                for pool, sc in ((self.k, self.ks), (self.v, self.vs)):
                    pool[pages[s], :, :m] = np.clip(np.rint(rng.standard_normal((H, m, hd)) * 40), -127, 127)
                    sc[pages[s]] = np.exp(rng.standard_normal(H) * spread) / 40

    def upload(self):
        c = super().upload()
        D = self.hip.DeviceArray.from_numpy
        self.d["ks"], self.d["vs"] = D(self.ks), D(self.vs)
        self.q8 = self.hip.KvCacheQ8(c, self.d["ks"].ptr, self.d["vs"].ptr)
        return self.q8

    def values(self, pool):
        sc = self.ks if pool is self.k else self.vs
        with np.errstate(invalid="ignore"):
            return pool.astype(np.float64) * np.where(np.isfinite(sc) & (sc > 0), sc, 0).astype(np.float64)[:, :, None, None]

    def keys(self, pool, i):
        val = self.values(pool)
        out, ok = np.zeros((self.P + self.lens[i], self.H, self.hd)), np.zeros(self.P + self.lens[i], bool)
        for x in range(self.P + self.lens[i]):
            y = x - self.P
            pages = self.prefix if y < 0 else self.table[i]
            y = x if y < 0 else y
            e = int(pages[y // self.page])
            if 0 <= e < self.npages:
                out[x], ok[x] = val[e, :, y % self.page], True
        return out, ok

    def bound(self, o, a, n, smax, scale):
        good = self.vs[np.isfinite(self.vs) & (self.vs > 0)].astype(np.float64)
        lmax = np.abs(np.log2(good)).max(initial=64.0)
        ks = self.ks[np.isfinite(self.ks) & (self.ks > 0)].astype(np.float64)
        kmax = 127 * ks.max(initial=0.0) * scale if self.dtype == BF16 else 0.0
        return attend_q8_bound(o, a, 127 * good.max(initial=0.0), n, self.hd, smax, lmax, kmax, self.dtype)


def append(c, k, v, gain, eps, freq, layout, T):
    """What the append leaves of cache c, sequence by sequence and page by page, in 64 bits (v: by the definition's 32-bit steps): (bytes, scales and bounds on the
    keys' values) as dict(k, ks, v, vs, kval, kbound). Keys are checked by their values: a byte at a border may go either way."""
    r = dict(k=c.k.copy(), v=c.v.copy(), ks=c.ks.copy(), vs=c.vs.copy(), kval={}, shift={})
    H, hd, page = c.H, c.hd, c.page
    for i, b in enumerate(c.cu[:-1]):
        e = min(int(c.cu[i + 1]), T)
        for s in range(c.ldt):
            pos = [p for p in range(max(0, c.lens[i] - (e - b)), c.lens[i]) if p // page == s]
            pg = int(c.table[i, s])
            if not pos or not 0 <= pg < c.npages:
                continue
            rows = [b + p - (c.lens[i] - (e - b)) for p in pos]
            x, mag = norm_rope(widen(k[rows, :H * hd], c.dtype).reshape(-1, H, hd), gain, eps, [c.P + p for p in pos], freq, layout)
            y = widen(v[rows, :H * hd], c.dtype).reshape(-1, H, hd)
            r0 = pos[0] % page
            for h in range(H):
                fin = lambda z: np.where(np.isfinite(z), np.abs(z), 0).max()
                old = c.vs[pg, h] if r0 and c.vs[pg, h] < np.inf else 0.0
                sc, j = grow(old, page_scale(fin(y[:, h])))
                r["vs"][pg, h] = sc
                if j:
                    r["v"][pg, h, :r0] = np.rint(c.v[pg, h, :r0] * 2.0 ** -j)
                with np.errstate(all="ignore"):
                    inv = np.float32(1) / np.float32(sc) if sc > 0 else np.float32(0)
                    r["v"][pg, h, r0:r0 + len(pos)] = to_byte(y[:, h].astype(np.float32) * inv)
                old = c.ks[pg, h] if r0 and c.ks[pg, h] < np.inf else 0.0
                sc, j = grow(old, float(fin(x[:, h])) / 127)
                r["ks"][pg, h] = sc
                if j:
                    r["k"][pg, h, :r0] = np.rint(c.k[pg, h, :r0] * 2.0 ** -j)
                r["kval"][pg, h] = (r0, x[:, h], mag[:, h], sc, old)
    return r
