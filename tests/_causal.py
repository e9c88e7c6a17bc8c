"""Helpers of the causal attention path's tests: 16-bit types in numpy, the operators in 64 bits, and packed / paged inputs."""
import ctypes as C

import numpy as np

F16, BF16 = 1, 2
HALF_STEP = {F16: 2.0 ** -11, BF16: 2.0 ** -8}  # a rounding is off by at most this, relative to the value
TINY = {F16: 2.0 ** -25, BF16: 2.0 ** -134}     # or by this, where the result is subnormal
U24 = 2.0 ** -24


def narrow(x, dtype):
    """fp32 -> the type's bits, round to nearest even"""
    x = np.asarray(x, np.float32, order="C")
    if dtype == F16:
        with np.errstate(over="ignore"):
            return x.astype(np.float16).view(np.uint16)
    b = x.view(np.uint32).astype(np.uint64)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def widen(b, dtype):
    """bits -> float64"""
    if dtype == F16:
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def norm_rope(x, gain, eps, pos, freq, layout, mscale=1.0):
    """x [T][H][hd] float64 -> (result, sum of the absolute values that enter each result)"""
    u = x
    if gain is not None:
        u = u / np.sqrt(np.mean(u * u, -1, keepdims=True) + eps) * gain.astype(np.float64)
    mag = np.abs(u)
    if freq is None or len(freq) == 0:
        return u, mag
    r = len(freq)
    th = np.asarray(pos, np.float64)[:, None] * freq.astype(np.float64)
    cs, sn = (np.cos(th) * mscale)[:, None], (np.sin(th) * mscale)[:, None]
    i, j = (slice(0, r), slice(r, 2 * r)) if layout == 0 else (slice(0, 2 * r, 2), slice(1, 2 * r, 2))
    out, m = u.copy(), mag.copy()
    a, b = u[..., i], u[..., j]
    out[..., i], out[..., j] = a * cs - b * sn, a * sn + b * cs
    m[..., i] = m[..., j] = (np.abs(a) + np.abs(b)) * abs(mscale)
    return out, m


def attend(q, k, v, scale, seen):
    """one head: q [n][hd], k, v [m][hd], seen [n][m] -> (o, sum of p |v| / sum of p), zeros for a row that sees nothing; what is
    hidden has no part in it"""
    with np.errstate(all="ignore"):
        s = np.where(seen, q @ k.T * scale, -np.inf)
        top = s.max(-1, initial=-np.inf, keepdims=True)
        p = np.where(seen, np.exp(s - np.where(np.isneginf(top), 0.0, top)), 0.0)
        l = p.sum(-1, keepdims=True)
        p = np.divide(p, l, out=p, where=l != 0)
        fin = np.isfinite(v).all(-1)
        o, a = p[:, fin] @ v[fin], p[:, fin] @ np.abs(v[fin])
        for t in np.flatnonzero(~fin):
            w = np.where(seen[:, t:t + 1], p[:, t:t + 1] * v[t], 0.0)
            o, a = o + w, a + np.abs(w)
    return o, a


def attend_bound(o, a, vmax, n, hd, smax, dtype):
    """How far an attention output may be from its value: its own rounding; the rounding of the probabilities to the type, as the matrix
    product takes them (relative, and for fp16 also 2^-25 where they are subnormal: the largest is at least 1 and so is their sum);
    the fp32 sums of hd products in a score (smax: the largest sum of absolute products, scaled) and of n values, the exponential of
    arguments up to that size and its base change, and the joins of partial results."""
    u = HALF_STEP[dtype]
    return u * np.abs(o) + (u + (n + (hd + 8) * smax + 256) * U24) * a + n * TINY[dtype] * vmax + TINY[dtype]


class Packed:
    """a packed batch of q, k, v with extra columns and rows that no sequence owns (NaN)"""

    def __init__(self, hip, rng, lens, Hq, Hk, hd, dtype, tail=3, gap=8, qstd=1.5):
        self.lens, self.Hq, self.Hk, self.hd, self.dtype = lens, Hq, Hk, hd, dtype
        self.cu = np.cumsum([0] + list(lens)).astype(np.int32)
        self.n = int(self.cu[-1])
        self.T = self.n + tail
        self.ldq, self.ldk, self.ldv, self.ldo = Hq * hd + gap, Hk * hd + 2 * gap, Hk * hd + gap, Hq * hd + 3 * gap
        mk = lambda ld, w, std: self._rows(rng, ld, w, std)
        self.q, self.k, self.v = mk(self.ldq, Hq * hd, qstd), mk(self.ldk, Hk * hd, 1.0), mk(self.ldv, Hk * hd, 1.0)

    def _rows(self, rng, ld, w, std):
        x = np.full((self.T, ld), np.nan, np.float32)
        x[:self.n, :w] = rng.standard_normal((self.n, w)) * std
        return narrow(x, self.dtype)

    def heads(self, x, H):
        """[n][H][hd] float64"""
        return widen(x[:self.n, :H * self.hd], self.dtype).reshape(self.n, H, self.hd)


class Cache:
    """a paged cache of sequences (new, past) behind a prefix. Every pool value outside the tokens' own is NaN. bad: {(sequence or
    'prefix', slot): entry} replaces entries of the tables (their keys are then left out)."""

    def __init__(self, hip, rng, new, past, prefix, page, H, hd, dtype, bad=None, extra=2, empty=False):
        self.hip, self.new, self.past, self.P, self.page, self.H, self.hd, self.dtype = hip, list(new), list(past), prefix, page, H, hd, dtype
        self.lens = [a + b for a, b in zip(new, past)]
        own = [-(-n // page) for n in self.lens]
        npre = -(-prefix // page)
        self.npages = npre + sum(own) + extra
        self.ldt = max(own + [1]) + 1
        order = rng.permutation(self.npages).astype(np.int32)
        self.prefix = order[:npre].copy()
        self.table = np.full((len(own), self.ldt), -1, np.int32)
        at = npre
        for i, n in enumerate(own):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.cu = np.cumsum([0] + self.new).astype(np.int32)
        shape = (self.npages, H, page, hd)
        self.k, self.v = (narrow(np.full(shape, np.nan, np.float32), dtype) for _ in range(2))
        if not empty:
            for pool in (self.k, self.v):
                for i in range(-1, len(own)):
                    n, pages = (prefix, self.prefix) if i < 0 else (self.lens[i], self.table[i])
                    x = narrow(rng.standard_normal((n, H, hd)).astype(np.float32), dtype)
                    for t in range(n):
                        pool[pages[t // page], :, t % page] = x[t]
        self.good = (self.prefix.copy(), self.table.copy())
        for (i, slot), e in (bad or {}).items():
            (self.prefix if i == "prefix" else self.table[i])[slot] = e

    def upload(self):
        D = self.hip.DeviceArray.from_numpy
        self.d = {n: D(getattr(self, n) if getattr(self, n).size else np.zeros(1, np.int32)) for n in ("prefix", "table", "cu")}
        self.d["len"] = D(np.asarray(self.lens, np.int32))
        self.d["k"], self.d["v"] = D(self.k), D(self.v)
        d = self.d
        self.c = self.hip.KvCache(self.dtype, self.H, self.hd, self.page, self.npages, d["k"].ptr, d["v"].ptr, d["prefix"].ptr, self.P,
                                  d["table"].ptr, self.ldt, d["len"].ptr, d["cu"].ptr, len(self.new))
        return self.c

    def keys(self, pool, i):
        """(values [P + len][H][hd] float64, which of them are there) of sequence i"""
        out, ok = np.zeros((self.P + self.lens[i], self.H, self.hd)), np.zeros(self.P + self.lens[i], bool)
        for x in range(self.P + self.lens[i]):
            y = x - self.P
            pages = self.prefix if y < 0 else self.table[i]
            y = x if y < 0 else y
            e = int(pages[y // self.page])
            if 0 <= e < self.npages:
                out[x], ok[x] = widen(pool[e, :, y % self.page], self.dtype), True
        return out, ok

    def expect(self, q, scale):
        """q [n][Hq][hd] float64 -> (o, sum p |v|, keys, largest scaled sum of |q k|, largest |v|) per row"""
        Hq, G = q.shape[1], q.shape[1] // self.H
        o, a = np.zeros_like(q), np.zeros_like(q)
        smax, vmax, nmax = 0.0, 0.0, 1
        for i, b in enumerate(self.cu[:-1]):
            n = self.new[i]
            if n == 0:
                continue
            (k, ok), (v, _) = self.keys(self.k, i), self.keys(self.v, i)
            p = np.maximum(self.past[i] + np.arange(n), -1)  # a query before its sequence's start sees the prefix
            seen = (np.arange(self.P + self.lens[i])[None] <= self.P + p[:, None]) & ok[None]
            for h in range(Hq):
                qh = q[b:b + n, h]
                o[b:b + n, h], a[b:b + n, h] = attend(qh, k[:, h // G], v[:, h // G], scale, seen)
                if len(k):
                    smax = max(smax, float((np.abs(qh) @ np.abs(np.nan_to_num(k[:, h // G], posinf=0, neginf=0)).T).max()) * scale)
            if len(v):
                vmax = max(vmax, float(np.abs(np.nan_to_num(v, posinf=0, neginf=0)).max()))
            nmax = max(nmax, len(k))
        return o, a, nmax, smax, vmax


def close(got, want, bound, what):
    """got within bound of want; where want is not finite it is the same kind of value"""
    fin = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what + ": NaN elsewhere"
    assert np.array_equal(got[np.isinf(want)], want[np.isinf(want)]), what + ": infinities"
    over = np.abs(got[fin] - want[fin]) - bound[fin]
    assert over.size == 0 or over.max() <= 0, f"{what}: {over.max():.3g} over a bound of {bound[fin].flat[over.argmax()]:.3g}"


def ptr(a):
    return a.ctypes.data_as(C.c_void_p)
