"""The causal text model in 8 bits (row quantiser, int8 product, append to a cache of int8, attention over it) against the operators' definitions in
64 bits. Bounds are worst cases of the roundings named in _q8."""
import ctypes as C

import numpy as np
import pytest

from tests._causal import BF16, F16, HALF_STEP, TINY, U24, close, narrow, norm_rope, widen
from tests._q8 import CacheQ8, append, linear_bound, quantize, round128
from tests.test_gpu_causal import CACHED, EPS, MIXED, dev, head_bound, queries, say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    from hexanima_amd import hip as h
    h.init(0)
    return h


# ------------------------------------------------------------------------------------------------------------- rows
def run_quant(hip, x, K, dtype, stream=None):
    """x [M][ldx] bits -> (q [M][ldq], scales); what lies behind the written columns stays"""
    M, ldx = x.shape
    ldq = round128(K) + 32
    d = [dev(hip, x), dev(hip, np.full((M + 1, ldq), 85, np.int8)), dev(hip, np.full(M + 1, 7, np.float32))]
    hip.check(hip.lib().hxa_quantize_rows(dtype, d[0].ptr, ldx, M, K, d[1].ptr, ldq, d[2].ptr, stream), "quantize_rows")
    hip.sync()
    q, s = d[1].numpy(), d[2].numpy()
    assert (q[M] == 85).all() and s[M] == 7 and (q[:M, round128(K):] == 85).all() and (q[:M, K:round128(K)] == 0).all()
    return q[:M, :K], s[:M]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 2048), (3, 7), (5, 129), (2, 2049), (7, 1000), (3, 8192), (2, 8200), (2, 16384), (3, 16391),
                                 (2, 40001), (1, 130944), (1030, 64), (1025, 2047), (1024, 2048)])
def test_quantize_rows(hip, dtype, M, K):
    say("quant", dtype, M, K)
    rng = np.random.default_rng(M + K)
    x = np.full((M, -(-K // 8) * 8 + 16), np.nan, np.float32)
    x[:, :K] = rng.standard_normal((M, K)) * np.exp(rng.standard_normal((M, 1)) * 4)
    b = narrow(x, dtype)
    q, s = run_quant(hip, b, K, dtype)
    wq, ws = quantize(widen(b[:, :K], dtype))
    assert np.array_equal(s, ws) and np.array_equal(q, wq)
    # a byte stands for its value to within half a step (and the two 32-bit products), where the value is finite
    v, step = widen(b[:, :K], dtype), s[:, None].astype(np.float64)
    fin = np.isfinite(v)
    assert (np.abs(q * step - np.where(fin, v, 0))[fin] <= (step * (0.5 + 127 * 4 * U24) * np.ones_like(v))[fin]).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,K,ldx,off", [(5, 1003, 1003, 0), (1100, 229, 229, 1), (3, 8191, 8195, 3), (4, 16, 17, 5), (2, 20001, 20001, 7)])
def test_quantize_rows_that_begin_anywhere(hip, dtype, M, K, ldx, off):
    """row strides and first values of no alignment, the last row ending with the buffer"""
    say("quant", dtype, M, K, ldx, off)
    b = narrow(np.random.default_rng(K).standard_normal(off + (M - 1) * ldx + K), dtype)
    rows = np.stack([b[off + m * ldx:off + m * ldx + K] for m in range(M)])
    d = [dev(hip, b), dev(hip, np.full((M, round128(K)), 85, np.int8)), dev(hip, np.zeros(M, np.float32))]
    hip.check(hip.lib().hxa_quantize_rows(dtype, d[0].at(2 * off), ldx, M, K, d[1].ptr, round128(K), d[2].ptr, None), "quantize_rows")
    hip.sync()
    wq, ws = quantize(widen(rows, dtype))
    assert np.array_equal(d[2].numpy(), ws) and np.array_equal(d[1].numpy()[:, :K], wq) and not d[1].numpy()[:, K:].any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,K", [(6, 300), (1100, 96)])
def test_quantize_special_rows(hip, dtype, M, K):
    """zeros, infinities, NaN, subnormal and largest values, ties"""
    rng = np.random.default_rng(3)
    x = rng.standard_normal((M, -(-K // 8) * 8)).astype(np.float32)
    x[0] = 0
    x[1, 5], x[1, 9], x[1, 17] = np.inf, -np.inf, np.nan
    x[2] = np.nan
    x[2, 3] = -np.inf
    b = narrow(x, dtype)
    b[3] = 1                                                       # the least subnormal
    b[4] = narrow(np.full(x.shape[1], 65504 if dtype == F16 else 3e38, np.float32) * np.sign(x[4]), dtype)
    b[5] = narrow(np.resize(np.array([127, 0.5, 1.5, 2.5, -0.5, -63.5], np.float32), x.shape[1]), dtype)
    q, s = run_quant(hip, b, K, dtype)
    wq, ws = quantize(widen(b[:, :K], dtype))
    assert np.array_equal(s, ws) and np.array_equal(q, wq)
    assert s[0] == 0 and not q[0].any() and s[2] == 0 and not q[2].any()
    assert list(q[1, [5, 9, 17]]) == [127, -127, 0] and list(q[5, :6]) == [127, 0, 2, 2, 0, -64]


def test_quantize_offsets_past_32_bits(hip):
    """rows 2^31 values and bytes apart"""
    K, ld = 100, 2 ** 31
    x = hip.DeviceArray((ld + 128,), np.uint16)
    q = hip.DeviceArray((ld + 128,), np.int8)
    s = hip.DeviceArray((2,), np.float32)
    rows = narrow(np.random.default_rng(0).standard_normal((2, K)), F16)
    for i in range(2):
        hip.check(hip.lib().hxa_h2d(x.at(2 * i * ld), rows[i].ctypes.data, 2 * K))
    hip.check(hip.lib().hxa_quantize_rows(F16, x.ptr, ld, 2, K, q.ptr, ld, s.ptr, None))
    hip.sync()
    wq, ws = quantize(widen(rows, F16))
    got = np.zeros((2, K), np.int8)
    for i in range(2):
        hip.check(hip.lib().hxa_d2h(got[i].ctypes.data, q.at(i * ld), K))
    assert np.array_equal(got, wq) and np.array_equal(s.numpy(), ws)


def test_quantize_more_rows_than_a_grid_holds(hip):
    """2^24 + 3 rows of a workgroup each"""
    M, K, ldq = 2 ** 24 + 3, 2056, 2176
    x, q, s = hip.DeviceArray((M, K), np.uint16), hip.DeviceArray((M, ldq), np.int8), hip.DeviceArray((M,), np.float32)
    at = [0, 1, 2 ** 23 - 1, 2 ** 23, 2 ** 24 - 1, 2 ** 24, M - 1]
    rows = narrow(np.random.default_rng(1).standard_normal((len(at), K)), F16)
    for i, m in enumerate(at):
        hip.check(hip.lib().hxa_h2d(x.at(m * K * 2), rows[i].ctypes.data, 2 * K))
    hip.check(hip.lib().hxa_quantize_rows(F16, x.ptr, K, M, K, q.ptr, ldq, s.ptr, None))
    hip.sync()
    wq, ws = quantize(widen(rows, F16))
    got, gs = np.zeros((len(at), ldq), np.int8), np.zeros(len(at), np.float32)
    for i, m in enumerate(at):
        hip.check(hip.lib().hxa_d2h(got[i].ctypes.data, q.at(m * ldq), ldq))
        hip.check(hip.lib().hxa_d2h(gs[i:].ctypes.data, s.at(m * 4), 4))
    assert np.array_equal(got[:, :K], wq) and not got[:, K:].any() and np.array_equal(gs, ws)


# ------------------------------------------------------------------------------------------------------------- product
class Linear:
    def __init__(self, hip, M, N, K, bias=True, seed=0, junk="a", gap=(16, 48, 8)):
        """junk: the operand whose columns past K hold anything (the other's are zeros)"""
        rng = np.random.default_rng(seed + M + N + K)
        self.hip, self.M, self.N, self.K = hip, M, N, K
        self.lda, self.ldw, self.ldo = round128(K) + gap[0], round128(K) + gap[1], N + gap[2]
        self.a, self.w = (rng.integers(-128, 128, (r, ld), np.int64).astype(np.int8) for r, ld in ((M, self.lda), (N, self.ldw)))
        (self.w if junk == "a" else self.a)[:, K:round128(K)] = 0
        self.sa, self.sw = (np.exp(rng.standard_normal(n)).astype(np.float32) / 500 for n in (M, N))
        self.bias = rng.standard_normal(N).astype(np.float32) if bias else None
        self.d = [dev(hip, x) for x in (self.a, self.sa, self.w, self.sw)]
        self.db = dev(hip, self.bias) if bias else None

    def expect(self, dtype):
        dot = self.a[:, :self.K].astype(np.float64) @ self.w[:, :self.K].astype(np.float64).T * self.sa[:, None].astype(np.float64) * self.sw.astype(np.float64)
        want = dot + (self.bias.astype(np.float64) if self.bias is not None else 0)
        return want, linear_bound(dot, want, dtype)

    def run(self, dtype, with_ws=True, tile=None, stream=None):
        L, hip = self.hip.lib(), self.hip
        o = dev(hip, np.full((self.M + 1, self.ldo), 0x5555, np.uint16))
        args = [dtype, self.d[0].ptr, self.lda, self.d[1].ptr, self.M, self.d[2].ptr, self.ldw, self.d[3].ptr, self.N, self.K,
                self.db.ptr if self.db else None, o.ptr, self.ldo]
        if tile:
            nb = tile[2] * self.M * self.N * 4 if tile[2] > 1 else 0
            ws = hip.DeviceArray((max(nb, 16),), np.uint8)
            hip.check(L.hxa_linear_i8_tile(*args, *tile, ws.ptr, nb, stream), "tile")
        else:
            nb = L.hxa_linear_i8_ws_bytes(self.M, self.N, self.K) if with_ws else 0
            ws = hip.DeviceArray((max(nb, 16),), np.uint8)
            hip.check(L.hxa_linear_i8(*args, ws.ptr if with_ws else None, nb, stream), "linear_i8")
        hip.sync()
        o = o.numpy()
        assert (o[self.M:] == 0x5555).all() and (o[:, self.N:] == 0x5555).all()
        return o[:self.M, :self.N]


SHAPES = [(1, 8, 1), (1, 4096, 2048), (3, 24, 130), (16, 264, 1000), (17, 2048, 256), (33, 40, 4096), (64, 2048, 8192), (65, 520, 384), (100, 1000, 129),
          (128, 128, 128), (255, 256, 640), (300, 776, 2000), (1000, 2048, 1024), (1031, 1544, 131), (2000, 264, 3968), (700, 4104, 256), (2, 16, 130944)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_i8(hip, dtype, M, N, K):
    say("linear", dtype, M, N, K)
    for bias, junk in ((True, "a"), (False, "w")):
        p = Linear(hip, M, N, K, bias, junk=junk)
        want, bound = p.expect(dtype)
        got = p.run(dtype)
        close(widen(got, dtype), want, bound, "linear")
        assert np.array_equal(p.run(dtype, with_ws=False), got)  # the same bits in every form


def test_linear_i8_widest_strides(hip):
    """rows just below 2^23 bytes apart, of the result 2^23 values: the tiles' offsets in 32 bits, all others past them"""
    M, N, K, ld, ldo = 300, 264, 256, 2 ** 23 - 16, 2 ** 23
    p = Linear(hip, M, N, K)
    want, bound = p.expect(F16)
    a, w, o = hip.DeviceArray((M, ld), np.int8), hip.DeviceArray((N, ld), np.int8), hip.DeviceArray((M, ldo), np.uint16)
    for d, rows in ((a, p.a), (w, p.w)):
        for i in range(len(rows)):
            hip.check(hip.lib().hxa_h2d(d.at(i * ld), rows[i].ctypes.data, K))
    for tile in ((256, 256), (192, 192), (128, 128), (64, 64), (64, 32), (32, 16), (16, 16)):
        for i in range(M):
            hip.check(hip.lib().hxa_memset(o.at(i * ldo * 2), 0x55, (N + 8) * 2))
        hip.check(hip.lib().hxa_linear_i8_tile(F16, a.ptr, ld, p.d[1].ptr, M, w.ptr, ld, p.d[3].ptr, N, K, p.db.ptr, o.ptr, ldo, *tile, 1, None, 0, None))
        hip.sync()
        got = np.zeros((M, N + 8), np.uint16)
        for i in range(M):
            hip.check(hip.lib().hxa_d2h(got[i].ctypes.data, o.at(i * ldo * 2), (N + 8) * 2))
        assert (got[:, N:] == 0x5555).all()
        close(widen(got[:, :N], F16), want, bound, f"strides {tile}")


TILES = [(256, 256), (256, 192), (192, 256), (192, 192), (256, 128), (128, 256), (192, 128), (128, 128), (64, 128), (128, 64), (64, 64), (64, 32), (32, 32), (32, 16), (16, 16)]


@pytest.mark.parametrize("M,N,K", [(1, 8, 128), (70, 200, 640), (300, 520, 1280), (513, 264, 256), (40, 40, 5120)])
def test_linear_i8_tiles(hip, M, N, K):
    """every tile and number of slices gives the same bits"""
    p = Linear(hip, M, N, K)
    want, bound = p.expect(BF16)
    first = p.run(BF16)
    close(widen(first, BF16), want, bound, "linear")
    for bm, bn in TILES:
        for S in (1, 2, 5):
            if K % (128 * S) or (bn <= 32 and S > 1):
                continue
            say("tile", bm, bn, S)
            assert np.array_equal(p.run(BF16, tile=(bm, bn, S)), first), (bm, bn, S)


def test_linear_i8_largest_sums(hip):
    """every product 2^14, K as long as it may be: the sum just fits; scales and bias that are not finite reach their row and column alone"""
    p = Linear(hip, 40, 48, hip.I8_MAX_K, gap=(0, 0, 0))
    p.a[:], p.w[:] = -128, -128
    p.d[0].upload(p.a), p.d[2].upload(p.w)
    want, bound = p.expect(F16)
    assert np.isinf(widen(narrow(want, F16), F16)).any()
    for tile in (None, (64, 64, 1), (128, 128, 3), (32, 32, 1)):
        got = widen(p.run(BF16, tile=tile), BF16)
        close(got, *p.expect(BF16), "largest")
    p.sa[3], p.sw[5], p.bias[7] = np.nan, np.inf, -np.inf
    p.d[1].upload(p.sa), p.d[3].upload(p.sw), p.db.upload(p.bias)
    got = widen(p.run(BF16), BF16)
    assert np.isnan(got[3]).all() and (got[:3, 5] == np.inf).all() and (got[:3, 7] == -np.inf).all()
    assert np.isfinite(np.delete(np.delete(got, 3, 0), [5, 7], 1)).all()


# ------------------------------------------------------------------------------------------------------------- append
def run_append(hip, c, k, v, T, gain, freq, rot, layout, stream=None, mscale=1.0):
    plan = c.q8
    d = [dev(hip, k), dev(hip, v), dev(hip, gain) if gain is not None else None, dev(hip, freq)]
    rope = hip.Rope(d[3].ptr, rot, layout, mscale)
    hip.check(hip.lib().hxa_kv_append_q8(C.byref(plan), d[0].ptr, k.shape[1], d[1].ptr, v.shape[1], T, d[2].ptr if d[2] else None, EPS,
                                         C.byref(rope) if rot else None, stream), "append")
    hip.sync()


def check_append(hip, c, k, v, T, gain, freq, layout, what):
    """the cache on the device after an append to c; c takes its bytes and scales over"""
    want = append(c, k, v, gain, EPS, freq, layout, T)
    got = {n: c.d[n].numpy() for n in ("k", "v", "ks", "vs")}
    assert np.array_equal(got["v"], want["v"]) and np.array_equal(got["vs"], want["vs"], equal_nan=True), what + ": values"
    seen = np.ones(c.k.shape, bool)
    for (pg, h), (r0, x, mag, sc, old) in want["kval"].items():
        n, s = len(x), float(got["ks"][pg, h])
        err = head_bound(x, mag, c.hd, F16) - HALF_STEP[F16] * np.abs(x) - TINY[F16]  # the 32-bit steps alone
        # the scale is the largest magnitude / 127, or the earlier one doubled
        assert abs(s - sc) <= err.max() / 127 + 4 * U24 * sc, what + ": key scale"
        if old > 0:
            assert np.log2(s / old) % 1 == 0
        y = got["k"][pg, h, r0:r0 + n] * s
        close(y, np.clip(x, -127 * s, 127 * s), np.full(x.shape, s / 2) + err + 127 * s * 4 * U24, what + ": keys")
        seen[pg, h, r0:r0 + n] = False
    assert np.array_equal(got["k"][seen], want["k"][seen]), what + ": earlier keys"
    assert np.array_equal(np.isnan(got["ks"]), np.isnan(want["ks"]))
    untouched = [(pg, h) for pg in range(c.npages) for h in range(c.H) if (pg, h) not in want["kval"]]
    assert all(got["ks"][at] == c.ks[at] or np.isnan(c.ks[at]) for at in untouched)
    c.k, c.v, c.ks, c.vs = got["k"], got["v"], got["ks"], got["vs"]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,H,new,past,prefix,page,rot,layout", [
    (128, 8, [1] * 70, [0, 5, 15, 16, 17] * 14, 100, 16, 128, 0), (64, 3, [0, 40, 1, 0, 129], [7, 0, 33, 4, 1], 0, 32, 32, 1),
    (256, 2, [5], [1234], 1000, 1, 256, 1), (128, 1, [64, 64, 200], [0, 1, 63], 3, 64, 128, 0), (64, 1, [1, 0, 2] * 100, [0, 0, 3] * 100, 0, 4, 0, 0),
    (256, 2, [130, 70, 1], [0, 100, 127], 0, 128, 64, 0), (128, 2, [300, 3], [11, 250], 7, 256, 16, 1), (64, 2, [500], [77], 0, 300, 64, 0)])
def test_kv_append_q8(hip, dtype, hd, H, new, past, prefix, page, rot, layout):
    say("append", dtype, hd, H, len(new), prefix, page)
    rng = np.random.default_rng(hd + len(new))
    c = CacheQ8(hip, rng, new, past, prefix, page, H, hd, dtype, spread=1.0)
    n, tail = int(c.cu[-1]), 2
    if len(new) > 2:  # tokens of a page that is not in the pool, and negative positions, stay out
        c.table[2, past[2] // page] = c.npages
        i = 3 if len(new) > 3 and new[3] else 1
        c.lens[i] = 0 if i == 3 else new[1] - 2
    ldk, ldv = H * hd + 8, H * hd + 24
    k, v = (narrow(rng.standard_normal((n + tail, ld)) * np.exp(rng.standard_normal((n + tail, 1))), dtype) for ld in (ldk, ldv))
    g = (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32)
    freq = hip.rope_freqs(rot, 1e6)[0] if rot else np.zeros(1, np.float32)
    c.upload()
    run_append(hip, c, k, v, n + tail, g, freq, rot, layout)
    check_append(hip, c, k, v, n + tail, g, freq[:rot // 2], layout, "append")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,page", [(64, 5), (128, 16), (256, 70)])
def test_a_page_filled_token_by_token(hip, dtype, hd, page):
    """values that grow over the calls: every call by the definition, and at the end each value within one step of what went in"""
    rng = np.random.default_rng(page)
    H, n = 2, 2 * page + 3
    c = CacheQ8(hip, rng, [1], [0], 0, page, H, hd, dtype, empty=True)
    c.lens = [n]
    c = CacheQ8(hip, rng, [1], [n - 1], 0, page, H, hd, dtype, empty=True)
    x = rng.standard_normal((n, H * hd)) * np.exp2(rng.uniform(-1, 5, (n, 1)) * np.linspace(0, 1, n)[:, None])
    x[0] = 0  # a page that begins with zeros
    k = narrow(x, dtype)
    freq = np.zeros(1, np.float32)
    for t in range(n):
        c.lens, c.past = [t + 1], [t]
        c.upload()
        run_append(hip, c, k[t:t + 1], k[t:t + 1], 1, None, freq, 0, 0)
        check_append(hip, c, k[t:t + 1], k[t:t + 1], 1, None, freq[:0], 0, f"token {t}")
    grown = 0
    val = widen(k, dtype).reshape(n, H, hd)
    for pool, sc in ((c.k, c.ks), (c.v, c.vs)):
        for t in range(n):
            pg = c.table[0, t // page]
            s = sc[pg].astype(np.float64)[:, None]
            d = np.abs(pool[pg, :, t % page] * s - val[t])
            assert (d < s * (1 + 127 * 8 * U24)).all()
            grown += int((d > 0.51 * s).any())
    assert grown  # some were rounded more than once


def test_append_special_values(hip):
    """NaN and infinities take no part in a scale; old scales that are none; growth by many doublings; a scale's least value"""
    hd, H, page = 64, 4, 16
    rng = np.random.default_rng(4)
    c = CacheQ8(hip, rng, [3], [5], 0, page, H, hd, BF16)
    pg = c.table[0, 0]
    c.ks[pg], c.vs[pg] = [np.nan, np.inf, -1.0, 2.0 ** -60], [0.0, np.nan, 1e-30, 2.0 ** -64]
    x = rng.standard_normal((3, H * hd)).astype(np.float32)
    x[0, 3], x[1, 70], x[2, 140] = np.nan, np.inf, -np.inf
    x[:, 192:] *= 1e30
    k = narrow(x, BF16)
    c.upload()
    run_append(hip, c, k, k, 3, None, np.zeros(1, np.float32), 0, 0)
    for pool, sc, was, sold in (("k", "ks", c.k, c.ks), ("v", "vs", c.v, c.vs)):
        q, s = c.d[pool].numpy()[pg], c.d[sc].numpy()[pg].astype(np.float64)
        val = widen(k, BF16).reshape(3, H, hd).transpose(1, 0, 2)
        fin = np.where(np.isfinite(val), val, 0)
        assert (s >= np.abs(fin).max((1, 2)) / 127 * (1 - 4 * U24)).all() and (s <= 2 * np.abs(fin).max((1, 2)) / 127).all()
        want = np.where(np.isnan(val), 0, np.clip(val, -127 * s[:, None, None], 127 * s[:, None, None]))
        assert (np.abs(q[:, 5:8] * s[:, None, None] - want) <= s[:, None, None] * (0.5 + 127 * 8 * U24)).all()
        assert not q[3, :5].any()  # shifted out
        held = [h for h in range(3) if not (np.isfinite(sold[pg, h]) and sold[pg, h] > 0)]
        assert np.array_equal(q[held, :5], was[pg][held][:, :5]) and np.array_equal(q[:, 8:], was[pg][:, 8:])
    # values below the least scale become zeros
    c = CacheQ8(hip, rng, [2], [0], 0, page, 1, hd, BF16, empty=True)
    k = narrow(np.full((2, hd), 1e-25, np.float32), BF16)
    c.upload()
    run_append(hip, c, k, k, 2, None, np.zeros(1, np.float32), 0, 0)
    assert c.d["ks"].numpy()[c.table[0, 0], 0] == np.float32(2.0 ** -64) and not c.d["k"].numpy()[c.table[0, 0], 0, :2].any()


# ------------------------------------------------------------------------------------------------------------- attention
def run_cached(hip, c, q, scale, with_ws=True, stream=None):
    n, Hq = q.shape[0], q.shape[1]
    hd, tail = c.hd, 2
    qn = np.full((n + tail, Hq * hd + 8), np.nan, np.float32)
    qn[:n, :Hq * hd] = q.reshape(n, -1)
    plan = c.upload()
    dq, do = dev(hip, narrow(qn, c.dtype)), dev(hip, np.full((n + tail, Hq * hd + 16), 0x5555, np.uint16))
    L = hip.lib()
    nb = L.hxa_attention_cached_q8_ws_bytes(C.byref(plan), n + tail, Hq)
    ws = dev(hip, np.full(max(nb, 16), 0xff, np.uint8))
    hip.check(L.hxa_attention_cached_q8(C.byref(plan), dq.ptr, Hq * hd + 8, do.ptr, Hq * hd + 16, n + tail, Hq, scale,
                                        ws.ptr if with_ws else None, nb if with_ws else 0, stream), "cached")
    hip.sync()
    o = do.numpy()
    assert (o[n:] == 0x5555).all() and (o[:, Hq * hd:] == 0x5555).all()
    return widen(o[:n, :Hq * hd], c.dtype).reshape(n, Hq, hd)


def check_cached(hip, c, q, scale, with_ws, what):
    got = run_cached(hip, c, q, scale, with_ws)
    o, a, n, smax, _ = c.expect(q, scale)
    close(got, o, c.bound(o, a, n, smax, scale), what)
    return got


@pytest.mark.parametrize("with_ws", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,Hq,H,new,past,prefix,page", CACHED + MIXED)
def test_attention_cached_q8(hip, dtype, hd, Hq, H, new, past, prefix, page, with_ws):
    say("cached", dtype, hd, Hq, H, len(new), prefix, page, with_ws)
    rng = np.random.default_rng(hd + prefix + len(new))
    c = CacheQ8(hip, rng, new, past, prefix, page, H, hd, dtype)
    q = queries(rng, int(c.cu[-1]), Hq, hd, dtype)
    got = check_cached(hip, c, q, hd ** -0.5, with_ws, "cached")
    assert np.array_equal(run_cached(hip, c, q, hd ** -0.5, with_ws), got)


FORMS = [(128, 8, 4, [1] * 6, [0, 10, 100, 64, 33, 2], 300), (64, 2, 1, [70, 40], [30, 0], 64), (256, 4, 2, [1] * 40, [7] * 40, 300),
         (128, 96, 48, [130, 90], [20, 300], 40)]


@pytest.mark.parametrize("with_ws", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,Hq,H,new,past,prefix", FORMS)
def test_cached_q8_bad_pages_and_empty_rows(hip, dtype, hd, Hq, H, new, past, prefix, with_ws):
    say("bad pages", dtype, hd, with_ws)
    rng = np.random.default_rng(1)
    page = 16
    c = CacheQ8(hip, rng, new, past, prefix, page, H, hd, dtype, bad={("prefix", 1): -1, ("prefix", 2): 10 ** 6, (1, 0): 2 ** 31 - 1})
    q = queries(rng, int(c.cu[-1]), Hq, hd, dtype)
    check_cached(hip, c, q, hd ** -0.5, with_ws, "bad pages")
    bad = {("prefix", s): -5 for s in range(-(-prefix // page))} | {(0, s): 99999 for s in range(c.ldt)}
    c = CacheQ8(hip, rng, new, past, prefix, page, H, hd, dtype, bad=bad)
    got = run_cached(hip, c, q, hd ** -0.5, with_ws)
    assert (got[:new[0]] == 0).all() and (got[new[0]:] != 0).any()


@pytest.mark.parametrize("with_ws", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,Hq,H,new,past,prefix", FORMS)
def test_cached_q8_scales(hip, dtype, hd, Hq, H, new, past, prefix, with_ws):
    """value scales from 2^-40 to 2^8 side by side; scales that are 0, negative, infinite or NaN: pages of zeros"""
    rng = np.random.default_rng(2)
    c = CacheQ8(hip, rng, new, past, prefix, 16, H, hd, dtype)
    q = queries(rng, int(c.cu[-1]), Hq, hd, dtype)
    c.vs = np.where(np.isfinite(c.vs), np.exp2(rng.uniform(-40, 8, c.vs.shape)), np.nan).astype(np.float32)
    check_cached(hip, c, q, hd ** -0.5, with_ws, "wide value scales")
    for sc in (c.ks, c.vs):
        sc[rng.random(sc.shape) < 0.2] = 0
        sc[rng.random(sc.shape) < 0.1] = np.inf
        sc[rng.random(sc.shape) < 0.1] = -1
        sc[rng.random(sc.shape) < 0.1] = np.nan
    check_cached(hip, c, q, hd ** -0.5, with_ws, "no scales")
    c.vs[:] = 0
    assert (run_cached(hip, c, q, hd ** -0.5, with_ws) == 0).all()


@pytest.mark.parametrize("hd,Hq,H,new,past,prefix", FORMS)
def test_cached_q8_small_values_count(hip, hd, Hq, H, new, past, prefix):
    """a row whose weight lies on keys of small values keeps their bits beside pages of large ones"""
    rng = np.random.default_rng(6)
    c = CacheQ8(hip, rng, new, past, prefix, 16, H, hd, F16, spread=0.0)
    c.vs[:] = np.where(rng.random(c.vs.shape) < 0.5, 1e-5, 1.0) * np.ones_like(c.vs)
    big = c.vs > 0.5
    c.k[big] = np.clip(c.k[big], -127, 0)
    c.k[~big] = np.clip(c.k[~big], 0, 127)
    q = np.abs(queries(rng, int(c.cu[-1]), Hq, hd, F16))
    check_cached(hip, c, q, 2.0 * hd ** -0.5, True, "small values")
    check_cached(hip, c, q, 2.0 * hd ** -0.5, False, "small values")


@pytest.mark.parametrize("with_ws", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,Hq,H,new,past,prefix", FORMS)
def test_cached_q8_steep_scores_and_wide_queries(hip, dtype, hd, Hq, H, new, past, prefix, with_ws):
    rng = np.random.default_rng(31)
    c = CacheQ8(hip, rng, new, past, prefix, 16, H, hd, dtype)
    q = queries(rng, int(c.cu[-1]), Hq, hd, dtype, std=8.0)
    check_cached(hip, c, q, 1.0, with_ws, "steep")
    # queries of very different sizes, scores as before
    f = np.exp2(np.round(rng.uniform(-100, 100, q.shape[:2]))) if dtype == BF16 else np.exp2(np.round(rng.uniform(-6, 10, q.shape[:2])))
    q = widen(narrow(q * f[..., None], dtype), dtype)
    c.ks[:] = c.ks * (np.float32(2.0 ** -100) if dtype == BF16 else np.float32(2.0 ** -10))
    check_cached(hip, c, q, 1.0, with_ws, "wide queries")
    q[0] = 0
    check_cached(hip, c, q, 1.0, with_ws, "a query of zeros")


@pytest.mark.parametrize("with_ws", [True, False])
@pytest.mark.parametrize("hd,Hq,H,new,past,prefix,page", [
    (128, 4, 2, [100, 3], [1500, 700], 600, 1), (64, 8, 2, [40, 90], [1300, 0], 1111, 2), (256, 2, 1, [64, 1, 30], [1700, 5, 64], 0, 3),
    (128, 8, 1, [17, 1], [5000, 4200], 40, 8)])
def test_cached_q8_more_pages_than_the_table(hip, hd, Hq, H, new, past, prefix, page, with_ws):
    """ranges of several times 512 pages, of the prefix and of the sequences, in every mode; pages that are not there and scales that are none in the later ones"""
    say("many pages", hd, page, with_ws)
    rng = np.random.default_rng(hd + page)
    c = CacheQ8(hip, rng, new, past, prefix, page, H, hd, F16)
    q = queries(rng, int(c.cu[-1]), Hq, hd, F16)
    check_cached(hip, c, q, hd ** -0.5, with_ws, "many pages")
    c = CacheQ8(hip, rng, new, past, prefix, page, H, hd, F16, bad={(0, 513): -1, (0, 514): 10 ** 6, (0, 580): 2 ** 31 - 1})
    c.vs[rng.random(c.vs.shape) < 0.1] = 0
    c.ks[rng.random(c.ks.shape) < 0.1] = np.nan
    check_cached(hip, c, q, hd ** -0.5, with_ws, "many pages, some bad")


def test_cached_q8_queries_not_finite(hip):
    """a NaN or infinite query makes its own row NaN and no other"""
    rng = np.random.default_rng(3)
    for dtype in (F16, BF16):
        for hd, Hq, H, new, past, prefix in FORMS:
            c = CacheQ8(hip, rng, new, past, prefix, 16, H, hd, dtype)
            q = queries(rng, int(c.cu[-1]), Hq, hd, dtype)
            clean = run_cached(hip, c, q, hd ** -0.5)
            q[1, 0, 3], q[2, Hq - 1, 1] = np.nan, np.inf
            got = run_cached(hip, c, q, hd ** -0.5)
            assert np.isnan(got[1, 0]).all()
            hit = np.zeros(q.shape[:2], bool)
            hit[1, 0] = hit[2, Hq - 1] = True
            assert np.array_equal(got[~hit], clean[~hit])


def test_cached_q8_lengths_out_of_range(hip):
    """len below the new tokens and past the table, a prefix alone, cu past the rows"""
    rng = np.random.default_rng(4)
    hd, Hq, H, page = 128, 4, 2, 16
    for prefix in (0, 100, 400):
        c = CacheQ8(hip, rng, [3, 2, 2], [0, 30, 5], prefix, page, H, hd, F16)
        c.ldt = 2
        c.table = np.ascontiguousarray(c.table[:, :2])
        q = queries(rng, 7, Hq, hd, F16)
        held = CacheQ8.__new__(CacheQ8)
        held.__dict__.update(c.__dict__)
        held.lens, held.past = [1, 32, 7], [-2, 10 ** 6, 5]
        c.lens = [1, 10 ** 9, 7]
        o, a, n, smax, _ = held.expect(q, hd ** -0.5)
        for ws in (True, False):
            got = run_cached(hip, c, q, hd ** -0.5, ws)
            close(got, o, held.bound(o, a, n, smax, hd ** -0.5), "lengths")
            assert prefix or (got[:2] == 0).all()
    c = CacheQ8(hip, rng, [1, 2], [0, 0], 300, page, H, hd, F16)
    q = queries(rng, 3, Hq, hd, F16)
    c.ldt, c.table = 0, np.zeros((2, 0), np.int32)
    none = CacheQ8.__new__(CacheQ8)
    none.__dict__.update(c.__dict__)
    none.lens, none.past = [0, 0], [10 ** 6] * 2
    o, a, n, smax, _ = none.expect(q, hd ** -0.5)
    for ws in (True, False):
        close(run_cached(hip, c, q, hd ** -0.5, ws), o, none.bound(o, a, n, smax, hd ** -0.5), "prefix alone")


def test_q8_offsets_past_32_bits(hip):
    """pools of 5 GB with the pages at their end: append, then attention"""
    L, rng = hip.lib(), np.random.default_rng(6)
    Hq, H, hd, page, n = 4, 2, 128, 64, 130
    npages = 5 * 2 ** 30 // (H * page * hd)
    kc, vc = (hip.DeviceArray((npages * H * page * hd,), np.int8) for _ in range(2))
    ks, vs = (hip.DeviceArray((npages, H), np.float32, zero=True) for _ in range(2))
    pages = np.array([npages - 1, npages - 3, npages - 2], np.int32)
    k, v, q = (narrow(rng.standard_normal((n, w * hd)), F16) for w in (H, H, Hq))
    d = [dev(hip, np.array(a, np.int32)) for a in ([0, n], pages, [n])]
    x = [dev(hip, a) for a in (k, v, q, np.zeros((n, Hq * hd), np.uint16))]
    plan = hip.KvCacheQ8(hip.KvCache(F16, H, hd, page, npages, kc.ptr, vc.ptr, None, 0, d[1].ptr, 3, d[2].ptr, d[0].ptr, 1), ks.ptr, vs.ptr)
    hip.check(L.hxa_kv_append_q8(C.byref(plan), x[0].ptr, H * hd, x[1].ptr, H * hd, n, None, 0.0, None, None))
    hip.check(L.hxa_attention_cached_q8(C.byref(plan), x[2].ptr, Hq * hd, x[3].ptr, Hq * hd, n, Hq, hd ** -0.5, None, 0, None))
    hip.sync()
    c = CacheQ8(hip, rng, [n], [0], 0, page, H, hd, F16, empty=True)
    c.table[0, :3] = c.npages - 1, c.npages - 3, c.npages - 2
    at = npages - c.npages
    one = H * page * hd
    for p in c.table[0, :3]:
        for big, pool in ((kc, c.k), (vc, c.v)):
            hip.check(L.hxa_d2h(pool[p].ctypes.data, big.at((int(p) + at) * one), one))
    c.ks, c.vs = ks.numpy()[at:], vs.numpy()[at:]
    for pool, rows in ((c.k, k), (c.v, v)):
        val = c.values(pool)
        got = np.stack([val[c.table[0, t // page], :, t % page] for t in range(n)])
        s = (c.ks if pool is c.k else c.vs).max()
        assert np.abs(got - widen(rows, F16).reshape(n, H, hd)).max() <= s * 0.5001
    o, a, m, smax, _ = c.expect(widen(q, F16).reshape(n, Hq, hd), hd ** -0.5)
    close(widen(x[3].numpy(), F16).reshape(n, Hq, hd), o, c.bound(o, a, m, smax, hd ** -0.5), "cached")


def test_q8_two_streams_at_once(hip):
    """calls in flight on two streams, each with its own workspace and output, give what they give alone, bit for bit"""
    rng = np.random.default_rng(77)
    L, hd, Hq, H = hip.lib(), 128, 8, 2
    jobs = []
    for new, past, prefix in (([1] * 20, [400] * 20, 600), ([1] * 3, [3000, 20, 900], 256)):
        c = CacheQ8(hip, rng, new, past, prefix, 16, H, hd, BF16)
        st = C.c_void_p()
        hip.check(L.hxa_stream_create(C.byref(st)))
        plan = c.upload()
        n = len(new)
        nb = L.hxa_attention_cached_q8_ws_bytes(C.byref(plan), n, Hq)
        p = Linear(hip, n, 256, Hq * hd, seed=n)
        lb = L.hxa_linear_i8_ws_bytes(n, 256, Hq * hd)
        bufs = dict(q=dev(hip, narrow(queries(rng, n, Hq, hd, BF16), BF16)), o=dev(hip, np.zeros((n, Hq * hd), np.uint16)), ws=hip.DeviceArray((nb,), np.uint8),
                    b=hip.DeviceArray((n, Hq * hd), np.int8), s=hip.DeviceArray((n,), np.float32), y=dev(hip, np.zeros((n, 256), np.uint16)),
                    lw=hip.DeviceArray((max(lb, 16),), np.uint8))
        jobs.append((c, plan, n, nb, lb, p, bufs, st))

    def go(j, st):
        c, plan, n, nb, lb, p, b, _ = j
        hip.check(L.hxa_attention_cached_q8(C.byref(plan), b["q"].ptr, Hq * hd, b["o"].ptr, Hq * hd, n, Hq, hd ** -0.5, b["ws"].ptr, nb, st))
        hip.check(L.hxa_quantize_rows(BF16, b["o"].ptr, Hq * hd, n, Hq * hd, b["b"].ptr, Hq * hd, b["s"].ptr, st))
        hip.check(L.hxa_linear_i8(BF16, b["b"].ptr, Hq * hd, b["s"].ptr, n, p.d[2].ptr, p.ldw, p.d[3].ptr, 256, Hq * hd, p.db.ptr, b["y"].ptr, 256,
                                  b["lw"].ptr, lb, st))

    alone = []
    for j in jobs:
        go(j, None)
        hip.sync()
        alone.append([j[6][n].numpy().copy() for n in ("o", "y")])
        j[6]["o"].upload(np.zeros_like(alone[-1][0]))
    for _ in range(10):
        for j in jobs:
            go(j, j[7])
    hip.sync()
    for j, want in zip(jobs, alone):
        assert all(np.array_equal(j[6][n].numpy(), w) and w.any() for n, w in zip(("o", "y"), want))
        hip.check(L.hxa_stream_destroy(j[7]))


# --------------------------------------------------------------------------------------------------------- as it is used
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_a_layer_in_8_bits(hip, dtype):
    """Hidden states to int8, the fused qkv product, queries normed and turned, keys and values into the cache, attention, its result to int8 and the output
    product: prompts behind a template, then single-token steps, eager and as one captured graph whose replays follow the lengths on the device. Each
    operator's result is checked by its definition on what the one before it left."""
    rng = np.random.default_rng(12)
    L, Hq, H, hd, D, page, P = hip.lib(), 8, 2, 128, 500, 16, 70
    W, scale = (Hq + 2 * H) * hd, hd ** -0.5
    rest, steps = [5, 1, 40], 3
    c = CacheQ8(hip, rng, [n + steps for n in rest], [0] * 3, P, page, H, hd, dtype)
    c.k[c.table[c.table >= 0]] = -128
    plan = c.upload()
    gq, gk = ((1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2))
    freq, _ = hip.rope_freqs(hd, 10000.0)
    dgq, dgk, df = dev(hip, gq), dev(hip, gk), dev(hip, freq)
    rope = hip.Rope(df.ptr, hd, 0, 1.0)
    st = C.c_void_p()
    hip.check(L.hxa_stream_create(C.byref(st)))
    weights = {}
    for name, N, K in (("qkv", W, D), ("o", D // 8 * 8, Hq * hd)):
        w = narrow(np.pad(rng.standard_normal((N, K)) * 0.05, ((0, 0), (0, -K % 8))), dtype)
        dw, q, s = dev(hip, w), hip.DeviceArray((N, round128(K)), np.int8), hip.DeviceArray((N,), np.float32)
        hip.check(L.hxa_quantize_rows(dtype, dw.ptr, w.shape[1], N, K, q.ptr, round128(K), s.ptr, st))
        hip.sync()
        weights[name] = (q, s, N, K)

    def buffers(n):
        A = hip.DeviceArray
        b = dict(x=A((n, 504), np.uint16), xq=A((n, 512), np.int8), xs=A((n,), np.float32), qkv=A((n, W), np.uint16), q=A((n, Hq * hd), np.uint16),
                 o=A((n, Hq * hd), np.uint16), oq=A((n, Hq * hd), np.int8), os=A((n,), np.float32), y=A((n, 496), np.uint16),
                 pos=A((n,), np.int32), cu=A((4,), np.int32))
        p = hip.KvCacheQ8.from_buffer_copy(plan)
        p.c.cu, p.c.len = b["cu"].ptr, c.d["len"].ptr
        b["plan"], b["n"] = p, n
        sizes = [L.hxa_attention_cached_q8_ws_bytes(C.byref(p), n, Hq)] + [L.hxa_linear_i8_ws_bytes(n, w[2], w[3]) for w in weights.values()]
        b["nb"] = max(sizes + [16])
        b["ws"] = A((b["nb"],), np.uint8)
        return b

    def linear(b, q, ld, s, name, out, ldo):
        wq, ws, N, K = weights[name]
        hip.check(L.hxa_linear_i8(dtype, b[q].ptr, ld, b[s].ptr, b["n"], wq.ptr, round128(K), ws.ptr, N, K, None, b[out].ptr, ldo, b["ws"].ptr, b["nb"], st))

    def calls(b):
        n, p, x = b["n"], b["plan"], b["qkv"]
        hip.check(L.hxa_quantize_rows(dtype, b["x"].ptr, 504, n, D, b["xq"].ptr, 512, b["xs"].ptr, st))
        linear(b, "xq", 512, "xs", "qkv", "qkv", W)
        hip.check(L.hxa_qk_norm_rope(dtype, x.ptr, W, Hq, None, 0, 0, n, hd, dgq.ptr, None, EPS, b["pos"].ptr, C.byref(rope), b["q"].ptr, Hq * hd,
                                     None, 0, st))
        hip.check(L.hxa_kv_append_q8(C.byref(p), x.at(Hq * hd * 2), W, x.at((Hq + H) * hd * 2), W, n, dgk.ptr, EPS, C.byref(rope), st))
        hip.check(L.hxa_attention_cached_q8(C.byref(p), b["q"].ptr, Hq * hd, b["o"].ptr, Hq * hd, n, Hq, scale, b["ws"].ptr, b["nb"], st))
        hip.check(L.hxa_quantize_rows(dtype, b["o"].ptr, Hq * hd, n, Hq * hd, b["oq"].ptr, Hq * hd, b["os"].ptr, st))
        linear(b, "oq", Hq * hd, "os", "o", "y", 496)

    def load(b, lo, hi):
        x = np.concatenate([states[i][a:e] for i, (a, e) in enumerate(zip(lo, hi))])
        b["x"].upload(x)
        c.cu = np.cumsum([0] + [e - a for a, e in zip(lo, hi)]).astype(np.int32)
        c.lens, c.new, c.past = list(hi), [e - a for a, e in zip(lo, hi)], list(lo)
        b["cu"].upload(c.cu)
        c.d["len"].upload(np.array(hi, np.int32))
        b["pos"].upload(np.concatenate([P + np.arange(a, e) for a, e in zip(lo, hi)]).astype(np.int32))

    def check(b, what):
        n = b["n"]
        g = {k: b[k].numpy() for k in ("x", "xq", "xs", "qkv", "q", "o", "oq", "os", "y", "pos")}
        for x, K, q, s in (("x", D, "xq", "xs"), ("o", Hq * hd, "oq", "os")):
            wq, ws = quantize(widen(g[x][:, :K], dtype))
            assert np.array_equal(g[q][:, :K], wq) and np.array_equal(g[s], ws) and not g[q][:, K:].any(), what
        for q, s, name, out in (("xq", "xs", "qkv", "qkv"), ("oq", "os", "o", "y")):
            wq, ws, N, K = weights[name]
            want = g[q].astype(np.float64) @ wq.numpy().astype(np.float64).T * g[s].astype(np.float64)[:, None] * ws.numpy().astype(np.float64)
            close(widen(g[out][:, :N], dtype), want, linear_bound(want, want, dtype), what + " " + name)
        u, mag = norm_rope(widen(g["qkv"][:, :Hq * hd], dtype).reshape(n, Hq, hd), gq, EPS, g["pos"], freq, 0)
        close(widen(g["q"], dtype).reshape(n, Hq, hd), u, head_bound(u, mag, hd, dtype), what + " queries")
        check_append(hip, c, np.ascontiguousarray(g["qkv"][:, Hq * hd:(Hq + H) * hd]), np.ascontiguousarray(g["qkv"][:, (Hq + H) * hd:]), n, gk, freq, 0,
                     what + " append")
        qh = widen(g["q"], dtype).reshape(n, Hq, hd)
        o, a, m, smax, _ = c.expect(qh, scale)
        close(widen(g["o"], dtype).reshape(n, Hq, hd), o, c.bound(o, a, m, smax, scale), what + " attention")

    states = [narrow(rng.standard_normal((n + steps, 504)), dtype) for n in rest]
    b = buffers(sum(rest))
    load(b, [0, 0, 0], rest)
    calls(b)
    hip.sync()
    check(b, "prompts")
    b = buffers(3)
    g = C.c_void_p()
    load(b, rest, [n + 1 for n in rest])
    hip.check(L.hxa_stream_begin_capture(st, 1))
    calls(b)
    hip.check(L.hxa_stream_end_capture(st, C.byref(g)))
    for step in range(steps):
        load(b, [n + step for n in rest], [n + step + 1 for n in rest])
        hip.check(L.hxa_graph_launch(g, st))
        hip.sync()
        check(b, f"step {step}")
        y = b["y"].numpy()
        b["y"].upload(np.zeros_like(y))
        calls(b)  # the same tokens again change nothing
        hip.sync()
        assert np.array_equal(b["y"].numpy(), y) and all(np.array_equal(c.d[n].numpy(), getattr(c, n), equal_nan=n in ("ks", "vs")) for n in ("k", "v", "ks", "vs"))
    hip.check(L.hxa_graph_exec_destroy(g))
    hip.check(L.hxa_stream_destroy(st))
