"""The causal text model's attention path (q / k norm with rotation, the paged cache, causal attention over packed prompts and over the
cache) against the operators' definitions in 64 bits. The bounds are worst cases of the roundings named in _causal.attend_bound."""
import ctypes as C

import numpy as np
import pytest

from tests._causal import BF16, F16, HALF_STEP, TINY, U24, Cache, Packed, attend, attend_bound, close, narrow, norm_rope, widen

pytestmark = pytest.mark.gpu
EPS = 1e-6


def say(*a):
    print(*a, flush=True)


@pytest.fixture(scope="module")
def hip():
    from hexanima_amd import hip as h
    h.init(0)
    return h


def dev(hip, a):
    return hip.DeviceArray.from_numpy(a)


# ------------------------------------------------------------------------------------------------- norm and rotation
def head_bound(want, mag, hd, dtype, th_turns=0.0):
    """the output's rounding; the fp32 sum of hd squares, its root and three products; sine and cosine of an angle whose turns were
    rounded to 32 bits (pi 2^-24) plus 4 half steps of their own"""
    return HALF_STEP[dtype] * np.abs(want) + TINY[dtype] + (hd / 2 + 32) * U24 * mag


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,Hq,Hk,T,rot,layout,first", [
    (128, 16, 8, 1, 128, 0, 70000), (128, 32, 8, 37, 128, 0, 0), (64, 5, 1, 130, 32, 1, 11), (256, 10, 2, 33, 64, 0, 2 ** 30),
    (64, 3, 3, 1030, 64, 0, 5), (256, 1, 1, 9, 256, 1, 1000000), (128, 7, 0, 5, 16, 0, -3), (128, 0, 3, 5, 112, 1, 2 ** 31 - 6),
    (128, 2, 2, 6, 0, 0, 0)])
def test_qk_norm_rope(hip, dtype, hd, Hq, Hk, T, rot, layout, first):
    say("qk", dtype, hd, Hq, Hk, T, rot, layout, first)
    rng = np.random.default_rng(hd + T)
    L = hip.lib()
    freq, _ = hip.rope_freqs(rot, 10000.0) if rot else (np.zeros(1, np.float32), 1)
    pos = (first + np.arange(T)).astype(np.int32)
    ins, outs, gains = [], [], []
    for H in (Hq, Hk):
        ld = max(H, 1) * hd + 16
        x = narrow(rng.standard_normal((T, ld)) * 3.0, dtype)
        ins.append((x, ld, H))
        gains.append((1.0 + 0.2 * rng.standard_normal(hd)).astype(np.float32))
        outs.append(np.full((T, ld + 8), 0x5555, np.uint16))
    d = [dev(hip, a) for a in (ins[0][0], ins[1][0], gains[0], gains[1], pos, freq, outs[0], outs[1])]
    rope = hip.Rope(d[5].ptr, rot, layout, 1.0)
    p = lambda i, H: d[i].ptr if H else None
    hip.check(L.hxa_qk_norm_rope(dtype, p(0, Hq), ins[0][1], Hq, p(1, Hk), ins[1][1], Hk, T, hd, d[2].ptr, d[3].ptr, EPS, d[4].ptr,
                                 C.byref(rope), p(6, Hq), ins[0][1] + 8, p(7, Hk), ins[1][1] + 8, None), "qk")
    hip.sync()
    for (x, ld, H), g, o in zip(ins, gains, (d[6].numpy(), d[7].numpy())):
        assert (o[:, H * hd:] == 0x5555).all()  # columns past the heads stay
        if H == 0:
            continue
        want, mag = norm_rope(widen(x[:, :H * hd], dtype).reshape(T, H, hd), g, EPS, pos, freq[:rot // 2], layout)
        close(widen(o[:, :H * hd], dtype).reshape(T, H, hd), want, head_bound(want, mag, hd, dtype), "qk")


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_qk_in_place_without_gains_or_positions(hip, dtype):
    """in place on the columns of one projection, no norm, rows as positions, scaled cosines; then a norm without a rotation"""
    rng = np.random.default_rng(3)
    T, Hq, Hk, hd = 19, 6, 2, 64
    ld = (Hq + 2 * Hk) * hd
    x = narrow(rng.standard_normal((T, ld)), dtype)
    freq, m = hip.rope_freqs(hd, 10000.0, hip.ROPE_PARTS, 4.0, 4096.0)
    dx, df = dev(hip, x), dev(hip, freq)
    rope = hip.Rope(df.ptr, hd, 0, m)
    k = dx.at(Hq * hd * 2)
    hip.check(hip.lib().hxa_qk_norm_rope(dtype, dx.ptr, ld, Hq, k, ld, Hk, T, hd, None, None, EPS, None, C.byref(rope), dx.ptr, ld, k, ld,
                                         None), "qk")
    hip.sync()
    got = dx.numpy()
    H = Hq + Hk
    want, mag = norm_rope(widen(x[:, :H * hd], dtype).reshape(T, H, hd), None, EPS, np.arange(T), freq, 0, m)
    close(widen(got[:, :H * hd], dtype).reshape(T, H, hd), want, head_bound(want, mag, hd, dtype), "in place")
    assert np.array_equal(got[:, H * hd:], x[:, H * hd:])
    g = (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32)
    dg = dev(hip, g)
    hip.check(hip.lib().hxa_qk_norm_rope(dtype, dx.ptr, ld, Hq, None, 0, 0, T, hd, dg.ptr, None, 0.0, None, None, dx.ptr, ld, None, 0, None), "qk")
    hip.sync()
    want, mag = norm_rope(widen(got[:, :Hq * hd], dtype).reshape(T, Hq, hd), g, 0.0, np.arange(T), None, 0)
    close(widen(dx.numpy()[:, :Hq * hd], dtype).reshape(T, Hq, hd), want, head_bound(want, mag, hd, dtype), "norm alone")


# ------------------------------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,H,new,past,prefix,page", [
    (128, 8, [1] * 70, [0, 5, 15, 16, 17] * 14, 100, 16), (64, 3, [0, 40, 1, 0, 129], [7, 0, 33, 4, 1], 0, 32),
    (256, 2, [5], [12345], 1000, 1), (128, 1, [64, 64], [0, 1], 3, 64), (64, 1, [1, 0, 2] * 1500, [0, 0, 3] * 1500, 0, 4)])
def test_kv_append(hip, dtype, hd, H, new, past, prefix, page):
    say("append", dtype, hd, H, len(new), prefix, page)
    rng = np.random.default_rng(hd + len(new))
    c = Cache(hip, rng, new, past, prefix, page, H, hd, dtype)
    n, tail = int(c.cu[-1]), 2
    if len(new) > 2:  # two tokens of a page that is not in the pool, and two negative positions, stay out
        c.table[2, (past[2]) // page] = c.npages
        c.lens[3 if new[3] else 1] = 0 if new[3] else new[1] - 2
    ldk, ldv = H * hd + 8, H * hd + 24
    k, v = narrow(rng.standard_normal((n + tail, ldk)), dtype), narrow(rng.standard_normal((n + tail, ldv)), dtype)
    g = (1 + 0.1 * rng.standard_normal(hd)).astype(np.float32)
    freq, _ = hip.rope_freqs(hd // 2, 1e6)
    plan = c.upload()
    dk, dv, dg, df = dev(hip, k), dev(hip, v), dev(hip, g), dev(hip, freq)
    rope = hip.Rope(df.ptr, hd // 2, hip.ROPE_PAIRS, 1.0)
    hip.check(hip.lib().hxa_kv_append(C.byref(plan), dk.ptr, ldk, dv.ptr, ldv, n + tail, dg.ptr, EPS, C.byref(rope), None), "append")
    hip.sync()
    gk, gv = c.d["k"].numpy(), c.d["v"].numpy()
    wk, wv, bound = widen(c.k, dtype), c.v.copy(), np.zeros(c.k.shape)
    for i, b in enumerate(c.cu[:-1]):
        for j in range(new[i]):
            p = c.lens[i] - new[i] + j
            if p < 0 or not 0 <= c.table[i, p // page] < c.npages:
                continue
            at = (c.table[i, p // page], slice(None), p % page)
            x, mag = norm_rope(widen(k[b + j:b + j + 1, :H * hd], dtype).reshape(1, H, hd), g, EPS, [prefix + p], freq, 1)
            wk[at], bound[at] = x[0], head_bound(x[0], mag[0], hd, dtype)
            wv[at] = v[b + j, :H * hd].reshape(H, hd)
    close(widen(gk, dtype), wk, bound, "keys")  # everything else as it was: bound 0
    assert np.array_equal(gv, wv)


# ------------------------------------------------------------------------------------------------------------- causal
def run_causal(hip, b, scale, stream=None):
    o = np.full((b.T, b.ldo), 0x5555, np.uint16)
    d = [dev(hip, x) for x in (b.q, b.k, b.v, b.cu, o)]
    hip.check(hip.lib().hxa_attention_causal(b.dtype, d[0].ptr, b.ldq, d[1].ptr, b.ldk, d[2].ptr, b.ldv, d[4].ptr, b.ldo, b.T, d[3].ptr,
                                             len(b.lens), b.Hq, b.Hk, b.hd, scale, stream), "causal")
    hip.sync()
    o = d[4].numpy()
    assert (o[b.n:] == 0x5555).all() and (o[:, b.Hq * b.hd:] == 0x5555).all()  # rows behind the last sequence, columns past the heads
    return b.heads(o, b.Hq)


def expect_causal(b, scale):
    q, k, v = b.heads(b.q, b.Hq), b.heads(b.k, b.Hk), b.heads(b.v, b.Hk)
    o, bound = np.zeros_like(q), np.zeros_like(q)
    G = b.Hq // b.Hk
    for s, e in zip(b.cu, b.cu[1:]):
        n = e - s
        seen = np.tril(np.ones((n, n), bool))
        for h in range(b.Hq if n else 0):
            kk, vv = k[s:e, h // G], v[s:e, h // G]
            o[s:e, h], a = attend(q[s:e, h], kk, vv, scale, seen)
            smax = float((np.abs(q[s:e, h]) @ np.abs(np.where(np.isfinite(kk), kk, 0)).T).max()) * scale
            bound[s:e, h] = attend_bound(o[s:e, h], a, np.abs(np.where(np.isfinite(vv), vv, 0)).max(), n, b.hd, smax, b.dtype)
    return o, bound


# 64-row workgroups, then (from 512 workgroup places on; 256 with heads of 256) 128-row ones; one to many query heads a key head;
# empty, single-token and tile-crossing sequences
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,Hq,Hk,lens", [
    (128, 16, 8, [77]), (128, 2, 2, [1]), (128, 4, 1, [0, 1, 63, 64, 65, 0, 129, 2]), (64, 6, 2, [200, 33]), (256, 3, 1, [130, 5]),
    (64, 7, 1, [19, 128, 0]), (256, 2, 2, [64, 1]), (128, 40, 1, [50, 3]), (128, 1, 1, [3] * 90), (64, 2, 1, [700]),
    (128, 128, 128, [400]), (64, 96, 48, [11, 700, 64, 0, 300]), (256, 64, 64, [260, 200]), (128, 300, 100, [150, 140])])
def test_attention_causal(hip, dtype, hd, Hq, Hk, lens):
    say("causal", dtype, hd, Hq, Hk, lens)
    b = Packed(hip, np.random.default_rng(sum(lens) + hd), lens, Hq, Hk, hd, dtype)
    scale = hd ** -0.5
    got = run_causal(hip, b, scale)
    want, bound = expect_causal(b, scale)
    close(got, want, bound, "causal")
    assert np.array_equal(run_causal(hip, b, scale), got)  # the same bits again


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,Hq,Hk", [(128, 4, 2), (64, 256, 128), (256, 64, 64), (128, 128, 128)])
def test_causal_steep_scores(hip, dtype, hd, Hq, Hk):
    """scores of hundreds: the maximum moves along the row, and sums are those of one or two keys"""
    b = Packed(hip, np.random.default_rng(5), [210, 90], Hq, Hk, hd, dtype, qstd=8.0)
    want, bound = expect_causal(b, 1.0)
    close(run_causal(hip, b, 1.0), want, bound, "steep")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,Hq,Hk", [(128, 4, 2), (64, 3, 1), (256, 2, 1), (128, 128, 128), (64, 256, 256), (256, 64, 64)])
def test_causal_infinities_and_nan_stay_behind_the_mask(hip, dtype, hd, Hq, Hk):
    """keys and values of later tokens that are not finite leave the rows before them alone, and reach the rows after"""
    b = Packed(hip, np.random.default_rng(9), [150, 140], Hq, Hk, hd, dtype)
    inf, nan = narrow(np.float32(np.inf), dtype), narrow(np.float32(np.nan), dtype)
    b.v[40, 3], b.v[41, hd - 1], b.v[100, 5], b.v[149, :hd] = inf, inf | 0x8000, nan, inf
    b.v[150 + 70, 9] = nan
    b.k[120, 0], b.k[150 + 139, 1] = nan, nan
    want, bound = expect_causal(b, hd ** -0.5)
    got = run_causal(hip, b, hd ** -0.5)
    close(got[:40], want[:40], bound[:40], "rows before")
    close(got, want, bound, "all rows")
    assert np.isfinite(want[150:220]).all() and np.isnan(want[220:, :, 9]).any()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_scores_of_minus_infinity(hip, dtype, hd):
    """a row that sees nothing but scores of -infinity gets zeros; beside finite ones such a key weighs nothing"""
    b = Packed(hip, np.random.default_rng(2), [3], 1, 1, hd, dtype)
    b.q[:, 0] = narrow(np.float32(-1), dtype)
    b.q[0, 1:hd] = 0
    b.k[0, :hd] = 0
    b.k[0, 0] = narrow(np.float32(np.inf), dtype)
    got = run_causal(hip, b, 0.1)
    q, k, v = (b.heads(x, 1)[:, 0] for x in (b.q, b.k, b.v))
    k[0] = 0
    o, a = attend(q, k, v, 0.1, np.tril(np.ones((3, 3), bool)) & (np.arange(3) > 0))
    smax = float((np.abs(q) @ np.abs(k).T).max()) * 0.1
    close(got[:, 0], o, attend_bound(o, a, np.abs(v).max(), 3, hd, smax, dtype), "without the first key")
    assert (got[0] == 0).all() and (o[1:] != 0).any()


# ------------------------------------------------------------------------------------------------------------- cached
def run_cached(hip, c, q, scale, with_ws=True, stream=None):
    n, Hq = q.shape[0], q.shape[1]
    hd, tail = c.hd, 2
    qn = np.full((n + tail, Hq * hd + 8), np.nan, np.float32)
    qn[:n, :Hq * hd] = q.reshape(n, -1)
    qb = narrow(qn, c.dtype)
    plan = c.upload()
    dq, do = dev(hip, qb), dev(hip, np.full((n + tail, Hq * hd + 16), 0x5555, np.uint16))
    L = hip.lib()
    nb = L.hxa_attention_cached_ws_bytes(C.byref(plan), n + tail, Hq)
    ws = dev(hip, np.full(max(nb, 16), 0xff, np.uint8))
    hip.check(L.hxa_attention_cached(C.byref(plan), dq.ptr, Hq * hd + 8, do.ptr, Hq * hd + 16, n + tail, Hq, scale,
                                     ws.ptr if with_ws else None, nb if with_ws else 0, stream), "cached")
    hip.sync()
    o = do.numpy()
    assert (o[n:] == 0x5555).all() and (o[:, Hq * hd:] == 0x5555).all()
    return widen(o[:n, :Hq * hd], c.dtype).reshape(n, Hq, hd), nb


def queries(rng, n, Hq, hd, dtype, std=1.5):
    return widen(narrow(rng.standard_normal((n, Hq, hd)) * std, dtype), dtype)


CACHED = [  # hd, Hq, H, new, past, prefix, page
    (128, 16, 8, [1], [700], 0, 16),                        # one token, keys split
    (128, 16, 8, [1], [0], 0, 16),                          # its own key alone
    (128, 2, 1, [1], [0], 1, 1),
    (64, 8, 2, [1] * 9, [0, 1, 62, 63, 64, 200, 999, 5, 127], 0, 32),
    (128, 4, 1, [1] * 5, [10, 0, 300, 64, 127], 1000, 16),  # shared prefix, 20 rows: 64-row blocks over it
    (128, 8, 4, [1] * 5, [10, 0, 300, 64, 127], 777, 7),    # 10 rows: 16-row blocks
    (128, 8, 2, [1] * 40, [3 * i for i in range(40)], 515, 64),  # 160 rows: 128-row blocks, two of them
    (64, 4, 2, [1] * 70, [i % 9 for i in range(70)], 300, 128),
    (256, 4, 2, [1] * 6, [0, 40, 64, 100, 9, 1], 320, 16),
    (256, 6, 3, [1] * 50, [2 * i for i in range(50)], 258, 32),
    (128, 16, 8, [1, 3, 0, 2], [20, 100, 7, 300], 400, 16),  # a few tokens each, one sequence without
    (128, 4, 2, [20, 1, 33, 0], [50, 3, 0, 9], 130, 16),    # pieces of prompts, 64-row blocks
    (64, 3, 1, [90, 40], [0, 500], 65, 32),
    (256, 2, 1, [70, 31], [10, 0], 100, 16),
    (128, 256, 128, [130, 70], [30, 0], 70, 16),            # 128-row blocks
    (256, 96, 96, [129, 200], [30, 0], 0, 64),
    (64, 140, 140, [300], [100], 20, 16),
    (128, 2, 1, [40] + [1] * 30, [5] + [40] * 30, 70, 16),  # on average few rows, one sequence with five blocks of them
    (128, 4, 2, [1], [3000], 0, 16),                        # more tiles than a row has partial results
    (64, 4, 2, [1, 1, 1], [2500, 0, 70], 2500, 32),         # and a shared prefix of more
    (128, 8, 8, [1] * 200, [i % 50 for i in range(200)], 0, 8),  # more blocks than run at once
    (64, 8, 4, [1] * 150, [(i * 37) % 300 for i in range(150)], 280, 16),
]


@pytest.mark.parametrize("with_ws", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,Hq,H,new,past,prefix,page", CACHED)
def test_attention_cached(hip, dtype, hd, Hq, H, new, past, prefix, page, with_ws):
    say("cached", dtype, hd, Hq, H, new, past, prefix, page, with_ws)
    rng = np.random.default_rng(hd + prefix + len(new))
    c = Cache(hip, rng, new, past, prefix, page, H, hd, dtype)
    q = queries(rng, int(c.cu[-1]), Hq, hd, dtype)
    got, _ = run_cached(hip, c, q, hd ** -0.5, with_ws)
    o, a, n, smax, vmax = c.expect(q, hd ** -0.5)
    close(got, o, attend_bound(o, a, vmax, n, hd, smax, dtype), "cached")
    assert np.array_equal(run_cached(hip, c, q, hd ** -0.5, with_ws)[0], got)


@pytest.mark.parametrize("with_ws", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,Hq,H,new,past,prefix", [(128, 8, 4, [1] * 6, [0, 10, 100, 64, 33, 2], 300), (64, 2, 1, [70, 40], [30, 0], 64),
                                                     (256, 4, 2, [1] * 40, [7] * 40, 300)])
def test_cached_bad_pages_and_empty_rows(hip, dtype, hd, Hq, H, new, past, prefix, with_ws):
    """entries outside the pool leave their keys out; a sequence whose keys are all out gets zeros"""
    say("bad pages", dtype, hd, with_ws)
    rng = np.random.default_rng(1)
    page = 16
    bad = {("prefix", 1): -1, ("prefix", 2): 10 ** 6, (1, 0): 2 ** 31 - 1}
    c = Cache(hip, rng, new, past, prefix, page, H, hd, dtype, bad=bad)
    q = queries(rng, int(c.cu[-1]), Hq, hd, dtype)
    got, _ = run_cached(hip, c, q, hd ** -0.5, with_ws)
    o, a, n, smax, vmax = c.expect(q, hd ** -0.5)
    close(got, o, attend_bound(o, a, vmax, n, hd, smax, dtype), "bad pages")
    bad = {("prefix", s): -5 for s in range(-(-prefix // page))} | {(0, s): 99999 for s in range(c.ldt)}
    c = Cache(hip, rng, new, past, prefix, page, H, hd, dtype, bad=bad)
    got, _ = run_cached(hip, c, q, hd ** -0.5, with_ws)
    assert (got[:new[0]] == 0).all() and (got[new[0]:] != 0).any()


@pytest.mark.parametrize("with_ws", [True, False])
def test_cached_infinities_and_nan(hip, with_ws):
    """a value that is not finite reaches the queries that see it and no other; so does a key that is NaN"""
    rng = np.random.default_rng(8)
    for hd, Hq, H, new, past, prefix in [(128, 4, 2, [5, 1, 1], [30, 9, 64], 300), (128, 4, 2, [40, 50], [30, 0], 70),
                                         (64, 130, 130, [200, 170], [3, 0], 10)]:
        c = Cache(hip, rng, new, past, prefix, 16, H, hd, F16)
        last = lambda i, p: (c.table[i, p // 16], 0, p % 16)
        c.v.view(np.float16)[last(0, c.lens[0] - 2)] = np.inf
        c.v.view(np.float16)[last(0, c.lens[0] - 1)] = np.nan
        c.k.view(np.float16)[last(1, c.lens[1] - 1)] = np.nan
        q = queries(rng, int(c.cu[-1]), Hq, hd, F16)
        o, a, n, smax, vmax = c.expect(q, hd ** -0.5)
        close(run_cached(hip, c, q, hd ** -0.5, with_ws)[0], o, attend_bound(o, a, vmax, n, hd, smax, F16), "not finite")
        assert np.isfinite(o[0]).all() and np.isinf(o[new[0] - 2, 0]).all() and np.isnan(o[new[0] - 1, 0]).all()


def test_cached_lengths_out_of_range(hip):
    """len below the new tokens (negative own positions: the prefix alone) and past the table (what the table holds)"""
    rng = np.random.default_rng(4)
    hd, Hq, H, page = 128, 4, 2, 16
    for prefix in (0, 100, 400):
        c = Cache(hip, rng, [3, 2, 2], [0, 30, 5], prefix, page, H, hd, F16)
        c.ldt = 2
        c.table = np.ascontiguousarray(c.table[:, :2])
        q = queries(rng, 7, Hq, hd, F16)
        c.lens = [1, 10 ** 9, 7]
        plan = c.upload()
        held = Cache.__new__(Cache)
        held.__dict__.update(c.__dict__)
        held.lens, held.past = [1, 32, 7], [-2, 10 ** 6, 5]
        o, a, n, smax, vmax = held.expect(q, hd ** -0.5)
        for ws in (True, False):
            got, _ = run_cached(hip, c, q, hd ** -0.5, ws)
            close(got, o, attend_bound(o, a, vmax, n, hd, smax, F16), "lengths")
            assert prefix or (got[:2] == 0).all()


MIXED = [  # hd, Hq, H, new, past, prefix, page: prompts beside single tokens, whole blocks of rows and rests of every kind
    (128, 8, 2, [130, 1, 64, 1, 0, 33, 1, 4, 5], [20, 300, 0, 64, 10, 100, 0, 7, 9], 70, 16),   # 128-row blocks; rests of 8, 4, 16, 20 rows
    (64, 4, 1, [150] + [1] * 70 + [17, 33], [0] + [30] * 70 + [5, 0], 300, 32),                # 64-row blocks, more than 64 sequences
    (128, 64, 64, [80, 1, 64, 16, 128, 17], [3, 90, 0, 200, 64, 1], 0, 16),                    # one row a token and head
    (256, 4, 2, [70, 1, 1, 8, 9], [40, 500, 0, 1, 63], 130, 64),
]


@pytest.mark.parametrize("with_ws", [True, False])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,Hq,H,new,past,prefix,page", MIXED)
def test_cached_prompts_beside_single_tokens(hip, dtype, hd, Hq, H, new, past, prefix, page, with_ws):
    say("mixed", dtype, hd, Hq, H, with_ws)
    rng = np.random.default_rng(hd + Hq)
    c = Cache(hip, rng, new, past, prefix, page, H, hd, dtype)
    q = queries(rng, int(c.cu[-1]), Hq, hd, dtype)
    got, _ = run_cached(hip, c, q, hd ** -0.5, with_ws)
    o, a, n, smax, vmax = c.expect(q, hd ** -0.5)
    close(got, o, attend_bound(o, a, vmax, n, hd, smax, dtype), "mixed")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,Hq,H,new,past,prefix", [(128, 8, 4, [1] * 7, [900, 0, 64, 300, 1, 20, 500], 400), (64, 4, 2, [60, 3], [200, 700], 100)])
def test_cached_steep_scores(hip, dtype, hd, Hq, H, new, past, prefix):
    """scores of tens to hundreds: the maximum moves from range to range, and most partial results weigh nothing"""
    rng = np.random.default_rng(31)
    c = Cache(hip, rng, new, past, prefix, 16, H, hd, dtype)
    q = queries(rng, int(c.cu[-1]), Hq, hd, dtype, std=8.0)
    o, a, n, smax, vmax = c.expect(q, 1.0)
    close(run_cached(hip, c, q, 1.0)[0], o, attend_bound(o, a, vmax, n, hd, smax, dtype), "steep")


def test_sequences_past_the_last_row_end_there(hip):
    """cu[nseq] above T, as a graph captured for fewer rows may find it: the last sequence has the rows that there are"""
    rng = np.random.default_rng(23)
    hd, Hq, H = 128, 4, 2
    b = Packed(hip, rng, [70, 90], Hq, H, hd, F16, tail=0)
    want = run_causal(hip, b, 0.1)
    b.cu = np.array([0, 70, 10 ** 6], np.int32)
    assert np.array_equal(run_causal(hip, b, 0.1), want) and (want[159] != 0).any()
    L = hip.lib()
    pools = []
    for end in (160, 2 ** 31 - 1):
        c = Cache(hip, np.random.default_rng(5), [70, 90], [5, 0], 30, 16, H, hd, F16, empty=True)
        c.cu[2] = end
        c.lens = [75, 90]
        plan = c.upload()
        k, v = dev(hip, b.k), dev(hip, b.v)
        hip.check(L.hxa_kv_append(C.byref(plan), k.ptr, b.ldk, v.ptr, b.ldv, 160, None, 0.0, None, None))
        dq, do = dev(hip, b.q), dev(hip, np.zeros((160, b.ldo), np.uint16))
        hip.check(L.hxa_attention_cached(C.byref(plan), dq.ptr, b.ldq, do.ptr, b.ldo, 160, Hq, 0.1, None, 0, None))
        hip.sync()
        pools.append((c.d["k"].numpy().copy(), c.d["v"].numpy().copy(), do.numpy().copy()))
    assert all(np.array_equal(x, y) for x, y in zip(*pools))


def test_cached_prefix_alone(hip):
    """a table without entries: every query sees the prefix, and without a prefix nothing"""
    rng = np.random.default_rng(14)
    hd, Hq, H = 128, 4, 2
    for prefix, new in ((300, [1, 1, 2]), (40, [50, 30]), (0, [1, 3])):
        c = Cache(hip, rng, new, [0] * len(new), prefix, 16, H, hd, F16)
        q = queries(rng, int(c.cu[-1]), Hq, hd, F16)
        c.ldt, c.table = 0, np.zeros((len(new), 0), np.int32)
        none = Cache.__new__(Cache)
        none.__dict__.update(c.__dict__)
        none.lens, none.past = [0] * len(new), [10 ** 6] * len(new)
        o, a, n, smax, vmax = none.expect(q, hd ** -0.5)
        for ws in (True, False):
            got, _ = run_cached(hip, c, q, hd ** -0.5, ws)
            close(got, o, attend_bound(o, a, vmax, n, hd, smax, F16), "prefix alone")
            assert prefix or (got == 0).all()


def test_two_streams_at_once(hip):
    """calls in flight on two streams, each with its own workspace and output, give what they give alone, bit for bit"""
    rng = np.random.default_rng(77)
    L, hd, Hq, H = hip.lib(), 128, 8, 2
    jobs = []
    for new, past, prefix in (([1] * 20, [400] * 20, 600), ([1] * 3, [3000, 20, 900], 256)):
        c = Cache(hip, rng, new, past, prefix, 16, H, hd, BF16)
        q = queries(rng, len(new), Hq, hd, BF16)
        st = C.c_void_p()
        hip.check(L.hxa_stream_create(C.byref(st)))
        plan = c.upload()
        nb = L.hxa_attention_cached_ws_bytes(C.byref(plan), len(new), Hq)
        jobs.append((c, plan, dev(hip, narrow(q, BF16)), dev(hip, np.zeros((len(new), Hq * hd), np.uint16)), hip.DeviceArray((nb,), np.uint8), nb, st,
                     len(new)))
    go = lambda j, st: hip.check(L.hxa_attention_cached(C.byref(j[1]), j[2].ptr, Hq * hd, j[3].ptr, Hq * hd, j[7], Hq, hd ** -0.5, j[4].ptr, j[5], st))
    alone = []
    for j in jobs:
        go(j, None)
        hip.sync()
        alone.append(j[3].numpy().copy())
        j[3].upload(np.zeros_like(alone[-1]))
    for _ in range(10):
        for j in jobs:
            go(j, j[6])
    hip.sync()
    for j, want in zip(jobs, alone):
        assert np.array_equal(j[3].numpy(), want) and (want != 0).any()
        hip.check(L.hxa_stream_destroy(j[6]))


# ------------------------------------------------------------------------------------------------- far ends of large buffers
def test_offsets_past_32_bits(hip):
    """pools of 5 GB with the pages at their end, and key rows 16 MB apart: append, then attention over the cache and over the prompt"""
    L, rng = hip.lib(), np.random.default_rng(6)
    Hq, H, hd, page, n = 4, 2, 128, 64, 130
    npages = 5 * 2 ** 30 // (H * page * hd * 2)
    kc, vc = hip.DeviceArray((npages * H * page * hd,), np.uint16), hip.DeviceArray((npages * H * page * hd,), np.uint16)
    pages = np.array([npages - 1, npages - 3, npages - 2], np.int32)
    ld = 2 ** 23
    k, v = narrow(rng.standard_normal((n, H * hd)), F16), narrow(rng.standard_normal((n, H * hd)), F16)
    q = narrow(rng.standard_normal((n, Hq * hd)), F16)
    big = hip.DeviceArray((n * ld,), np.uint16)  # k and v of a row side by side, 2.2 GB
    big2 = hip.DeviceArray((300 * ld,), np.uint16)  # 5 GB: rows 170 .. 299
    for t in range(n):
        row = np.concatenate([k[t], v[t]])
        hip.check(L.hxa_h2d(big.at(2 * t * ld), row.ctypes.data, row.nbytes))
        hip.check(L.hxa_h2d(big2.at(2 * (170 + t) * ld), row.ctypes.data, row.nbytes))
    dq, do, do2 = dev(hip, q), hip.DeviceArray((n, Hq * hd), np.uint16), hip.DeviceArray((300, Hq * hd), np.uint16)
    d = [dev(hip, np.array(a, np.int32)) for a in ([0, n], pages, [n], [170, 300])]
    c = hip.KvCache(F16, H, hd, page, npages, kc.ptr, vc.ptr, None, 0, d[1].ptr, 3, d[2].ptr, d[0].ptr, 1)
    hip.check(L.hxa_kv_append(C.byref(c), big.ptr, ld, big.at(2 * H * hd), ld, n, None, 0.0, None, None))
    hip.check(L.hxa_attention_cached(C.byref(c), dq.ptr, Hq * hd, do.ptr, Hq * hd, n, Hq, hd ** -0.5, None, 0, None))
    q2 = np.zeros((300, Hq * hd), np.uint16)
    q2[170:] = q
    dq2 = dev(hip, q2)
    hip.check(L.hxa_attention_causal(F16, dq2.ptr, Hq * hd, big2.ptr, ld, big2.at(2 * H * hd), ld, do2.ptr, Hq * hd, 300, d[3].ptr, 1, Hq, H, hd,
                                     hd ** -0.5, None))
    hip.sync()
    qq, kk, vv = (widen(x, F16).reshape(n, -1, hd) for x in (q, k, v))
    o, bound = np.zeros((n, Hq, hd)), np.zeros((n, Hq, hd))
    for h in range(Hq):
        o[:, h], a = attend(qq[:, h], kk[:, h // 2], vv[:, h // 2], hd ** -0.5, np.tril(np.ones((n, n), bool)))
        smax = (np.abs(qq[:, h]) @ np.abs(kk[:, h // 2]).T).max() * hd ** -0.5
        bound[:, h] = attend_bound(o[:, h], a, np.abs(vv).max(), n, hd, smax, F16)
    close(widen(do.numpy(), F16).reshape(n, Hq, hd), o, bound, "cached")
    close(widen(do2.numpy()[170:], F16).reshape(n, Hq, hd), o, bound, "causal")


# --------------------------------------------------------------------------------------------------------- as it is used
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_decoding_with_the_cache_equals_the_whole_prompt(hip, dtype):
    """A template goes into the cache once; prompts of different lengths are appended behind it and attended, then two single-token steps
    follow. Each row agrees with causal attention over the whole sequence at once; the steps run as one captured graph
    whose replays follow the lengths on the device."""
    rng = np.random.default_rng(12)
    L, Hq, H, hd, page, P = hip.lib(), 8, 2, 128, 16, 300
    rest = [5, 1, 40]
    steps = 2
    total = [P + n + steps for n in rest]
    W = (Hq + 2 * H) * hd
    template = rng.standard_normal((P, W))
    seqs = [narrow(np.concatenate([template, rng.standard_normal((n + steps, W))]), dtype) for n in rest]
    for s in seqs:
        s[:P] = seqs[0][:P]
    gq, gk = ((1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2))
    freq, _ = hip.rope_freqs(hd, 10000.0)
    dgq, dgk, df = dev(hip, gq), dev(hip, gk), dev(hip, freq)
    rope = hip.Rope(df.ptr, hd, 0, 1.0)
    scale = hd ** -0.5
    # everything at once
    packed = np.concatenate(seqs)
    T = len(packed)
    cu = np.cumsum([0] + total).astype(np.int32)
    pos = np.concatenate([np.arange(n) for n in total]).astype(np.int32)
    dx, dcu, dpos, do = dev(hip, packed), dev(hip, cu), dev(hip, pos), dev(hip, np.zeros((T, Hq * hd), np.uint16))
    kp = dx.at(Hq * hd * 2)
    hip.check(L.hxa_qk_norm_rope(dtype, dx.ptr, W, Hq, kp, W, H, T, hd, dgq.ptr, dgk.ptr, EPS, dpos.ptr, C.byref(rope), dx.ptr, W, kp, W, None))
    hip.check(L.hxa_attention_causal(dtype, dx.ptr, W, kp, W, dx.at((Hq + H) * hd * 2), W, do.ptr, Hq * hd, T, dcu.ptr, 3, Hq, H, hd, scale, None))
    hip.sync()
    turned = dx.numpy()
    heads = widen(turned, dtype).reshape(T, Hq + 2 * H, hd)
    exact, bound = np.zeros((T, Hq, hd)), np.zeros((T, Hq, hd))
    for s, e in zip(cu, cu[1:]):
        for h in range(Hq):
            qh, kh, vh = heads[s:e, h], heads[s:e, Hq + h // (Hq // H)], heads[s:e, Hq + H + h // (Hq // H)]
            exact[s:e, h], a = attend(qh, kh, vh, scale, np.tril(np.ones((e - s, e - s), bool)))
            smax = (np.abs(qh) @ np.abs(kh).T).max() * scale
            bound[s:e, h] = attend_bound(exact[s:e, h], a, np.abs(vh).max(), e - s, hd, smax, dtype)
    close(widen(do.numpy(), dtype).reshape(T, Hq, hd), exact, bound, "at once")
    # through the cache
    c = Cache(hip, rng, [n + steps for n in rest], [0] * 3, P, page, H, hd, dtype, empty=True)
    plan = c.upload()
    st = C.c_void_p()
    hip.check(L.hxa_stream_create(C.byref(st)))
    dlen, dcu1 = dev(hip, np.array([P], np.int32)), dev(hip, np.array([0, P], np.int32))
    once = hip.KvCache(dtype, H, hd, page, c.npages, plan.k, plan.v, None, 0, plan.prefix, len(c.prefix), dlen.ptr, dcu1.ptr, 1)
    dt = dev(hip, seqs[0][:P])
    hip.check(L.hxa_kv_append(C.byref(once), dt.at(Hq * hd * 2), W, dt.at((Hq + H) * hd * 2), W, P, dgk.ptr, EPS, C.byref(rope), st))
    hip.sync()

    def feed(lo, hi):
        """rows lo .. hi - 1 of each sequence's rest"""
        rows = [s[P + a:P + b] for s, a, b in zip(seqs, lo, hi)]
        return np.concatenate(rows), np.cumsum([0] + [len(r) for r in rows]).astype(np.int32), np.array(hi, np.int32)

    def check(out, lo, hi, what):
        at = 0
        for i, (a, b) in enumerate(zip(lo, hi)):
            rows = slice(cu[i] + P + a, cu[i] + P + b)
            got = out[at:at + b - a].reshape(b - a, Hq, hd)
            at += b - a
            close(got, exact[rows], bound[rows], what)

    def buffers(n):
        bufs = dict(x=hip.DeviceArray((n, W), np.uint16), q=hip.DeviceArray((n, Hq * hd), np.uint16), o=hip.DeviceArray((n, Hq * hd), np.uint16),
                    pos=hip.DeviceArray((n,), np.int32), cu=hip.DeviceArray((4,), np.int32))
        p = hip.KvCache.from_buffer_copy(plan)
        p.cu, p.len = bufs["cu"].ptr, c.d["len"].ptr
        nb = L.hxa_attention_cached_ws_bytes(C.byref(p), n, Hq)
        bufs["ws"], bufs["nb"], bufs["plan"] = hip.DeviceArray((max(nb, 16),), np.uint8), nb, p
        return bufs

    def calls(b, n):
        p = b["plan"]
        x = b["x"]
        hip.check(L.hxa_qk_norm_rope(dtype, x.ptr, W, Hq, None, 0, 0, n, hd, dgq.ptr, None, EPS, b["pos"].ptr, C.byref(rope), b["q"].ptr, Hq * hd,
                                     None, 0, st))
        hip.check(L.hxa_kv_append(C.byref(p), x.at(Hq * hd * 2), W, x.at((Hq + H) * hd * 2), W, n, dgk.ptr, EPS, C.byref(rope), st))
        hip.check(L.hxa_attention_cached(C.byref(p), b["q"].ptr, Hq * hd, b["o"].ptr, Hq * hd, n, Hq, scale, b["ws"].ptr, b["nb"], st))

    def load(b, lo, hi):
        x, cu1, ln = feed(lo, hi)
        b["x"].upload(x)
        b["cu"].upload(cu1)
        c.d["len"].upload(ln)
        b["pos"].upload(np.concatenate([P + np.arange(a, e) for a, e in zip(lo, hi)]).astype(np.int32))

    lo, hi = [0, 0, 0], rest
    b = buffers(sum(rest))
    load(b, lo, hi)
    calls(b, sum(rest))
    hip.sync()
    check(widen(b["o"].numpy(), dtype), lo, hi, "prompts")
    # the cached keys are the turned ones, bit for bit
    kd = c.d["k"].numpy()
    for t in (0, 17, P - 1):
        assert np.array_equal(kd[c.prefix[t // page], :, t % page].reshape(-1), turned[t, Hq * hd:(Hq + H) * hd])
    t = cu[2] + P + 33
    assert np.array_equal(kd[c.table[2, 33 // page], :, 33 % page].reshape(-1), turned[t, Hq * hd:(Hq + H) * hd])
    # steps: eager, then captured and replayed for each step, with the step's own eager result between the replays
    b = buffers(3)
    g = C.c_void_p()
    load(b, hi, [n + 1 for n in hi])
    hip.check(L.hxa_stream_begin_capture(st, 1))
    calls(b, 3)
    hip.check(L.hxa_stream_end_capture(st, C.byref(g)))
    for rep in range(2):
        for step in range(steps):
            lo1, hi1 = [n + step for n in rest], [n + step + 1 for n in rest]
            load(b, lo1, hi1)
            hip.check(L.hxa_graph_launch(g, st))
            hip.sync()
            out = b["o"].numpy()
            check(widen(out, dtype), lo1, hi1, f"step {step}")
            b["o"].upload(np.zeros_like(out))
            calls(b, 3)
            hip.sync()
            assert np.array_equal(b["o"].numpy(), out)
    hip.check(L.hxa_graph_exec_destroy(g))
    hip.check(L.hxa_stream_destroy(st))
