"""Attention over the int8 cache where scales, queries and weights are far apart, against its definition in 64 bits, with a bound for each row and head."""
import numpy as np
import pytest

from tests._causal import BF16, F16, HALF_STEP, TINY, U24, close
from tests._q8 import CacheQ8
from tests.test_gpu_causal import queries, say
from tests.test_gpu_q8 import FORMS, run_cached

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    from hexanima_amd import hip as h
    h.init(0)
    return h


def scales_of(c, i):
    """(key scales, value scales) [keys][H] of sequence i's keys, 0 where they count as none"""
    pages = [int((c.prefix if x < c.P else c.table[i])[(x if x < c.P else x - c.P) // c.page]) for x in range(c.P + c.lens[i])]
    at = [e if 0 <= e < c.npages else -1 for e in pages]
    with np.errstate(invalid="ignore"):
        return [np.where((np.array(at) >= 0)[:, None] & np.isfinite(s[at]) & (s[at] > 0), s[at], 0).astype(np.float64) for s in (c.ks, c.vs)]


def rows_of(c, q, scale):
    """(o, bound) per row, head and dim, in 64 bits. In natural units of the score, with w the softmax's weights, vs a key's value scale:
      - every weight carries the same relative error rel at most, of numerator and denominator: the score's 32-bit sum of hd products and its scaling ((hd + 8)
        half steps of the sum of |q k|), the logarithm of vs (8 half steps of it), exponential, rescales and joins (256); the sums themselves n;
      - the numerator's weights are rounded to fp16, half a step 2^-11, or 2^-25 below 2^-14, where the largest w vs of the row is 2^-25 / FLOOR at least (a
        page without a scale stands there with 2^-64, the least scale): n keys of bytes up to 127;
      - bf16 queries lose at most 2^-25 a dim where the row's largest is 1 or more (2^-39 of it otherwise, which the 256 hold);
      - the output's own rounding."""
    n_q, Hq, hd = q.shape
    G = Hq // c.H
    o, bound = np.zeros_like(q), np.zeros_like(q)
    pools = c.values(c.k), c.values(c.v)
    c.values = lambda pool: pools[pool is c.v]  # once for all sequences
    for i, b in enumerate(c.cu[:-1]):
        n = c.new[i]
        if n == 0 or c.P + c.lens[i] == 0:
            continue
        (k, ok), (v, _), (_, vs) = c.keys(c.k, i), c.keys(c.v, i), scales_of(c, i)
        seen = (np.arange(len(k))[None] <= c.P + c.past[i] + np.arange(n)[:, None]) & ok[None]
        for h in range(Hq):
            kh, vh, qh = k[:, h // G], v[:, h // G], q[b:b + n, h]
            s = np.where(seen, qh @ kh.T * scale, -np.inf)
            p = np.exp(s - np.where(seen.any(1), s.max(1), 0)[:, None])
            w = p / np.maximum(p.sum(1, keepdims=True), 1e-300)  # a row that sees nothing: zeros
            keys = seen.sum(1)[:, None]
            size = (np.where(seen, np.abs(qh) @ np.abs(kh).T, 0).max(1) * scale)[:, None]
            lmax = np.abs(np.log2(vs[:, h // G], out=np.full(len(vs), -64.0), where=vs[:, h // G] > 0)).max()
            rel = (keys + (hd + 8) * size + 8 * lmax + 256) * U24
            if c.dtype == BF16:
                rel = rel + hd * 2.0 ** -25 * np.abs(kh).max() * scale
            a = w @ np.abs(vh)
            o[b:b + n, h] = w @ vh
            bound[b:b + n, h] = (HALF_STEP[c.dtype] * np.abs(o[b:b + n, h]) + (2.0 ** -11 + 2 * rel) * a +
                                 keys * FLOOR * 127 * (w * np.maximum(vs[:, h // G], 2.0 ** -64)).max(1)[:, None] + TINY[c.dtype])
    del c.values
    if c.dtype == F16:  # from 65520 on the nearest fp16 value is infinity
        o = np.where(np.abs(o) >= 65520, np.copysign(np.inf, o), o)
    return o, bound


FLOOR = 2.0 ** -32  # the largest weight of a row stands as 2^7 or more before its byte


@pytest.mark.parametrize("with_ws", [True, False])
@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("hd,Hq,H,new,past,prefix", FORMS)
def test_small_values_keep_their_bits(hip, hd, Hq, H, new, past, prefix, page, with_ws):
    """rows whose weight lies on pages of small values, beside pages of values 10^5 times as large: the bound is well below most results"""
    say("small values", hd, page, with_ws)
    rng = np.random.default_rng(6)
    c = CacheQ8(hip, rng, new, past, prefix, page, H, hd, F16, spread=0.0)
    c.vs[:] = np.where(rng.random(c.vs.shape) < 0.5, 0.01, 1000.0)
    big = c.vs > 1
    c.k[big], c.k[~big] = np.clip(c.k[big], -127, 0), np.clip(c.k[~big], 0, 127)
    q = np.abs(queries(rng, int(c.cu[-1]), Hq, hd, F16))
    o, bound = rows_of(c, q, 2.0 * hd ** -0.5)
    few = [r for i, b in enumerate(c.cu[:-1]) for r in range(b, c.cu[i + 1])]
    assert (bound[few] < np.abs(o[few]) / 8).mean() > 0.8
    close(run_cached(hip, c, q, 2.0 * hd ** -0.5, with_ws), o, bound, "small values")


@pytest.mark.parametrize("with_ws", [True, False])
@pytest.mark.parametrize("dtype,page", [(F16, 16), (BF16, 16), (BF16, 5)])
@pytest.mark.parametrize("hd,Hq,H,new,past,prefix", FORMS)
def test_wide_value_scales_row_by_row(hip, dtype, hd, Hq, H, new, past, prefix, page, with_ws):
    """value scales from 2^-40 to 2^8 side by side, some of none: each row by the largest scale that it gives weight to"""
    say("wide value scales", dtype, hd, page, with_ws)
    rng = np.random.default_rng(9)
    c = CacheQ8(hip, rng, new, past, prefix, page, H, hd, dtype)
    c.vs[:] = np.exp2(rng.uniform(-40, 8, c.vs.shape))
    q = queries(rng, int(c.cu[-1]), Hq, hd, dtype, std=6.0)
    close(run_cached(hip, c, q, hd ** -0.5, with_ws), *rows_of(c, q, hd ** -0.5), "wide value scales")
    kinds = rng.integers(0, 12, c.vs.shape)
    for n, none in enumerate((0.0, -1.0, np.inf, np.nan)):
        c.vs[kinds == n] = none
    close(run_cached(hip, c, q, hd ** -0.5, with_ws), *rows_of(c, q, hd ** -0.5), "some without")


@pytest.mark.parametrize("with_ws", [True, False])
@pytest.mark.parametrize("page", [16, 5])
@pytest.mark.parametrize("hd,Hq,H,new,past,prefix", FORMS)
@pytest.mark.parametrize("power", [92, 112, 122])
def test_wide_queries_beside_pages_without_a_key_scale(hip, power, hd, Hq, H, new, past, prefix, page, with_ws):
    """bf16 queries of about 2^power over keys of about 2^-power: keys whose scale is 0, negative, infinite or NaN score 0, whatever their bytes"""
    say("wide queries, no key scale", power, hd, page, with_ws)
    rng = np.random.default_rng(power)
    c = CacheQ8(hip, rng, new, past, prefix, page, H, hd, BF16, spread=0.0)
    c.k[:] = np.clip(np.rint(c.k / 32.0), -4, 4)
    c.ks[:] = np.float32(2.0 ** -power)
    kinds = rng.integers(0, 12, c.ks.shape)
    for n, none in enumerate((0.0, -1.0, np.inf, np.nan)):
        c.ks[kinds == n] = none
    c.k[kinds < 4] = rng.integers(-128, 128, c.k[kinds < 4].shape)
    q = queries(rng, int(c.cu[-1]), Hq, hd, BF16) * 2.0 ** power
    o, bound = rows_of(c, q, hd ** -0.5)
    close(run_cached(hip, c, q, hd ** -0.5, with_ws), o, bound, "wide queries")


LONG = [(128, 8, 4, [1, 1], [3000, 2500], 0), (64, 4, 4, [40], [2000], 0), (256, 2, 1, [1] * 3, [1500] * 3, 300), (128, 2, 2, [130], [1500], 0),
        (128, 8, 2, [1] * 20, [700] * 20, 1000)]


@pytest.mark.parametrize("with_ws", [True, False])
@pytest.mark.parametrize("dtype,page", [(F16, 16), (BF16, 16), (F16, 5)])
@pytest.mark.parametrize("hd,Hq,H,new,past,prefix", LONG)
def test_a_long_tail_of_small_weights(hip, dtype, hd, Hq, H, new, past, prefix, page, with_ws):
    """the first key, whose value is 0, has nearly all the weight; thousands behind it have 2^-27 of it each and make up the result"""
    say("tail", dtype, hd, page, with_ws)
    rng = np.random.default_rng(13)
    c = CacheQ8(hip, rng, new, past, prefix, page, H, hd, dtype, spread=0.0)
    c.k[:], c.v[:] = rng.integers(-8, 9, c.k.shape), rng.integers(64, 128, c.v.shape)
    for pg in [c.prefix[0]] if prefix else c.table[:, 0]:
        c.k[pg, :, 0], c.v[pg, :, 0] = 127, 0
    c.ks[:], c.vs[:] = 1 / 127, 1.0
    q = 1 + queries(rng, int(c.cu[-1]), Hq, hd, dtype, std=0.0)
    scale = 27 * np.log(2) / hd
    o, bound = rows_of(c, q, scale)
    assert (bound < np.abs(o) / 8).mean() > 0.9
    close(run_cached(hip, c, q, scale, with_ws), o, bound, "tail")


@pytest.mark.parametrize("with_ws", [True, False])
@pytest.mark.parametrize("dtype,page", [(F16, 16), (BF16, 16), (F16, 5)])
@pytest.mark.parametrize("hd,Hq,H,new,past,prefix", LONG)
@pytest.mark.parametrize("power", [10, 19, 26, 40, 80])
def test_scores_far_from_zero(hip, power, hd, Hq, H, new, past, prefix, dtype, page, with_ws):
    """The largest score is about 2^power in powers of two and the others at most 4/5 of it, or (of the other sign) -2^power and the others 5/4 of it: the key's value and
    nothing else. The sums of products are multiples of 2^10 below 2^25, exact; whatever is rounded after them is the key's weight, the same above and
    below the line but for its rounding to fp16. The others' weights are 2^-190 or less."""
    say("far scores", power, dtype, hd, page, with_ws)
    rng = np.random.default_rng(14)
    for sign in (1, -1):
        c = CacheQ8(hip, rng, new, past, prefix, page, H, hd, dtype, spread=0.0)
        c.k[:] = rng.integers(0, 101, c.k.shape) if sign > 0 else rng.integers(125, 128, c.k.shape)
        c.v[:] = rng.integers(-127, 128, c.v.shape)
        c.ks[:], c.vs[:] = 1.0, np.exp2(rng.uniform(-3, 3, c.vs.shape))
        want = np.zeros((int(c.cu[-1]), Hq, hd))
        for i, b in enumerate(c.cu[:-1]):
            x = int(rng.integers(0, past[i] + 1))
            pg = c.table[i, x // page]
            c.k[pg, :, x % page] = 127 if sign > 0 else 100
            want[b:b + new[i]] = np.repeat(c.v[pg, :, x % page] * c.vs[pg, :, None].astype(np.float64), Hq // H, 0)
        q = np.full(want.shape, sign * 1024.0)
        got = run_cached(hip, c, q, 2.0 ** power / (1024 * 127 * hd * np.log2(np.e)), with_ws)
        close(got, want, (HALF_STEP[dtype] + 2.0 ** -11 + 256 * U24) * np.abs(want) + TINY[dtype], "far scores")


@pytest.mark.parametrize("hd,Hq,H,new,past,prefix,page", [
    (64, 80, 40, [1] * 420, [(7 * i) % 90 for i in range(420)], 300, 16), (128, 160, 40, [1, 3, 2, 0, 4] * 20, [(11 * i) % 200 for i in range(100)], 520, 64),
    (256, 64, 32, [2] * 130, [(5 * i) % 130 for i in range(130)], 260, 5)])
def test_large_batches_behind_a_prefix(hip, hd, Hq, H, new, past, prefix, page):
    """the prefix's blocks are half the places of a key head and more"""
    say("large batch", hd, Hq, len(new))
    rng = np.random.default_rng(hd)
    c = CacheQ8(hip, rng, new, past, prefix, page, H, hd, BF16)
    q = queries(rng, int(c.cu[-1]), Hq, hd, BF16)
    close(run_cached(hip, c, q, hd ** -0.5), *rows_of(c, q, hd ** -0.5), "large batch")
