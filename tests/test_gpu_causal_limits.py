"""The causal text model's attention path at the far ends of what its calls take: many blocks, values that are not finite, weights of one kind."""
import numpy as np
import pytest

from tests._causal import BF16, F16, Cache, Packed, attend_bound, close, narrow, widen
from tests.test_gpu_causal import expect_causal, hip, queries, run_cached, run_causal, say  # noqa: F401 (hip is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,Hq,lens", [(F16, 1000, [80, 81, 83, 79, 120, 1, 137, 59]), (BF16, 1024, [330, 0, 310])])
def test_more_than_4096_blocks_a_key_head(hip, dtype, Hq, lens):
    """a few sequences of 5000 blocks of 128 rows: each block's rows are written, with their own values"""
    say("many blocks", dtype, Hq, lens)
    assert sum(lens) * Hq > 4096 * 128
    b = Packed(hip, np.random.default_rng(Hq), lens, Hq, 1, 64, dtype)
    want, bound = expect_causal(b, 0.125)
    close(run_causal(hip, b, 0.125), want, bound, "many blocks")


def bits(x, dtype):
    return narrow(np.float32(x), dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,Hq,Hk", [(64, 3, 1), (128, 4, 2), (256, 2, 1), (64, 256, 256), (128, 128, 128), (256, 64, 64)])
def test_scores_of_minus_infinity_over_values_that_are_not_finite(hip, dtype, hd, Hq, Hk):
    """a row whose scores are all -infinity is zeros, whatever the values; beside finite scores such a key adds 0 times its value"""
    say("-inf", dtype, hd, Hq, Hk)
    n = 150
    b = Packed(hip, np.random.default_rng(3), [n, 70], Hq, Hk, hd, dtype)
    b.q[:b.n, np.arange(Hq) * hd] = bits(-1, dtype)
    b.k[:100, np.arange(Hk) * hd] = bits(np.inf, dtype)
    b.v[5, 3], b.v[50, 7], b.v[90, hd - 1] = bits(np.inf, dtype), bits(np.nan, dtype), bits(-np.inf, dtype)
    want, bound = expect_causal(b, hd ** -0.5)
    want[:100], bound[:100] = 0, 0
    got = run_causal(hip, b, hd ** -0.5)
    close(got, want, bound, "-inf")
    assert np.isnan(want[100:n, 0][:, [3, 7, hd - 1]]).all() and np.isfinite(want[100:n, 0, 0]).all()


MINUS_INF = [  # hd, Hq, H, new, past, prefix: partial results of 16 rows; of 64 and 128 rows over a shared prefix; of 64 rows
    (128, 16, 8, [1, 1], [1500, 700], 0), (64, 4, 1, [1, 2], [1500, 700], 0), (256, 4, 2, [1, 1], [1500, 700], 300),
    (128, 8, 2, [1] * 8, [100, 300] * 4, 1000), (64, 8, 2, [1] * 40, [100, 300] * 20, 515), (256, 6, 2, [1] * 50, [100, 30] * 25, 400),
    (128, 4, 2, [20, 30], [1500, 200], 0), (256, 2, 1, [40, 30], [700, 200], 100), (128, 128, 128, [150, 130], [300, 20], 0)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,Hq,H,new,past,prefix", MINUS_INF)
def test_cached_scores_of_minus_infinity_over_values_that_are_not_finite(hip, dtype, hd, Hq, H, new, past, prefix):
    """the same over the cache, and the same with and without a workspace: the prefix and the older half of each sequence score -infinity; then
    everything does"""
    say("cached -inf", dtype, hd, Hq, H, prefix)
    page = 16
    for all_keys in (False, True):
        c = Cache(hip, np.random.default_rng(7), new, past, prefix, page, H, hd, dtype)
        q = queries(np.random.default_rng(8), sum(new), Hq, hd, dtype)
        q[:, :, 0] = -1
        c.k[c.prefix, :, :, 0] = bits(np.inf, dtype)
        c.v[c.prefix[3:4], 0, 2, 9] = bits(np.inf, dtype)
        for i, n in enumerate(c.lens):
            for t in range(n if all_keys else past[i] // 2):
                c.k[c.table[i, t // page], :, t % page, 0] = bits(np.inf, dtype)
            c.v[c.table[i, 0], 0, 1, 4] = bits([np.inf, np.nan][i % 2], dtype)
        scale = hd ** -0.5
        o, a, m, smax, vmax = c.expect(q, scale)
        bound = attend_bound(o, a, vmax, m, hd, smax, dtype)
        if all_keys:
            o[:], bound[:] = 0, 0
        else:
            assert np.isnan(o[:, 0, 4]).all() and np.isfinite(o[:, 0, 0]).all() and (prefix == 0 or np.isnan(o[:, 0, 9]).all())
        for ws in (True, False):
            got, nb = run_cached(hip, c, q, scale, ws)
            close(got, o, bound, f"all={all_keys} ws={ws}")


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,Hq,H", [(64, 16, 8), (128, 16, 16), (256, 8, 2), (128, 64, 2)])
def test_equal_values_come_out_as_they_are(hip, dtype, hd, Hq, H):
    """the weights' sum is that of the weights as they are multiplied: rounded alike, they cancel. 64 scores of 0, then 64 of up to 5.4 (below the
    growth that rescales, so weights are not near 1), over one value just below 2, where half a step of the result is half of what
    a weight's rounding may be: the sums are off by 128 2^-24 of it, so every result is the value"""
    say("equal values", dtype, hd, Hq, H)
    v = bits(2, dtype) - 1
    rng = np.random.default_rng(hd)
    B = 12
    q = np.zeros((B, Hq, hd))
    q[:, :, 0] = rng.uniform(3.0, 5.4, (B, Hq))
    q = widen(narrow(q, dtype), dtype)
    c = Cache(hip, rng, [1] * B, [127] * B, 0, 16, H, hd, dtype)
    c.k[:] = 0
    for i in range(B):
        c.k[c.table[i, 4:8], :, :, 0] = bits(1, dtype)
        c.v[c.table[i, :8]] = v
    for ws in (True, False):
        got, _ = run_cached(hip, c, q, 1.0, ws)
        assert (got == widen(np.uint16(v), dtype)).all(), (ws, np.unique(got))
    b = Packed(hip, rng, [128], Hq, H, hd, dtype)
    b.q[:b.n, :Hq * hd], b.k[:b.n, :H * hd], b.v[:b.n, :H * hd] = 0, 0, v
    b.q[:b.n, np.arange(Hq) * hd] = narrow(rng.uniform(3.0, 5.4, (b.n, Hq)), dtype)
    b.k[64:128, np.arange(H) * hd] = bits(1, dtype)
    assert (run_causal(hip, b, 1.0) == widen(np.uint16(v), dtype)).all()


@pytest.mark.parametrize("hd,Hq,H", [(64, 2, 1), (128, 4, 2), (256, 2, 1)])
def test_many_small_weights_count(hip, hd, Hq, H):
    """weights of 2^-15 (subnormal in fp16) beside one of 1: 3000 of them are a tenth of the sum"""
    say("small weights", hd)
    n = 3000
    s = float(15 * np.log(2))
    b = Packed(hip, np.random.default_rng(1), [n], Hq, H, hd, F16)
    b.q[:n, :Hq * hd], b.k[:n, :H * hd] = 0, 0
    b.q[:n, np.arange(Hq) * hd] = bits(s, F16)
    b.k[0, np.arange(H) * hd] = bits(1, F16)
    want, bound = expect_causal(b, 1.0)
    close(run_causal(hip, b, 1.0), want, bound, "causal")
    c = Cache(hip, np.random.default_rng(2), [1, 2], [n, 100], 0, 16, H, hd, F16)
    c.k[:] = 0
    for i in range(2):
        c.k[c.table[i, 0], :, 0, 0] = bits(1, F16)
    q = np.zeros((3, Hq, hd))
    q[:, :, 0] = widen(np.array([bits(s, F16)]), F16)[0]
    o, a, m, smax, vmax = c.expect(q, 1.0)
    for ws in (True, False):
        close(run_cached(hip, c, q, 1.0, ws)[0], o, attend_bound(o, a, vmax, m, hd, smax, F16), f"ws={ws}")
