"""The text model's calls in 8 bits without a GPU: what they refuse before any device call, their workspaces, and the definitions that the GPU tests
compare with."""
import ctypes as C

import numpy as np
import pytest

from tests._causal import BF16, F16, narrow, widen
from tests._q8 import LEAST, grow, page_scale, quantize
from tests.test_causal_cpu import BAD_PLANS, FAKE, hip, plan  # noqa: F401 (hip is a fixture)


def quant(hip, **kw):
    a = dict(dtype=1, x=FAKE, ldx=136, M=3, K=130, q=FAKE, ldq=256, scale=FAKE)
    a.update(kw)
    return hip.lib().hxa_quantize_rows(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=0), -11), (dict(dtype=3), -11), (dict(M=-1), -12), (dict(M=2 ** 25 + 1), -12), (dict(K=0), -12), (dict(K=-5), -12),
    (dict(K=130945, ldx=140000, ldq=140032), -12), (dict(x=None), -12), (dict(q=None), -12), (dict(scale=None), -12), (dict(x=FAKE + 1), -12),
    (dict(q=FAKE + 8), -12), (dict(scale=FAKE + 2), -12), (dict(ldx=128), -12), (dict(ldx=129), -12), (dict(ldq=240), -12), (dict(ldq=264), -12)])
def test_quantize_rows_refuses(hip, kw, rc):
    assert quant(hip, **kw) == rc and hip.last_error().startswith("quantize_rows")


def linear(hip, tile=None, **kw):
    a = dict(dtype=1, a=FAKE, lda=256, sa=FAKE, M=3, w=FAKE, ldw=256, sw=FAKE, N=16, K=130, bias=FAKE, out=FAKE, ldo=16, ws=None, nb=0)
    a.update(kw)
    v = list(a.values())
    if tile:
        return hip.lib().hxa_linear_i8_tile(*v[:-2], *tile, *v[-2:], None)
    return hip.lib().hxa_linear_i8(*v, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=0), -11), (dict(M=-1), -12), (dict(N=-8), -12), (dict(N=12), -12), (dict(K=0), -12), (dict(K=130945, lda=131072, ldw=131072), -12),
    (dict(a=None), -12), (dict(w=None), -12), (dict(out=None), -12), (dict(sa=None), -12), (dict(sw=None), -12), (dict(a=FAKE + 8), -12),
    (dict(w=FAKE + 8), -12), (dict(out=FAKE + 8), -12), (dict(sw=FAKE + 4), -12), (dict(bias=FAKE + 4), -12), (dict(sa=FAKE + 2), -12),
    (dict(lda=240), -12), (dict(lda=264), -12), (dict(ldw=240), -12), (dict(lda=2 ** 23), -12), (dict(ldw=2 ** 23), -12), (dict(ldo=8), -12),
    (dict(ldo=20), -12)])
def test_linear_i8_refuses(hip, kw, rc):
    assert linear(hip, **kw) == rc and hip.last_error().startswith("linear_i8")
    assert linear(hip, (64, 64, 1), **kw) == rc and hip.last_error().startswith("linear_i8_tile")


def test_linear_i8_workspace_tiles_and_empty_calls(hip):
    L = hip.lib()
    assert linear(hip, ws=FAKE + 8, nb=1 << 20) == -12
    for tile in ((96, 64, 1), (64, 64, 0), (64, 64, 65), (64, 64, 3), (32, 32, 2), (0, 0, 1), (-64, 64, 1)):
        assert linear(hip, tile) == -12
    assert linear(hip, (64, 64, 2)) == -12 and linear(hip, (64, 64, 2), ws=FAKE, nb=2 * 3 * 16 * 4 - 1) == -12  # no workspace, one byte short
    assert linear(hip, M=0, a=None) == 0 and linear(hip, N=0, w=None) == 0 and quant(hip, M=0, x=None) == 0
    assert L.hxa_linear_i8_ws_bytes(0, 8, 8) == 0 and L.hxa_linear_i8_ws_bytes(8, 12, 8) == 0 and L.hxa_linear_i8_ws_bytes(8, 8, 0) == 0
    for M, N, K in ((1, 4096, 2048), (64, 2048, 8192), (1000, 2048, 8192), (6500, 16384, 2048)):
        nb = L.hxa_linear_i8_ws_bytes(M, N, K)
        assert nb >= 0 and nb % (4 * M * N) == 0 and nb <= 64 * 4 * M * N


def q8(hip, ks=FAKE, vs=FAKE, **kw):
    return hip.KvCacheQ8(plan(hip, **kw), ks, vs)


@pytest.mark.parametrize("kw,rc", BAD_PLANS + [(dict(nseq=2 ** 30 + 1), -12)])
def test_q8_plans_refused(hip, kw, rc):
    L, c = hip.lib(), q8(hip, **kw)
    assert L.hxa_kv_append_q8(C.byref(c), FAKE, 256, FAKE, 256, 4, None, 1e-6, None, None) == rc and hip.last_error().startswith("kv_append_q8")
    Hq = 4 if kw.get("H") != 5000 else 5000
    assert L.hxa_attention_cached_q8(C.byref(c), FAKE, 512, FAKE, 512, 4, Hq, 0.1, None, 0, None) == rc
    assert hip.last_error().startswith("attention_cached_q8")
    assert L.hxa_attention_cached_q8_ws_bytes(C.byref(c), 4, Hq) == 0


def test_q8_calls_refuse(hip):
    L = hip.lib()
    run = lambda c, k=FAKE, ldk=256, v=FAKE, ldv=256, T=4, g=None, eps=1e-6, rope=None: L.hxa_kv_append_q8(
        C.byref(c), k, ldk, v, ldv, T, g, eps, C.byref(rope) if rope else None, None)
    c = q8(hip)
    assert [run(c, k=None), run(c, v=None), run(c, ldk=248), run(c, ldv=260), run(c, k=FAKE + 2), run(c, T=-1), run(c, g=FAKE + 4),
            run(c, eps=float("nan")), run(q8(hip, ks=None)), run(q8(hip, vs=None)), run(q8(hip, ks=FAKE + 2)),
            run(q8(hip, nseq=2 ** 22), T=4), run(q8(hip, page=1), T=2 ** 23)] == [-12] * 13
    assert run(c, rope=hip.Rope(FAKE, 24, 0, 1.0)) == -12 and run(c, rope=hip.Rope(FAKE, 32, 5, 1.0)) == -11
    assert L.hxa_kv_append_q8(None, FAKE, 256, FAKE, 256, 4, None, 1e-6, None, None) == -12
    assert run(c, T=0, k=None) == 0 and run(q8(hip, nseq=0), k=None) == 0 and run(q8(hip, ldt=0), k=None) == 0
    att = lambda c, q=FAKE, ldq=512, o=FAKE, ldo=512, T=4, Hq=4, scale=0.1, ws=None, nb=0: L.hxa_attention_cached_q8(
        C.byref(c), q, ldq, o, ldo, T, Hq, scale, ws, nb, None)
    assert [att(c, q=None), att(c, o=None), att(c, ldq=504), att(c, ldo=516), att(c, T=-1), att(c, Hq=3), att(c, Hq=0), att(c, scale=0.0),
            att(c, scale=float("nan")), att(c, ws=FAKE + 8, nb=1 << 20), att(c, T=2 ** 25, Hq=64, ldq=8192, ldo=8192),
            att(q8(hip, ks=None)), att(q8(hip, vs=FAKE + 1))] == [-12] * 13
    assert att(c, T=0, q=None) == 0 and att(q8(hip, nseq=0), q=None) == 0
    assert L.hxa_attention_cached_q8(None, FAKE, 512, FAKE, 512, 4, 4, 0.1, None, 0, None) == -12


def test_q8_workspace_follows_the_sizes(hip):
    L = hip.lib()
    size = lambda T, Hq, **kw: L.hxa_attention_cached_q8_ws_bytes(C.byref(q8(hip, **kw)), T, Hq)
    assert size(1, 4, nseq=1, prefix_len=0, ldt=1) == 0 and size(100000, 4, nseq=8) == 0
    assert size(1, 4, nseq=1, ldt=512) > 0 and size(1, 4, nseq=1, ldt=512) % ((128 * 4 + 8) * 4) == 0
    assert size(64, 4, nseq=64, prefix_len=4096) > 0
    row = 8 * (128 * 4 + 8)
    for n in (64, 5000, 200000):
        nb = size(n, 8, nseq=n, prefix_len=4096, ldt=500)
        assert nb % (n * row) == 0 and nb <= max(2 ** 30, 4 * n * row)


def test_the_tests_own_definitions():
    """the row quantiser and a page's growth against values written out"""
    q, s = quantize(np.array([[127.0, 0.5, 1.5, -63.5, np.nan, np.inf], [0, 0, 0, 0, 0, -np.inf], [np.nan] * 6]))
    assert list(s) == [1, 0, 0] and list(q[0]) == [127, 0, 2, -64, 0, 127] and not q[1:].any()
    q, s = quantize(np.array([[1e-30, -1e-31]]))
    assert s[0] == LEAST and not q.any()
    assert page_scale(254.0) == 2 and page_scale(0.0) == 0 and page_scale(1e-30) == LEAST
    assert grow(0.0, 3.0) == (3.0, 0) and grow(1.0, 0.7) == (1.0, 0) and grow(1.0, 1.0) == (1.0, 0) and grow(1.0, 1.01) == (2.0, 1) and grow(0.5, 4.0) == (4.0, 3)
    x = np.random.default_rng(0).standard_normal((4, 100))
    q, s = quantize(widen(narrow(x, BF16), BF16))
    assert (np.abs(q * s[:, None] - widen(narrow(x, BF16), BF16)) <= s[:, None] * 0.50001).all() and (np.abs(q).max(1) == 127).all()
    assert (np.abs(x - widen(narrow(x, F16), F16)) <= 2.0 ** -11 * np.abs(x)).all()


def test_linear_i8_refuses_grids_past_32_bits(hip):
    assert linear(hip, (16, 16, 1), M=1 << 27, N=8, ldo=8) == -12 and "too many tiles" in hip.last_error()


@pytest.mark.parametrize("M,N,tiles", [
    (2 ** 31 - 1, 8, (None, (256, 256, 1), (128, 64, 1), (64, 64, 1), (16, 16, 1))), (8, 2 ** 31 - 8, ((256, 256, 1), (64, 128, 1), (16, 16, 1))),
    (2 ** 31 - 128, 8, ((256, 256, 1), (192, 128, 1), (16, 16, 1))), (2 ** 31 - 255, 8, ((256, 256, 1),)), (17, 2 ** 31 - 128, ((256, 256, 1),))])
def test_linear_i8_refuses_rows_and_columns_near_2_31(hip, M, N, tiles):
    """rounding them up to whole tiles passes 32 bits (threads: 512 a tile, 256 up to 128 x 128 and 64 columns)"""
    for tile in tiles:
        rc = linear(hip, tile, M=M, N=N, ldo=N)
        assert rc == -12 and "too many tiles" in hip.last_error(), (tile, hip.last_error())


def test_linear_i8_workspaces_of_large_products(hip):
    """the K slices that pay for no product of many tiles, up to the largest sizes"""
    for p in range(13, 31):
        assert hip.lib().hxa_linear_i8_ws_bytes(2 ** p + 77, 4096, 8192) == 0 and hip.lib().hxa_linear_i8_ws_bytes(4096, 2 ** p + 8, 8192) == 0
