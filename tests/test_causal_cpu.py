"""The causal text model's attention path without a GPU: rotary frequencies, what its calls refuse before any device call, and the
64-bit definitions the GPU tests compare with."""
import ctypes as C
import math

import numpy as np
import pytest

from tests._causal import BF16, F16, attend, narrow, norm_rope, widen

FAKE = 1 << 20  # a pointer that a refused call never follows


@pytest.fixture(scope="module")
def hip():
    from hexanima_amd import hip as h
    h.lib()
    return h


def test_rope_freqs(hip):
    rot, base = 96, 5e5
    i = np.arange(rot // 2)
    plain = base ** (-2.0 * i / rot)
    f, m = hip.rope_freqs(rot, base)
    assert np.array_equal(f, plain.astype(np.float32)) and m == 1.0
    f, m = hip.rope_freqs(rot, base, hip.ROPE_LINEAR, 8.0)
    np.testing.assert_allclose(f, plain / 8, rtol=2 ** -24 + 1e-12)
    f, m = hip.rope_freqs(rot, base, hip.ROPE_BASE, 8.0)
    np.testing.assert_allclose(f[0], 1.0)
    np.testing.assert_allclose(f[-1], plain[-1] / 8, rtol=1e-6)
    f, m = hip.rope_freqs(rot, base, hip.ROPE_PARTS, 8.0, 4096.0, 32.0, 1.0)
    assert m == pytest.approx(0.1 * math.log(8) + 1, rel=1e-6)
    turns = 4096 * plain / (2 * np.pi)
    np.testing.assert_allclose(f[turns >= 32], plain[turns >= 32], rtol=2 ** -23)
    np.testing.assert_allclose(f[turns <= 1], plain[turns <= 1] / 8, rtol=2 ** -23)
    mid = (turns < 32) & (turns > 1)
    # between the borders linear in the pair index, whose real-valued places the borders have
    place = lambda r: rot * math.log(4096 / (r * 2 * np.pi)) / (2 * math.log(base))
    ramp = (i - place(32)) / (place(1) - place(32))
    np.testing.assert_allclose(f[mid], (plain / 8 * ramp + plain * (1 - ramp))[mid], rtol=1e-6)
    assert mid.any() and np.all(np.diff(f) < 0)


@pytest.mark.parametrize("args,rc", [((0, 1e4, 0, 1, 0, 32, 1), -12), ((15, 1e4, 0, 1, 0, 32, 1), -12), ((16, 1.0, 0, 1, 0, 32, 1), -12),
                                     ((16, float("nan"), 0, 1, 0, 32, 1), -12), ((16, 1e4, 4, 1, 0, 32, 1), -11),
                                     ((16, 1e4, 1, 0.5, 0, 32, 1), -12), ((2, 1e4, 2, 2, 0, 32, 1), -12), ((16, 1e4, 3, 2, 0, 32, 1), -12),
                                     ((16, 1e4, 3, 2, 4096, 1, 32), -12), ((16, 1e4, 3, float("inf"), 4096, 32, 1), -12)])
def test_rope_freqs_refuses(hip, args, rc):
    f = np.zeros(64, np.float32)
    assert hip.lib().hxa_rope_freqs(*args, f.ctypes.data, None) == rc and not f.any()
    assert hip.lib().hxa_rope_freqs(16, 1e4, 0, 1, 0, 32, 1, None, None) == -12


def qk(hip, **kw):
    a = dict(dtype=1, q=FAKE, ldq=1024, Hq=8, k=FAKE, ldk=256, Hk=2, T=3, hd=128, gq=FAKE, gk=FAKE, eps=1e-6, pos=FAKE,
             rope=hip.Rope(FAKE, 128, 0, 1.0), qo=FAKE, ldqo=1024, ko=FAKE, ldko=256)
    a.update(kw)
    rope = a["rope"]
    return hip.lib().hxa_qk_norm_rope(a["dtype"], a["q"], a["ldq"], a["Hq"], a["k"], a["ldk"], a["Hk"], a["T"], a["hd"], a["gq"], a["gk"],
                                      a["eps"], a["pos"], C.byref(rope) if rope else None, a["qo"], a["ldqo"], a["ko"], a["ldko"], None)


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=0), -11), (dict(dtype=3), -11), (dict(hd=96), -11), (dict(T=-1), -12), (dict(T=2 ** 25 + 1), -12), (dict(Hq=-1), -12),
    (dict(eps=float("nan")), -12), (dict(eps=-1.0), -12), (dict(q=None), -12), (dict(ko=None), -12), (dict(q=FAKE + 8), -12),
    (dict(ldq=1016), -12), (dict(ldq=1028), -12), (dict(ldqo=1032), -12), (dict(gq=FAKE + 4), -12), (dict(pos=FAKE + 2), -12)])
def test_qk_norm_rope_refuses(hip, kw, rc):
    assert qk(hip, **kw) == rc and hip.last_error().startswith("qk_norm_rope")


def test_rotations_refused_and_empty_calls(hip):
    R = hip.Rope
    for rope, rc in [(R(FAKE, 8, 0, 1.0), -12), (R(FAKE, 144, 0, 1.0), -12), (R(FAKE, -16, 0, 1.0), -12), (R(FAKE, 64, 2, 1.0), -11),
                     (R(None, 64, 0, 1.0), -12), (R(FAKE, 64, 0, float("inf")), -12)]:
        assert qk(hip, rope=rope) == rc
    assert qk(hip, T=0, q=None) == 0 and qk(hip, Hq=0, Hk=0, q=None, k=None) == 0


def plan(hip, **kw):
    a = dict(dtype=1, H=2, hd=128, page=16, npages=100, k=FAKE, v=FAKE, prefix=FAKE, prefix_len=40, table=FAKE, ldt=8, len=FAKE, cu=FAKE, nseq=4)
    a.update(kw)
    return hip.KvCache(*[a[f] for f, _ in hip.KvCache._fields_])


BAD_PLANS = [(dict(dtype=0), -11), (dict(hd=32), -11), (dict(H=0), -12), (dict(H=5000), -12), (dict(page=0), -12), (dict(page=65537), -12),
             (dict(npages=0), -12), (dict(nseq=-1), -12), (dict(ldt=-1), -12), (dict(prefix_len=-1), -12),
             (dict(npages=2 ** 30, page=64), -12), (dict(ldt=2 ** 28), -12), (dict(k=None), -12), (dict(v=FAKE + 8), -12), (dict(cu=None), -12),
             (dict(len=None), -12), (dict(table=None), -12), (dict(prefix=None), -12), (dict(cu=FAKE + 1), -12)]


@pytest.mark.parametrize("kw,rc", BAD_PLANS)
def test_plans_refused(hip, kw, rc):
    L, c = hip.lib(), plan(hip, **kw)
    assert L.hxa_kv_append(C.byref(c), FAKE, 256, FAKE, 256, 4, None, 1e-6, None, None) == rc
    assert hip.last_error().startswith("kv_append")
    Hq = 4 if kw.get("H") != 5000 else 5000
    assert L.hxa_attention_cached(C.byref(c), FAKE, 512, FAKE, 512, 4, Hq, 0.1, None, 0, None) == rc
    assert hip.last_error().startswith("attention_cached")
    assert L.hxa_attention_cached_ws_bytes(C.byref(c), 4, Hq) == 0


def test_append_refuses(hip):
    L, c = hip.lib(), plan(hip)
    run = lambda k=FAKE, ldk=256, v=FAKE, ldv=256, T=4, g=None, eps=1e-6, rope=None: L.hxa_kv_append(
        C.byref(c), k, ldk, v, ldv, T, g, eps, C.byref(rope) if rope else None, None)
    assert [run(k=None), run(v=None), run(ldk=248), run(ldv=260), run(k=FAKE + 2), run(T=-1), run(g=FAKE + 4), run(eps=float("nan"))] == [-12] * 8
    assert run(rope=hip.Rope(FAKE, 24, 0, 1.0)) == -12 and run(rope=hip.Rope(FAKE, 32, 5, 1.0)) == -11
    assert L.hxa_kv_append(None, FAKE, 256, FAKE, 256, 4, None, 1e-6, None, None) == -12
    assert run(T=0, k=None) == 0
    c = plan(hip, nseq=0)
    assert run(k=None) == 0


def causal(hip, **kw):
    a = dict(dtype=2, q=FAKE, ldq=1024, k=FAKE, ldk=256, v=FAKE, ldv=256, o=FAKE, ldo=1024, T=9, cu=FAKE, nseq=2, Hq=8, Hk=2, hd=128, scale=0.1)
    a.update(kw)
    return hip.lib().hxa_attention_causal(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=0), -11), (dict(hd=80), -11), (dict(T=-1), -12), (dict(nseq=-1), -12), (dict(Hk=3), -12), (dict(Hq=0), -12), (dict(Hk=0), -12),
    (dict(T=2 ** 24, Hq=256, Hk=1, ldq=2 ** 15, ldo=2 ** 15), -12), (dict(scale=0.0), -12), (dict(scale=-1.0), -12), (dict(scale=float("inf")), -12),
    (dict(scale=float("nan")), -12), (dict(q=None), -12), (dict(o=FAKE + 4), -12), (dict(ldk=248), -12), (dict(ldo=1020), -12),
    (dict(ldk=2 ** 24), -12), (dict(ldv=2 ** 24), -12), (dict(cu=None), -12), (dict(cu=FAKE + 2), -12), (dict(nseq=2 ** 30), -12)])
def test_attention_causal_refuses(hip, kw, rc):
    assert causal(hip, **kw) == rc and hip.last_error().startswith("attention_causal")


def test_attention_cached_refuses(hip):
    L, c = hip.lib(), plan(hip)
    run = lambda q=FAKE, ldq=512, o=FAKE, ldo=512, T=4, Hq=4, scale=0.1, ws=None, nb=0: L.hxa_attention_cached(
        C.byref(c), q, ldq, o, ldo, T, Hq, scale, ws, nb, None)
    assert [run(q=None), run(o=None), run(ldq=504), run(ldo=516), run(T=-1), run(Hq=3), run(Hq=0), run(scale=0.0), run(scale=float("nan")),
            run(ws=FAKE + 8, nb=1 << 20), run(T=2 ** 25, Hq=64, ldq=8192, ldo=8192)] == [-12] * 11
    assert run(T=0, q=None) == 0
    assert L.hxa_attention_cached(None, FAKE, 512, FAKE, 512, 4, 4, 0.1, None, 0, None) == -12
    assert causal(hip, T=0, q=None) == 0 and causal(hip, nseq=0, cu=None) == 0


def test_workspace_follows_the_sizes(hip):
    """few rows over long keys and a prefix that a batch shares need partials; many rows need none"""
    L = hip.lib()
    size = lambda T, Hq, **kw: L.hxa_attention_cached_ws_bytes(C.byref(plan(hip, **kw)), T, Hq)
    assert size(1, 4, nseq=1, prefix_len=0, ldt=1) == 0
    assert size(1, 4, nseq=1, ldt=512) > 0 and size(1, 4, nseq=1, ldt=512) % ((128 * 4 + 8) * 4) == 0
    assert size(64, 4, nseq=64, prefix_len=4096) > 0
    assert size(100000, 4, nseq=8) == 0


def test_short_tables_are_not_split(hip):
    """up to 6 tiles of 64 keys take no workspace, nor up to 16 where the blocks are many; a prefix counts with them"""
    L = hip.lib()
    size = lambda T, Hq, **kw: L.hxa_attention_cached_ws_bytes(C.byref(plan(hip, **kw)), T, Hq)
    assert size(1, 4, nseq=1, prefix_len=0, ldt=24) == 0 and size(1, 4, nseq=1, prefix_len=0, ldt=25) > 0
    assert size(1, 4, nseq=1, prefix_len=65, ldt=20) > 0 and size(1, 4, nseq=1, prefix_len=64, ldt=20) == 0
    assert size(64, 4, nseq=64, prefix_len=0, ldt=64, H=4) == 0 and size(64, 4, nseq=64, prefix_len=0, ldt=65, H=4) > 0
    assert size(8, 4, nseq=8, prefix_len=0, ldt=64, H=4) > 0 and size(64, 4, nseq=64, prefix_len=256, ldt=48, H=4) > 0


def test_workspace_stays_bounded(hip):
    """many rows: fewer partial results a row instead of more memory, down to one for the prefix's first ranges and one for the own keys"""
    L = hip.lib()
    row = lambda Hq: Hq * (128 * 4 + 8)
    for n in (64, 1000, 5000, 40000, 200000):
        for P in (0, 4096):
            nb = L.hxa_attention_cached_ws_bytes(C.byref(plan(hip, nseq=n, prefix_len=P, ldt=500)), n, 8)
            assert nb % (n * row(8)) == 0 and nb <= max(2 ** 30, 4 * n * row(8)), (n, P, nb)
            assert n > 64 or nb > 0
    assert cached_call(hip, 2 ** 18) == 0 and cached_call(hip, 2 ** 20) == -12  # 2^15 (2^17) blocks of 64 rows for each of 32 heads


def cached_call(hip, T):
    """the error of a call over the cache with T tokens of 256 heads, refused for its pointers where the size is not"""
    L, c = hip.lib(), plan(hip, H=32)
    rc = L.hxa_attention_cached(C.byref(c), None, 2 ** 15, FAKE, 2 ** 15, T, 256, 0.1, None, 0, None)
    return 0 if "pointers" in hip.last_error() else rc


def test_the_tests_own_definitions():
    """attend and norm_rope against sums written out; narrow and widen against numpy's and a known bf16 rounding"""
    rng = np.random.default_rng(0)
    q, k, v = rng.standard_normal((3, 4)), rng.standard_normal((5, 4)), rng.standard_normal((5, 4))
    seen = np.tril(np.ones((3, 5), bool), 1)
    seen[2] = False
    o, _ = attend(q, k, v, 0.5, seen)
    for r in range(2):
        e = [math.exp(0.5 * float(q[r] @ k[s])) if seen[r, s] else 0.0 for s in range(5)]
        np.testing.assert_allclose(o[r], sum(e[s] * v[s] for s in range(5)) / sum(e))
    assert (o[2] == 0).all()
    v[4] = np.inf
    assert np.isfinite(attend(q, k, v, 0.5, seen)[0]).all()
    x = rng.standard_normal((2, 1, 8))
    f = np.array([1.0, 0.1], np.float32)
    y, _ = norm_rope(x, None, 0.0, [0, 3], f, 1)
    np.testing.assert_allclose(y[0], x[0])
    z = (x[1, 0, 2] + 1j * x[1, 0, 3]) * np.exp(1j * 3 * float(f[1]))
    np.testing.assert_allclose([y[1, 0, 2], y[1, 0, 3]], [z.real, z.imag])
    np.testing.assert_allclose(y[1, 0, 4:], x[1, 0, 4:])
    assert widen(narrow(np.float32(1.00390625), BF16), BF16) == 1.0 and widen(narrow(np.float32(1.01171875), BF16), BF16) == 1.015625
    assert widen(narrow(np.float32(0.1), F16), F16) == float(np.float16(0.1))
