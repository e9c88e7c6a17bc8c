"""Which rows and keys the workgroups of the causal attention kernels take (csrc/causal_walk.h), on the CPU: the kernels' own source with a wave
of 64 values in an array. Every block of every sequence is taken once, every tile of every block lies in one piece, every piece has a slot
of its own, and no work lies behind the grid."""
import ctypes as C
import os
import random
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("walk") / "walk.so")
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-o", so, os.path.join(HERE, "causal_walk_host.cpp")], check=True)
    lib = C.CDLL(so)
    lib.host_find_block.restype = lib.host_cached.restype = C.c_long
    return lib


def ints(x):
    return np.asarray(x, np.int32)


def ptr(a):
    return a.ctypes.data_as(C.c_void_p)


def prompts(host, lens, G, RB, first, T=None):
    """mistakes in the blocks of sequences of these lengths, and each block's place in its sequence (-1: none)"""
    cu = ints(np.cumsum([0] + list(lens)))
    T = int(cu[-1]) if T is None else T
    grid = T * G // RB + len(lens)
    order = np.empty(max(grid, 1), np.int32)
    return host.host_find_block(ptr(cu), len(lens), T, G, RB, first, C.c_long(grid), ptr(order)), order[:grid]


def parts(r, total, n):
    """total into n parts, some of them empty"""
    cut = sorted(r.randint(0, total) for _ in range(n - 1))
    return [b - a for a, b in zip([0] + cut, cut + [total])]


@pytest.mark.parametrize("nseq", [1, 2, 3, 7, 15, 16, 17, 63, 64, 65, 130])
@pytest.mark.parametrize("RB", [64, 128])
def test_every_block_of_prompts_once(host, nseq, RB):
    r = random.Random(nseq * RB)
    for total in [0, 1, RB - 1, RB, RB + 1, 63 * RB, 64 * RB, 64 * RB + 1, 65 * RB, 300 * RB, 1000 * RB + 7, 4000 * RB - 5] + [
            r.randint(1, 3000 * RB) for _ in range(10)]:
        G = r.choice([1, 2, 5, 8])
        lens = parts(r, total // G, nseq)
        for first in (256 // r.choice([1, 2, 8, 12]), 1):
            bad, _ = prompts(host, lens, G, RB, first)
            assert bad == 0, (lens, G, RB, first)


@pytest.mark.parametrize("nseq", [2, 3, 5, 8, 16])
def test_every_block_of_long_batches_once(host, nseq):
    """more blocks than one round of the place search tells apart (64), and than two do (4096), on both sides of the borders"""
    r = random.Random(nseq)
    for total in (64, 65, 4095, 4096, 4097, 64 * 65 - 1, 64 * 65, 64 * 65 + 1, 5000, 8192, 9999):
        even = [total // nseq + (i < total % nseq) for i in range(nseq)]
        for blocks in (even, [total - 2 * (nseq - 1)] + [2] * (nseq - 1), parts(r, total, nseq), parts(r, total, nseq)):
            for first in (256, 32, 1):
                bad, _ = prompts(host, [64 * b - (b > 1) for b in blocks], 1, 64, first)
                assert bad == 0, (blocks, first)


@pytest.mark.parametrize("hd,RB", [(64, 128), (128, 64), (128, 128), (256, 64), (256, 128)])
@pytest.mark.parametrize("Hk", [1, 2, 8, 12, 300])
def test_longest_blocks_first_with_a_reversed_layer_only_where_two_share_a_cu(host, hd, RB, Hk):
    first = host.host_second_layer(hd, 256, Hk)
    for lens in ([4096], [6500, 300, 1], [900] * 16):
        bad, order = prompts(host, lens, 4, RB, first)
        order = order[order >= 0]
        assert bad == 0
        if hd != 256:
            assert first == max(1, 256 // Hk)
            order[first:2 * first] = order[first:2 * first][::-1].copy()
        assert (np.diff(order) <= 0).all()


def test_prompts_past_the_rows(host):
    """entries of cu past T count as T"""
    for lens in ([100, 200], [50] * 20, [10] * 70):
        for T in (0, 60, 299):
            assert prompts(host, lens, 3, 64, 32, T)[0] == 0


def cached(host, hd, Hq, H, new, length, page, ldt, prefix, ws=1, places=None, rcp=0, behind=0):
    """mistakes in a key head's items over the cache, and the host's plan"""
    cu, ln = ints(np.cumsum([0] + list(new))), ints(length)
    plan = np.zeros(9, np.int32)
    bad = host.host_cached(hd, Hq, H, int(cu[-1]) + behind, len(new), ptr(cu), ptr(ln), page, ldt, prefix, ws,
                           C.c_long(places or (256 if hd == 256 else 512)), rcp, ptr(plan))
    names = ("np_mode", "np_blocks", "sp_max", "rb_log", "s_max", "x_first", "budget", "least", "n_blocks")
    return bad, dict(zip(names, plan.tolist()))


@pytest.mark.parametrize("seed", range(12))
def test_every_tile_over_the_cache_once(host, seed):
    """batches of one to many tokens a sequence, short and long, with and without a prefix; reciprocals rounded either way"""
    r = random.Random(seed)
    split = shared = 0
    for _ in range(120):
        nseq = r.choice([1, 2, 3, 16, 17, 63, 64, 65, 128, 200])
        hd, H = r.choice([64, 128, 256]), r.choice([1, 2, 3, 4, 8, 12, 40, 64, 128])
        G, page = r.choice([1, 2, 4, 5, 8]), r.choice([1, 7, 16, 64, 128])
        kind = r.random()
        new = [1] * nseq if kind < 0.4 else [r.choice([0, 1, 2, 5, 40, 129, 400]) for _ in range(nseq)] if kind < 0.8 else parts(r, r.randint(1, 2000), nseq)
        if sum(new) == 0:
            new[0] = 1
        most = r.choice([10, 300, 4000, 60000])
        length = [n + r.randint(0, most) if r.random() < 0.9 else r.choice([-5, 0, 10 ** 9]) for n in new]
        ldt = -(-max([1] + [x for x in length if x < 10 ** 9]) // page) + r.randint(0, 3)
        prefix = r.choice([0, 0, r.randint(1, 300), r.randint(256, 40000)])
        ws = r.random() < 0.8
        for rcp in (-1, 0, 1):
            bad, plan = cached(host, hd, G * H, H, new, length, page, ldt, prefix, ws, rcp=rcp)
            assert bad == 0, (hd, G, H, new, length, page, ldt, prefix, ws, rcp, plan)
        split += plan["s_max"] > 1
        shared += plan["sp_max"] > 0
    assert split > 20 and shared > 5


@pytest.mark.parametrize("seed", range(4))
def test_pieces_of_very_long_lists_fit_the_grid(host, seed):
    """few places a key head and tiles by the hundred million: whatever the plan, its items cover them"""
    r = random.Random(100 + seed)
    todo = [(256, 64, 1, 2048, 50000, 0), (256, 256, 4, 100, 400000, 0), (128, 512, 1, 31, 2 ** 20, 10 ** 6), (64, 64, 2, 2, 2 ** 24 - 1, 0),
            (128, 4, 1, 2, 1, 2 ** 30 - 65), (64, 8, 1, 31, 2 ** 24 - 2 ** 23, 2 ** 29 - 64)]
    for _ in range(60):
        tiles = int(2 ** r.uniform(10, 24)) - 1
        todo.append((r.choice([64, 128, 256]), r.choice([1, 8, 64, 256, 512, 2048]), r.choice([1, 3, 8]), r.choice([1, 2, 40, 300, 3000]), max(tiles, 1),
                     r.choice([0, r.randint(256, 2 ** 30 - 64 * tiles - 65) if 2 ** 30 - 64 * tiles > 400 else 0])))
    sizes = []
    for hd, H, G, nseq, tiles, prefix in todo:
        new = [r.choice([1, 1, 1, 3]) for _ in range(nseq)]
        for length in ([64 * tiles] * nseq, [r.randint(n, max(64 * tiles, n)) for n in new]):
            for rcp in (-1, 1):
                bad, plan = cached(host, hd, G * H, H, new, length, 64, tiles, prefix, rcp=rcp)
                assert bad == 0, (hd, H, G, nseq, tiles, prefix, rcp, plan)
        sizes.append((plan["s_max"] > 1, plan["n_blocks"] * tiles / plan["budget"]))
    assert any(x and n > 2 ** 21 for x, n in sizes) and any(not x and n > 2 ** 24 for x, n in sizes)


@pytest.mark.parametrize("seed", range(4))
def test_plans_for_more_rows_than_there_are(host, seed):
    """a launch captured for a full batch, replayed with fewer tokens, down to none"""
    r = random.Random(200 + seed)
    for _ in range(60):
        nseq, H, G, hd = r.choice([1, 2, 40, 64, 65, 130]), r.choice([1, 2, 8, 40]), r.choice([1, 2, 8]), r.choice([64, 128, 256])
        new = [r.choice([0, 0, 1, 3]) if r.random() < 0.7 else 0 for _ in range(nseq)] if r.random() < 0.7 else [0] * nseq
        length = [n + r.randint(0, 3000) for n in new]
        prefix, behind = r.choice([0, r.randint(256, 9000)]), r.choice([1, nseq, 700])
        for rcp in (-1, 1):
            bad, plan = cached(host, hd, G * H, H, new, length, 16, 300, prefix, r.random() < 0.8, rcp=rcp, behind=behind)
            assert bad == 0, (hd, G, H, new, length, prefix, behind, rcp, plan)
