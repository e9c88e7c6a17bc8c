"""The items over a cache of int8, whose plan counts setups and tiles otherwise: the checks of test_causal_walk on its plans, on the CPU. Ranges of the prefix and
pieces together are no more than the places."""
import ctypes as C
import os
import random
import subprocess

import numpy as np
import pytest

from tests.test_causal_walk import (cached, ints, ptr, test_every_tile_over_the_cache_once, test_pieces_of_very_long_lists_fit_the_grid,  # noqa: F401
                                    test_plans_for_more_rows_than_there_are)

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("walk") / "q8_walk.so")
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-o", so, os.path.join(HERE, "q8_walk_host.cpp")], check=True)
    lib = C.CDLL(so)
    lib.host_find_block.restype = lib.host_cached.restype = C.c_long
    return lib


@pytest.mark.parametrize("seed", range(3))
def test_a_piece_never_waits_for_a_place(host, seed):
    """where there is a budget for it: np_blocks + budget + 1 items at most, the last of them empty or not, fit the places a key head"""
    r = random.Random(seed)
    for _ in range(100):
        nseq, H, G = r.choice([2, 16, 64, 128]), r.choice([1, 2, 4, 8]), r.choice([1, 2, 4, 8])
        length = [r.randint(1, 4000) for _ in range(nseq)]
        prefix = r.choice([0, 300, 4096, 30000])
        bad, p = cached(host, 128, G * H, H, [1] * nseq, length, 16, 250, prefix)
        assert bad == 0 and (p["s_max"] == 1 or p["budget"] == 1 or p["budget"] + p["np_blocks"] + 1 <= 512 // H)


@pytest.fixture(scope="module")
def load(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("walk") / "q8_load.so")
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-o", so, os.path.join(HERE, "q8_walk_load_host.cpp")], check=True)
    lib = C.CDLL(so)

    def run(hd, Hq, H, new, length, page, ldt, prefix, places):
        cu, ln, x = ints(np.cumsum([0] + list(new))), ints(length), np.zeros(6)
        lib.host_load(hd, Hq, H, int(cu[-1]), len(new), ptr(cu), ptr(ln), page, ldt, prefix, C.c_long(places), ptr(x))
        return x.tolist()
    return run


MANY = [(128, 32, 8, 2048, 1, 4096, 500), (128, 32, 8, 512, 4, 1000, 500), (128, 64, 16, 1024, 1, 1000, 300), (256, 16, 16, 128, 16, 4096, 300),
        (128, 32, 8, 1024, 1, 4096, 470), (128, 32, 8, 256, 4, 16000, 300), (64, 32, 8, 512, 1, 1000, 1000), (128, 8, 1, 4096, 1, 300, 2000)]


def is_shared_out(x, places, prefix):
    """The pieces have half the places or more to themselves, and so no item takes more than about twice its share of the work. A piece has chunk tiles of the
    list, the largest of ceil(list / budget), 1 and a block's tiles over its slots but one, or (pieces within their blocks) fewer than SEG = 6 more; and a
    block's own start, 6. A range of the prefix, two for a tile, takes no more with two roundings up, or its slots' share of the tiles."""
    most, total, block, slots, budget, shared = x
    chunk = max(2 * total / places, 1, block / max(slots - 1, 1)) + 1 + 6
    assert shared and 2 * budget >= places and most <= max(chunk + 6, 2 * -(-(-(-prefix // 64)) // shared)), x


@pytest.mark.parametrize("hd,Hq,H,nseq,n,prefix,past", MANY)
def test_large_batches_behind_a_prefix_are_shared_out(load, hd, Hq, H, nseq, n, prefix, past):
    """many blocks of the prefix leave the sequences' own keys their places"""
    r = random.Random(nseq)
    places = 256 if hd == 256 else 512
    for length in ([n + past] * nseq, [n + int(r.expovariate(1 / past)) for _ in range(nseq)]):
        ldt = -(-max(length) // 16)
        is_shared_out(load(hd, Hq, H, [n] * nseq, length, 16, ldt, prefix, places), places // H, prefix)


@pytest.mark.parametrize("seed", range(4))
def test_batches_behind_a_prefix_are_shared_out(load, seed):
    """one to some thousands of sequences of one to several tokens, any number of heads"""
    r = random.Random(300 + seed)
    for _ in range(60):
        hd, H, G = r.choice([64, 128, 256]), r.choice([1, 2, 4, 8, 16, 40]), r.choice([1, 2, 4, 8])
        nseq, n = int(2 ** r.uniform(1, 11)), r.choice([1, 1, 1, 2, 4])
        n = min(n, 16 // G)
        most = r.choice([100, 1000, 6000])
        length = [n + r.randint(0, most) for _ in range(nseq)]
        ldt, places = -(-max(length) // 16), 256 if hd == 256 else 512
        prefix = int(2 ** r.uniform(9.4, 15))
        is_shared_out(load(hd, G * H, H, [n] * nseq, length, 16, ldt, prefix, places), places // H, prefix)
