"""The items over a cache of int8, whose plan counts setups and tiles otherwise: the checks of test_causal_walk on its plans, on the CPU. Ranges of the prefix and
pieces together are no more than the places."""
import ctypes as C
import os
import random
import subprocess

import pytest

from tests.test_causal_walk import (cached, test_every_tile_over_the_cache_once, test_pieces_of_very_long_lists_fit_the_grid,  # noqa: F401
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
