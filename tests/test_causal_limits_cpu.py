"""Limits that the causal attention path's calls state, without a GPU."""
import ctypes as C

import pytest

from tests.test_causal_cpu import FAKE, hip, plan  # noqa: F401 (hip is a fixture)


@pytest.mark.parametrize("nseq", [2 ** 30 + 1, 2 ** 31 - 1])
def test_more_sequences_than_the_search_counts_are_refused(hip, nseq):
    """the search of a token's sequence steps by up to 64 (nseq + 63) / 64, which has to stay below 2^31"""
    L, c = hip.lib(), plan(hip, nseq=nseq)
    assert L.hxa_kv_append(C.byref(c), FAKE, 256, FAKE, 256, 4, None, 1e-6, None, None) == -12 and "nseq" in hip.last_error()
    assert L.hxa_attention_cached(C.byref(c), FAKE, 512, FAKE, 512, 4, 4, 0.1, None, 0, None) == -12
