"""The causal text model's attention path at the far ends of what its calls take: many blocks, values that are not finite, weights of one kind."""
import numpy as np
import pytest

from tests._causal import BF16, F16, Packed, close
from tests.test_gpu_causal import expect_causal, hip, run_causal, say  # noqa: F401 (hip is a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,Hq,lens", [(F16, 1000, [80, 81, 83, 79, 120, 1, 137, 59]), (BF16, 1024, [330, 0, 310])])
def test_more_than_4096_blocks_a_key_head(hip, dtype, Hq, lens):
    """a few sequences of 5000 blocks of 128 rows: each block's rows are written, with their own values"""
    say("many blocks", dtype, Hq, lens)
    assert sum(lens) * Hq > 4096 * 128
    b = Packed(hip, np.random.default_rng(Hq), lens, Hq, 1, 64, dtype)
    want, bound = expect_causal(b, 0.125)
    close(run_causal(hip, b, 0.125), want, bound, "many blocks")
