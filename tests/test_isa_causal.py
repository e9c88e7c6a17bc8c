"""The built gfx950 code of the causal attention kernels at their barriers: like the other kernels that fill LDS by direct loads, they wait
for their own LDS reads before a barrier that frees a buffer, on every path."""
from tests.test_isa_barriers import _kernels, _reads_at_barriers


def test_no_barrier_is_passed_with_a_fragment_read_in_flight(tmp_path):
    kernels = _kernels(r"causal_kernel|cached_kernel", str(tmp_path))
    assert len(kernels) == 18  # 2 types x 3 head widths x (64 rows, 128 rows, over the cache)
    bad = {n: [r for r in _reads_at_barriers(ins) if r[1] > 0] for n, ins in kernels.items()}
    assert not {n: r for n, r in bad.items() if r}
