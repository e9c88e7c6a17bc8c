"""The built gfx950 code of the 8-bit kernels at their barriers: a barrier that frees LDS for another wave's writes or loads is not passed with a read of this wave in
flight, on any path."""
from tests.test_isa_barriers import _kernels, _reads_at_barriers


def test_no_barrier_is_passed_with_a_read_in_flight(tmp_path):
    # heads of 128, both types and page forms; a GEMM of each loop form, the decoding tiles
    kernels = _kernels(r"cached_q8_kernel\w*Li128E|gemm_kernelILi(256ELi256|128ELi128|64ELi64)ELi3E|gemm_skinny_kernelILi(16|32|64)ELi3E", str(tmp_path))
    assert len(kernels) >= 4 + 3 + 3
    bad = {n: [r for r in _reads_at_barriers(ins) if r[1] > 0] for n, ins in kernels.items()}
    assert not {n: r for n, r in bad.items() if r}


def test_no_barrier_is_passed_with_a_read_in_flight_in_the_other_widths(tmp_path):
    kernels = _kernels(r"cached_q8_kernel\w*Li(64|256)E|kv_append_q8_kernel|quant_rows_kernel", str(tmp_path))
    names = " ".join(kernels)
    assert sum("cached_q8" in n for n in kernels) == 8 and sum("kv_append_q8" in n for n in kernels) == 18 and "quant_rows" in names
    bad = {n: [r for r in _reads_at_barriers(ins) if r[1] > 0] for n, ins in kernels.items()}
    assert not {n: r for n, r in bad.items() if r}
