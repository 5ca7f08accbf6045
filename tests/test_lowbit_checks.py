"""What the low-bit layers and the filtered draws check on the host, and what their sources have to hold (no GPU needed)."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "clavaddpm_amd", "csrc")


def test_a_waves_lds_reads_have_returned_before_it_passes_a_barrier_of_the_product():
    """The stages of `mx4_tile_kernel` are overwritten behind its barriers.  The compiler orders LDS reads before a written-out
    barrier but not the wait for them, which belongs to the instruction that uses the value: the barrier has to hold it."""
    text = open(os.path.join(CSRC, "gemm_mx4.hip")).read()
    barriers = re.findall(r'asm volatile\("([^"]*s_barrier[^"]*)"', text)
    assert len(barriers) == 3
    for b in barriers:
        assert re.fullmatch(r"s_waitcnt vmcnt\((%0|0)\) lgkmcnt\(0\)\\n\\ts_barrier", b), b
