"""What the low-bit layers and the filtered draws check on the host, and what their sources have to hold (no GPU needed)."""
import ctypes
import os
import re

from clavaddpm_amd import ops
from clavaddpm_amd._lib import lib

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "clavaddpm_amd", "csrc")


def test_a_waves_lds_reads_have_returned_before_it_passes_a_barrier_of_the_product():
    """The stages of `mx4_tile_kernel` are overwritten behind its barriers.  The compiler orders LDS reads before a written-out
    barrier but not the wait for them, which belongs to the instruction that uses the value: the barrier has to hold it."""
    text = open(os.path.join(CSRC, "gemm_mx4.hip")).read()
    barriers = re.findall(r'asm volatile\("([^"]*s_barrier[^"]*)"', text)
    assert len(barriers) == 3
    for b in barriers:
        assert re.fullmatch(r"s_waitcnt vmcnt\((%0|0)\) lgkmcnt\(0\)\\n\\ts_barrier", b), b


def c_refuses(name, types, *args):
    rc = ops._function(name, types)(*args, None)
    assert rc < 0
    return lib().clava_last_error().decode()


def test_codes_have_to_start_where_their_loads_and_stores_do():
    p, off = ctypes.c_void_p(4096), ctypes.c_void_p(4096 + 2)
    assert "codes" in c_refuses("clava_mx4_pack", "pillippp", p, 0, 40, 4, 40, off, p)
    assert "codes" in c_refuses("clava_mx4_unpack", "pplipilp", off, p, 4, 40, p, 0, 40)
    layer = [p, 3, 0, p, p, p, None, 0, p, 3, 0, p, 4, 8, 40, None]
    for at in (0, 4, 8):                                         # x, w, y
        args = list(layer)
        args[at] = ctypes.c_void_p(4096 + 4)
        assert "16 bytes" in c_refuses("clava_linear_mx4", "pilppppipilpiiipp", *args), at


def test_a_workspace_that_is_too_small_is_refused():
    """Float rows are packed into the workspace: 17 rows of 40 columns need 17 * 68 bytes."""
    p = ctypes.c_void_p(4096)
    need = ops._mx4_workspace(17, 40, 0)
    assert need == 17 * 68
    args = [p, 0, 40, None, p, p, None, 0, p, 0, 8, None, 17, 8, 40, p]
    for size in (0, need - 1, -1):
        said = c_refuses("clava_linear_mx4_sized", "pilppppipilpiiiplp", *args, size)
        assert f"{need} bytes" in said and str(size) in said
    assert f"{need} bytes" in c_refuses("clava_linear_mx4", "pilppppipilpiiipp", *args)      # of a size that nobody gave
    small = list(args)
    small[12], small[15] = 0, None                               # no rows: nothing to do
    assert ops._function("clava_linear_mx4_sized", "pilppppipilpiiiplp")(*small, 0, None) == 0
