"""What the low-bit layers and the filtered draws check on the host, and what their sources have to hold (no GPU needed)."""
import ctypes
import math
import os
import re

import pytest
import torch
from torch.autograd import forward_ad

from clavaddpm_amd import ops
from clavaddpm_amd._lib import ClavaHipError, lib
from clavaddpm_amd.tab_ddpm import CategoryChoice

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


def some_mx4(codes, scales, rows, cols):
    """An Mx4Tensor at made-up addresses: calls on it are refused before anything reads them."""
    q = ops.Mx4Tensor.__new__(ops.Mx4Tensor)
    q.codes_ptr, q.scales_ptr, q.rows, q.cols, q.device = codes, scales, rows, cols, torch.device("cpu")
    return q


def test_a_result_over_anything_that_is_read_is_refused():
    """64 x 128 matrices: codes of 4096 bytes, scales of 256."""
    x, w = some_mx4(0x10000, 0x20000, 64, 128), some_mx4(0x30000, 0x40000, 64, 128)
    for codes, scales, word in ((0x30000, 0x50000, "w"), (0x31000 - 16, 0x50000, "w"), (0x40000, 0x50000, "w"), (0x50000, 0x40000 + 255, "w"),
                                (0x50000, 0x20000, "x"), (0x10000 - 4080, 0x50000, "x"), (0x20000, 0x30000, "x"), (0x50000, 0x30000 - 255, "w")):
        with pytest.raises(ClavaHipError, match=f"overlaps {word},"):
            ops.linear_mx4(x, w, out=some_mx4(codes, scales, 64, 64))
    far = ops._parts(some_mx4(0x50000, 0x51000, 64, 128), 64, 128, 0)
    ops._not_over("", far, x=ops._parts(x, 64, 128, 0), w=ops._parts(w, 64, 128, 0), bias=())
    ops._not_over("", far, bias=((0x50000 - 512, 512, 512, 1),), b2=((0x51100, 512, 512, 1),))
    for bias in ((0x50000 - 511, 512, 512, 1), (0x51100 - 1, 512, 512, 1), (0x50100, 4, 4, 1), (0x40000, 0x20000, 0x20000, 1)):
        with pytest.raises(ClavaHipError, match="overlaps bias"):
            ops._not_over("", far, bias=(bias,))


def test_shared_bytes_of_rows_and_of_one_piece():
    """Against the bytes themselves: rows of 6 bytes every 10 and pieces of every size and place, and other rows."""
    def own(start, row, step, rows):
        return {start + i * step + k for i in range(rows) for k in range(row)}
    rows = (100, 6, 10, 4)
    for start in range(90, 150):
        for size in range(1, 25):
            piece = (start, size, size, 1)
            want = bool(own(*rows) & own(*piece))
            assert ops._share(rows, piece) == want and ops._share(piece, rows) == want, piece
        other = (start, 3, 10, 4)
        assert ops._share(rows, other) == bool(own(*rows) & own(*other)) or start >= 130 or start < 73, start
        assert ops._share(rows, (start, 3, 7, 2)) >= bool(own(*rows) & own(start, 3, 7, 2)), start
    t = torch.zeros(5, 4)[:, 1:3]
    assert ops._spread(t) == ((t.data_ptr(), 72, 72, 1),) and ops._spread(torch.zeros(1).expand(9)) [0][1] == 4


def test_a_derivative_that_is_asked_for_is_refused():
    x = torch.ones(3)
    ops._no_gradient("f has no backward", x, None)
    with pytest.raises(ClavaHipError, match="f has no backward: call"):
        ops._no_gradient("f has no backward", None, x.clone().requires_grad_())
    with torch.no_grad():
        ops._no_gradient("f has no backward", x.clone().requires_grad_())
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        ops._no_gradient("f has no backward", x, None)
        ops._no_gradient("f has no backward", forward_ad.unpack_dual(dual).primal)
        for grad in (True, False):                               # (no_grad does not stop tangents)
            with torch.set_grad_enabled(grad), pytest.raises(ClavaHipError, match="no forward derivative"):
                ops._no_gradient("f has no backward", x, dual)
        w = some_mx4(0x30000, 0x40000, 3, 3)
        with pytest.raises(ClavaHipError, match="no forward derivative"):
            ops.linear_mx4(some_mx4(0x10000, 0x20000, 4, 3), w, dual)


def test_numbers_that_no_parameter_holds():
    for bad in (dict(top_k=math.inf), dict(top_k=[1, math.inf]), dict(top_k=math.nan), dict(temperature=10 ** 400), dict(temperature=[1.0, 10 ** 400])):
        with pytest.raises(ValueError, match="CategoryChoice"):
            CategoryChoice(**bad)
    cpu = torch.device("cpu")
    assert CategoryChoice(top_k=[2 ** 40, 3.0, 0]).arguments(3, cpu)["top_k"].tolist() == [2 ** 31 - 1, 3, 0]
    assert CategoryChoice(top_k=10 ** 30).arguments(3, cpu)["top_k"] == 2 ** 31 - 1
    for name in ("temperature", "top_p"):
        with pytest.raises(ClavaHipError, match=name):
            ops._choice_args(cpu, 1, 1, ((name, 10 ** 400),))
    assert ops._choice_args(cpu, 1, 1, (("temperature", 10 ** 300),)).temperature == 1e300
