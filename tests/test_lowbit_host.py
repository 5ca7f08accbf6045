"""What the low-bit layers and the filtered draws refuse before any GPU work, and their host-side settings (no GPU needed)."""
import ctypes

import numpy as np
import pytest
import torch

from clavaddpm_amd import _lib, mx4_nets, ops, split_nets
from clavaddpm_amd._lib import ClavaHipError, lib
from clavaddpm_amd.tab_ddpm import CategoryChoice, GaussianMultinomialDiffusion, MLPDiffusion


def refused(call, *words):
    with pytest.raises(ClavaHipError) as e:
        call()
    for w in words:
        assert w in str(e.value), str(e.value)


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 40)
    refused(lambda: ops.mx4_pack(x), "device")
    refused(lambda: ops.Mx4Tensor(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 4, dtype=torch.uint8), 40), "device")
    refused(lambda: ops.sample_categories(x), "device")
    refused(lambda: ops.linear_mx4(x, x), "Mx4Tensor")
    refused(lambda: mx4_nets.Mx4Stack([x], [x[0]], [0]), "first and a last")


def c_refuses(name, types, *args):
    rc = ops._function(name, types)(*args, None)
    assert rc < 0
    return lib().clava_last_error().decode()


def test_c_entries_refuse_before_they_launch():
    p = ctypes.c_void_p(4096)          # never read: every call below is refused first
    pack, unpack, layer = ("clava_mx4_pack", "pillippp"), ("clava_mx4_unpack", "pplipilp"), ("clava_linear_mx4", "pilppppipilpiiipp")
    assert "null" in c_refuses(*pack, None, 0, 40, 4, 40, p, p)
    assert "dtype" in c_refuses(*pack, p, 3, 40, 4, 40, p, p)
    assert "leading" in c_refuses(*pack, p, 0, 39, 4, 40, p, p)
    assert "-1 x 40" in c_refuses(*pack, p, 0, 40, -1, 40, p, p)
    assert "x 0" in c_refuses(*pack, p, 0, 40, 4, 0, p, p)
    assert "dtype" in c_refuses(*unpack, p, p, 4, 40, p, 7, 40)
    assert "leading" in c_refuses(*unpack, p, p, 4, 40, p, 0, 3)
    good = [p, 3, 0, p, p, p, None, 0, p, 0, 8, None, 4, 8, 40, None]
    for at, value, word in ((0, None, "null"), (3, None, "null"), (4, None, "null"), (8, None, "null"), (1, 9, "dtypes"), (9, -1, "dtypes"), (9, 3, "null"),
                            (7, 4, "activation"), (10, 7, "leading"), (12, -1, "M -1"), (13, 0, "N 0"), (14, 0, "K 0"), (0, ctypes.c_void_p(4104), "16 bytes"),
                            (4, ctypes.c_void_p(4097), "16 bytes")):
        args = list(good)
        args[at] = value
        assert word in c_refuses(*layer, *args), (at, value)
    floats = list(good)
    floats[1], floats[2], floats[12] = 0, 40, 17
    assert "null" in c_refuses(*layer, *floats)                          # no workspace
    floats[15], floats[2] = p, 39
    assert "leading" in c_refuses(*layer, *floats)
    choice = ctypes.byref(ops._choice_args(torch.device("cpu"), 2, 1, (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))))
    draw = ("clava_sample_categories", "piliiipipplUUuppplp")
    good = [p, 0, 10, 2, 2, 10, p, 5, choice, p, 2, 0, 0, 0, p, None, None, 0]
    for at, value, word in ((0, None, "null"), (1, 3, "dtype"), (2, 9, "leading"), (3, -1, "B -1"), (4, 0, "m 0"), (6, None, "offsets"), (8, None, "choice"),
                            (10, 1, "uniforms"), (14, None, "null"), (5, 1 << 31 - 1, "")):
        args = list(good)
        args[at] = value
        if at == 5:
            args[2], args[7] = value, 5
        c_refuses(*draw, *args)
        assert word in lib().clava_last_error().decode(), (at, value)
    wide = list(good)
    wide[2] = wide[5] = wide[7] = 5000
    assert "workspace" in c_refuses(*draw, *wide)
    assert c_refuses(*draw, *(wide[:16] + [ctypes.c_void_p(4100), 1 << 40]))


def test_workspace_sizes():
    need = ops._function("clava_choice_workspace_bytes", "iiii", ops.c_ll)
    assert need(4, 3, 2048, 2048) == 0 and need(4, 3, 10000, 2048) == 0 and need(0, 1, 10000, 10000) == 0
    assert need(4, 1, 10000, 10000) > 0 and need(8, 1, 10000, 10000) == 2 * need(4, 1, 10000, 10000)
    assert need(10 ** 6, 1, 10000, 10000) < 1 << 28                      # large batches go in turns
    ws = ops._function("clava_linear_mx4_workspace_bytes", "iii", ops.c_ll)
    assert ws(100, 130, 0) == 100 * 2 * 68 and ws(100, 130, 3) == 0 and ws(0, 130, 0) == 0
    assert ws(16, 2048, 1) == 0 and ws(16, 2049, 1) == 16 * 17 * 68 and ws(17, 2048, 1) == 17 * 16 * 68


def test_category_choice_checks_its_parameters():
    for bad in (dict(temperature=-1), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(top_k=-1), dict(top_k=2.5), dict(top_p=1.1),
                dict(top_p=-0.1), dict(min_p=2), dict(min_p="a"), dict(top_p=[0.5, 3.0]), dict(top_k=True)):
        with pytest.raises(ValueError):
            CategoryChoice(**bad)
    c = CategoryChoice(temperature=0.7, top_k=[1, 0, 3])
    assert "0.7" in repr(c)
    got = c.arguments(3, torch.device("cpu"))
    assert got["temperature"] == 0.7 and got["top_k"].tolist() == [1, 0, 3] and got["top_k"].dtype == torch.int32
    with pytest.raises(ValueError):
        c.arguments(2, torch.device("cpu"))


def test_sample_refuses_a_choice_that_cannot_apply():
    net = MLPDiffusion(3, 0, "none", {"d_layers": [32], "dropout": 0.0})
    d = GaussianMultinomialDiffusion(np.array([0]), 3, net, num_timesteps=10)
    with pytest.raises(ValueError, match="no categorical"):
        d.sample(2, torch.ones(1), choice=CategoryChoice())


def test_mx4_is_a_gemm_mode():
    before = split_nets.get_gemm_mode()
    try:
        split_nets.set_gemm_mode("mx4")
        assert split_nets.get_gemm_mode() == "mx4"
        with pytest.raises(ValueError):
            split_nets.set_gemm_mode("mx5")
    finally:
        split_nets.set_gemm_mode(before)
    assert _lib.declared_symbols()


def test_matrices_that_share_memory_are_told_from_columns_of_one_buffer():
    # (start, bytes of a row, row stride) twice, rows
    assert ops._overlap(0, 16, 64, 8, 16, 64, 4) and ops._overlap(8, 16, 64, 0, 16, 64, 4)
    assert not ops._overlap(0, 16, 64, 16, 48, 64, 4) and not ops._overlap(16, 48, 64, 0, 16, 64, 4)
    assert ops._overlap(0, 16, 64, 16, 49, 64, 4) and ops._overlap(0, 16, 64, 60, 8, 64, 4)
    assert ops._overlap(0, 16, 64, 16, 16, 32, 4)                        # strides that differ
    assert not ops._overlap(0, 16, 64, 208, 16, 32, 4) and not ops._overlap(208, 16, 32, 0, 16, 64, 4)
    assert ops._overlap(0, 16, 16, 15, 1, 1, 1) and not ops._overlap(0, 16, 16, 16, 1, 1, 1)


def test_more_columns_than_a_product_takes():
    p = ctypes.c_void_p(4096)
    assert "33554433" in c_refuses("clava_linear_mx4", "pilppppipilpiiipp", p, 3, 0, p, p, p, None, 0, p, 0, 8, None, 4, 8, (1 << 25) + 1, None)


def test_the_workspace_is_for_blocks_as_wide_as_the_caller_says():
    need = ops._function("clava_choice_workspace_bytes", "iiii", ops.c_ll)
    assert need(64, 400, 10 ** 6, 5000) < need(64, 400, 10 ** 6, 10 ** 6) // 4
    assert need(64, 400, 10 ** 6, 10 ** 6) == need(64, 400, 10 ** 6, 2 ** 31 - 1)
    assert need(64, 1, 10 ** 6, 5000) == need(64, 1, 10 ** 6, 10 ** 6)   # one feature: its own width
