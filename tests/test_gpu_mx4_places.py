"""`ops.linear_mx4` with operands and results at the places in memory that its argument checks allow."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu

from clavaddpm_amd import ops
from clavaddpm_amd._lib import ClavaHipError
from test_gpu_mx4 import product_case, tolerance

DEV = "cuda"
TILES = [(70, 90), (2050, 2100), (5000, 6700)]                    # products that take tiles of 64 x 64, 128 x 128, 256 x 256


def with_scales_at(q, start):
    """The same matrix with its scales `start` bytes behind a multiple of 256."""
    room = torch.full((q.scales.numel() + 64,), 77, device=DEV, dtype=torch.uint8)
    assert room.data_ptr() % 256 == 0
    room[start:start + q.scales.numel()] = q.scales.reshape(-1)
    return ops.Mx4Tensor(q.codes, room[start:start + q.scales.numel()].view(q.scales.shape), q.cols)


@pytest.mark.parametrize("K", [512, 300])                         # scales of whole 16 bytes a row, and not
@pytest.mark.parametrize("M, N", TILES[:2])
def test_scales_at_every_place_of_16_bytes(M, N, K):
    x, w, bias, want, mag = product_case(M, K, N, M + K)
    xq, wq, b = ops.mx4_pack(x.to(DEV)), ops.mx4_pack(w.to(DEV)), bias.to(DEV)
    want = want + bias.double().numpy()
    whole = ops.linear_mx4(xq, wq, b)
    for start in range(0, 17):
        xs, ws = with_scales_at(xq, start), with_scales_at(wq, start)
        assert torch.equal(ops.mx4_unpack(xs), ops.mx4_unpack(xq))
        for left, right in ((xs, wq), (xq, ws), (xs, ws)):
            y = ops.linear_mx4(left, right, b)
            if start % 4 == 0:
                assert torch.equal(y, whole), start
            assert (np.abs(y.cpu().double().numpy() - want) <= tolerance(M, K, N, mag + np.abs(bias.numpy()), want, torch.float32)).all(), start
        out = ops.linear_mx4(xs, ws, b, act="relu", out=with_scales_at(ops.mx4_empty(M, N, DEV), start))
        again = ops.mx4_pack(ops.linear_mx4(xs, ws, b, act="relu"))
        assert torch.equal(out.codes, again.codes) and torch.equal(out.scales, again.scales), start
        few = ops.linear_mx4(ops.mx4_pack(x[:9].to(DEV)), ws, b)
        assert torch.equal(few, ops.linear_mx4(ops.mx4_pack(x[:9].to(DEV)), wq, b)), start


def test_results_over_weights_bias_and_scales():
    x, w, bias = torch.randn(128, 128, device=DEV), ops.mx4_pack(torch.randn(128, 128, device=DEV)), torch.randn(128, device=DEV)
    q = ops.mx4_pack(x)
    both = torch.zeros(128, 256, device=DEV)
    both[7, 200:] = 1.0
    square = torch.randn(128, 128, device=DEV)
    want = ops.linear_mx4(x, w, both[7, 128:].contiguous())
    for f in (lambda: ops.linear_mx4(x, w, out=w), lambda: ops.linear_mx4(q, w, bias, out=w), lambda: ops.linear_mx4(x, w, square[3], out=square),
              lambda: ops.linear_mx4(q, w, out=ops.Mx4Tensor(ops.mx4_empty(128, 128, DEV).codes, q.scales, 128)),
              lambda: ops.linear_mx4(x, w, both[7, 100:228], out=both[:, :128]),
              lambda: ops.mx4_pack(square, out=ops.Mx4Tensor(square.view(torch.uint8).view(-1)[:8192].view(128, 64), w.scales, 128)),
              lambda: ops.mx4_unpack(ops.Mx4Tensor(square.view(torch.uint8).view(-1)[:8192].view(128, 64), w.scales, 128), out=square)):
        with pytest.raises(ClavaHipError, match="overlaps"):
            f()
    # beside each other in one buffer
    ops.linear_mx4(x, w, both[7, 128:], out=both[:, :128])
    assert torch.equal(both[:, :128], want)


def test_draws_over_what_they_read():
    z, u = torch.randn(8, 8, device=DEV), torch.rand(8, 4, device=DEV)
    off = torch.arange(0, 10, 2, device=DEV, dtype=torch.int32)
    k = torch.full((8, 4), 2, device=DEV, dtype=torch.int32)
    for f in (lambda: ops.sample_categories(z, u, off, out=z.view(torch.int32).view(-1)[16:48].view(8, 4)), lambda: ops.sample_categories(z, u, off, out=u.view(torch.int32)),
              lambda: ops.sample_categories(z[:1], u[:1], off, out=off[1:].view(1, 4)), lambda: ops.sample_categories(z, u, off, top_k=k, out=k)):
        with pytest.raises(ClavaHipError, match="overlaps"):
            f()
    out = torch.empty(8, 4, device=DEV, dtype=torch.int32)
    assert torch.equal(ops.sample_categories(z, u, off, top_k=k, out=out), ops.sample_categories(z, u, off, top_k=2))


def test_tangents_are_refused_not_lost():
    x, w = torch.randn(4, 40, device=DEV), ops.mx4_pack(torch.randn(8, 40, device=DEV))
    t = torch.ones(4, 1, device=DEV)
    want = ops.linear_mx4(x, w), ops.sample_categories(x, seed=3)
    with forward_ad.dual_level():
        dx, db, dt = (forward_ad.make_dual(v, torch.ones_like(v)) for v in (x, torch.zeros(8, device=DEV), t))
        for f in (lambda: ops.mx4_pack(dx), lambda: ops.linear_mx4(dx, w), lambda: ops.linear_mx4(x, w, db),
                  lambda: ops.sample_categories(dx, log_prob=True), lambda: ops.sample_categories(x, temperature=dt, log_prob=True)):
            with pytest.raises(ClavaHipError, match="forward"):
                f()
        # whole numbers have no derivative, and inputs without a tangent are as ever
        assert torch.equal(ops.sample_categories(dx, temperature=dt, seed=3), want[1]) and torch.equal(ops.linear_mx4(x, w), want[0])
    with pytest.raises(ClavaHipError, match="backward"):
        ops.sample_categories(x, temperature=t.clone().requires_grad_(), log_prob=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M, N", [(70, 201), (2050, 2101), (5000, 6701)])
def test_16_bit_results_of_odd_rows_at_odd_places(M, N, dtype):
    """Rows of the three tiles' results that start at any 2 bytes and end inside a dword: the float32 result's rounding, and
    nothing beside it."""
    for K in (300, 512):
        x, w, bias, _, _ = product_case(M, K, N, M)
        xq, wq, b = ops.mx4_pack(x.to(DEV)), ops.mx4_pack(w.to(DEV)), bias.to(DEV)
        want = ops.linear_mx4(xq, wq, b, act="relu").to(dtype)
        assert torch.equal(ops.linear_mx4(xq, wq, b, act="relu", out_dtype=dtype), want)
        for start, gap in ((1, 10), (3, 4), (8, 1), (5, 7)):
            big = torch.full((M + 2, N + gap + start), 9.0, device=DEV, dtype=dtype)
            ops.linear_mx4(xq, wq, b, act="relu", out=big[1:M + 1, start:start + N])
            assert torch.equal(big[1:M + 1, start:start + N], want), (K, start)
            assert (big[0] == 9).all() and (big[M + 1] == 9).all() and (big[:, :start] == 9).all() and (big[:, start + N:] == 9).all(), (K, start)
