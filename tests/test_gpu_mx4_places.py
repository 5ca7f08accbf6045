"""`ops.linear_mx4` with operands and results at the places in memory that its argument checks allow."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from clavaddpm_amd import ops
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
