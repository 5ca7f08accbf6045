"""`ops.sample_categories` where two rules meet: masks laid over each other, features that overlap, results over inputs."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from clavaddpm_amd import ops
from clavaddpm_amd._lib import ClavaHipError
from test_gpu_choice import check, choose, uniforms

DEV = "cuda"


def masked_twice(classes, ordinary, low, value, dtype, rows, seed):
    """Every feature: `ordinary` logits, `low` ones of `value`, the rest -inf, each row in another order."""
    g = torch.Generator().manual_seed(seed)
    z = torch.full((rows, sum(classes)), -math.inf)
    at = 0
    for K in classes:
        for b in range(rows):
            where = at + torch.randperm(K, generator=g)[:ordinary + low]
            z[b, where[:ordinary]] = 5.0 + 2 * torch.randn((ordinary,), generator=g)
            z[b, where[ordinary:]] = value
        at += K
    return z.to(dtype)


@pytest.mark.parametrize("temperature", [1e-30, 0.3, 1.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("value", ["lowest", -3e38, -1e38, -2e5])
def test_a_mask_of_the_lowest_value_under_a_mask_of_minus_infinity(value, dtype, temperature):
    """A finite logit so far below the maximum that its distance in bins passes float32 is a class like any other: it counts for
    top-k, and its index is its own.  Blocks without it come in between, so that what one leaves behind is not the next one's."""
    classes = [100, 65, 300, 70, 1024, 129, 1025, 2000, 2048, 40, 2600]
    for ordinary, low in ((20, 10), (30, 30), (1, 20), (5, 59)):
        low = min(low, 35)                                       # (the narrowest feature has 40 classes)
        z = masked_twice(classes, ordinary, low, torch.finfo(dtype).min if value == "lowest" else value, dtype, 4, ordinary)
        z[1] = masked_twice(classes, ordinary, 0, 0.0, dtype, 1, 7)[0]
        u = uniforms(4, len(classes), low)
        for top_k in (ordinary - 1 or 1, ordinary, ordinary + 3, ordinary + low, ordinary + low + 5, 200):
            check(z, u, classes, max(classes), temperature=temperature, top_k=top_k)
            check(z, u, classes, 2048, temperature=temperature, top_k=top_k, top_p=0.9, min_p=0.01)


@pytest.mark.parametrize("K", [65, 100, 900, 2048])
def test_only_lowest_values_and_minus_infinities(K):
    """All classes that are left share the mass; the largest finite value beside the lowest one leaves its own."""
    low, high = torch.finfo(torch.float32).min, torch.finfo(torch.float32).max
    z = torch.full((5, K), -math.inf)
    z[0, 3:40], z[1, ::2], z[2, 1], z[3, K - 30:], z[4, 5:25] = low, low, low, low, low
    z[3, 2], z[4, 50] = high, 0.0
    for p in ({"top_k": 3}, {"top_k": 30}, {"top_k": 500}, {"top_k": 30, "top_p": 0.5}, {"top_k": 30, "temperature": 1e-40}, {"top_k": 30, "temperature": 1e30}):
        for dtype in (torch.float32, torch.bfloat16):
            check(z if dtype is torch.float32 else z.clamp(torch.finfo(dtype).min, torch.finfo(dtype).max).where(z.isfinite(), z).to(dtype),
                  uniforms(5, 1, K), [K], **p)


@pytest.mark.parametrize("off", [[0, 5000, 0, 5000, 0, 5000, 100, 4000], [0, 2100, 0, 2200, 3, 2300, 9, 60, 0, 2049], [4999, 5000, 0, 5000, 0, 50, 0, 4500, 1, 2800, 2, 4700]])
@pytest.mark.parametrize("p", [{}, {"top_k": 30, "top_p": 0.9}, {"top_k": 1500}])
def test_features_that_overlap_are_drawn_or_marked(off, p):
    """More wide features than a row of that many classes has side by side: nothing is left as it was.  Those there is room for
    have their class, as all others do, and the rest -1."""
    m, B = len(off) - 1, 5
    z = 2 * torch.randn((B, max(off)), generator=torch.Generator().manual_seed(m))
    u = uniforms(B, m, m)
    out = torch.full((B, m), 777777, device=DEV, dtype=torch.int32)
    _, lp = ops.sample_categories(z.to(DEV), u.to(DEV), torch.tensor(off, device=DEV, dtype=torch.int32), out=out, log_prob=True, **p)
    full = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, **p}
    wide = [f for f in range(m) if off[f + 1] - off[f] > 2048]
    left = wide[max(off) // 2049:]
    assert left
    want = [[-1 if f in left else choose(z[b, off[f]:max(off[f], off[f + 1])].double().numpy(), float(u[b, f]), **full)[0] for f in range(m)]
            for b in range(B)]
    assert out.cpu().tolist() == want
    assert torch.equal(lp.isnan(), out < 0)
