"""`ops.sample_categories`: temperature, top-k, top-p, min-p and the draw against their definition in 64 bits on the host."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from clavaddpm_amd import ops
from clavaddpm_amd._lib import ClavaHipError

DEV = "cuda"


def filtered(z, temperature, top_k, top_p, min_p):
    """Kept masses of one block in index order (float64), or None where nothing can be drawn."""
    z = np.asarray(z, dtype=np.float64)
    K = len(z)
    if K == 0 or np.isnan(z).any() or z.max() == -math.inf or math.isnan(temperature) or temperature < 0:
        return None
    if temperature < 1e-290:
        temperature, top_k = 1.0, 1
    top = z.max()
    if top == math.inf:
        a = (z == math.inf).astype(np.float64)
    else:
        with np.errstate(under="ignore"):
            a = np.exp((z - top) / temperature)
    order = np.argsort(-z, kind="stable")
    k = top_k if 0 < top_k < K else K
    keep = np.zeros(K, bool)
    mass = math.fsum(a[order[:k]])
    # The masses before each are summed in more than 64 bits, so that a border is where it is; the goal is the float64 product
    # that the definition names (0.26 * 3000 is 780 in float64, and 780 + 2.7e-14 in more bits, which is another border).
    goal = np.longdouble(float(top_p) * mass)
    before = np.concatenate([[0.0], np.cumsum(a[order[:k]], dtype=np.longdouble)[:-1]])
    for n, i in enumerate(order[:k]):
        keep[i] = (top_p >= 1 or n == 0 or before[n] < goal) and a[i] >= min(max(min_p, 0.0), 1.0)
    return a * keep


def choose(z, u, **p):
    w = filtered(z, **p)
    if w is None or math.isnan(u):
        return -1, math.nan
    run = np.cumsum(w, dtype=np.longdouble)
    total = run[-1]
    hits = np.nonzero((run > np.longdouble(max(u, 0.0)) * total) & (w > 0))[0]
    i = hits[0] if len(hits) else np.nonzero(w > 0)[0][-1]
    return int(i), float(np.log(w[i] / float(total)))


def expect(logits, u, classes, **p):
    z, at = logits.double().cpu().numpy(), np.concatenate([[0], np.cumsum(classes)])
    B, m = u.shape
    idx, lp = np.zeros((B, m), np.int32), np.zeros((B, m))
    pick = lambda v, b, f: float(v[b, f]) if isinstance(v, np.ndarray) else v
    for b in range(B):
        for f in range(m):
            idx[b, f], lp[b, f] = choose(z[b, at[f]:at[f + 1]], float(u[b, f]), **{k: pick(v, b, f) for k, v in p.items()})
    return idx, lp


def offsets(classes):
    return torch.tensor(np.concatenate([[0], np.cumsum(classes)]), device=DEV, dtype=torch.int32)


def same(got, want, widest=0):
    """Equal classes; log-probabilities within the float32 rounding (half a step), the float64 arithmetic's 1e-12 and, for
    features of more than 2048 classes, what the masses lose as whole units of 2^-s, s = min(51, 62 - ceil(log2 K)): half a
    unit a class, K 2^-(s + 1) in all, of a sum that is at least 1."""
    idx, lp = got
    assert np.array_equal(idx.cpu().numpy(), want[0])
    g, w = lp.cpu().double().numpy(), want[1]
    assert np.array_equal(np.isnan(g), np.isnan(w))
    ok = ~np.isnan(w)
    units = widest * 2.0 ** -(min(51, 62 - math.ceil(math.log2(widest))) + 1) if widest > 2048 else 0.0
    assert (np.abs(g[ok] - w[ok]) <= np.abs(w[ok]) * 2.0 ** -24 + 1e-12 + units).all()


def check(logits, u, classes, max_classes=None, **p):
    got = ops.sample_categories(logits.to(DEV), u.to(DEV), offsets(classes), max_classes, log_prob=True, **p)
    same(got, expect(logits, u, classes, **{"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, **p}), max(classes))
    return got


def uniforms(B, m, seed):
    u = torch.from_numpy(np.random.RandomState(seed).uniform(size=(B, m))).float()
    return u.clamp(max=1 - 2.0 ** -24)


FILTERS = [{}, {"temperature": 0.3}, {"top_k": 1}, {"top_k": 5}, {"top_p": 0.5}, {"top_p": 0.95, "temperature": 1.7}, {"min_p": 0.05},
           {"top_k": 12, "top_p": 0.8, "min_p": 0.01, "temperature": 0.9}, {"temperature": 0.0}, {"top_p": 0.0}, {"min_p": 1.0}]
CLASSES = [1, 2, 3, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 300, 511, 513, 1000, 1024, 1025]


@pytest.mark.parametrize("p", FILTERS, ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_many_features_of_every_width(p, dtype):
    g = torch.Generator().manual_seed(len(str(p)))
    z = (3 * torch.randn((6, sum(CLASSES)), generator=g)).to(dtype)
    check(z, uniforms(6, len(CLASSES), 1), CLASSES, max(CLASSES), **p)


@pytest.mark.parametrize("p", FILTERS, ids=str)
@pytest.mark.parametrize("K", [1500, 2047, 2048, 2049, 4097, 10000, 40001, 131072])
def test_one_wide_feature(p, K):
    g = torch.Generator().manual_seed(K)
    rows = 3 if K < 50000 else 2
    z = 3 * torch.randn((rows, K), generator=g)
    check(z, uniforms(rows, 1, K), [K], **p)
    check(z.bfloat16(), uniforms(rows, 1, K + 1), [K], **p)


@pytest.mark.parametrize("K", [1, 5, 40, 64, 200, 1000, 3001, 9000, 70000])
def test_equal_logits_keep_the_lowest_indexes(K):
    z = torch.zeros(4, K)
    z[1] = torch.randint(0, 3, (K,), generator=torch.Generator().manual_seed(K)).float()
    z[2, ::2] = -0.0                                              # the two zeros are equal
    u = torch.tensor([[0.0], [0.5], [0.999], [0.3]])
    for p in ({}, {"top_k": 3}, {"top_k": max(1, K // 2)}, {"top_p": 0.5}, {"top_p": 0.26, "top_k": max(2, K - 1)}, {"temperature": 0.0}):
        check(z, u, [K], **p)


@pytest.mark.parametrize("K", [4, 50, 700, 5000])
def test_masks_infinities_and_nan(K):
    low = torch.finfo(torch.float32).min
    g = torch.Generator().manual_seed(K)
    z = torch.randn((12, K), generator=g)
    z[0] = -math.inf                                              # nothing left
    z[1] = -math.inf
    z[1, K - 1] = -3.0                                            # one class left
    z[2] = low                                                    # the lowest value everywhere: all alike
    z[3, ::2] = low
    z[4, 1] = math.inf
    z[5, 1::2] = math.inf
    z[6, K // 2] = math.nan
    z[7, 0], z[7, 1] = math.nan, -math.inf
    z[8] = torch.finfo(torch.float32).max
    z[9, ::3] = -math.inf
    z[10] *= 1e30
    z[11] = torch.linspace(-80, 0, K)
    u = uniforms(12, 1, K)
    for p in FILTERS:
        check(z, u, [K], **p)


@pytest.mark.parametrize("K", [6, 90, 3000])
def test_uniforms_at_their_ends(K):
    z = torch.randn((7, K), generator=torch.Generator().manual_seed(K))
    z[:, 0] = -math.inf
    u = torch.tensor([[0.0], [1.0 - 2.0 ** -24], [1.0], [5.0], [-1.0], [math.nan], [2.0 ** -24]])
    for p in ({}, {"top_k": 2}, {"top_p": 0.7}):
        idx, _ = check(z, u, [K], **p)
        assert (idx[:5] > 0).all() and idx[5] == -1


def test_parameters_for_every_row_and_feature():
    B, classes = 9, [3, 40, 64, 300, 2500]
    m = len(classes)
    r = np.random.RandomState(4)
    z = 2 * torch.randn((B, sum(classes)), generator=torch.Generator().manual_seed(1))
    u = uniforms(B, m, 6)
    t = torch.from_numpy(r.uniform(0, 1.5, (B, m))).float()
    t[0, 0], t[1, 1], t[2, 2] = 0.0, math.nan, -1.0
    k = torch.from_numpy(r.randint(-1, 20, (1, m))).int()
    p = torch.from_numpy(r.uniform(0.1, 1.1, (B, 1))).float()
    mn = torch.from_numpy(r.uniform(-0.1, 0.1, (m,))).float()
    got = ops.sample_categories(z.to(DEV), u.to(DEV), offsets(classes), log_prob=True, temperature=t.to(DEV), top_k=k.to(DEV), top_p=p.to(DEV),
                                min_p=mn.to(DEV))
    full = lambda v: np.broadcast_to(v.numpy(), (B, m)).astype(np.float64 if v.dtype == torch.float32 else np.int64)
    want_k = full(k)
    z64, at = z.double().numpy(), np.concatenate([[0], np.cumsum(classes)])
    idx, lp = np.zeros((B, m), np.int32), np.zeros((B, m))
    for b in range(B):
        for f in range(m):
            idx[b, f], lp[b, f] = choose(z64[b, at[f]:at[f + 1]], float(u[b, f]), temperature=full(t)[b, f], top_k=int(want_k[b, f]),
                                         top_p=full(p)[b, f], min_p=full(mn)[b, f])
    same(got, (idx, lp), max(classes))


def test_features_without_classes_strides_and_a_wrong_hint():
    classes = [0, 5, 0, 70, 2300, 0]
    big = torch.randn((8, sum(classes) + 11), generator=torch.Generator().manual_seed(2))
    z = big[::2, 3:3 + sum(classes)]
    ub = uniforms(4, len(classes) + 3, 2)
    u = ub[:, 1:1 + len(classes)]
    want = expect(z, u, classes, temperature=0.8, top_k=9, top_p=0.9, min_p=0.0)
    zd, ud = big.to(DEV)[::2, 3:3 + sum(classes)], ub.to(DEV)[:, 1:1 + len(classes)]
    for hint in (None, 0, 1, 70, 2300, 10 ** 6):
        same(ops.sample_categories(zd, ud, offsets(classes), hint, temperature=0.8, top_k=9, top_p=0.9, log_prob=True), want, max(classes))
    # offsets outside of the row are cut to it
    off = torch.tensor([-5, 4, 10 ** 6, 2], device=DEV, dtype=torch.int32)
    got = ops.sample_categories(zd, ud[:, :3], off)
    assert got[:, 0].ge(0).all() and got[:, 0].lt(4).all() and got[:, 1].ge(0).all() and (got[:, 2] == -1).all()


def test_many_classes_with_almost_all_logits_in_a_narrow_band():
    """Keys that share their high bits, so that a coarse first cut of the order keeps nearly every class."""
    for K in (900, 2000, 8000, 100000):
        g = torch.Generator().manual_seed(K)
        z = 5.0 + 1e-5 * torch.randn((3, K), generator=g)
        z[1, 7] = 40.0
        z[2, 5] = -1e30
        for p in ({"top_k": K // 3}, {"top_p": 0.37}, {"top_k": K // 2, "top_p": 0.5}):
            check(z, uniforms(3, 1, K), [K], **p)


def test_own_random_numbers_do_not_depend_on_how_rows_are_cut():
    classes = [4, 50, 900]
    z = torch.randn((40, sum(classes)), device=DEV)
    off = offsets(classes)
    a = ops.sample_categories(z, None, off, seed=9, row_offset=100, step_index=3)
    b = torch.cat([ops.sample_categories(z[:13], None, off, seed=9, row_offset=100, step_index=3),
                   ops.sample_categories(z[13:], None, off, seed=9, row_offset=113, step_index=3)])
    assert torch.equal(a, b)
    assert not torch.equal(a, ops.sample_categories(z, None, off, seed=9, row_offset=100, step_index=4))
    # they are uniform: shares of a two-class feature within six standard deviations
    n = 1 << 16
    p = 0.3
    two = torch.tensor([[math.log(1 - p), math.log(p)]], device=DEV).expand(n, 2).contiguous()
    share = ops.sample_categories(two, None, seed=5).float().mean().item()
    assert abs(share - p) < 6 * math.sqrt(p * (1 - p) / n)


def test_the_same_bits_again_on_another_stream_and_from_replayed_graphs():
    classes = [5, 300, 6000]
    z = torch.randn((16, sum(classes)), device=DEV)
    u = uniforms(16, 3, 8).to(DEV)
    off = offsets(classes)
    args = dict(temperature=0.9, top_k=30, top_p=0.8, log_prob=True)
    want = ops.sample_categories(z, u, off, **args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.sample_categories(z, u, off, **args)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs, outs, ins = [], [], []
    for k in range(2):
        zin = z.clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.sample_categories(zin, u, off, **args))
        graphs.append(g)
        ins.append(zin)
    for rep in range(3):
        for k in (0, 1):
            ins[k].copy_(torch.roll(z, 1 + rep + 3 * k, 1))
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for k in (0, 1):
            want = ops.sample_categories(ins[k], u, off, **args)
            assert torch.equal(outs[k][0], want[0]) and torch.equal(outs[k][1], want[1])


def test_no_rows_no_columns():
    assert ops.sample_categories(torch.empty(0, 5, device=DEV)).shape == (0, 1)
    assert ops.sample_categories(torch.empty(3, 0, device=DEV)).eq(-1).all()


def test_refusals():
    z, off = torch.randn(4, 10, device=DEV), offsets([4, 6])
    u = torch.rand(4, 2, device=DEV)
    bad = [lambda: ops.sample_categories(z.cpu(), u, off), lambda: ops.sample_categories(z, u.double(), off),
           lambda: ops.sample_categories(z, u[:, :1], off), lambda: ops.sample_categories(z, u.cpu(), off),
           lambda: ops.sample_categories(z, u, off.long()), lambda: ops.sample_categories(z, u, off.cpu()),
           lambda: ops.sample_categories(z[0], u, off), lambda: ops.sample_categories(z.double(), u, off),
           lambda: ops.sample_categories(z.t().contiguous().t(), u, off), lambda: ops.sample_categories(z, u, off, temperature=-1.0),
           lambda: ops.sample_categories(z, u, off, temperature=math.nan), lambda: ops.sample_categories(z, u, off, top_p=-0.1),
           lambda: ops.sample_categories(z, u, off, min_p=1.5), lambda: ops.sample_categories(z, u, off, min_p=-0.5),
           lambda: ops.sample_categories(z, u, off, temperature=torch.ones(3, device=DEV)),
           lambda: ops.sample_categories(z, u, off, temperature=torch.ones(2)),
           lambda: ops.sample_categories(z, u, off, top_k=torch.ones(2, device=DEV)),
           lambda: ops.sample_categories(z, u, off, -1), lambda: ops.sample_categories(z, u, off, out=torch.empty(4, 2, device=DEV)),
           lambda: ops.sample_categories(z, u.t().contiguous().t(), off)]
    for f in bad:
        with pytest.raises(ClavaHipError):
            f()


@pytest.mark.parametrize("K", [0, 1, 5, 64, 65, 2048, 2049, 4500])
def test_one_feature_inside_a_wider_row(K):
    z = torch.randn((3, 5000), generator=torch.Generator().manual_seed(K))
    u = uniforms(3, 1, K)
    off = torch.tensor([17, 17 + K], device=DEV, dtype=torch.int32)
    for p in ({}, {"top_k": 7, "top_p": 0.9}, {"min_p": 0.2}):
        want = expect(z[:, 17:17 + K], u, [K], **{"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, **p})
        same(ops.sample_categories(z.to(DEV), u.to(DEV), off, log_prob=True, **p), want, max(K, 1))


@pytest.mark.parametrize("B, classes", [(1100, [2100]), (530, [2100, 30, 2200])])
def test_more_wide_rows_than_one_launch_takes(B, classes):
    z = 2 * torch.randn((B, sum(classes)), generator=torch.Generator().manual_seed(B))
    u = uniforms(B, len(classes), B)
    check(z, u, classes, max(classes), top_k=40, top_p=0.9)
    # parameters and outputs of the rows behind the first launch are theirs too
    k = torch.from_numpy(np.random.RandomState(1).randint(1, 60, (B, 1))).int()
    idx = ops.sample_categories(z.to(DEV), u.to(DEV), offsets(classes), top_k=k.to(DEV))
    cut = ops.sample_categories(z[-9:].to(DEV), u[-9:].to(DEV), offsets(classes), top_k=k[-9:].to(DEV))
    assert torch.equal(idx[-9:], cut)


def test_more_features_than_their_table_holds():
    classes = [1 + i % 70 for i in range(1300)] + [300, 2500]
    z = torch.randn((2, sum(classes)), generator=torch.Generator().manual_seed(3))
    for p in ({}, {"top_k": 3, "top_p": 0.8}):
        check(z, uniforms(2, len(classes), 4), classes, 2500, **p)
        check(z, uniforms(2, len(classes), 4), classes, None, **p)


def test_features_wider_than_the_caller_said():
    classes = [2060, 9, 2500, 6000]
    z = torch.randn((5, sum(classes)), generator=torch.Generator().manual_seed(3))
    for hint in (2049, 2060, 2499, 2500, 5999):
        check(z, uniforms(5, 4, 4), classes, hint, top_k=30, top_p=0.8)


def test_parameters_that_are_no_numbers():
    z = torch.randn(4, 50, device=DEV)
    for name in ("temperature", "top_p", "min_p"):
        v = torch.tensor([[0.5], [math.nan], [0.5], [math.nan]], device=DEV)
        idx, lp = ops.sample_categories(z, None, log_prob=True, **{name: v})
        assert (idx[1::2] == -1).all() and lp[1::2].isnan().all() and (idx[::2] >= 0).all()
    for bad in (dict(top_k=2.5), dict(top_k=math.inf), dict(top_k=math.nan), dict(top_p=math.nan)):
        with pytest.raises(ClavaHipError):
            ops.sample_categories(z, None, **bad)
    grad = z.clone().requires_grad_()
    with pytest.raises(ClavaHipError):
        ops.sample_categories(grad, None, log_prob=True)
    with torch.no_grad():
        ops.sample_categories(grad, None, log_prob=True)
    ops.sample_categories(grad, None)


def test_offsets_that_pass_32_bits():
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    classes = [4, 100, 900, 3000]
    n = sum(classes)
    z = torch.randn((3, n), generator=torch.Generator().manual_seed(3)).bfloat16()
    far = torch.empty((1 << 32) + n, device=DEV, dtype=torch.bfloat16).as_strided((3, n), (1 << 31, 1))
    far.copy_(z)
    u = uniforms(3, 4, 4).to(DEV)
    for p in ({}, {"top_k": 30, "top_p": 0.8}):
        a = ops.sample_categories(far, u, offsets(classes), log_prob=True, **p)
        b = ops.sample_categories(z.to(DEV), u, offsets(classes), log_prob=True, **p)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("left", [2, 10, 64, 65, 200, 1500])
def test_fewer_classes_left_than_top_k(left):
    K = 5000
    z = torch.full((4, K), -math.inf)
    g = torch.Generator().manual_seed(left)
    for b in range(4):
        z[b, torch.randperm(K, generator=g)[:left]] = 2 * torch.randn((left,), generator=g)
    for k in (left - 1, left, left + 1, 1024, 1025, 3000):
        for p in ({"top_k": k}, {"top_k": k, "top_p": 0.6}, {"top_k": k, "top_p": 0.9, "min_p": 0.05}):
            check(z, uniforms(4, 1, left), [K], **p)
            check(z, torch.zeros(4, 1), [K], **p)
