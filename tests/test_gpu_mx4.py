"""Microscaled 4-bit matrices (`ops.mx4_pack`, `mx4_unpack`, `linear_mx4`) against their definition in 64 bits on the host."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from clavaddpm_amd import ops
from clavaddpm_amd._lib import ClavaHipError

DEV = "cuda"
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # half a step of each type


def quantise(x):
    """(codes, scale bytes) of float64 rows: the nearest grid value, ties to the even code."""
    rows, cols = x.shape
    kp = (cols + 127) // 128 * 128
    b = np.zeros((rows, kp))
    b[:, :cols] = x
    b = b.reshape(rows, -1, 32)
    bad = ~np.isfinite(b).all(axis=2)
    b = np.where(bad[:, :, None], 0.0, b)
    top = np.abs(b).max(axis=2)
    e = np.where(top > 0, np.floor(np.log2(np.where(top > 0, top, 1.0))), -200).astype(np.int64)
    e = np.where(np.ldexp(1.0, e) > top, e - 1, np.where(np.ldexp(1.0, e + 1) <= top, e + 1, e))      # log2 rounds
    e = np.where(top > 0, np.clip(e - 2, -127, 127), -127)
    v = np.abs(np.ldexp(b, -e[:, :, None]))
    c = np.abs(v[..., None] - GRID)
    near = c.min(axis=-1)
    hits = c == near[..., None]
    first = hits.argmax(axis=-1)
    code = np.where((hits.sum(axis=-1) == 2) & (first % 2 == 1), first + 1, first)
    code = np.minimum(code, 7)
    code = np.where(np.signbit(b), code + 8, code)
    code = np.where(bad[:, :, None], 0, code).reshape(rows, kp).astype(np.uint8)
    return code[:, 0::2] | code[:, 1::2] << 4, np.where(bad, 255, e + 127).astype(np.uint8)


def values(codes, scales, cols):
    q = np.stack([codes & 15, codes >> 4], axis=2).reshape(codes.shape[0], -1)
    v = np.where(q > 7, -GRID[q & 7], GRID[q & 7])
    s = np.repeat(scales.astype(np.int64), 32, axis=1)
    v = np.where(s == 255, np.nan, np.ldexp(v, s - 127))
    return v[:, :cols]


def rand(rows, cols, seed, dtype=torch.float32, spread=3.0):
    r = np.random.RandomState(seed)
    x = r.standard_normal((rows, cols)) * np.exp(spread * r.standard_normal((rows, 1 + (cols - 1) // 32)).repeat(32, axis=1)[:, :cols])
    return torch.from_numpy(x).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 31), (5, 32), (2, 33), (7, 127), (4, 128), (129, 130), (33, 1000), (1, 70001)])
def test_pack_and_unpack_are_the_definition(rows, cols, dtype):
    x = rand(rows, cols, rows * 1000 + cols, dtype)
    x[0, 0] = 0.0
    want = quantise(x.double().numpy())
    q = ops.mx4_pack(x.to(DEV))
    assert np.array_equal(q.scales.cpu().numpy(), want[1])
    got = q.codes.cpu().numpy()
    assert np.array_equal(values(got, want[1], cols), values(*want, cols))
    assert np.array_equal(got, want[0])                          # the sign of a zero and the zeros behind the last column too
    for out in DTYPES:
        v = torch.from_numpy(values(*want, cols)).to(out)
        assert torch.equal(ops.mx4_unpack(q, dtype=out).cpu(), v)


def test_pack_ties_saturation_and_the_ends_of_float32():
    halves = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.999, 6.0, 4.0, -0.25, -5.0, -7.5, 0.0, -0.0] * 2)
    rows = [halves * 2.0 ** k for k in (0, -3, 40, 124, -100, -126, -140, -149)]
    rows += [torch.full((32,), 2.0 ** -149), torch.full((32,), torch.finfo(torch.float32).max), torch.zeros(32)]
    x = torch.stack(rows)
    want = quantise(x.double().numpy())
    q = ops.mx4_pack(x.to(DEV))
    assert np.array_equal(q.scales.cpu().numpy(), want[1]) and np.array_equal(q.codes.cpu().numpy(), want[0])
    assert torch.equal(ops.mx4_unpack(q).cpu().double(), torch.from_numpy(values(*want, 32)))


def test_a_block_with_a_nan_or_an_infinity_reads_as_nan_and_poisons_its_rows_of_a_product():
    x = torch.ones(4, 200)
    x[1, 40], x[2, 199], x[3, 0] = math.nan, math.inf, -math.inf
    q = ops.mx4_pack(x.to(DEV))
    v = ops.mx4_unpack(q).cpu()
    assert v[0].isfinite().all()
    for r, (lo, hi) in ((1, (32, 64)), (2, (192, 200)), (3, (0, 32))):
        assert v[r, lo:hi].isnan().all() and v[r, :lo].isfinite().all() and v[r, hi:].isfinite().all()
    for m in (4, 300):                                           # few rows and many
        xs = torch.ones(m, 200)
        xs[:4] = x
        y = ops.linear_mx4(xs.to(DEV), ops.mx4_pack(torch.ones(70, 200, device=DEV)))
        assert y[0].isfinite().all() and y[1:4].isnan().all() and y[4:].isfinite().all()
        y4 = ops.linear_mx4(xs.to(DEV), ops.mx4_pack(torch.ones(70, 200, device=DEV)), act="relu", out=ops.mx4_empty(m, 70, DEV))
        y = ops.mx4_unpack(y4)
        assert y[0].isfinite().all() and y[1:4].isnan().all()


def test_rows_with_a_stride_and_an_odd_start():
    big = rand(40, 301, 3).to(DEV)
    for dtype in DTYPES:
        b = big.to(dtype)
        x = b[::2, 3:270]
        q = ops.mx4_pack(x)
        ref = ops.mx4_pack(x.contiguous())
        assert torch.equal(q.codes, ref.codes) and torch.equal(q.scales, ref.scales)
        out = torch.full((20, 301), 7.0, device=DEV, dtype=dtype)
        ops.mx4_unpack(q, out=out[:, 1:268])
        assert torch.equal(out[:, 1:268], ops.mx4_unpack(q, dtype=dtype))
        assert (out[:, 0] == 7).all() and (out[:, 268:] == 7).all()
    one = torch.randn(64, 1, device=DEV)
    assert torch.equal(ops.mx4_pack(one.t()).codes, ops.mx4_pack(one.t().contiguous()).codes)


def act64(y, act):
    with np.errstate(over="ignore"):
        return {"none": lambda: y, "relu": lambda: np.maximum(y, 0), "leaky_relu": lambda: np.where(y > 0, y, 0.01 * y),
                "silu": lambda: y / (1 + np.exp(-y))}[act]()


def product_case(M, K, N, seed, dtype=torch.float32):
    """Operands, the float64 product of their 4-bit values and, for every output, the sum of the products' magnitudes."""
    x, w = rand(M, K, seed, dtype, 0.7), rand(N, K, seed + 1, spread=0.7) / math.sqrt(K)
    bias = torch.from_numpy(np.random.RandomState(seed + 2).standard_normal(N)).float()
    xv, wv = values(*quantise(x.double().numpy()), K), values(*quantise(w.double().numpy()), K)
    return x, w, bias, xv @ wv.T, np.abs(xv) @ np.abs(wv).T


SIZES = [(1, 1, 1), (1, 128, 16), (2, 33, 7), (7, 4099, 130), (15, 512, 1024), (16, 128, 129), (17, 640, 31), (33, 257, 70),
         (64, 2048, 96), (127, 384, 255), (128, 1024, 512), (129, 100, 257), (256, 256, 256), (300, 1000, 300), (511, 96, 513), (1030, 512, 384)]


def tolerance(M, K, N, mag, y, out):
    """Float32 accumulation of K products of magnitude sum `mag`: one instruction adds 128 exact products to its sum with at
    most a step (2^-23) of the largest partial sum lost for each of its additions, which are K / 128 instructions of at most
    128 + 1 terms in a tree, and up to 16 partial sums are added: (K / 128 + 8 + 16) steps of the magnitude sum; the
    activation and the bias a few half steps of the result; the output's own rounding."""
    steps = K / 128 + 24
    return mag * steps * 2.0 ** -23 + np.abs(y) * (8 * 2.0 ** -24 + EPS[out]) + 2.0 ** -24 + (2.0 ** -24 if out == torch.float16 else 0)


@pytest.mark.parametrize("M, K, N", SIZES)
@pytest.mark.parametrize("act, biased", [("none", False), ("relu", True)])
def test_linear_sizes(M, K, N, act, biased):
    x, w, bias, want, mag = product_case(M, K, N, M + K + N)
    wq = ops.mx4_pack(w.to(DEV))
    y = ops.linear_mx4(x.to(DEV), wq, bias.to(DEV) if biased else None, act=act)
    ref = act64(want + bias.double().numpy() if biased else want, act)
    err = np.abs(y.cpu().double().numpy() - ref)
    assert (err <= tolerance(M, K, N, mag + np.abs(bias.numpy()), ref, torch.float32)).all()
    # the packed operand gives the same bits as the float one, and a row the same bits in every batch of its kind
    assert torch.equal(y, ops.linear_mx4(ops.mx4_pack(x.to(DEV)), wq, bias.to(DEV) if biased else None, act=act))


@pytest.mark.parametrize("M, K, N", [(3, 130, 50), (200, 300, 200)])
@pytest.mark.parametrize("act", ["none", "relu", "leaky_relu", "silu"])
@pytest.mark.parametrize("dtype, out", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float16), (torch.float16, torch.float32),
                                        (torch.bfloat16, torch.bfloat16)])
def test_linear_types_and_activations(M, K, N, act, dtype, out):
    x, w, bias, want, mag = product_case(M, K, N, 5, dtype)
    y = ops.linear_mx4(x.to(DEV), ops.mx4_pack(w.to(DEV)), bias.to(DEV), act=act, out_dtype=out)
    ref = act64(want + bias.double().numpy(), act)
    assert y.dtype == out
    # silu's slope is below 1.1
    assert (np.abs(y.cpu().double().numpy() - ref) <= tolerance(M, K, N, 1.1 * (mag + np.abs(bias.numpy())), ref, out)).all()


@pytest.mark.parametrize("M, K, N", [(1, 128, 32), (3, 100, 33), (16, 512, 1024), (64, 257, 127), (130, 300, 128), (300, 640, 513), (520, 512, 512)])
def test_linear_result_as_the_next_layers_operand(M, K, N):
    """Codes of the fused result against the float32 result packed by itself: the accumulators are the same ones."""
    x, w, bias, _, _ = product_case(M, K, N, 11)
    wq, b = ops.mx4_pack(w.to(DEV)), bias.to(DEV)
    for act in ("relu", "silu", "none"):
        ref = ops.mx4_pack(ops.linear_mx4(x.to(DEV), wq, b, act=act))
        out = ops.mx4_empty(M, N, DEV)
        out.codes.fill_(0x5a)                                    # the padding has to be written too
        out.scales.fill_(0x5a)
        got = ops.linear_mx4(x.to(DEV), wq, b, act=act, out=out)
        assert got is out and torch.equal(out.scales, ref.scales) and torch.equal(out.codes, ref.codes)


def test_linear_leaves_what_is_not_its_own():
    x, w, _, _, _ = product_case(70, 300, 90, 3)
    wq = ops.mx4_pack(w.to(DEV))
    for M in (5, 70):
        big = torch.full((M + 2, 100), 9.0, device=DEV)
        ops.linear_mx4(x[:M].to(DEV), wq, out=big[1:M + 1, 3:93])
        assert torch.equal(big[1:M + 1, 3:93], ops.linear_mx4(x[:M].to(DEV), wq))
        assert (big[0] == 9).all() and (big[-1] == 9).all() and (big[:, :3] == 9).all() and (big[:, 93:] == 9).all()


def test_no_rows():
    w = ops.mx4_pack(torch.randn(8, 40, device=DEV))
    x = torch.empty(0, 40, device=DEV)
    assert ops.mx4_pack(x).codes.shape == (0, 64) and ops.mx4_unpack(ops.mx4_pack(x)).shape == (0, 40)
    assert ops.linear_mx4(x, w).shape == (0, 8)
    assert ops.linear_mx4(x, w, out=ops.mx4_empty(0, 8, DEV)).rows == 0


def test_another_stream_and_a_captured_graph_that_is_replayed():
    x, w, bias, _, _ = product_case(40, 512, 256, 21)
    xd, wq, b = x.to(DEV), ops.mx4_pack(w.to(DEV)), bias.to(DEV)
    want = ops.linear_mx4(xd, wq, b, act="relu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.linear_mx4(xd, wq, b, act="relu")
    side.synchronize()
    assert torch.equal(got, want)
    graphs, outs, ins = [], [], []
    for k in range(2):                                           # two graphs that live together
        xin = xd.clone()
        ops.linear_mx4(xin, wq, b, act="relu")
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            h = ops.linear_mx4(xin, wq, b, act="relu", out=ops.mx4_empty(40, 256, DEV))
            outs.append(ops.mx4_unpack(h))
        graphs.append(g)
        ins.append(xin)
    for rep in range(3):
        for k in (0, 1):
            ins[k].copy_(xd * (1 + rep + 2 * k))
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for k in (0, 1):
            assert torch.equal(outs[k], ops.mx4_unpack(ops.mx4_pack(ops.linear_mx4(ins[k], wq, b, act="relu"))))


def test_refusals():
    x, w = torch.randn(4, 40, device=DEV), ops.mx4_pack(torch.randn(8, 40, device=DEV))
    bad = [lambda: ops.linear_mx4(torch.randn(4, 41, device=DEV), w), lambda: ops.linear_mx4(x, torch.randn(8, 40, device=DEV)),
           lambda: ops.linear_mx4(x, w, act="gelu"), lambda: ops.linear_mx4(x, w, bias=torch.zeros(9, device=DEV)),
           lambda: ops.linear_mx4(x, w, bias=torch.zeros(8, device=DEV, dtype=torch.float64)),
           lambda: ops.linear_mx4(x.double(), w), lambda: ops.linear_mx4(x, w, out_dtype=torch.float64),
           lambda: ops.linear_mx4(x.cpu(), w), lambda: ops.linear_mx4(x, w, out=torch.empty(4, 9, device=DEV)),
           lambda: ops.linear_mx4(x, w, out=ops.mx4_empty(5, 8, DEV)), lambda: ops.linear_mx4(x[0], w),
           lambda: ops.linear_mx4(torch.randn(40, 4, device=DEV).t(), w), lambda: ops.linear_mx4(x.clone().requires_grad_(), w),
           lambda: ops.mx4_pack(x.expand(4, 40)[:1].expand(4, 40)), lambda: ops.mx4_pack(x, out=ops.mx4_empty(4, 41, DEV)),
           lambda: ops.mx4_unpack(w, dtype=torch.int32), lambda: ops.mx4_unpack(w, out=torch.empty(8, 41, device=DEV)),
           lambda: ops.Mx4Tensor(w.codes, w.scales, 300), lambda: ops.Mx4Tensor(w.codes.int(), w.scales, 40),
           lambda: ops.Mx4Tensor(w.codes, w.scales, 0),
           lambda: ops.Mx4Tensor(torch.zeros(8 * 64 + 1, device=DEV, dtype=torch.uint8)[1:].view(8, 64), w.scales, 40)]
    for f in bad:
        with pytest.raises(ClavaHipError):
            f()
    with torch.no_grad():
        ops.linear_mx4(x.clone().requires_grad_(), w)


@pytest.mark.parametrize("M, N", [(2050, 2100), (5000, 6700)])            # tiles of 128 x 128, of 256 x 256
@pytest.mark.parametrize("K", [40, 300, 512, 1030])                       # one step of 128 columns, an odd number, whole groups of four, nine
def test_large_products(M, N, K):
    x, w, bias, want, mag = product_case(M, K, N, K)
    xq, wq, b = ops.mx4_pack(x.to(DEV)), ops.mx4_pack(w.to(DEV)), bias.to(DEV)
    y = ops.linear_mx4(x.to(DEV), wq, b, act="relu")
    ref = np.maximum(want + bias.double().numpy(), 0)
    assert (np.abs(y.cpu().double().numpy() - ref) <= tolerance(M, K, N, mag + np.abs(bias.numpy()), ref, torch.float32)).all()
    assert torch.equal(y, ops.linear_mx4(xq, wq, b, act="relu"))
    assert torch.equal(y.bfloat16(), ops.linear_mx4(xq, wq, b, act="relu", out_dtype=torch.bfloat16))
    out, again = ops.linear_mx4(xq, wq, b, act="relu", out=ops.mx4_empty(M, N, DEV)), ops.mx4_pack(y)
    assert torch.equal(out.codes, again.codes) and torch.equal(out.scales, again.scales)
    big = torch.full((M + 1, N + 9), 9.0, device=DEV)
    ops.linear_mx4(xq, wq, b, act="relu", out=big[:M, 5:5 + N])
    assert torch.equal(big[:M, 5:5 + N], y) and (big[M] == 9).all() and (big[:, :5] == 9).all() and (big[:, 5 + N:] == 9).all()


@pytest.mark.parametrize("M", [1, 16, 17, 64, 65])
@pytest.mark.parametrize("K", [2047, 2048, 2049])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_and_columns_at_which_the_way_changes(M, K, dtype):
    x, w, _, want, mag = product_case(M, K, 45, M + K, dtype)
    wq = ops.mx4_pack(w.to(DEV))
    wide = torch.randn(M, K + 5, device=DEV).to(dtype)
    wide[:, 3:3 + K] = x.to(DEV)
    y = ops.linear_mx4(wide[:, 3:3 + K], wq)
    assert (np.abs(y.cpu().double().numpy() - want) <= tolerance(M, K, 45, mag, want, torch.float32)).all()
    assert torch.equal(y, ops.linear_mx4(ops.mx4_pack(x.to(DEV)), wq))


def test_result_beside_its_operand_but_not_on_it():
    x, w = torch.randn(70, 128, device=DEV), ops.mx4_pack(torch.randn(128, 128, device=DEV))
    want = ops.linear_mx4(x, w)
    both = torch.cat([x, torch.zeros_like(x)], 1)
    ops.linear_mx4(both[:, :128], w, out=both[:, 128:])
    assert torch.equal(both[:, 128:], want)
    stack = torch.cat([x, torch.zeros_like(x)])
    ops.linear_mx4(stack[:70], w, out=stack[70:])
    assert torch.equal(stack[70:], want)
    q = ops.mx4_pack(x)
    for f in (lambda: ops.linear_mx4(x, w, out=x), lambda: ops.linear_mx4(both[:, :128], w, out=both[:, 127:255]), lambda: ops.linear_mx4(q, w, out=q),
              lambda: ops.linear_mx4(stack[:70], w, out=stack[69:139]), lambda: ops.linear_mx4(x[:1], w, out=x[:1]),
              lambda: ops.mx4_pack(x.clone().requires_grad_())):
        with pytest.raises(ClavaHipError):
            f()


def test_offsets_that_pass_32_bits():
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    x, w = torch.randn(66, 200, device=DEV), ops.mx4_pack(torch.randn(72, 200, device=DEV))
    step = (1 << 32) // 60 // 128 * 128                                   # rows end past 2^32 elements
    far = torch.empty(66 * step, device=DEV, dtype=torch.bfloat16)
    for M in (2, 66):
        s = step if M == 66 else 60 * step
        xs = far.as_strided((M, 200), (s, 1))
        xs.copy_(x[:M])
        near = x[:M].bfloat16()
        assert torch.equal(ops.mx4_pack(xs).codes, ops.mx4_pack(near).codes)
        want = ops.linear_mx4(near, w, out_dtype=torch.bfloat16)
        assert torch.equal(ops.linear_mx4(xs, w, out_dtype=torch.bfloat16), want)
        ys = far.as_strided((M, 72), (s, 1), 300)
        assert torch.equal(ops.linear_mx4(near, w, out=ys), want)
        ops.mx4_unpack(ops.mx4_pack(want), out=ys)
        assert torch.equal(ys, ops.mx4_unpack(ops.mx4_pack(want), dtype=torch.bfloat16))
    del far, xs, ys
    # more than 2^31 groups of eight columns: several launches
    rows = (1 << 31) // 16 + 5
    q = ops.mx4_empty(rows, 128, DEV)
    tail = torch.randn(9, 128, device=DEV)
    flat = torch.zeros(rows, 128, device=DEV, dtype=torch.bfloat16)
    flat[-9:] = tail
    ops.mx4_pack(flat, out=q)
    ref = ops.mx4_pack(tail.bfloat16())
    assert torch.equal(q.codes[-9:], ref.codes) and torch.equal(q.scales[-9:], ref.scales) and (q.codes[-20:-9] == 0).all()
    ops.mx4_unpack(q, out=flat)
    assert torch.equal(flat[-9:], ops.mx4_unpack(ref, dtype=torch.bfloat16)) and (flat[-20:-9] == 0).all()


def test_two_streams_at_once():
    x, y, w = torch.randn(3000, 700, device=DEV), torch.randn(9, 3001, device=DEV), ops.mx4_pack(torch.randn(1000, 700, device=DEV))
    v = ops.mx4_pack(torch.randn(77, 3001, device=DEV))
    want = ops.linear_mx4(x, w), ops.linear_mx4(y, v)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(5):
        with torch.cuda.stream(a):
            got.append((0, ops.linear_mx4(x, w)))
        with torch.cuda.stream(b):
            got.append((1, ops.linear_mx4(y, v)))
    torch.cuda.synchronize()
    for k, t in got:
        assert torch.equal(t, want[k])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows, cols", [(1, 5), (1, 600), (2, 9), (3, 127), (37, 129), (300, 513), (64, 1999)])
def test_rows_at_every_place_of_16_bytes(rows, cols, dtype):
    """Rows that start anywhere in 16 bytes, of a tensor of their own (nothing before or behind) and inside a wider one."""
    x = rand(rows, cols, cols).to(DEV)
    ref = ops.mx4_pack(x.to(dtype).float())
    for start in range(9):
        for gap in (0, 1, 3, 8):
            flat = torch.full((start + rows * (cols + gap) + 16,), math.nan, device=DEV, dtype=dtype)
            view = flat[start:].as_strided((rows, cols), (cols + gap, 1), flat.storage_offset() + start)
            view.copy_(x)
            q = ops.mx4_pack(view)
            assert torch.equal(q.codes, ref.codes) and torch.equal(q.scales, ref.scales), (start, gap)
    own = x.to(dtype)
    q = ops.mx4_pack(own)
    assert torch.equal(q.codes, ref.codes) and torch.equal(q.scales, ref.scales)
