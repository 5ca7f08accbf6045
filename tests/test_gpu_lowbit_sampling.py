"""The 4-bit layers and the filtered draw as the sampler uses them: a denoiser's stack, single steps and whole chains."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from clavaddpm_amd import mx4_nets, ops, split_nets
from clavaddpm_amd.pipeline_utils import Classifier, make_cond_fn
from clavaddpm_amd.tab_ddpm import CategoryChoice, GaussianMultinomialDiffusion, MLPDiffusion
from clavaddpm_amd.tab_ddpm.modules import run_stack
from test_gpu_choice import choose, uniforms

DEV = "cuda"


@pytest.fixture
def mx4():
    before = split_nets.get_gemm_mode()
    split_nets.set_gemm_mode("mx4")
    yield
    split_nets.set_gemm_mode(before)


def model(K=(3, 40, 7), n_num=4, layers=(96, 160, 160, 96), T=20, seed=0):
    torch.manual_seed(seed)
    net = MLPDiffusion(n_num + sum(K), 0, "none", {"d_layers": list(layers), "dropout": 0.0}).to(DEV).eval()
    return net, GaussianMultinomialDiffusion(np.array(K), n_num, net, num_timesteps=T, device=torch.device(DEV)).to(DEV).eval()


@pytest.mark.parametrize("rows", [1, 13, 70, 300])
def test_every_hidden_layer_of_a_stack_against_64_bits(rows):
    """Each layer from the operand it was given: exact products in 64 bits, and what the 4-bit result may be off by: half a step
    of its grid (steps of 1/2 below 2, 1 below 4, 2 below 6, and what lies beyond 6), all times the block's scale, and the
    float32 accumulation (128 steps of 2^-23 of the magnitude sum, K <= 160: two instructions, 8 partial sums)."""
    net, _ = model()
    ws, bs, acts = net.stack()
    stack = mx4_nets.Mx4Stack(ws, bs, acts)
    x = torch.randn(rows, ws[0].shape[1], device=DEV)
    emb = torch.randn(128, device=DEV)
    with torch.no_grad():
        h = ops.mx4_pack(ops.linear(x, stack.first, stack.biases[0], rowadd=emb))
        for l, w in enumerate(stack.hidden, start=1):
            q = ops.mx4_empty(rows, w.rows, DEV)
            ops.linear_mx4(h, w, stack.biases[l], act="relu", out=q)
            xv, wv = ops.mx4_unpack(h).double().cpu(), ops.mx4_unpack(w).double().cpu()
            y = torch.relu(xv @ wv.t() + stack.biases[l].detach().double().cpu())
            mag = xv.abs() @ wv.abs().t() + stack.biases[l].detach().double().cpu().abs()
            got = ops.mx4_unpack(q).double().cpu()
            scale = torch.ldexp(torch.ones(()).double(), q.scales.cpu().int() - 127).repeat_interleave(32, 1)[:, :w.rows]
            size = y / scale
            step = torch.where(size < 2, 0.25, torch.where(size < 4, 0.5, torch.where(size < 6, 1.0, size - 6 + 1e-9)))
            assert ((got - y).abs() <= step * scale + 128 * 2.0 ** -23 * mag).all(), l
            # no block is scaled larger than its maximum asks for, nor smaller than saturation at 8 allows
            assert (size < 8 + 1e-3).all()
            h = q


def test_a_stack_is_its_layers_and_near_the_float_network():
    net, _ = model()
    ws, bs, acts = net.stack()
    stack = mx4_nets.Mx4Stack(ws, bs, acts)
    x, emb = torch.randn(200, ws[0].shape[1], device=DEV), torch.randn(128, device=DEV)
    with torch.no_grad():
        out = stack.forward(x, emb)
        h = ops.linear(x, ws[0], bs[0], rowadd=emb)
        for l in range(1, len(ws) - 1):
            h = ops.linear_mx4(h, ops.mx4_pack(ws[l]), bs[l].detach(), act="relu")      # float between the layers: packed again
        assert torch.equal(out, ops.linear(h, ws[-1], bs[-1]))
        assert torch.equal(out, stack.forward(x, emb, stack.buffers(200)))
        ref = run_stack(ws, bs, acts, x, rowadd0=emb)[-1]
        # a 4-bit rounding is off by at most a quarter of its value (1/2 a step of 1/2 at 1, of 2 at 4 .. 6), two of them a
        # product, over the hidden layers: well correlated with the float network, and nothing like it at random
        c = torch.corrcoef(torch.stack([out.flatten(), ref.flatten()]))[0, 1]
        assert c > 0.9
        assert stack.forward(x[:0], emb).shape == (0, ws[-1].shape[0])


@pytest.mark.parametrize("K, n_num", [((3, 40, 7), 4), ((0,), 5), ((300, 2), 0)])
def test_chain_on_4_bit_layers(mx4, K, n_num):
    _, d = model(K, n_num)
    x, out = d.sample(57, torch.ones(1), seed=3)
    assert x.shape == (57, n_num + sum(k > 0 for k in K)) and torch.isfinite(x).all() and len(out["y"]) == 57
    for f, k in enumerate(K if K[0] else ()):
        col = x[:, n_num + f]
        assert (col == col.round()).all() and col.min() >= 0 and col.max() < k
    # reproducible, independent of how rows are cut, and resumable
    assert torch.equal(x, d.sample(57, torch.ones(1), seed=3)[0])
    parts = torch.cat([d.sample(20, torch.ones(1), seed=3)[0], d.sample(37, torch.ones(1), seed=3, row_offset=20)[0]])
    assert torch.equal(x, parts)


def test_guided_chain_on_4_bit_layers(mx4):
    net, d = model((0,), 5)
    torch.manual_seed(1)
    clf = Classifier(d_in=5, d_out=6, dim_t=128, hidden_sizes=[32, 32]).to(DEV).eval()
    ys = torch.arange(40).remainder(6).reshape(-1, 1)
    a, _ = d.conditional_sample(ys, {"y": ys}, make_cond_fn(clf, 1.0), seed=4)
    assert torch.isfinite(a).all() and torch.equal(a, d.conditional_sample(ys, {"y": ys}, make_cond_fn(clf, 1.0), seed=4)[0])
    # One step.  A scale of 0 guides nowhere: it adds a zero, which only makes the first step's float32 arithmetic float64 (a
    # chain's first step is float32; over more steps that rounding moves values over 4-bit borders).  The guidance itself adds
    # variance * gradient, as the float64 step says.
    kw = dict(seed=4, n_steps=1)
    b, c = d.conditional_sample(ys, {"y": ys}, make_cond_fn(clf, 0.0), **kw)[0], d.conditional_sample(ys, **kw)[0]
    assert ((b - c).abs() <= 1e-5 * c.abs().max()).all()
    g = d.conditional_sample(ys, {"y": ys}, make_cond_fn(clf, 2.0), **kw)[0]
    x, _ = d._initial_state(40, None, 4, 0)
    t = torch.full((40,), d.num_timesteps - 1, device=DEV, dtype=torch.long)
    push = make_cond_fn(clf, 2.0)(x.float(), t, y=ys.to(DEV)).double().cpu() * d._model_variance[-1].double().cpu()
    assert ((g - b - push).abs() <= 1e-5 * c.abs().max()).all() and push.abs().max() > 0


def test_p_sample_index_with_a_choice():
    _, d = model((3, 40, 300), 0)
    B, m = 30, 3
    logits = 2 * torch.randn(B, 343, device=DEV)
    idx = torch.zeros(B, m, device=DEV, dtype=torch.int32)
    t = torch.randint(0, 20, (B,), device=DEV)
    u = uniforms(B, m, 3)
    got, lp = d.p_sample_index(logits, idx, t, u.to(DEV), return_log_prob=True, choice=CategoryChoice(temperature=[0.5, 1.0, 2.0], top_k=5, top_p=0.9))
    _, want_lp = d.p_sample_index(logits, idx, t, None, return_log_prob=True)
    assert torch.equal(lp, want_lp)
    z, at, temps = lp.double().cpu().numpy(), [0, 3, 43, 343], [0.5, 1.0, 2.0]
    for b in range(B):
        for f in range(m):
            i, _ = choose(z[b, at[f]:at[f + 1]], float(u[b, f]), temperature=temps[f], top_k=5, top_p=0.9, min_p=0.0)
            assert got[b, f] == i
    greedy, none = d.p_sample_index(logits, idx, t, choice=CategoryChoice(temperature=0.0))
    assert none is None
    for f in range(m):
        assert torch.equal(greedy[:, f].long(), lp[:, at[f]:at[f + 1]].argmax(1))


@pytest.mark.parametrize("mode", ["f16x3", "f32", "mx4"])
def test_sample_with_a_choice_ends_in_its_last_step(mode):
    before = split_nets.get_gemm_mode()
    split_nets.set_gemm_mode(mode)
    try:
        _, d = model((3, 40, 7), 4)
        m, T = 3, d.num_timesteps
        plain, _ = d.sample(33, torch.ones(1), seed=8)
        got, _ = d.sample(33, torch.ones(1), seed=8, choice=CategoryChoice(temperature=0.0))
        assert got.shape == plain.shape and torch.isfinite(got).all()
        # by hand: all steps but the last, then the posterior's most likely classes
        x, idx = d._initial_state(33, None, 8, 0)
        d._run_chain(x, idx, None, torch.zeros(33), None, 8, 0, T - 1, None)
        assert torch.equal(torch.cat([plain[:0], got])[:, 4:], _last(d, x, idx))
        # rows do not depend on how they are cut
        c = CategoryChoice(temperature=0.8, top_p=0.7, top_k=[2, 9, 0])
        whole, _ = d.sample(33, torch.ones(1), seed=8, choice=c)
        cut = torch.cat([d.sample(10, torch.ones(1), seed=8, choice=c)[0], d.sample(23, torch.ones(1), seed=8, row_offset=10, choice=c)[0]])
        if mode != "f16x3":                          # (its layers pick tiles by batch; the float columns may differ in the last bit)
            assert torch.equal(whole, cut)
        assert torch.equal(whole[:, 4:], cut[:, 4:])
        xs, ys = d.sample_all(50, 25, torch.ones(1), seed=2, choice=c)
        assert xs.shape == (50, 7) and torch.isfinite(xs).all()
        with pytest.raises(ValueError):
            d.sample(4, torch.ones(1), n_steps=3, choice=c)
        one, _ = d.sample(5, torch.ones(1), seed=1, t_start=0, choice=c, noise=None)
        assert one.shape == (5, 7)
    finally:
        split_nets.set_gemm_mode(before)


def _last(d, x, idx):
    net = d._denoise_fn
    with torch.no_grad():
        out = net(d._denoiser_input(x, idx), torch.zeros(x.shape[0], device=DEV, dtype=torch.long))
    t = torch.zeros(x.shape[0], device=DEV, dtype=torch.long)
    _, lp = d.p_sample_index(out[:, 4:], idx, t, None, return_log_prob=True)
    return torch.stack([lp[:, a:b].argmax(1) for a, b in ((0, 3), (3, 43), (43, 50))], 1).double().cpu()


def test_logits_that_are_no_numbers_end_as_nan_in_the_table():
    net, d = model((3, 5), 2, T=4)
    with torch.no_grad():
        net.mlp.head.weight[2:].fill_(float("nan"))
    before = split_nets.get_gemm_mode()
    split_nets.set_gemm_mode("f32")
    try:
        x, _ = d.sample(6, torch.ones(1), seed=1, t_start=0, choice=CategoryChoice(top_k=2))
    finally:
        split_nets.set_gemm_mode(before)
    assert x[:, 2:].isnan().all()


def test_a_4_bit_heads_logits_go_straight_into_the_draw():
    """The run of the operators as a server would make it, captured as one graph: packed rows, layers, logits, classes."""
    K = [5, 60, 900]
    net, d = model(tuple(K), 2, layers=(128, 256, 128))
    ws, bs, acts = net.stack()
    layers = [ops.mx4_pack(w.detach()) for w in ws]
    off = d._offsets_i32
    x = torch.randn(50, ws[0].shape[1], device=DEV)
    u = uniforms(50, 3, 9).to(DEV)

    def run(x):
        h = x
        for w, b in zip(layers[:-1], bs[:-1]):
            h = ops.linear_mx4(h, w, b.detach(), act="relu", out=ops.mx4_empty(x.shape[0], w.rows, DEV))
        logits = ops.linear_mx4(h, layers[-1], bs[-1].detach(), out_dtype=torch.bfloat16)[:, 2:]
        return ops.sample_categories(logits, u, off, max(K), temperature=0.7, top_k=20, top_p=0.95, log_prob=True), logits

    (idx, lp), logits = run(x)
    z, at = logits.double().cpu().numpy(), np.concatenate([[0], np.cumsum(K)])
    for b in range(50):
        for f in range(3):
            i, p = choose(z[b, at[f]:at[f + 1]], float(u[b, f]), temperature=0.7, top_k=20, top_p=0.95, min_p=0.0)
            assert idx[b, f] == i and abs(float(lp[b, f]) - p) <= abs(p) * 2.0 ** -24 + 1e-12
    xin = x.clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, _ = run(xin)
    for rep in range(3):
        xin.copy_(x * (rep + 1))
        g.replay()
        torch.cuda.synchronize()
        (i, p), _ = run(xin)
        assert torch.equal(out[0], i) and torch.equal(out[1], p)
