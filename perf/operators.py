"""The low-bit layers and the filtered categorical draw, as cases: their plain form in elementary torch operations, the calls
that a user makes of the kernels, and what each case cannot do without.

A microscaled 4-bit matrix (OCP MX, E2M1 elements) holds blocks of 32 columns: `codes` uint8 [rows, Kp / 2], element 2 i in
the low four bits of byte i, and `scales` uint8 [rows, Kp / 32], a power of two with bias 127; Kp = the columns rounded up to
128, with zero codes behind the last column.
"""
import math

import numpy as np
import torch

own = False

_DTYPE = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
_GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


# ---------------------------------------------------------------------------------------------------------------- cases
def _quant(name, rows, cols, dtype):
    return {"name": name, "op": "quantise", "rows": rows, "cols": cols, "dtype": dtype}


def _product(name, m, k, n, dtype, out, act, bias):
    return {"name": name, "op": "product", "m": m, "k": k, "n": n, "dtype": dtype, "out": out, "act": act, "bias": bias}


def _draw(name, rows, features, k_low, k_high, dtype, temperature, top_k, top_p, min_p, masked):
    return {"name": name, "op": "sample", "rows": rows, "features": features, "k_low": k_low, "k_high": k_high, "dtype": dtype,
            "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p, "masked": masked}


def listed():
    return [
        # a training batch's hidden activations, written as 4 bits and read back
        _quant("quantise 4096x1024", 4096, 1024, "float32"),
        # a sampling batch of 16-bit activations whose width ends inside a block
        _quant("quantise 20000x1999 bf16", 20000, 1999, "bfloat16"),
        # one record through one hidden layer: latency
        _product("product 1x1024x1024", 1, 1024, 1024, "float32", "float32", "relu", True),
        # a few records through a wide layer, odd sizes: the weights' bytes count
        _product("product 7x4099x8001 bf16", 7, 4099, 8001, "bfloat16", "bfloat16", "silu", True),
        # a hidden layer at the training batch
        _product("product 4096x1024x1024", 4096, 1024, 1024, "float32", "float32", "relu", True),
        # the last hidden layer of a sampling batch
        _product("product 20000x1024x512", 20000, 1024, 512, "bfloat16", "bfloat16", "relu", True),
        # a large square layer: the matrix cores count
        _product("product 16384x8192x8192", 16384, 8192, 8192, "bfloat16", "bfloat16", "none", False),
        # one record with fifty small columns: latency
        _draw("sample 1x50", 1, 50, 2, 64, "float32", 0.8, 0, 0.9, 0.0, False),
        # the sampling step of a wide table, temperature alone
        _draw("sample 4096x50", 4096, 50, 2, 1000, "float32", 0.7, 0, 1.0, 0.0, False),
        # a large sampling batch of it with every filter, some classes forbidden
        _draw("sample 20000x50 filtered", 20000, 50, 2, 1000, "float32", 0.9, 40, 0.9, 0.01, True),
        # a column with very many classes, 16-bit logits, nucleus
        _draw("sample 64x131071 bf16", 64, 1, 131071, 131071, "bfloat16", 0.8, 0, 0.95, 0.0, False),
        # one record of a column with very many classes
        _draw("sample 1x262144", 1, 1, 262144, 262144, "float32", 1.0, 50, 1.0, 0.02, False),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["quantise", "product", "product", "sample", "sample"])
    if op == "quantise":
        rows = _log_int(rng, 1, 32768)
        cols = _log_int(rng, 1, min(16384, max(8, (1 << 25) // rows)))
        c = _quant("", rows, cols, rng.choice(list(_DTYPE)))
    elif op == "product":
        m, k = _log_int(rng, 1, 16384), _log_int(rng, 32, 8192)
        c = _product("", m, k, _log_int(rng, 16, 8192), rng.choice(list(_DTYPE)), rng.choice(["float32", "bfloat16"]),
                     rng.choice(["none", "relu", "leaky_relu", "silu"]), rng.choice([True, False]))
    else:
        if rng.random() < 0.5:
            features, low, high = _log_int(rng, 1, 50), 2, _log_int(rng, 8, 1000)
            rows = _log_int(rng, 1, 20000)
        else:
            low = high = _log_int(rng, 1000, 262144)
            features = 1
            rows = _log_int(rng, 1, max(2, (1 << 23) // high))
        c = _draw("", rows, features, low, high, rng.choice(["float32", "bfloat16"]), round(rng.uniform(0.3, 1.5), 3),
                  rng.choice([0, 0, _log_int(rng, 1, 200)]), rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                  rng.choice([0.0, round(rng.uniform(0.001, 0.1), 4)]), rng.choice([False, True]))
    del c["name"]
    return c


def _classes(case):
    """Classes of every feature: log-uniform between the case's bounds, the same list every time."""
    r = np.random.RandomState(case["features"])
    u = r.uniform(math.log(case["k_low"]), math.log(case["k_high"]), case["features"])
    return [int(min(case["k_high"], max(case["k_low"], round(math.exp(v))))) for v in u]


# --------------------------------------------------------------------------------------------------------------- inputs
def _activations(g, rows, cols, dtype):
    """Hidden activations: half of them zero (ReLU), a few columns far larger than the rest."""
    x = torch.randn((rows, cols), generator=g, device="cuda")
    gain = torch.exp(0.7 * torch.randn((1, cols), generator=g, device="cuda"))
    return torch.relu(x * gain).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = _DTYPE[case["dtype"]]
    if case["op"] == "quantise":
        return {"op": "quantise", "x": _activations(g, case["rows"], case["cols"], dtype)}
    if case["op"] == "product":
        w = torch.randn((case["n"], case["k"]), generator=g, device="cuda") / math.sqrt(case["k"])
        codes, scales = _plain_codes(w)
        bias = 0.1 * torch.randn(case["n"], generator=g, device="cuda") if case["bias"] else None
        return {"op": "product", "x": _activations(g, case["m"], case["k"], dtype), "codes": codes, "scales": scales, "cols": case["k"],
                "bias": bias, "act": case["act"], "out": _DTYPE[case["out"]]}
    classes = _classes(case)
    offsets = torch.tensor([0] + list(np.cumsum(classes)), device="cuda", dtype=torch.int32)
    z = 3.0 * torch.randn((case["rows"], sum(classes)), generator=g, device="cuda")
    if case["masked"]:     # forbidden classes: about one in twenty
        z = z.masked_fill(torch.rand(z.shape, generator=g, device="cuda") < 0.05, -math.inf)
        z[:, offsets[:-1].long()] = 0.5
    u = torch.rand((case["rows"], len(classes)), generator=g, device="cuda")
    feature = torch.repeat_interleave(torch.arange(len(classes), device="cuda"), torch.tensor(classes, device="cuda"))
    return {"op": "sample", "logits": z.to(dtype), "u": u, "offsets": offsets, "feature": feature, "widest": max(classes),
            **{k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")}}


# ----------------------------------------------------------------------------------------------------------- plain form
def _blocks(x):
    """float32 [rows, Kp / 32, 32] with zeros behind the last column (Kp: a multiple of 128)."""
    rows, cols = x.shape
    padded = -(-cols // 128) * 128
    out = torch.zeros((rows, padded), device=x.device, dtype=torch.float32)
    out[:, :cols] = x
    return out.view(rows, padded // 32, 32)


def _plain_quantise(x):
    """(elements on the E2M1 grid, exponent of the scale): both of [rows, Kp / 32, ...]."""
    b = _blocks(x)
    top = b.abs().amax(dim=2)
    e = torch.where(top > 0, torch.frexp(top).exponent - 3, -127).clamp(-127, 127)
    v = torch.ldexp(b, -e[:, :, None])
    size = v.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    return torch.clamp(torch.round(size / step) * step, max=6.0) * torch.sign(v), e


def _plain_codes(x):
    q, e = _plain_quantise(x)
    size = q.abs()
    code = torch.where(size < 2, 2 * size, torch.where(size < 4, size + 2, size / 2 + 4)).to(torch.uint8)
    code = (code + 8 * (q < 0).to(torch.uint8)).view(x.shape[0], -1)
    return code[:, 0::2] + 16 * code[:, 1::2], (e + 127).to(torch.uint8)


def _plain_values(codes, scales):
    grid = torch.tensor(_GRID + [-v for v in _GRID], device=codes.device)
    q = torch.stack([codes & 15, codes >> 4], dim=2).long()
    q = grid[q].view(codes.shape[0], -1, 32)
    return torch.ldexp(q, scales.int()[:, :, None] - 127).view(codes.shape[0], -1)


def _plain_product(s):
    q, e = _plain_quantise(s["x"].float())
    x = torch.ldexp(q, e[:, :, None]).view(s["x"].shape[0], -1)
    y = torch.mm(x, _plain_values(s["codes"], s["scales"]).t())
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["act"] == "relu":
        y = torch.clamp(y, min=0)
    elif s["act"] == "leaky_relu":
        y = torch.where(y > 0, y, 0.01 * y)
    elif s["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    return y.to(s["out"])


def _plain_sample(s):
    """In 64 bits: a draw next to a border has to fall on the right side. Blocks stay side by side, as they come."""
    z, u, f = s["logits"].double(), s["u"].double(), s["feature"]
    off = s["offsets"].long()
    first, last = off[:-1], off[1:] - 1
    # the blocks' elements in falling order, equal ones by their index
    order = torch.argsort(z, dim=1, descending=True, stable=True)
    order = order.gather(1, torch.argsort(f[order], dim=1, stable=True))
    rank = torch.arange(z.shape[1], device=z.device) - first[f]
    top = z.gather(1, order[:, first])
    a = torch.exp((z - top[:, f]) / s["temperature"])
    falling = a.gather(1, order)
    keep = falling >= s["min_p"]
    if s["top_k"] > 0:
        keep = keep & (rank < s["top_k"])
        falling = falling * (rank < s["top_k"])
    if s["top_p"] < 1:
        run = torch.cumsum(falling, dim=1)
        base = run[:, first] - falling[:, first]
        keep = keep & (run - falling - base[:, f] < s["top_p"] * (run[:, last] - base)[:, f])
    kept = torch.zeros_like(a).scatter(1, order, keep.to(a.dtype)) * a
    run = torch.cumsum(kept, dim=1)
    base = run[:, first] - kept[:, first]
    mass = run[:, last] - base
    goal = torch.minimum(u * mass, mass * (1 - 2.0 ** -50))
    count = torch.cumsum(run - base[:, f] <= goal[:, f], dim=1)
    index = count[:, last] - count[:, first] + (kept[:, first] <= goal)
    return {"index": index.int(), "log_prob": torch.log(kept.gather(1, index + first) / mass).float()}


def run(state):
    if own:
        from clavaddpm_amd import ops
        if state["op"] == "quantise":
            return ops.mx4_unpack(ops.mx4_pack(state["x"]), dtype=state["x"].dtype)
        if state["op"] == "product":
            w = ops.Mx4Tensor(state["codes"], state["scales"], state["cols"])
            return ops.linear_mx4(state["x"], w, state["bias"], act=state["act"], out_dtype=state["out"])
        index, log_prob = ops.sample_categories(state["logits"], state["u"], state["offsets"], state["widest"], temperature=state["temperature"],
                                                top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"], log_prob=True)
        return {"index": index, "log_prob": log_prob}
    if state["op"] == "quantise":
        x = state["x"]
        q, e = _plain_quantise(x.float())
        return torch.ldexp(q, e[:, :, None]).view(x.shape[0], -1)[:, :x.shape[1]].to(x.dtype)
    if state["op"] == "product":
        return _plain_product(state)
    return _plain_sample(state)


# ------------------------------------------------------------------------------------------------------- work and truth
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "quantise":      # x read, the codes and scales written, their values written
        n = case["rows"] * case["cols"]
        return {"bytes": n * (2 * size + 17 / 32), "flops": 3 * n}
    if case["op"] == "product":
        m, k, n = case["m"], case["k"], case["n"]
        y = 4 if case["out"] == "float32" else 2
        return {"bytes": m * k * size + n * k * 17 / 32 + m * n * y + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    n, draws = case["rows"] * sum(_classes(case)), case["rows"] * case["features"]
    return {"bytes": n * size + draws * 12, "flops": 4 * n}


def _exact_values(x):
    """Nearest E2M1 value of every element over its block's scale, in 64 bits: by the borders between neighbours."""
    rows, cols = x.shape
    b = torch.nn.functional.pad(x.double(), (0, -cols % 32)).view(rows, -1, 32)
    top = b.abs().amax(dim=2, keepdim=True)
    scale = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.where(top > 0, top, 1.0))) - 2, -127, 127))
    scale = torch.where(scale * 8 <= top, scale * 2, torch.where(scale * 4 > top, scale / 2, scale)) if bool((top > 0).any()) else scale
    v = (b / scale).abs()
    at = ((v > 0.25).long() + (v >= 0.75) + (v > 1.25) + (v >= 1.75) + (v > 2.5) + (v >= 3.5) + (v > 5))
    q = torch.tensor(_GRID, device=x.device, dtype=torch.float64)[at] * scale
    return torch.where(b < 0, -q, q).view(rows, -1)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantise":
        return _exact_values(s["x"])
    if case["op"] == "product":
        codes = s["codes"].cpu().numpy()
        q = np.stack([codes & 15, codes >> 4], axis=2).reshape(case["n"], -1)[:, :case["k"]]
        power = np.repeat(s["scales"].cpu().numpy().astype(np.int64) - 127, 32, axis=1)[:, :case["k"]]
        size = np.array(_GRID)[q & 7]
        w = torch.from_numpy(np.ldexp(np.where(q > 7, -size, size), power)).cuda()
        y = _exact_values(s["x"]) @ w.t()
        if s["bias"] is not None:
            y += s["bias"].double()
        return {"none": lambda v: v, "relu": lambda v: v.clamp(min=0), "leaky_relu": lambda v: torch.maximum(v, 0.01 * v),
                "silu": lambda v: v * torch.sigmoid(v)}[case["act"]](y)
    index, log_prob, at = [], [], 0
    for j, k in enumerate(_classes(case)):
        logits = s["logits"][:, at:at + k].double() / case["temperature"]
        at += k
        falling, order = torch.sort(logits, dim=1, descending=True, stable=True)
        if case["top_k"] > 0:
            falling[:, case["top_k"]:] = -math.inf
        p = torch.softmax(falling, dim=1)
        drop = p < case["min_p"] * p[:, :1]
        if case["top_k"] > 0:
            drop[:, case["top_k"]:] = True
        if case["top_p"] < 1:
            drop |= p.cumsum(1) - p >= case["top_p"]
        p = torch.softmax(torch.zeros_like(p).scatter(1, order, falling.masked_fill(drop, -math.inf)), dim=1)
        i = torch.searchsorted(p.cumsum(1), s["u"][:, j:j + 1].double().contiguous(), right=True).clamp(max=k - 1)
        index.append(i.int())
        log_prob.append(torch.log(p.gather(1, i)))
    return {"index": torch.cat(index, 1), "log_prob": torch.cat(log_prob, 1)}
