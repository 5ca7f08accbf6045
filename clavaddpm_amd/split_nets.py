"""Host-side preparation of Linear stacks for the split-f16 matrix-core path (csrc/split.h, clava_gemm_f16x3).

A stack (MLPDiffusion's proj+mlp, `tab_ddpm/modules.py:425-460`, or the eval-mode Classifier,
`pipeline_utils.py:584-630`) is prepared once per set of weights:
  * eval-mode BatchNorm below a layer is folded into that layer's weight and bias (W' = W diag(s), b' = b + W c);
  * weights are packed as split rows (hi/lo float16 planes), plus their transposes for the input-gradient chain;
  * the power-of-two scale of every activation / gradient plane is calibrated with a float32 pass of the same
    network (the float32 MFMA kernels) on a fixed synthetic batch, so that magnitudes sit near 2^6: a factor 1000 below
    the float16 limit.
The calibration batch depends only on the weights, never on the rows being sampled: a table sampled on 1 or 8 GPUs
is bit-identical.  If any intermediate still leaves the float16 range the kernels raise an overflow flag and the
caller reruns the chain on the float32 kernels (`GaussianMultinomialDiffusion._run_chain`).

`set_gemm_mode("f32")` (or CLAVA_GEMM=f32) selects the float32-input MFMA kernels for the sampling loop instead,
`set_gemm_mode("mx4")` microscaled 4-bit operands in the denoiser's hidden blocks (mx4_nets.py: a draft, not float32 accuracy;
training runs as under "f16x3").
"""
import ctypes
import math
import os

import torch

from . import _lib, _native, ops
from ._lib import ACT_LEAKY, ACT_NONE

_MODES = ("f16x3", "f32", "mx4")
_mode = os.environ.get("CLAVA_GEMM", "f16x3")
if _mode not in _MODES:
    raise _lib.ClavaHipError(f"CLAVA_GEMM={_mode!r}: expected one of {_MODES}")

# Calibrated activation / gradient magnitudes are scaled into (2^5, 2^6]: a factor 1000 below the float16 limit.  The low
# plane of the smaller elements then sits in the float16 subnormals, which costs nothing measurable: their absolute
# error stays 2^-31 of the largest element (tools/dbg_f16x3_range.py: the product's rms error moves from 3.6e-7 to
# 3.7e-7 between a 2^14 and a 2^6 target on heavy-tailed ReLU data; the float32 MFMA kernel is at the same level).
TARGET_LOG2 = 6
IN_TARGET_LOG2 = 5        # the chain state may grow more than hidden activations do
DLAST_LOG2 = 10           # |onehot - softmax| <= 1 always
W_TARGET_LOG2 = 12        # weights into (2^11, 2^12]
CAL_ROWS = 1024
fallback_count = 0        # chains that left the float16 range and were rerun on the float32 kernels (this process)


def set_gemm_mode(mode):
    """'f16x3' (default): split-f16 layers on the f16 matrix cores; 'f32': the float32-input MFMA kernels; 'mx4': the denoiser's
    hidden blocks on microscaled 4-bit operands (sampling only)."""
    global _mode
    if mode not in _MODES:
        raise ValueError(f"gemm mode must be one of {_MODES}")
    _mode = mode


def get_gemm_mode():
    return _mode


class CSplitNet(ctypes.Structure):
    _fields_ = [("n_layers", ctypes.c_int),
                ("dims", _native.c_int_p),
                ("w", ctypes.POINTER(ctypes.c_void_p)),
                ("wt", ctypes.POINTER(ctypes.c_void_p)),
                ("b", ctypes.POINTER(ctypes.c_void_p)),
                ("act", _native.c_int_p),
                ("shift_w", _native.c_int_p),
                ("shift_in", ctypes.c_int),
                ("shift_out", _native.c_int_p),
                ("shift_grad", _native.c_int_p),
                ("shift_dlast", ctypes.c_int),
                ("fs_front", ctypes.c_void_p),
                ("fs_tail", ctypes.c_void_p),
                ("fs_back", ctypes.c_void_p),
                ("fs_head", ctypes.c_void_p),
                ("bf", ctypes.POINTER(ctypes.c_void_p)),
                ("num_wt", ctypes.c_void_p),
                ("cat_wt", ctypes.c_void_p),
                ("cat_bias", ctypes.c_void_p),
                ("log_tiny", ctypes.c_float)]


def shift_for(maxabs, target=TARGET_LOG2):
    """Power-of-two exponent s with maxabs * 2^s in (2^(target-1), 2^target]."""
    if not (maxabs > 0.0) or not math.isfinite(maxabs):
        return 0
    return int(min(24, max(-24, target - math.ceil(math.log2(maxabs)))))


def fold_batchnorm(ws, bs, sc, sh):
    """Fold the eval BatchNorm applied to layer l-1's activated output into layer l: returns float32 (ws', bs')."""
    fw, fb = [], []
    for l, (w, b) in enumerate(zip(ws, bs)):
        w, b = w.detach().float().contiguous(), b.detach().float().contiguous()
        if l > 0 and sc is not None and sc[l - 1] is not None:
            b = ops.linear(sh[l - 1].reshape(1, -1).contiguous(), w, b)[0].contiguous()
            w = (w * sc[l - 1].reshape(1, -1)).contiguous()
        fw.append(w)
        fb.append(b)
    return fw, fb


_FUSED_IDX = {}
FUSED_CHUNK = 32768       # bytes per LDS ring chunk of the fused kernels (csrc/fused_narrow.hip: RING_CHUNK)


def pack_fused(w, shift, n_pad=None, k_pad=None, group=4):
    """float32 [N, K] -> the fragments of one layer for the fused narrow-stack kernels (csrc/fused_narrow.hip), a uint8 device
    tensor: v_mfma_f32_32x32x16_f16 fragments [group of <= `group` row tiles][k-step][row tile][plane hi/lo][lane 64][8
    halves] of the planes hi = f16(w 2^shift), lo = f16(w 2^shift - hi); lane (r = lane & 31, h = lane >> 5) holds row
    32 t + r, and its element j of step s is column 16 s + 8 (j >> 2) + 4 h + (j & 3): the order in which an accumulator
    tile of the previous layer is laid out, so that layers chain in registers.  Rows / columns are zero padded to n_pad /
    k_pad (default: multiples of 32 / 16)."""
    N, K = w.shape
    Np = n_pad if n_pad is not None else (N + 31) // 32 * 32
    Kp = k_pad if k_pad is not None else (K + 15) // 16 * 16
    nt, ks = Np // 32, Kp // 16
    if Np % 32 or Kp % 16 or Np < N or Kp < K or (nt > group and nt % group):
        raise _lib.ClavaHipError(f"pack_fused: padded shape [{Np}, {Kp}] does not hold [{N}, {K}] in groups of {group} tiles")
    dev = w.device
    wp = torch.zeros((Np, Kp), device=dev, dtype=torch.float32)
    wp[:N, :K] = w.detach().float() * (2.0 ** shift)
    if not bool((wp.abs() <= 65504.0).all()):
        raise _lib.ClavaHipError("pack_fused: a scaled weight leaves the float16 range")
    hi = wp.half()
    lo = (wp - hi.float()).half()
    g = min(group, nt)
    key = (Np, Kp, g, str(dev))
    idx = _FUSED_IDX.get(key)
    if idx is None:
        lane = torch.arange(64, device=dev)
        r, h = lane & 31, lane >> 5
        j = torch.arange(8, device=dev)
        koff = 8 * (j >> 2) + (j & 3)
        grp = torch.arange(nt // g, device=dev)
        tig = torch.arange(g, device=dev)
        s_ = torch.arange(ks, device=dev)
        shape = (nt // g, ks, g, 64, 8)
        rows = (32 * (g * grp[:, None, None, None, None] + tig[None, None, :, None, None]) + r[None, None, None, :, None]).expand(shape)
        cols = (16 * s_[None, :, None, None, None] + 4 * h[None, None, None, :, None] + koff[None, None, None, None, :]).expand(shape)
        idx = (rows * Kp + cols).reshape(-1)
        if len(_FUSED_IDX) >= 32:
            _FUSED_IDX.clear()
        _FUSED_IDX[key] = idx
    shape = (nt // g, ks, g, 1, 64, 8)
    out = torch.cat([hi.reshape(-1)[idx].reshape(shape), lo.reshape(-1)[idx].reshape(shape)], dim=3).contiguous()
    return out.view(torch.uint8).reshape(-1)


def fused_stream(parts):
    """One weight stream of a fused kernel: the layers' fragments in consumption order, zero padded to whole ring chunks."""
    buf = torch.cat(parts)
    pad = (-buf.numel()) % FUSED_CHUNK
    if pad:
        buf = torch.cat([buf, torch.zeros(pad, device=buf.device, dtype=torch.uint8)])
    return buf.contiguous()


def pad_bias(b, n_pad=None):
    n = b.numel()
    Np = n_pad if n_pad is not None else (n + 31) // 32 * 32
    out = torch.zeros(Np, device=b.device, dtype=torch.float32)
    out[:n] = b.detach().float()
    return out


def calibration_input(n_num, offsets, device):
    """Fixed synthetic denoiser input [CAL_ROWS, n_num + sumK]: N(0,1) numeric columns (the quantile-normalised scale of
    the chain state, lib/data.py:217-223) and the log-one-hot of a cycling category per feature."""
    g = torch.Generator().manual_seed(0)
    cols = [torch.randn(CAL_ROWS, n_num, generator=g)]
    if offsets is not None and len(offsets) > 1:
        log_tiny = math.log(1e-30)
        r = torch.arange(CAL_ROWS)
        for f in range(len(offsets) - 1):
            k = int(offsets[f + 1] - offsets[f])
            blk = torch.full((CAL_ROWS, k), log_tiny)
            blk[r, r % k] = 0.0
            cols.append(blk)
    x = torch.cat(cols, dim=1).float()
    return x.to(device).contiguous(), float(x.abs().max())


class SplitNet:
    """Packed weights, folded biases and calibrated shifts of one stack; `.c` is the clava_split_net to pass by reference."""

    def __init__(self, ws, bs, acts, sc, sh, emb_table, x_cal, shift_in, y_cal=None, need_grad=False, cat=None):
        from .tab_ddpm.modules import run_stack
        dev = ws[0].device
        n = len(ws)
        fw, fb = fold_batchnorm(ws, bs, sc, sh)
        wmax = torch.stack([w.abs().max() for w in fw])
        # ---- float32 calibration pass at the two ends and the middle of the chain
        T = emb_table.shape[0]
        omax = torch.zeros(n, device=dev)
        gmax = torch.zeros(n, device=dev)
        for t in sorted({T - 1, T // 2, 0}):
            outs = run_stack(fw, fb, acts, x_cal[:, :fw[0].shape[1]].contiguous(), rowadd0=emb_table[t])
            omax = torch.maximum(omax, torch.stack([o.abs().max() for o in outs]))
            if need_grad:
                from .pipeline_utils import logsoftmax_select_grad
                g = logsoftmax_select_grad(outs[-1], y_cal)
                for l in range(n - 1, 0, -1):
                    has_act = acts[l - 1] != ACT_NONE
                    g = ops.linear_dgrad(g, fw[l], act_out=outs[l - 1] if has_act else None,
                                         slope=0.01 if acts[l - 1] == ACT_LEAKY else 0.0)
                    gmax[l] = torch.maximum(gmax[l], g.abs().max())
        stats = torch.cat([wmax, omax, gmax]).cpu().tolist()      # the one host synchronisation of the preparation
        wmax, omax, gmax = stats[:n], stats[n:2 * n], stats[2 * n:]
        self.shift_w = [shift_for(v, W_TARGET_LOG2) for v in wmax]
        self.shift_out = [shift_for(v) for v in omax]
        self.shift_grad = [shift_for(v) for v in gmax]
        self.shift_in = shift_in
        self.shift_dlast = DLAST_LOG2
        self.w = [ops.split_pack(w, s) for w, s in zip(fw, self.shift_w)]
        self.wt = [ops.split_pack(w.t().contiguous(), s) for w, s in zip(fw, self.shift_w)] if need_grad else None
        self.b = fb
        self.acts = list(acts)
        self.dims = [fw[0].shape[1]] + [w.shape[0] for w in fw]

        c = CSplitNet()
        self._dims = (ctypes.c_int * (n + 1))(*self.dims)
        self._w = _native.void_array([s.buf for s in self.w])
        self._wt = _native.void_array([s.buf for s in self.wt]) if need_grad else None
        self._b = _native.void_array(self.b)
        self._act = (ctypes.c_int * n)(*self.acts)
        self._sw = (ctypes.c_int * n)(*self.shift_w)
        self._so = (ctypes.c_int * n)(*self.shift_out)
        self._sg = (ctypes.c_int * n)(*self.shift_grad)
        c.n_layers = n
        c.dims = ctypes.cast(self._dims, _native.c_int_p)
        c.w = ctypes.cast(self._w, ctypes.POINTER(ctypes.c_void_p))
        if need_grad:
            c.wt = ctypes.cast(self._wt, ctypes.POINTER(ctypes.c_void_p))
            c.shift_grad = ctypes.cast(self._sg, _native.c_int_p)
        c.b = ctypes.cast(self._b, ctypes.POINTER(ctypes.c_void_p))
        c.act = ctypes.cast(self._act, _native.c_int_p)
        c.shift_w = ctypes.cast(self._sw, _native.c_int_p)
        c.shift_in = shift_in
        c.shift_out = ctypes.cast(self._so, _native.c_int_p)
        c.shift_dlast = self.shift_dlast
        # ---- operands of the fused narrow-stack kernels, for the parts of the configs' architectures that they cover
        # (a <= 32-wide input, dim_t = 128; classifier: 128, 256, ..., 256, 128, <= 64 classes; denoiser: first / last hidden
        # width 256, 512 or 1024).  Other shapes simply get no stream: the chain runs every layer as its own product then.
        self.bf = [None] * n
        self.fs_front = self.fs_tail = self.fs_back = self.fs_head = None
        d = self.dims
        pk = lambda l, **kw: pack_fused(fw[l], self.shift_w[l], **kw)
        pkt = lambda l, **kw: pack_fused(fw[l].t().contiguous(), self.shift_w[l], **kw)
        narrow_in = d[0] <= 32 and d[1] == 128 and os.environ.get("CLAVA_FUSED", "1") != "0"
        if narrow_in and not need_grad and n >= 3 and d[2] in (256, 512, 1024) and d[n - 1] in (256, 512, 1024) and d[n] <= 32:
            self.fs_front = fused_stream([pk(0), pk(1)])                         # proj, first hidden block
            self.fs_head = fused_stream([pk(n - 1)])
            for l in (0, 1, n - 1):
                self.bf[l] = pad_bias(fb[l])
        if narrow_in and need_grad and n == 9 and d[2] == 128 and d[3] == 256 and d[7] == 256 and d[8] == 128 and d[9] <= 64:
            self.fs_front = fused_stream([pk(0), pk(1), pk(2)])
            self.fs_tail = fused_stream([pk(7), pk(8, n_pad=64), pkt(8, k_pad=64), pkt(7)])
            self.fs_back = fused_stream([pkt(2), pkt(1), pkt(0)])
            for l in (0, 1, 2, 7):
                self.bf[l] = pad_bias(fb[l])
            self.bf[8] = pad_bias(fb[8], 64)
        self._bf = _native.void_array(self.bf)
        c.bf = ctypes.cast(self._bf, ctypes.POINTER(ctypes.c_void_p))
        for name in ("fs_front", "fs_tail", "fs_back", "fs_head"):
            t = getattr(self, name)
            setattr(c, name, t.data_ptr() if t is not None else None)
        # ---- gather form of the first layer for tables with categorical columns (csrc/cat_input.hip): cat = (n_num, sum K)
        self.num_wt = self.cat_wt = self.cat_bias = None
        if cat is not None and not need_grad and cat[1] > 0 and d[1] % 128 == 0 and cat[0] + cat[1] == d[0]:
            n_num = cat[0]
            log_tiny = float(torch.log(torch.tensor(1e-30, dtype=torch.float32)))     # index_to_log_onehot's clamp (utils.py:131)
            w0 = fw[0]
            self.num_wt = w0[:, :n_num].t().contiguous() if n_num > 0 else None
            self.cat_wt = w0[:, n_num:].t().contiguous()
            self.cat_bias = (fb[0].double() + log_tiny * w0[:, n_num:].double().sum(dim=1)).float().contiguous()
            c.num_wt = self.num_wt.data_ptr() if self.num_wt is not None else None
            c.cat_wt = self.cat_wt.data_ptr()
            c.cat_bias = self.cat_bias.data_ptr()
            c.log_tiny = log_tiny
        self.c = c


_cache = {}
_generation = 0          # bumped by everything that rewrites weights through raw device pointers (see `invalidate`)
_POS = {}


def invalidate():
    """Declare every cached SplitNet possibly stale.  Called by the kernels' callers that update parameters or BatchNorm
    statistics through raw pointers (`Trainer._optimizer_step`, `ClassifierTrainer.step`), which torch's version counters
    do not see; call it yourself after writing weights through `.data` in place."""
    global _generation
    _generation += 1


def _pos_weights(n, device):
    key = (str(device), n)
    w = _POS.get(key)
    if w is None:
        if len(_POS) >= 64:
            _POS.clear()
        w = (torch.arange(n, device=device, dtype=torch.int64) * 0x9E3779B1 + 0x7F4A7C15) | 1
        _POS[key] = w
    return w


def _fingerprint(tensors):
    """Exact, position-weighted fingerprint of the weights' BIT PATTERNS: sum_i bits_i * odd_weight(i) in wrapping
    int64 arithmetic, tensors combined with distinct odd multipliers.  Unlike a sum of values / squares it changes when
    two values swap places or move between tensors, and there is no floating-point cancellation."""
    parts = []
    for j, t in enumerate(tensors):
        if t is None or t.numel() == 0:
            continue
        flat = t.detach().reshape(-1).contiguous()
        bits = flat.view(torch.int32 if flat.element_size() % 4 == 0 else torch.uint8).to(torch.int64)
        parts.append((bits * _pos_weights(bits.numel(), t.device)).sum() * (2 * j + 1))
    return torch.stack(parts).sum()


def _versions(tensors):
    return tuple((t.data_ptr(), t._version) for t in tensors if t is not None)


def prepare(ws, bs, acts, sc, sh, emb_table, x_cal, shift_in, y_cal=None, need_grad=False, watch=None, cat=None):
    """SplitNet for these weights, cached until a weight changes.

    `watch` = every tensor the prepared network depends on (the module's parameters and BatchNorm buffers, the
    time-embedding layers included); default: ws + bs.  A cache entry is reused without any device work while (a) no
    raw-pointer writer has run since (`invalidate()` generation) and (b) torch's version counter of every watched
    tensor is unchanged; otherwise the exact fingerprint decides (one small reduction + one host sync), and the entry
    is rebuilt if it differs.  Entries keep their tensors alive, so a cached device address cannot be handed to another
    tensor by the allocator while the entry exists."""
    watch = [t.detach() for t in (watch if watch is not None else list(ws) + list(bs)) if t is not None]
    key = tuple((t.data_ptr(), tuple(t.shape)) for t in watch) + (emb_table.shape[0], shift_in, need_grad, x_cal.shape[1],
                                                                   os.environ.get("CLAVA_FUSED", "1"), cat)
    hit = _cache.get(key)
    vers = _versions(watch)
    if hit is not None:
        if hit["gen"] == _generation and hit["vers"] == vers:
            return hit["net"]
        sig = _fingerprint(watch)
        if bool(hit["sig"] == sig):
            hit["gen"], hit["vers"] = _generation, vers
            return hit["net"]
    else:
        sig = _fingerprint(watch)
    net = SplitNet(ws, bs, acts, sc, sh, emb_table, x_cal, shift_in, y_cal, need_grad, cat)
    if key not in _cache and len(_cache) >= 8:
        _cache.pop(next(iter(_cache)))
    _cache[key] = {"net": net, "sig": sig, "gen": _generation, "vers": vers, "keep": watch}
    return net
