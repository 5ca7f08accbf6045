"""Thin torch-tensor wrappers over the C ABI (one function per `clava_*` entry point).

Only plumbing lives here: argument checking, output allocation through torch's
caching allocator, and the raw-pointer call.  All arithmetic is in the HIP
library.
"""
import ctypes
import functools
import math

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import c_float, c_int, check, lib, ptr, require_cuda, stream_ptr

_ACT = {None: 0, "none": 0, "relu": 1, "leaky_relu": 2, "silu": 3}


def _f32c(t, name):
    if t is None:
        return None
    if t.dtype != torch.float32:
        raise _lib.ClavaHipError(f"{name}: expected float32, got {t.dtype}")
    if t.stride(-1) != 1:
        raise _lib.ClavaHipError(f"{name}: innermost dimension must be contiguous")
    return t


def _ld(t):
    return t.stride(0) if t.dim() == 2 else 0


def _rs(t):
    """Row stride of a 2-D tensor as a leading dimension.  torch reports an arbitrary stride(0) for a one-row tensor (a
    [1, n] transpose of an [n, 1] weight has stride 1): any value >= the row length is equivalent there."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[-1])


def linear(x, w, bias=None, act=None, rowadd=None, in_scale=None, in_shift=None, out=None):
    """act((x*in_scale+in_shift) @ w.T + bias + rowadd) via clava_gemm_bias_act_f32.

    `rowadd` is [M, N] or a single row [N] / [1, N] broadcast over the batch."""
    require_cuda(x, w, bias, rowadd, in_scale, in_shift)
    x, w = _f32c(x, "x"), _f32c(w, "w")
    M, K = x.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise _lib.ClavaHipError(f"linear: x is [{M},{K}] but w is {tuple(w.shape)}")
    if out is None:
        out = torch.empty((M, N), device=x.device, dtype=torch.float32)
    ldr = 0
    if rowadd is not None:
        rowadd = _f32c(rowadd, "rowadd")
        if rowadd.dim() == 2 and rowadd.shape[0] == M and M > 1:
            ldr = rowadd.stride(0)
        if rowadd.shape[-1] != N:
            raise _lib.ClavaHipError("linear: rowadd width mismatch")
    if M == 0:
        return out
    check(lib().clava_gemm_bias_act_f32(ptr(x), c_int(_rs(x)), ptr(w), c_int(_rs(w)), ptr(_f32c(bias, "bias")),
                                        ptr(rowadd), c_int(ldr), ptr(_f32c(in_scale, "in_scale")),
                                        ptr(_f32c(in_shift, "in_shift")), ptr(out), c_int(_rs(out)), c_int(M),
                                        c_int(N), c_int(K), c_int(_ACT[act]), stream_ptr()), "clava_gemm_bias_act_f32")
    return out


def linear_dgrad(dy, w, act_out=None, slope=0.0, col_scale=None, alpha=1.0, out=None):
    """alpha * col_scale * act'(act_out) * (dy @ w) via clava_gemm_dgrad_f32."""
    require_cuda(dy, w, act_out, col_scale)
    dy, w = _f32c(dy, "dy"), _f32c(w, "w")
    M, N = dy.shape
    K = w.shape[1]
    if w.shape[0] != N:
        raise _lib.ClavaHipError("linear_dgrad: dy/w shape mismatch")
    if out is None:
        out = torch.empty((M, K), device=dy.device, dtype=torch.float32)
    if M == 0:
        return out
    check(lib().clava_gemm_dgrad_f32(ptr(dy), c_int(_rs(dy)), ptr(w), c_int(_rs(w)), ptr(_f32c(act_out, "act_out")),
                                     c_int(_rs(act_out) if act_out is not None else 0), c_float(slope),
                                     ptr(_f32c(col_scale, "col_scale")), c_float(alpha), ptr(out), c_int(_rs(out)),
                                     c_int(M), c_int(N), c_int(K), stream_ptr()), "clava_gemm_dgrad_f32")
    return out


def linear_wgrad(dy, x, splits=1, out=None, slab_stride=None):
    """Partial products of dy.T @ x over `splits` batch ranges: returns [splits, N_out, K_in] (or fills `out`, whose
    slabs are `slab_stride` floats apart)."""
    require_cuda(dy, x)
    dy, x = _f32c(dy, "dy"), _f32c(x, "x")
    M, N = dy.shape
    K = x.shape[1]
    if x.shape[0] != M:
        raise _lib.ClavaHipError("linear_wgrad: batch mismatch")
    if out is None:
        out = torch.empty((splits, N, K), device=dy.device, dtype=torch.float32)
    if slab_stride is None:
        slab_stride = N * K
    check(lib().clava_gemm_wgrad_f32(ptr(dy), c_int(_rs(dy)), ptr(x), c_int(_rs(x)), ptr(out), c_int(K),
                                     _lib.c_long(slab_stride), c_int(M), c_int(N), c_int(K), c_int(splits), stream_ptr()),
          "clava_gemm_wgrad_f32")
    return out


# ---- split-f16 family (csrc/split.h): float32 values as two float16 planes, products on the f16 matrix cores ----------
class SplitTensor:
    """A [rows, cols] matrix stored as split rows (see include/clava_hip.h): `buf` is a uint8 device tensor of
    rows * pitch bytes, `shift` the power-of-two scale of the planes."""
    __slots__ = ("buf", "rows", "cols", "shift", "pitch")

    def __init__(self, buf, rows, cols, shift, pitch):
        self.buf, self.rows, self.cols, self.shift, self.pitch = buf, rows, cols, shift, pitch


def split_pitch(cols):
    return 4 * ((cols + 31) // 32 * 32)


def split_empty(rows, cols, shift, device):
    pitch = split_pitch(cols)
    return SplitTensor(torch.zeros(max(rows * pitch, 1), device=device, dtype=torch.uint8), rows, cols, shift, pitch)


def overflow_flag(device):
    return torch.zeros(1, device=device, dtype=torch.int32)


def split_pack(x, shift=0, overflow=None, out=None):
    """float32 [rows, cols] -> SplitTensor (clava_split_pack_f32); `out` reuses a SplitTensor of the same shape."""
    require_cuda(x)
    x = _f32c(x, "x")
    rows, cols = x.shape
    if out is None:
        out = split_empty(rows, cols, shift, x.device)
    else:
        if (out.rows, out.cols) != (rows, cols):
            raise _lib.ClavaHipError("split_pack: `out` has another shape")
        out.shift = shift
    if rows:
        check(lib().clava_split_pack_f32(ptr(x), _lib.c_long(_rs(x)), _lib.c_long(rows), c_int(cols), c_int(shift),
                                         ptr(out.buf), _lib.c_long(out.pitch), ptr(overflow), stream_ptr()), "clava_split_pack_f32")
    return out


def split_pack_transposed(x, shift=0, overflow=None, out=None):
    """SplitTensor of x.T for a float32 [cols, rows] matrix x, without materialising the transpose."""
    require_cuda(x)
    x = _f32c(x, "x")
    cols, rows = x.shape
    if out is None:
        out = split_empty(rows, cols, shift, x.device)
    else:
        if (out.rows, out.cols) != (rows, cols):
            raise _lib.ClavaHipError("split_pack_transposed: `out` has another shape")
        out.shift = shift
    if rows:
        check(lib().clava_split_pack_transposed_f32(ptr(x), _lib.c_long(_rs(x)), _lib.c_long(rows), c_int(cols), c_int(shift),
                                                    ptr(out.buf), _lib.c_long(out.pitch), ptr(overflow), stream_ptr()),
              "clava_split_pack_transposed_f32")
    return out


class _PackDesc(ctypes.Structure):
    _fields_ = [("src", ctypes.c_void_p), ("ld", ctypes.c_longlong), ("rows", ctypes.c_int), ("cols", ctypes.c_int),
                ("scale", ctypes.c_float), ("dst", ctypes.c_void_p), ("pitch", ctypes.c_longlong), ("dst_t", ctypes.c_void_p),
                ("pitch_t", ctypes.c_longlong)]


class PackPlan:
    """A fixed list of (float32 matrix, shift, SplitTensor or None, SplitTensor of the transpose or None) packed by ONE
    launch (clava_split_pack_multi_f32).  The descriptors live in device memory and hold raw pointers: the plan is valid
    while every tensor named keeps its storage (`key` lets the owner notice when that changed)."""

    def __init__(self, items, device):
        arr = (_PackDesc * len(items))()
        self.keep = []
        self.max_tiles = 1
        for d, (src, shift, dst, dst_t) in zip(arr, items):
            require_cuda(src)
            if src.dtype != torch.float32 or src.dim() != 2 or src.stride(1) != 1:
                raise _lib.ClavaHipError("PackPlan: float32 row-major matrices expected")
            rows, cols = src.shape
            d.src, d.ld, d.rows, d.cols, d.scale = src.data_ptr(), _rs(src), rows, cols, 2.0 ** shift
            if dst is not None:
                if (dst.rows, dst.cols) != (rows, cols):
                    raise _lib.ClavaHipError("PackPlan: destination has another shape")
                dst.shift = shift
                d.dst, d.pitch = dst.buf.data_ptr(), dst.pitch
            if dst_t is not None:
                if (dst_t.rows, dst_t.cols) != (cols, rows):
                    raise _lib.ClavaHipError("PackPlan: transposed destination has another shape")
                dst_t.shift = shift
                d.dst_t, d.pitch_t = dst_t.buf.data_ptr(), dst_t.pitch
            self.max_tiles = max(self.max_tiles, ((rows + 63) // 64) * ((cols + 63) // 64))
            self.keep.append((src, dst, dst_t, shift))
        self.n = len(items)
        raw = torch.frombuffer(bytearray(bytes(arr)), dtype=torch.uint8)
        self.dev = raw.to(device)
        self.key = tuple((s.data_ptr(), sh) for s, sh, _, _ in items)

    def run(self, overflow=None):
        for _, dst, dst_t, shift in self.keep:       # a cached plan may run again after another plan re-scaled its destinations
            if dst is not None:
                dst.shift = shift
            if dst_t is not None:
                dst_t.shift = shift
        check(lib().clava_split_pack_multi_f32(ptr(self.dev), c_int(self.n), c_int(self.max_tiles), ptr(overflow), stream_ptr()),
              "clava_split_pack_multi_f32")


def split_transpose(s, out=None):
    """SplitTensor of the transpose (clava_split_transpose): planes moved as they are, same shift."""
    if out is None:
        out = split_empty(s.cols, s.rows, s.shift, s.buf.device)
    elif (out.rows, out.cols) != (s.cols, s.rows):
        raise _lib.ClavaHipError("split_transpose: `out` has another shape")
    out.shift = s.shift
    if s.rows and s.cols:
        check(lib().clava_split_transpose(ptr(s.buf), _lib.c_long(s.pitch), _lib.c_long(s.rows), c_int(s.cols), ptr(out.buf),
                                          _lib.c_long(out.pitch), stream_ptr()), "clava_split_transpose")
    return out


def linear_wgrad_f16x3(dyt, xt, splits, out, slab_stride, tile_config=-1):
    """Partial products of dy.T @ x over `splits` batch ranges on the f16 matrix cores (clava_gemm_wgrad_f16x3):
    dyt = dy^T [N_out, M], xt = x^T [K_in, M] as SplitTensors; fills `out` (slabs `slab_stride` floats apart, rows K_in apart)."""
    n_out, M = dyt.rows, dyt.cols
    k_in = xt.rows
    if xt.cols != M:
        raise _lib.ClavaHipError("linear_wgrad_f16x3: batch mismatch")
    nkb = (M + 31) // 32
    while splits > 1 and (splits - 1) * ((nkb + splits - 1) // splits) >= nkb:
        splits -= 1
    check(lib().clava_gemm_wgrad_f16x3(ptr(dyt.buf), _lib.c_long(dyt.pitch), c_int(dyt.shift), ptr(xt.buf), _lib.c_long(xt.pitch),
                                       c_int(xt.shift), ptr(out), c_int(k_in), _lib.c_long(slab_stride), c_int(M), c_int(n_out),
                                       c_int(k_in), c_int(splits), c_int(tile_config), stream_ptr()), "clava_gemm_wgrad_f16x3")
    return splits


def linear_wgrad_f16x3_tn(dy, x, splits, out, slab_stride, bias_out=None, ldw=None):
    """`linear_wgrad_f16x3` from the batch-major SplitTensors themselves (clava_gemm_wgrad_f16x3_tn): dy [M, N_out],
    x [M, K_in], M a multiple of 32; no transposed copies.  `bias_out` (slabs, same stride) also receives the column sums
    of dy (the bias gradient).  `ldw`: row stride of the gradient in `out` (default K_in; larger when x holds only the
    first columns of the layer's input)."""
    M, n_out = dy.rows, dy.cols
    k_in = x.cols
    if x.rows != M or M % 32:
        raise _lib.ClavaHipError("linear_wgrad_f16x3_tn: batch mismatch or batch not a multiple of 32")
    nkb = M // 32
    while splits > 1 and (splits - 1) * ((nkb + splits - 1) // splits) >= nkb:
        splits -= 1
    check(lib().clava_gemm_wgrad_f16x3_tn(ptr(dy.buf), _lib.c_long(dy.pitch), c_int(dy.shift), ptr(x.buf), _lib.c_long(x.pitch),
                                          c_int(x.shift), ptr(out), c_int(k_in if ldw is None else ldw), _lib.c_long(slab_stride), ptr(bias_out), c_int(M),
                                          c_int(n_out), c_int(k_in), c_int(splits), stream_ptr()), "clava_gemm_wgrad_f16x3_tn")
    return splits


def split_unpack(s):
    out = torch.empty((s.rows, s.cols), device=s.buf.device, dtype=torch.float32)
    if s.rows:
        check(lib().clava_split_unpack_f32(ptr(s.buf), _lib.c_long(s.pitch), _lib.c_long(s.rows), c_int(s.cols), c_int(s.shift),
                                           ptr(out), _lib.c_long(_rs(out)), stream_ptr()), "clava_split_unpack_f32")
    return out


def linear_f16x3(x, w, bias=None, act=None, rowadd=None, act_out=None, slope=0.0, alpha=1.0, out_shift=None, out_f32=False,
                 overflow=None, tile_config=-1, out=None, both=False, out2=None):
    """alpha * act'(act_out) * act(x @ w.T + bias + rowadd) with x, w SplitTensors (clava_gemm_f16x3).
    Returns a SplitTensor with shift `out_shift`, or a float32 tensor when out_f32, or (SplitTensor, float32) when `both`
    (`out` = the SplitTensor to fill, `out2` = the float32 tensor to fill)."""
    M, K = x.rows, x.cols
    N = w.rows
    if w.cols != K:
        raise _lib.ClavaHipError(f"linear_f16x3: x is [{M},{K}] but w is [{w.rows},{w.cols}]")
    y_split = y_f32 = None
    if both:
        y_split = out if out is not None else split_empty(M, N, 0 if out_shift is None else out_shift, x.buf.device)
        if out is not None and out_shift is not None:
            y_split.shift = out_shift
        y_f32 = out2 if out2 is not None else torch.empty((M, N), device=x.buf.device, dtype=torch.float32)
    elif out_f32:
        y_f32 = out if out is not None else torch.empty((M, N), device=x.buf.device, dtype=torch.float32)
    else:
        y_split = out if out is not None else split_empty(M, N, 0 if out_shift is None else out_shift, x.buf.device)
        if out is not None and out_shift is not None:
            y_split.shift = out_shift
    check(lib().clava_gemm_f16x3(ptr(x.buf), _lib.c_long(x.pitch), c_int(x.shift), ptr(w.buf), _lib.c_long(w.pitch), c_int(w.shift),
                                 ptr(_f32c(bias, "bias")), ptr(_f32c(rowadd, "rowadd")), c_int(_ACT[act]),
                                 ptr(act_out.buf) if act_out is not None else None,
                                 _lib.c_long(act_out.pitch if act_out is not None else 0), c_float(slope), c_float(alpha),
                                 ptr(y_split.buf) if y_split is not None else None,
                                 _lib.c_long(y_split.pitch if y_split is not None else 0),
                                 c_int(y_split.shift if y_split is not None else 0), ptr(y_f32),
                                 c_int(_rs(y_f32) if y_f32 is not None else 0), c_int(M), c_int(N), c_int(K), ptr(overflow),
                                 c_int(tile_config), stream_ptr()), "clava_gemm_f16x3")
    if both:
        return y_split, y_f32
    return y_f32 if out_f32 else y_split


# ---- microscaled 4-bit matrices (OCP MX, E2M1 over blocks of 32 columns) and dense layers over them --------------------
# These calls take a few microseconds on the GPU at their smallest, so their host side counts: C functions with declared
# argument types (plain Python numbers, no ctypes objects), one look at a tensor's shape and strides.
_DT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MX4 = 3
c_ll = ctypes.c_longlong
_C_TYPES = {"p": ctypes.c_void_p, "i": ctypes.c_int, "l": c_ll, "u": ctypes.c_uint, "U": ctypes.c_ulonglong}
_FUNCTIONS = {}


def _function(name, types, result=ctypes.c_int):
    f = _FUNCTIONS.get(name)
    if f is None:
        f = getattr(lib(), name)
        f.argtypes = [_C_TYPES[c] for c in types]
        f.restype = result
        _FUNCTIONS[name] = f
    return f


def _refuse(message):
    raise _lib.ClavaHipError(message)


def _dt(t, name):
    d = _DT.get(t.dtype)
    if d is None:
        _refuse(f"{name}: expected float32, bfloat16 or float16, got {t.dtype}")
    return d


def _matrix(t, name):
    """(rows, columns, row stride) of a device tensor [rows, cols] with contiguous rows."""
    if not t.is_cuda:
        require_cuda(t)
    if t.dim() != 2:
        _refuse(f"{name}: expected [rows, cols], got {tuple(t.shape)}")
    (rows, cols), (ld, inner) = t.shape, t.stride()
    if inner != 1 and cols > 1:
        _refuse(f"{name}: innermost dimension must be contiguous")
    if rows > 1:
        if ld < cols:
            _refuse(f"{name}: rows overlap (stride {ld} for {cols} columns)")
    elif ld < cols:
        ld = cols                  # (torch reports any stride for a single row)
    return rows, cols, ld


def _no_gradient(message, *tensors):
    """Refuse tensors that a derivative is asked of: recorded for backward, or duals with a tangent."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        _refuse(message + ": call it under torch.no_grad() or detach its inputs")
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        _refuse(message + " and no forward derivative: give it the primal of a dual tensor")


def _launch(dev, name, f, *args):
    """f(*args, stream) on the current stream of the tensors' device."""
    index = dev.index
    if index == torch._C._cuda_getDevice():
        rc = f(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(dev):
            rc = f(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        check(rc, name)


class Mx4Tensor:
    """A [rows, cols] matrix in microscaled 4-bit form (see include/clava_hip.h): `codes` uint8 [rows, Kp / 2] and `scales`
    uint8 [rows, Kp / 32], Kp = cols rounded up to 128.  The codes behind the last column have to be zero."""
    __slots__ = ("rows", "cols", "device", "codes_ptr", "scales_ptr", "_codes", "_scales", "_buf")

    def __init__(self, codes, scales, cols):
        cols = int(cols)
        steps = (cols + 127) // 128
        if cols < 1:
            _refuse(f"Mx4Tensor: {cols} columns")
        rows = codes.shape[0]
        if codes.shape != (rows, 64 * steps) or codes.dtype is not torch.uint8 or not codes.is_contiguous():
            _refuse(f"Mx4Tensor: codes must be contiguous uint8 [{rows}, {64 * steps}], got {codes.dtype} {tuple(codes.shape)}")
        if scales.shape != (rows, 4 * steps) or scales.dtype is not torch.uint8 or not scales.is_contiguous():
            _refuse(f"Mx4Tensor: scales must be contiguous uint8 [{rows}, {4 * steps}], got {scales.dtype} {tuple(scales.shape)}")
        if not codes.is_cuda:
            require_cuda(codes)
        self.device = codes.device
        if scales.device != self.device:
            _refuse(f"Mx4Tensor: scales are on {scales.device}, codes on {self.device}")
        self.codes_ptr, self.scales_ptr = codes.data_ptr(), scales.data_ptr()
        if self.codes_ptr & 15:
            _refuse("Mx4Tensor: codes must start at a multiple of 16 bytes")
        self._codes, self._scales, self.rows, self.cols, self._buf = codes, scales, rows, cols, None

    # (mx4_empty's two parts share one allocation; the views are made when somebody looks at them)
    @property
    def codes(self):
        if self._codes is None:
            n = self.rows * 64 * ((self.cols + 127) // 128)
            self._codes = self._buf[:n].view(self.rows, -1) if n else self._buf.view(0, 64 * ((self.cols + 127) // 128))
        return self._codes

    @property
    def scales(self):
        if self._scales is None:
            steps = (self.cols + 127) // 128
            n = self.rows * 64 * steps
            self._scales = self._buf[n:].view(self.rows, -1) if n else self._buf.view(0, 4 * steps)
        return self._scales


def mx4_empty(rows, cols, device):
    """An uninitialised Mx4Tensor, for `out`."""
    q = Mx4Tensor.__new__(Mx4Tensor)
    steps = (cols + 127) // 128
    if cols < 1 or rows < 0:
        _refuse(f"mx4_empty: [{rows}, {cols}]")
    buf = torch.empty(rows * 68 * steps, device=device, dtype=torch.uint8)
    if not buf.is_cuda:
        require_cuda(buf)
    q.rows, q.cols, q.device, q._buf, q._codes, q._scales = rows, cols, buf.device, buf, None, None
    q.codes_ptr = buf.data_ptr()
    q.scales_ptr = q.codes_ptr + rows * 64 * steps
    return q


def mx4_pack(x, out=None):
    """[rows, cols] float32 / bfloat16 / float16 -> Mx4Tensor (clava_mx4_pack); `out` reuses one of the same shape.  A block
    that holds a NaN or an infinity reads as NaN.  No gradient is defined."""
    rows, cols, ld = _matrix(x, "mx4_pack: x")
    dt = _dt(x, "mx4_pack: x")
    if x.requires_grad or forward_ad._current_level >= 0:
        _no_gradient("mx4_pack has no backward", x)
    if out is None:
        out = mx4_empty(rows, cols, x.device)
    elif (out.rows, out.cols) != (rows, cols) or out.device != x.device:
        _refuse(f"mx4_pack: x is [{rows},{cols}] on {x.device} but out is [{out.rows},{out.cols}] on {out.device}")
    elif rows:
        _not_over("mx4_pack", _parts(out, rows, cols, 0), x=_parts(x, rows, cols, ld))
    _launch(out.device, "clava_mx4_pack", _function("clava_mx4_pack", "pillippp"),
            x.data_ptr(), dt, ld, rows, cols, out.codes_ptr, out.scales_ptr)
    return out


def mx4_unpack(q, dtype=torch.float32, out=None):
    """The values of an Mx4Tensor as float32, bfloat16 or float16 (clava_mx4_unpack); `out` may not overlap it."""
    own = out is None
    if own:
        if dtype not in _DT:
            _refuse(f"mx4_unpack: expected float32, bfloat16 or float16, got {dtype}")
        out = torch.empty((q.rows, q.cols), device=q.device, dtype=dtype)
    rows, cols, ld = _matrix(out, "mx4_unpack: out")
    if (rows, cols) != (q.rows, q.cols) or out.device != q.device:
        _refuse(f"mx4_unpack: q is [{q.rows},{q.cols}] on {q.device} but out is [{rows},{cols}] on {out.device}")
    if rows and not own:
        _not_over("mx4_unpack", _parts(out, rows, cols, ld), q=_parts(q, rows, cols, 0))
    _launch(q.device, "clava_mx4_unpack", _function("clava_mx4_unpack", "pplipilp"),
            q.codes_ptr, q.scales_ptr, rows, cols, out.data_ptr(), _dt(out, "mx4_unpack: out"), ld)
    return out


def _overlap(a, row_a, step_a, b, row_b, step_b, rows):
    """Whether two matrices share memory; of columns of one buffer only if they share columns."""
    if a + (rows - 1) * step_a + row_a <= b or b + (rows - 1) * step_b + row_b <= a:
        return False
    if rows == 1 or step_a != step_b:
        return True
    d = (b - a) % step_a
    return d < row_a or d + row_b > step_a


def _parts(t, rows, cols, ld):
    """The memory of an operand or result: (start, bytes of a row, of its stride, rows); codes and scales are one row each."""
    if isinstance(t, Mx4Tensor):
        steps = rows * ((cols + 127) // 128)
        return (t.codes_ptr, 64 * steps, 64 * steps, 1), (t.scales_ptr, 4 * steps, 4 * steps, 1)
    size = t.element_size()
    return ((t.data_ptr(), cols * size, ld * size, rows),)


def _ends(p, scales, rows, cols, ld, t):
    """Where a matrix at `p` begins and ends (scales: None for floats)."""
    if scales is None:
        return p, p + ((rows - 1) * ld + cols) * t.element_size()
    steps = rows * ((cols + 127) // 128)
    codes_end, scales_end = p + 64 * steps, scales + 4 * steps
    return (p if p < scales else scales), (codes_end if codes_end > scales_end else scales_end)


def _spread(t):
    """A tensor's memory as one part, with what lies between its elements."""
    size = t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))
    return ((t.data_ptr(), size, size, 1),)


def _share(p, q):
    """Whether two such parts have a byte in common (of two matrices with strides that differ: whether they may)."""
    (a, row_a, step_a, rows_a), (b, row_b, step_b, rows_b) = p, q
    if rows_a == 1 and rows_b == 1 or rows_a == rows_b:
        return _overlap(a, row_a, step_a, b, row_b, step_b, rows_a)
    if rows_a == 1:
        a, row_a, step_a, rows_a, b, row_b, rows_b = b, row_b, step_b, rows_b, a, row_a, rows_a
    if rows_b > 1:
        return a < b + (rows_b - 1) * step_b + row_b and b < a + (rows_a - 1) * step_a + row_a
    i = max(0, (b - a - row_a) // step_a + 1)                    # the first row that ends behind b
    return i < rows_a and a + i * step_a < b + row_b


def _not_over(name, out, **inputs):
    """Refuse a result that shares memory with what is read while it is written; all are tuples of parts."""
    low, high = min(p[0] for p in out), max(a + (n - 1) * step + row for a, row, step, n in out)
    for what, parts in inputs.items():
        for p in parts:
            if p[0] < high and low < p[0] + (p[3] - 1) * p[2] + p[1] and any(_share(p, q) for q in out):
                _refuse(f"{name}: out overlaps {what}, which is read while out is written")


@functools.lru_cache(maxsize=256)
def _mx4_workspace(rows, cols, dt):
    return _function("clava_linear_mx4_workspace_bytes", "iii", c_ll)(rows, cols, dt)


def linear_mx4(x, w, bias=None, act=None, out=None, out_dtype=torch.float32):
    """act(x @ w.T + bias) over 4-bit operands (clava_linear_mx4_sized): `w` an Mx4Tensor [N, K], `x` an Mx4Tensor [M, K] or a float
    matrix, which is packed first.  The result is a float matrix of `out_dtype`, or whatever `out` is: a float matrix or an
    Mx4Tensor (the next layer's operand); it may not overlap x, w or bias.  No gradient is defined."""
    if not isinstance(w, Mx4Tensor):
        _refuse("linear_mx4: w must be an Mx4Tensor")
    code = _ACT.get(act)
    if code is None:
        _refuse(f"linear_mx4: unknown activation {act!r}")
    N, dev, ws = w.rows, w.device, None
    if isinstance(x, Mx4Tensor):
        M, K, ldx, x_dt, xp, xs = x.rows, x.cols, 0, _MX4, x.codes_ptr, x.scales_ptr
    else:
        M, K, ldx = _matrix(x, "linear_mx4: x")
        x_dt, xp, xs = _dt(x, "linear_mx4: x"), x.data_ptr(), None
        if x.requires_grad or forward_ad._current_level >= 0:
            _no_gradient("linear_mx4 has no backward", x)
    if w.cols != K:
        _refuse(f"linear_mx4: x is [{M},{K}] but w is [{N},{w.cols}]")
    if N == 0:
        _refuse("linear_mx4: w has no rows")
    if x.device != dev:
        _refuse(f"linear_mx4: x is on {x.device}, w on {dev}")
    bp = None
    if bias is not None:
        if bias.dtype is not torch.float32 or bias.shape != (N,) or not bias.is_contiguous() or bias.device != dev:
            _refuse(f"linear_mx4: bias must be contiguous float32 [{N}] on {dev}")
        if bias.requires_grad or forward_ad._current_level >= 0:
            _no_gradient("linear_mx4 has no backward", bias)
        bp = bias.data_ptr()
    if out is None:
        if out_dtype not in _DT:
            _refuse(f"linear_mx4: expected float32, bfloat16 or float16, got {out_dtype}")
        out = torch.empty((M, N), device=dev, dtype=out_dtype)
        y_dt, ldy, yp, ys = _DT[out_dtype], N, out.data_ptr(), None
    else:
        if isinstance(out, Mx4Tensor):
            rows, cols, ldy, y_dt, yp, ys = out.rows, out.cols, 0, _MX4, out.codes_ptr, out.scales_ptr
        else:
            rows, cols, ldy = _matrix(out, "linear_mx4: out")
            y_dt, yp, ys = _dt(out, "linear_mx4: out"), out.data_ptr(), None
        if (rows, cols) != (M, N) or out.device != dev:
            _refuse(f"linear_mx4: the result is [{M},{N}] on {dev} but out is [{rows},{cols}] on {out.device}")
        if M:
            # first by the ends of each, which settles nearly every call
            low, high = _ends(yp, ys, M, N, ldy, out)
            x_low, x_high = _ends(xp, xs, M, K, ldx, x)
            w_low, w_high = _ends(w.codes_ptr, w.scales_ptr, N, K, 0, w)
            if low < x_high and x_low < high or low < w_high and w_low < high or bp is not None and low < bp + 4 * N and bp < high:
                _not_over("linear_mx4", _parts(out, M, N, ldy), x=_parts(x, M, K, ldx), w=_parts(w, N, K, 0),
                          bias=((bp, 4 * N, 4 * N, 1),) if bp else ())
    need = _mx4_workspace(M, K, x_dt) if x_dt != _MX4 else 0
    if need:
        ws = torch.empty(need, device=dev, dtype=torch.uint8)
    _launch(dev, "clava_linear_mx4_sized", _function("clava_linear_mx4_sized", "pilppppipilpiiiplp"),
            xp, x_dt, ldx, xs, w.codes_ptr, w.scales_ptr, bp, code, yp, y_dt, ldy, ys, M, N, K,
            None if ws is None else ws.data_ptr(), need)
    return out


# ---- one class per feature from its logits ----------------------------------------------------------------------------
class _CChoice(ctypes.Structure):
    _fields_ = [("temperature", ctypes.c_double), ("top_p", ctypes.c_double), ("min_p", ctypes.c_double), ("top_k", ctypes.c_int)] + \
               [(n + "_t", ctypes.c_void_p) for n in ("temperature", "top_p", "min_p", "top_k")] + \
               [(n + s, c_ll) for n in ("temperature", "top_p", "min_p", "top_k") for s in ("_rs", "_fs")]


_CHOICE_RANGE = {"temperature": (0.0, math.inf), "top_p": (0.0, math.inf), "min_p": (0.0, 1.0), "top_k": (-2 ** 63, 2 ** 63)}
_NUMBERS = {int, float}


def _choice_args(dev, rows, features, values):
    """The C struct of the four parameters: numbers, or tensors that broadcast to [rows, features]."""
    c = _CChoice()
    for name, v in values:
        if isinstance(v, torch.Tensor):
            want = torch.int32 if name == "top_k" else torch.float32
            if v.dtype is not want or v.device != dev:
                _refuse(f"sample_categories: {name} must be {want} on {dev}, got {v.dtype} on {v.device}")
            try:
                v = v.expand(rows, features)
            except RuntimeError:
                raise _lib.ClavaHipError(f"sample_categories: {name} {tuple(v.shape)} does not broadcast to [{rows},{features}]") from None
            setattr(c, name + "_t", v.data_ptr())
            rs, fs = v.stride()
            setattr(c, name + "_rs", rs)
            setattr(c, name + "_fs", fs)
            continue
        low, high = _CHOICE_RANGE[name]
        if not low <= v <= high or name == "top_k" and v != int(v) or isinstance(v, int) and v > 2 ** 1023:
            _refuse(f"sample_categories: {name} {v}, expected {'a whole number' if name == 'top_k' else f'in [{low}, {high}]'}")
        setattr(c, name, max(-1, min(int(v), 2 ** 31 - 1)) if name == "top_k" else v)
    return c


@functools.lru_cache(maxsize=64)
def _choice_numbers(*values):
    """The struct of four numbers, which C only reads (building it takes 2 of a small call's 11 us)."""
    return _choice_args(None, 0, 0, zip(_CHOICE_RANGE, values))


def sample_categories(logits, uniforms=None, offsets=None, max_classes=None, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                      log_prob=False, seed=0, row_offset=0, step_index=0, out=None):
    """One class per (row, feature) from `logits` [B, sumK] (float32, bfloat16 or float16) with temperature, top-k, top-p and
    min-p, as clava_sample_categories defines them; int32 [B, m], with `log_prob` also the log-probability of every drawn class
    under the filtered distribution, float32 [B, m] (no gradient is defined).

    Feature f owns columns offsets[f] .. offsets[f+1] (int32 device tensor [m + 1] that rises; None: one feature of all columns).
    `uniforms`: float32 [B, m] in [0, 1) ([B] for one feature), or None for the generator keyed by (seed, row_offset + row,
    feature, step_index).  `max_classes`: the largest number of classes of one feature, which picks the kernels and the workspace
    (any value is safe, a feature of more classes is slow; default: all columns).  Each parameter is a number or a device tensor (float32; top_k int32) that broadcasts to
    [B, m].  A feature with no class left to draw (none, all logits -inf, a NaN) or with a parameter that is no number yields -1
    and NaN.  A captured call repeats its own draws: give it `uniforms` that the program refills.  Features of more than 4096
    classes whose logits are nearly all equal are slow with top_k or top_p: one workgroup does each (64 rows of 131071: 2.2 ms)."""
    B, sumk, ld = _matrix(logits, "sample_categories: logits")
    dt = _dt(logits, "sample_categories: logits")
    if log_prob and (logits.requires_grad or isinstance(temperature, torch.Tensor) or forward_ad._current_level >= 0):
        _no_gradient("sample_categories: log_prob has no backward", logits, temperature if isinstance(temperature, torch.Tensor) else None)
    dev = logits.device
    m, op = 1, None
    if offsets is not None:
        if offsets.dtype is not torch.int32 or offsets.dim() != 1 or offsets.shape[0] < 2 or not offsets.is_contiguous() or offsets.device != dev:
            _refuse(f"sample_categories: offsets must be contiguous int32 [m + 1] on {dev}")
        m, op = offsets.shape[0] - 1, offsets.data_ptr()
    ld_u, up = 0, None
    if uniforms is not None:
        if uniforms.dim() == 1 and m == 1:
            uniforms = uniforms.reshape(-1, 1)
        rows, cols, ld_u = _matrix(uniforms, "sample_categories: uniforms")
        if uniforms.dtype is not torch.float32 or (rows, cols) != (B, m) or uniforms.device != dev:
            _refuse(f"sample_categories: uniforms must be float32 [{B},{m}] on {dev}, got {uniforms.dtype} [{rows},{cols}] on {uniforms.device}")
        up = uniforms.data_ptr()
    if max_classes is None or max_classes > sumk:
        max_classes = sumk
    elif max_classes < 0:
        _refuse(f"sample_categories: max_classes {max_classes}")
    if out is None:
        out = torch.empty((B, m), device=dev, dtype=torch.int32)
    elif out.dtype is not torch.int32 or out.shape != (B, m) or not out.is_contiguous() or out.device != dev:
        _refuse(f"sample_categories: out must be contiguous int32 [{B},{m}] on {dev}")
    elif B:
        row = 4 * m
        whole = {n: _spread(v) for n, v in zip(_CHOICE_RANGE, (temperature, top_p, min_p, top_k)) if isinstance(v, torch.Tensor) and v.numel()}
        _not_over("sample_categories", ((out.data_ptr(), B * row, B * row, 1),), logits=_parts(logits, B, sumk, ld) if sumk else (),
                  offsets=((op, row + 4, row + 4, 1),) if op else (), uniforms=_parts(uniforms, B, m, ld_u) if up else (), **whole)
    values = temperature, top_p, min_p, top_k
    c = _choice_numbers(*values) if _NUMBERS.issuperset(map(type, values)) else _choice_args(dev, B, m, zip(_CHOICE_RANGE, values))
    lp = torch.empty((B, m), device=dev, dtype=torch.float32) if log_prob else None
    need, ws = 0, None
    if max_classes > 2048:
        need = _function("clava_choice_workspace_bytes", "iiii", c_ll)(B, m, sumk, max_classes)
        if need:
            ws = torch.empty(need, device=dev, dtype=torch.uint8)
    _launch(dev, "clava_sample_categories", _function("clava_sample_categories", "piliiipipplUUuppplp"),
            logits.data_ptr(), dt, ld, B, m, sumk, op, max_classes, ctypes.byref(c), up, ld_u, seed & 0xFFFFFFFFFFFFFFFF,
            row_offset & 0xFFFFFFFFFFFFFFFF, step_index & 0xFFFFFFFF, out.data_ptr(), None if lp is None else lp.data_ptr(),
            None if ws is None else ws.data_ptr(), need)
    return (out, lp) if log_prob else out
