"""The root-mean-square norm in front of a block's linears, with the residual's
addition, its gradient, and its 8-bit form for linears that share their input:

    y, h = rms_norm(x, weight, residual)                          # h = x + residual goes on as the stream
    rows, h = rms_norm_int8(x, weight, residual, i8t=True)        # y rotated and quantized once
    q = convrot_w8a8_linear_rows(rows, wq, sq, qweight_i8t=wq8t)  # ... for each of its linears
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import native
from .experts import _no_tangent, _restored
from .mxfp4 import _check_dtype, _count, _no_grad, _same_device


class Int8Rows(NamedTuple):
    """Rows rotated and quantized to 8 bits: ``codes`` int8 times ``scales`` f32 [M],
    a row's.  ``codes`` is [M, K], or in the I8T layout (``i8t``) of the linear's
    matrix product, [M padded to 256, K].  ``shape`` [..., K] and ``dtype`` are the rows' before,
    M the product of the leading sizes; ``convrot_groupsize`` the rotation's."""
    codes: torch.Tensor
    scales: torch.Tensor
    shape: tuple
    dtype: torch.dtype
    convrot_groupsize: int
    i8t: bool

    def check(self) -> None:
        """Raises ValueError where the tensors are no such rows."""
        c, s = self.codes, self.scales
        K = self.shape[-1]
        M = 1
        for n in self.shape[:-1]:
            M *= n
        want = (native.i8t_rows(M) if self.i8t else M, K)
        if c.dtype != torch.int8 or s.dtype != torch.float32 or tuple(c.shape) != want or tuple(s.shape) != (M,) \
                or c.device != s.device:
            raise ValueError(f"8-bit rows of shape {tuple(self.shape)} (i8t={self.i8t}) are int8 {want} and float32 {(M,)} of one "
                             f"device, got {c.dtype} {tuple(c.shape)} and {s.dtype} {tuple(s.shape)}")
        if self.dtype not in native._IN_DTYPE_CODE:
            raise ValueError(f"rows must be of float32, bfloat16 or float16, got {self.dtype}")


def max_norm_width() -> int:
    """Widest row that the norm takes: 32768."""
    return native._limit("cr_max_norm_width")


def _check(x, weight, residual, eps):
    _check_dtype(x, "x")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"x must be [..., D], got shape {tuple(x.shape)}")
    D = x.shape[-1]
    _count(x.numel() // D, "rows")
    if weight is not None:
        _check_dtype(weight, "weight")
        if tuple(weight.shape) != (D,):
            raise ValueError(f"weight of shape {tuple(weight.shape)} does not fit: {(D,)} expected")
    if residual is not None and (residual.dtype != x.dtype or residual.shape != x.shape):
        raise ValueError(f"residual {residual.dtype} {tuple(residual.shape)} does not fit x {x.dtype} {tuple(x.shape)}")
    if not 0.0 <= float(eps) < float("inf"):
        raise ValueError(f"eps must be at least 0 and finite, got {eps}")
    _same_device(x, weight, residual)
    if D > max_norm_width():
        raise ValueError(f"rows of {D} are too wide: at most {max_norm_width()}")


def _code(t):
    return 0 if t is None else native._IN_DTYPE_CODE[t.dtype]


def _ready(t):
    return None if t is None else native._aligned(t)


def _norm(x, weight, residual, eps):
    lib = native.load_library()
    x2, w, r = native._aligned(x), _ready(weight), _ready(residual)
    D = x.shape[-1]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    h = None if r is None else torch.empty_like(y)
    with native.on_device(x.device):
        rc = lib.cr_rms_norm(x2.data_ptr(), _code(x), native._ptr(r), native._ptr(w), _code(w), native._ptr(h), y.data_ptr(),
                             x2.numel() // D, D, eps, native._stream(x.device))
    if rc != 0:
        raise RuntimeError(f"cr_rms_norm failed, hipError={rc}")
    return y, x2 if h is None else h


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, h = _norm(x, weight, residual, eps)
        ctx.save_for_backward(x if residual is None else h, weight)
        ctx.like, ctx.weight, ctx.eps = (x.dtype, x.shape, x.device), None if weight is None else weight.dtype, eps
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, h)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_y, d_h=None):
        (dtype, shape, dev), D = ctx.like, ctx.like[1][-1]
        need_x, need_w = ctx.needs_input_grad[0] or ctx.needs_input_grad[2], ctx.needs_input_grad[1]
        h, weight = ctx.saved_tensors
        if d_y is None:
            d_x, d_w = d_h, None
        else:
            h = _restored(h, "rows", dtype, shape, dev)
            w = None if ctx.weight is None else _restored(weight, "weight", ctx.weight, (D,), dev)
            d_x, d_w = _norm_grad(native._aligned(d_y), _ready(d_h), h, w, ctx.eps, need_x, need_w)
        return (d_x if ctx.needs_input_grad[0] else None, d_w, d_x if ctx.needs_input_grad[2] else None, None)


def _norm_grad(d_y, d_h, h, w, eps, need_x, need_w):
    lib = native.load_library()
    D, dev = h.shape[-1], h.device
    M = h.numel() // D
    d_x = torch.empty_like(h) if need_x else None
    d_w = torch.empty_like(w) if need_w else None
    if M == 0:
        return d_x, None if d_w is None else d_w.zero_()
    nbytes = lib.cr_rms_norm_grad_workspace(M, D) if need_w else 0
    st = native._stream(dev)
    with native.on_device(dev), native._call_lock(dev, st):
        work = native._workspace(dev, st, nbytes)
        rc = lib.cr_rms_norm_grad(d_y.data_ptr(), native._ptr(d_h), h.data_ptr(), _code(h), native._ptr(w), _code(w), native._ptr(d_x),
                                  native._ptr(d_w), M, D, eps, work.data_ptr(), nbytes, st)
    if rc != 0:
        raise RuntimeError(f"cr_rms_norm_grad failed, hipError={rc}")
    return d_x, d_w


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None, eps: float = 1e-6):
    """y = h / sqrt(mean(h^2) + eps) * weight over the last axis, with h = x; or, given a
    ``residual`` of x's shape and type, (y, h) with h = x + residual in their type, so
    that the norm is of the stream as it goes on.  weight [D] is of any of the three
    types (None: ones); y is of x's type, rounded once from 32 bits, the squares added in 64.

    Differentiable in x, weight and residual (x and residual share one gradient
    tensor, as those of a sum do).  The weight's is summed over rows in a fixed order."""
    if x.is_cuda:
        host = native.host_or_none()
        p = None if host is None else host.rms_norm(x, weight, residual, eps)
        if p is not None:
            return p
    native.check_runs("rms_norm", x, weight, residual)
    _check(x, weight, residual, eps)
    _no_tangent("rms_norm", x, weight, residual)
    eps = float(eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        return _Norm.apply(x, weight, residual, eps)
    y, h = _norm(x, weight, residual, eps)
    return y if residual is None else (y, h)


def rms_norm_int8(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None, eps: float = 1e-6,
                  convrot_groupsize: int = 256, *, i8t: bool = False):
    """:func:`rms_norm` with y rotated in groups of ``convrot_groupsize`` and quantized to
    8 bits, as :func:`convrot_w8a8_linear_rows` takes it: Int8Rows, or (Int8Rows, h)
    given a residual.  A row's scale is max(max|z|, 1e-10) / 127 in float32 of its
    rotated values z and its codes the nearest of z / scale, ties to even; z is held
    in 64 bits and y not rounded before.  A row with a value that is not finite gets
    scale NaN and codes 0.  ``i8t``: the codes in the layout of the linear's matrix
    product (rows in whole multiples of 64).  Without a gradient."""
    if x.is_cuda:
        host = native.host_or_none()
        p = None if host is None else host.rms_norm_int8(x, weight, residual, eps, convrot_groupsize, i8t)
        if p is not None:
            rows = Int8Rows(p[0], p[1], tuple(x.shape), x.dtype, convrot_groupsize, i8t)
            return rows if residual is None else (rows, p[2])
    native.check_runs("rms_norm_int8", x, weight, residual)
    if convrot_groupsize not in (16, 64, 256):
        raise ValueError(f"convrot_groupsize must be 16, 64 or 256, got {convrot_groupsize}")
    D = x.shape[-1] if x.dim() else 0
    if D % convrot_groupsize:
        raise ValueError(f"rows of {D} are not divisible by convrot_groupsize {convrot_groupsize}")
    if i8t and D % 64:
        raise ValueError(f"I8T rows are whole multiples of 64, got {D}")
    _check(x, weight, residual, eps)
    _no_grad("rms_norm_int8", x, weight, residual)
    lib = native.load_library()
    x2, w, r = native._aligned(x), _ready(weight), _ready(residual)
    M = x2.numel() // D
    codes = torch.empty((native.i8t_rows(M) if i8t else M, D), dtype=torch.int8, device=x.device)
    scales = torch.empty((M,), dtype=torch.float32, device=x.device)
    h = None if r is None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    with native.on_device(x.device):
        rc = lib.cr_rms_norm_int8(x2.data_ptr(), _code(x), native._ptr(r), native._ptr(w), _code(w), native._ptr(h), codes.data_ptr(),
                                  scales.data_ptr(), M, D, convrot_groupsize, bool(i8t), float(eps), native._stream(x.device))
    if rc != 0:
        raise RuntimeError(f"cr_rms_norm_int8 failed, hipError={rc}")
    rows = Int8Rows(codes, scales, tuple(x.shape), x.dtype, convrot_groupsize, bool(i8t))
    return rows if residual is None else (rows, h)


def convrot_w8a8_linear_rows(rows: Int8Rows, qweight: torch.Tensor, wscales: torch.Tensor, bias: torch.Tensor | None = None, *,
                             qweight_i8t: torch.Tensor | None = None) -> torch.Tensor:
    """``convrot_w8a8_linear`` of rows that are quantized already: [..., N] in the rows'
    type, the same matrix product and epilogue.  qweight int8 [N, K], rotated in the
    groups the rows were, with wscales [N] f32; bias [N].  ``qweight_i8t`` is
    ``prepare_convrot_w8a8_weight_i8t(qweight)``, made here when rows in the I8T layout
    come without it."""
    if rows.i8t and rows.codes.is_cuda and rows.dtype in native._IN_DTYPE_CODE:
        host = native.host_or_none()
        y = None if host is None else host.w8a8_rows(rows.codes, rows.scales, rows.shape, native._IN_DTYPE_CODE[rows.dtype], qweight,
                                                     wscales, bias, qweight_i8t)
        if y is not None:
            return y
    native.check_runs("convrot_w8a8_linear_rows", rows.codes, rows.scales, qweight, wscales, bias, qweight_i8t)
    rows.check()
    K = rows.shape[-1]
    if qweight.dtype != torch.int8 or qweight.dim() != 2 or qweight.shape[1] != K:
        raise ValueError(f"qweight {qweight.dtype} {tuple(qweight.shape)} does not fit rows of {K}: int8 [N, {K}] expected")
    N = qweight.shape[0]
    if wscales.dtype != torch.float32 or wscales.numel() != N:
        raise ValueError(f"wscales must be float32 of {N} elements, got {wscales.dtype} {tuple(wscales.shape)}")
    if bias is not None:
        _check_dtype(bias, "bias")
        if bias.numel() != N:
            raise ValueError(f"bias has {bias.numel()} elements, the weight has N={N} rows")
    if qweight_i8t is not None and (qweight_i8t.dtype != torch.int8 or tuple(qweight_i8t.shape) != (native.i8t_rows(N), K)):
        raise ValueError(f"qweight_i8t {qweight_i8t.dtype} {tuple(qweight_i8t.shape)} does not fit: int8 {(native.i8t_rows(N), K)} expected")
    _no_grad("convrot_w8a8_linear_rows", rows.scales, wscales, bias)
    _same_device(rows.codes, rows.scales, qweight, wscales, bias, qweight_i8t)
    dev, M = rows.codes.device, rows.scales.shape[0]
    out_shape = (*rows.shape[:-1], N)
    with native.on_device(dev):
        if not rows.i8t:
            f32 = rows.dtype == torch.float16
            out = native.int8_convrot_gemm(rows.codes, qweight, rows.scales, wscales.reshape(-1), None if bias is None else bias.reshape(-1),
                                           torch.float32 if f32 else rows.dtype)
            return (out.to(torch.float16) if f32 else out).reshape(out_shape)
        lib = native.load_library()
        w = native._aligned(native.int8_to_i8t(qweight) if qweight_i8t is None else qweight_i8t)
        out = torch.empty(out_shape, dtype=rows.dtype, device=dev)
        codes, xs, ws, b = native._aligned(rows.codes), native._aligned(rows.scales), native._aligned(wscales), _ready(bias)
        epi = {torch.float32: native.EPI_F32, torch.bfloat16: native.EPI_BF16, torch.float16: native.EPI_F16}[rows.dtype]
        nbytes = lib.cr_w8a8_rows_linear_workspace(M, N, K)
        st = native._stream(dev)
        with native._call_lock(dev, st):
            work = native._workspace(dev, st, nbytes)
            rc = lib.cr_w8a8_rows_linear(codes.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), native._ptr(b), _code(b),
                                         out.data_ptr(), epi, M, N, K, work.data_ptr(), nbytes, st)
    if rc != 0:
        raise RuntimeError(f"cr_w8a8_rows_linear failed, hipError={rc}")
    return out
