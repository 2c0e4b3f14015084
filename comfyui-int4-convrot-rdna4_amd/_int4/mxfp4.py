"""Microscaled 4-bit floats (MXFP4): the tier of linears whose weights and
activations are E2M1 codes with a power-of-two scale for every 32 values, which
gfx950's matrix cores multiply as they are.  0.53 bytes a weight, and no value
outside a block of 32 touches its scale.  The reference has no such tier; names,
rotation groups and calls follow the int4 one.

A quantized row of K values (K % 32 == 0) is K/2 bytes of codes (value 2j in the
low half of byte j) and K/32 scale bytes, byte s for 2^(s - 127), 255 for NaN.
``convrot_groupsize`` 16, 64 or 256 rotates x and W by the ConvRot Hadamard in
groups of that many values (the products stay the same, outliers are spread over
their group); None does not.

The forms here are for inference: they have no gradient, and refuse an input
that asks for one.  Their kernels are no torch operations, so a trace is refused
too.
"""
from __future__ import annotations

import torch

from . import native

_BLOCK = 32
_MAX_K = 1 << 24             # widest row that the library takes
_MAX_N = (1 << 31) - 256     # columns of a product


def _check_group(K: int, convrot_groupsize: int | None, what: str = "in_features") -> int:
    if K == 0 or K % _BLOCK:
        raise ValueError(f"{what} {K} is not a multiple of {_BLOCK}, the values that share a scale")
    if K > _MAX_K:
        raise ValueError(f"{what} {K} is too wide: at most {_MAX_K}")
    if convrot_groupsize is None:
        return 0
    if convrot_groupsize not in (16, 64, 256):
        raise ValueError(f"convrot_groupsize must be 16, 64, 256 or None, got {convrot_groupsize}")
    if K % convrot_groupsize:
        raise ValueError(f"{what} {K} not divisible by convrot_groupsize {convrot_groupsize}")
    return convrot_groupsize


def _check_dtype(t: torch.Tensor, what: str) -> int:
    code = native._IN_DTYPE_CODE.get(t.dtype)
    if code is None:
        raise ValueError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def _no_grad(what: str, *ts) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts) or native.has_tangent(*ts):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad() or on detached tensors")


def _same_device(*ts) -> None:
    native._check_cuda(*ts)
    devices = {t.device for t in ts if t is not None}
    if len(devices) > 1:
        raise RuntimeError(f"expected tensors on one device, got {sorted(map(str, devices))}")


def quantize_mxfp4(x: torch.Tensor, convrot_groupsize: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., K] -> (codes uint8 [..., K/2], scales uint8 [..., K/32]) on x's device.

    Per 32 values of a row (rotated first, in fp32, where a group size is given)
    the scale is 2^(floor(log2 max) - 2), not below 2^-127, and the codes are the
    nearest E2M1 values of y / scale, ties to even, magnitudes past 6 to 6.  A
    block that holds a NaN or an infinity is NaN as a whole (scale byte 255)."""
    if x.is_cuda:
        host = native.host_or_none()
        q = None if host is None else host.mx_quantize(x, convrot_groupsize)
        if q is not None:
            return q
    native.check_runs("quantize_mxfp4", x)
    dt = _check_dtype(x, "x")
    if x.dim() == 0:
        raise ValueError("x must have at least one dimension")
    K = x.shape[-1]
    G = _check_group(K, convrot_groupsize)
    M = _count(x.numel() // K, "rows")
    _no_grad("quantize_mxfp4", x)
    dev = x.device
    lib = native.load_library()
    xg = native._aligned(_on_gpu(x))
    codes = torch.empty((*x.shape[:-1], K // 2), dtype=torch.uint8, device=xg.device)
    scales = torch.empty((*x.shape[:-1], K // _BLOCK), dtype=torch.uint8, device=xg.device)
    with native.on_device(xg.device):
        rc = lib.cr_mxfp4_quant(xg.data_ptr(), dt, codes.data_ptr(), scales.data_ptr(), M, K, G,
                                native._stream(xg.device))
    if rc != 0:
        raise RuntimeError(f"cr_mxfp4_quant failed, hipError={rc}")
    return (codes, scales) if codes.device == dev else (codes.to(dev), scales.to(dev))


def dequantize_mxfp4(codes: torch.Tensor, scales: torch.Tensor, convrot_groupsize: int | None = None,
                     output_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values of codes [..., K/2] with scales [..., K/32], rotated back to the
    original basis where a group size is given: [..., K] in ``output_dtype``,
    rounded once, on the codes' device."""
    if codes.is_cuda and output_dtype in native._IN_DTYPE_CODE:
        host = native.host_or_none()
        x = None if host is None else host.mx_dequantize(codes, scales, convrot_groupsize,
                                                         native._IN_DTYPE_CODE[output_dtype])
        if x is not None:
            return x
    native.check_runs("dequantize_mxfp4", codes, scales)
    if output_dtype not in native._IN_DTYPE_CODE:
        raise ValueError(f"output_dtype must be float32, bfloat16 or float16, got {output_dtype}")
    _check_operand(codes, scales, codes.shape[:-1], codes.shape[-1] * 2 if codes.dim() else 0, "codes")
    K = codes.shape[-1] * 2
    G = _check_group(K, convrot_groupsize)
    M = _count(codes.numel() * 2 // K, "rows")
    dev = codes.device
    lib = native.load_library()
    c, s = native._aligned(_on_gpu(codes)), native._aligned(_on_gpu(scales))
    _same_device(c, s)
    out = torch.empty((*codes.shape[:-1], K), dtype=output_dtype, device=c.device)
    with native.on_device(c.device):
        rc = lib.cr_mxfp4_dequant(c.data_ptr(), s.data_ptr(), out.data_ptr(), native._IN_DTYPE_CODE[output_dtype],
                                  M, K, G, native._stream(c.device))
    if rc != 0:
        raise RuntimeError(f"cr_mxfp4_dequant failed, hipError={rc}")
    return out if out.device == dev else out.to(dev)


def mxfp4_linear(x: torch.Tensor, qweight: torch.Tensor, wscales: torch.Tensor, bias: torch.Tensor | None = None,
                 convrot_groupsize: int | None = None) -> torch.Tensor:
    """``x @ W.T + bias`` with x [..., K] quantized as :func:`quantize_mxfp4` does
    (rotated first where a group size is given) and W as that function returned it:
    qweight uint8 [N, K/2], wscales uint8 [N, K/32].  Products and sums in fp32;
    the output [..., N] has x's type and is rounded once.  bias [N] is float32,
    bfloat16 or float16."""
    if x.is_cuda:
        host = native.host_or_none()
        y = None if host is None else host.mx_linear(x, qweight, wscales, bias, convrot_groupsize)
        if y is not None:
            return y
    native.check_runs("mxfp4_linear", x, qweight, wscales, bias)
    dt = _check_dtype(x, "x")
    if x.dim() == 0:
        raise ValueError("x must have at least one dimension")
    K = x.shape[-1]
    if qweight.dim() != 2:
        raise ValueError(f"qweight must be 2-D, got shape {tuple(qweight.shape)}")
    if qweight.shape[-1] * 2 != K:
        raise ValueError(f"Input K={K} does not match qweight K={qweight.shape[-1] * 2}")
    G = _check_group(K, convrot_groupsize)
    M, N = _count(x.numel() // K, "rows"), _count(qweight.shape[0], "columns", _MAX_N)
    _check_operand(qweight, wscales, (N,), K, "qweight")
    bdt = _check_bias(bias, (N,))
    _no_grad("mxfp4_linear", x, bias)
    _same_device(x, qweight, wscales, bias)
    lib = native.load_library()
    x2 = native._aligned(x)
    w, ws = native._aligned(qweight), native._aligned(wscales)
    b = None if bias is None else native._aligned(bias)
    out = torch.empty((*x.shape[:-1], N), dtype=x.dtype, device=x.device)
    nbytes = lib.cr_mxfp4_linear_workspace(M, N, K, 1)
    st = native._stream(x.device)
    with native.on_device(x.device), native._call_lock(x.device, st):
        work = native._workspace(x.device, st, nbytes)
        rc = lib.cr_mxfp4_linear(x2.data_ptr(), dt, w.data_ptr(), ws.data_ptr(), native._ptr(b), bdt, out.data_ptr(), M,
                                 N, K, G, work.data_ptr(), nbytes, st)
    if rc != 0:
        raise RuntimeError(f"cr_mxfp4_linear failed, hipError={rc}")
    return out


def mxfp4_expert_linear(x: torch.Tensor, qweight: torch.Tensor, wscales: torch.Tensor, plan,
                        bias: torch.Tensor | None = None, convrot_groupsize: int | None = None, *,
                        sorted_rows: bool = False) -> torch.Tensor:
    """Every routed row times its expert's weights: [T k, N] in the plan's sorted order.

    qweight uint8 [E, N, K/2] and wscales uint8 [E, N, K/32] are the experts'
    weights, ``plan`` the :class:`ExpertPlan` of the router's choice
    (:func:`sort_tokens_by_expert`).  x is the tokens [T, K], whose rows are taken
    where the plan sends them (each is rotated and quantized once), or, with
    ``sorted_rows``, the T k rows [T k, K] already in the plan's order.  Row r of
    the output is x_r W_e^T + bias[e] for its expert e; rows past the last used
    one are zero.  Types and rounding as in :func:`mxfp4_linear`; bias is [E, N]."""
    if x.is_cuda:
        host = native.host_or_none()
        y = None if host is None else host.mx_expert_linear(x, qweight, wscales, plan.order, plan.position, plan.offsets,
                                                            bias, convrot_groupsize, sorted_rows)
        if y is not None:
            return y
    native.check_runs("mxfp4_expert_linear", x, qweight, wscales, bias, *plan)
    dt = _check_dtype(x, "x")
    if x.dim() != 2:
        raise ValueError(f"x must be 2-D, got shape {tuple(x.shape)}")
    K = x.shape[-1]
    if qweight.dim() != 3:
        raise ValueError(f"qweight must be 3-D, got shape {tuple(qweight.shape)}")
    if qweight.shape[-1] * 2 != K:
        raise ValueError(f"Input K={K} does not match qweight K={qweight.shape[-1] * 2}")
    G = _check_group(K, convrot_groupsize)
    E, N = qweight.shape[0], _count(qweight.shape[1], "columns", _MAX_N)
    _check_operand(qweight, wscales, (E, N), K, "qweight")
    plan.check(E)
    if E > native._limit("cr_max_experts"):
        raise ValueError(f"{E} experts are too many: at most {native._limit('cr_max_experts')} experts")
    T, k = plan.position.shape
    R = T * k
    if x.shape[0] != (R if sorted_rows else T):
        raise ValueError(f"x has {x.shape[0]} rows, the plan {R} sorted ones of {T} tokens "
                         f"(sorted_rows={sorted_rows})")
    bdt = _check_bias(bias, (E, N))
    _no_grad("mxfp4_expert_linear", x, bias)
    _same_device(x, qweight, wscales, bias, plan.order)
    lib = native.load_library()
    x2 = native._aligned(x)
    w, ws = native._aligned(qweight), native._aligned(wscales)
    b = None if bias is None else native._aligned(bias)
    out = torch.empty((R, N), dtype=x.dtype, device=x.device)
    nbytes = lib.cr_mxfp4_linear_workspace(x2.shape[0], N, K, E)
    st = native._stream(x.device)
    with native.on_device(x.device), native._call_lock(x.device, st):
        work = native._workspace(x.device, st, nbytes)
        rc = lib.cr_mxfp4_expert_linear(x2.data_ptr(), dt, None if sorted_rows else plan.order.data_ptr(), max(k, 1),
                                        plan.offsets.data_ptr(), E, w.data_ptr(), ws.data_ptr(), native._ptr(b), bdt,
                                        out.data_ptr(), R, N, K, G, work.data_ptr(), nbytes, st)
    if rc != 0:
        raise RuntimeError(f"cr_mxfp4_expert_linear failed, hipError={rc}")
    return out


def _on_gpu(t: torch.Tensor) -> torch.Tensor:
    if t.is_cuda:
        return t
    if not torch.cuda.is_available():
        raise RuntimeError("the MXFP4 kernels need a gfx950 GPU; none is visible")
    return t.to("cuda")


def _count(n: int, what: str, most: int = (1 << 31) - 1) -> int:
    if n > most:
        raise ValueError(f"{n} {what} are more than one call takes ({most})")
    return n


def _check_operand(codes, scales, rows, K: int, what: str) -> None:
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError(f"{what} and its scales must be uint8, got {codes.dtype} and {scales.dtype}")
    if codes.dim() == 0 or K % _BLOCK or K == 0:
        raise ValueError(f"{what} of shape {tuple(codes.shape)} hold no whole blocks of {_BLOCK} values")
    if tuple(scales.shape) != (*rows, K // _BLOCK):
        raise ValueError(f"scales of shape {tuple(scales.shape)} do not fit {what} of shape {tuple(codes.shape)}: "
                         f"{(*rows, K // _BLOCK)} expected")


def _check_bias(bias, shape) -> int:
    if bias is None:
        return 0
    if tuple(bias.shape) != tuple(shape):
        raise ValueError(f"bias of shape {tuple(bias.shape)} does not fit: {tuple(shape)} expected")
    return _check_dtype(bias, "bias")
