"""Expert routing: tokens sorted by expert, their rows gathered, the experts'
outputs added up per token with the router's weights, and the gradients of both.

    plan = sort_tokens_by_expert(ids, E)                  # ids [T, k]: the router's choice
    rows = gather_expert_rows(x, plan)                    # [T k, D], expert after expert
    ...                                                   # the experts, on rows offsets[e] .. offsets[e + 1] - 1
    y = combine_expert_rows(rows, weights, plan)          # [T, D]

Token t's slot j has the number t k + j; an id outside [0, E) leaves the slot
unused (a dropped or a padded token).  Sums run over a token's slots in order, in
fp32, without atomics: the same inputs give the same bits.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import native
from .mxfp4 import _check_dtype, _count, _same_device


class ExpertPlan(NamedTuple):
    """Where each slot's row goes.  ``order`` int32 [T k]: the slot of each sorted
    row, -1 past the last used one.  ``position`` int32 [T, k]: the sorted row of
    each slot, -1 for an unused one.  ``offsets`` int32 [E + 1]: expert e has the
    rows offsets[e] .. offsets[e + 1] - 1.  Rows of one expert are in slot order."""
    order: torch.Tensor
    position: torch.Tensor
    offsets: torch.Tensor

    @property
    def num_experts(self) -> int:
        return self.offsets.shape[0] - 1

    def check(self, E: int | None = None) -> None:
        """Raises ValueError where the tensors are no plan (of E experts)."""
        o, p, f = self.order, self.position, self.offsets
        if any(t.dtype != torch.int32 or not t.is_contiguous() or t.is_neg() for t in (o, p, f)) or p.dim() != 2 or o.dim() != 1 \
                or f.dim() != 1 or o.shape[0] != p.numel() or f.shape[0] < 2 or p.shape[1] < 1 \
                or not (o.device == p.device == f.device):
            raise ValueError("a plan is contiguous int32 tensors order [T k], position [T, k] and offsets [E + 1] of one "
                             f"device, got {tuple(o.shape)}, {tuple(p.shape)}, {tuple(f.shape)}")
        if o.shape[0] >= 1 << 31:
            raise ValueError(f"{o.shape[0]} slots are more than one plan holds (2^31 - 1)")
        if E is not None and f.shape[0] != E + 1:
            raise ValueError(f"the plan is of {f.shape[0] - 1} experts, the weights are of {E}")


def max_experts() -> int:
    """Most experts a plan can have: 1024."""
    return native._limit("cr_max_experts")


def sort_tokens_by_expert(expert_ids: torch.Tensor, num_experts: int) -> ExpertPlan:
    """The plan of expert_ids [T, k] (int32 or int64): a stable counting sort of the
    slots by expert, without a host synchronization."""
    if expert_ids.is_cuda:
        host = native.host_or_none()
        p = None if host is None else host.expert_sort(expert_ids, num_experts)
        if p is not None:
            return ExpertPlan(*p)
    native.check_runs("sort_tokens_by_expert", expert_ids)
    if expert_ids.dim() != 2 or expert_ids.shape[1] < 1:
        raise ValueError(f"expert_ids must be [T, k], got shape {tuple(expert_ids.shape)}")
    if expert_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"expert_ids must be int32 or int64, got {expert_ids.dtype}")
    native._check_cuda(expert_ids)
    lib = native.load_library()
    if not 1 <= num_experts <= max_experts():
        raise ValueError(f"num_experts must be 1 to {max_experts()}, got {num_experts}")
    ids = native._aligned(expert_ids)
    T, k = ids.shape
    R = T * k
    if R >= 1 << 31:
        raise ValueError(f"{R} slots are more than one plan holds (2^31 - 1)")
    dev = ids.device
    order = torch.empty((R,), dtype=torch.int32, device=dev)
    position = torch.empty((T, k), dtype=torch.int32, device=dev)
    offsets = torch.empty((num_experts + 1,), dtype=torch.int32, device=dev)
    nbytes = lib.cr_expert_sort_workspace(R, num_experts)
    st = native._stream(dev)
    with native.on_device(dev), native._call_lock(dev, st):
        work = native._workspace(dev, st, nbytes)
        rc = lib.cr_expert_sort(ids.data_ptr(), ids.element_size(), order.data_ptr(), position.data_ptr(),
                                offsets.data_ptr(), R, num_experts, work.data_ptr(), nbytes, st)
    if rc != 0:
        raise RuntimeError(f"cr_expert_sort failed, hipError={rc}")
    return ExpertPlan(order, position, offsets)


def _no_tangent(what, *ts):
    if native.has_tangent(*ts):
        raise RuntimeError(f"{what} has no forward-mode gradient")


def _gather(x, plan):
    lib = native.load_library()
    (T, k), D, E = plan.position.shape, x.shape[1], plan.num_experts
    x = native._aligned(x)
    rows = torch.empty((T * k, D), dtype=x.dtype, device=x.device)
    if D == 0:
        return rows
    with native.on_device(x.device):
        rc = lib.cr_expert_gather(x.data_ptr(), native._IN_DTYPE_CODE[x.dtype], plan.position.data_ptr(),
                                  plan.offsets.data_ptr(), rows.data_ptr(), T, k, E, D, native._stream(x.device))
    if rc != 0:
        raise RuntimeError(f"cr_expert_gather failed, hipError={rc}")
    return rows


def _combine(rows, weights, position):
    lib = native.load_library()
    (T, k), D = position.shape, rows.shape[1]
    rows = native._aligned(rows)
    out = torch.empty((T, D), dtype=rows.dtype, device=rows.device)
    if D == 0:
        return out
    with native.on_device(rows.device):
        rc = lib.cr_expert_combine(rows.data_ptr(), native._IN_DTYPE_CODE[rows.dtype], native._ptr(weights),
                                   position.data_ptr(), out.data_ptr(), T, k, D, native._stream(rows.device))
    if rc != 0:
        raise RuntimeError(f"cr_expert_combine failed, hipError={rc}")
    return out


def _restored(t, what, dtype, shape, device):
    """A saved tensor as the kernels take it: hooks on saved tensors may hand back
    another one than was saved."""
    if type(t) not in (torch.Tensor, torch.nn.Parameter) or t.layout != torch.strided or t.dtype != dtype \
            or tuple(t.shape) != tuple(shape) or t.device != device:
        raise RuntimeError(f"the saved {what} came back in another form: {dtype} {tuple(shape)} on {device} expected, got "
                           f"{t.dtype} {tuple(t.shape)} on {t.device}")
    return native._aligned(t)


class _Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        ctx.save_for_backward(plan.position)
        ctx.slots = plan.position.shape
        return _gather(x, plan)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_rows):
        position = _restored(ctx.saved_tensors[0], "positions", torch.int32, ctx.slots, d_rows.device)
        return _combine(d_rows, None, position), None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, plan):
        w = native._aligned(weights.to(torch.float32))
        ctx.save_for_backward(rows, w, plan.position, plan.offsets)
        ctx.slots, ctx.offsets, ctx.weights_dtype = plan.position.shape, plan.offsets.shape, weights.dtype
        return _combine(rows, w, plan.position)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        rows, w, position, offsets = ctx.saved_tensors
        (T, k), D, E, dev = ctx.slots, d_out.shape[1], ctx.offsets[0] - 1, d_out.device
        rows = _restored(rows, "rows", d_out.dtype, (T * k, D), dev)
        w = _restored(w, "weights", torch.float32, ctx.slots, dev)
        position = _restored(position, "positions", torch.int32, ctx.slots, dev)
        offsets = _restored(offsets, "offsets", torch.int32, ctx.offsets, dev)
        need_rows, need_weights = ctx.needs_input_grad[:2]
        d_out = native._aligned(d_out)
        d_rows = torch.empty_like(rows) if need_rows else None
        d_w = torch.empty((T, k), dtype=torch.float32, device=dev) if need_weights else None
        if D == 0:
            return d_rows, None if d_w is None else d_w.zero_().to(ctx.weights_dtype), None
        with native.on_device(dev):
            rc = native.load_library().cr_expert_combine_grad(
                rows.data_ptr(), native._IN_DTYPE_CODE[rows.dtype], w.data_ptr(), position.data_ptr(), offsets.data_ptr(),
                d_out.data_ptr(), native._ptr(d_rows), native._ptr(d_w), T, k, E, D, native._stream(dev))
        if rc != 0:
            raise RuntimeError(f"cr_expert_combine_grad failed, hipError={rc}")
        return d_rows, None if d_w is None else d_w.to(ctx.weights_dtype), None


def gather_expert_rows(x: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """x [T, D] -> rows [T k, D] in the plan's order (row r is token order[r] // k);
    rows past the last used one are zero.  Differentiable: a token's gradient is
    the sum of its rows', in fp32, rounded once."""
    if x.is_cuda:
        host = native.host_or_none()
        rows = None if host is None else host.expert_gather(x, plan.order, plan.position, plan.offsets)
        if rows is not None:
            return rows
    native.check_runs("gather_expert_rows", x, *plan)
    _check_dtype(x, "x")
    plan.check()
    if x.dim() != 2 or x.shape[0] != plan.position.shape[0]:
        raise ValueError(f"x of shape {tuple(x.shape)} does not fit a plan of {plan.position.shape[0]} tokens")
    _count(x.shape[1], "columns")
    _same_device(x, plan.order)
    _no_tangent("gather_expert_rows", x)
    if torch.is_grad_enabled() and x.requires_grad:
        return _Gather.apply(x, plan)
    return _gather(x, plan)


def combine_expert_rows(rows: torch.Tensor, weights: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """out[t] = sum_j weights[t, j] * rows[position[t, j]] over token t's used slots:
    rows [T k, D] in the plan's order, weights [T, k] of any of the three types,
    out [T, D] in the rows' type, summed in fp32 and rounded once.  A token without
    a used slot gets zeros.  Differentiable in the rows and the weights."""
    if rows.is_cuda:
        host = native.host_or_none()
        out = None if host is None else host.expert_combine(rows, weights, plan.order, plan.position, plan.offsets)
        if out is not None:
            return out
    native.check_runs("combine_expert_rows", rows, weights, *plan)
    _check_dtype(rows, "rows")
    _check_dtype(weights, "weights")
    plan.check()
    T, k = plan.position.shape
    if rows.dim() != 2 or rows.shape[0] != T * k:
        raise ValueError(f"rows of shape {tuple(rows.shape)} do not fit a plan of {T * k} rows")
    if tuple(weights.shape) != (T, k):
        raise ValueError(f"weights of shape {tuple(weights.shape)} do not fit: {(T, k)} expected")
    _count(rows.shape[1], "columns")
    _same_device(rows, weights, plan.order)
    _no_tangent("combine_expert_rows", rows, weights)
    if torch.is_grad_enabled() and (rows.requires_grad or weights.requires_grad):
        return _Combine.apply(rows, weights, plan)
    return _combine(rows, native._aligned(weights.to(torch.float32)), plan.position)
