"""A router's choice: the experts of each token and their weights, from the
router's logits, with the gradient of the weights.

    ids, weights = choose_experts(logits, 8, balance_bias, scoring="sigmoid", num_groups=8, top_groups=4)
    plan = sort_tokens_by_expert(ids, E)                  # experts.py goes on from here
"""
from __future__ import annotations

import math
import operator

import torch

from . import native
from .experts import _no_tangent, _restored, max_experts
from .mxfp4 import _check_dtype, _count, _same_device

_SCORING = ("softmax", "sigmoid")
_GROUP_SCORES = ("max", "sum2")


def _choose(logits, bias, k, sigmoid, groups, top_groups, sum2, renormalize, scale):
    lib = native.load_library()
    l2 = native._aligned(logits)
    T, E = logits.numel() // logits.shape[-1], logits.shape[-1]
    ids = torch.empty((*logits.shape[:-1], k), dtype=torch.int32, device=logits.device)
    weights = torch.empty((*logits.shape[:-1], k), dtype=torch.float32, device=logits.device)
    b = None if bias is None else native._aligned(bias.detach().to(torch.float32))
    with native.on_device(logits.device):
        rc = lib.cr_choose_experts(l2.data_ptr(), native._IN_DTYPE_CODE[logits.dtype], native._ptr(b), ids.data_ptr(),
                                   weights.data_ptr(), T, E, k, sigmoid, groups, top_groups, sum2, renormalize, scale,
                                   native._stream(logits.device))
    if rc != 0:
        raise RuntimeError(f"cr_choose_experts failed, hipError={rc}")
    return ids, weights


class _Choose(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, k, sigmoid, groups, top_groups, sum2, renormalize, scale):
        ids, weights = _choose(logits, bias, k, sigmoid, groups, top_groups, sum2, renormalize, scale)
        ctx.save_for_backward(logits, ids)
        ctx.shape, ctx.dtype, ctx.how = logits.shape, logits.dtype, (sigmoid, renormalize, scale)
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        return ids, weights

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, _, d_weights):
        if d_weights is None:
            return (None,) * 9
        logits, ids = ctx.saved_tensors
        dev, (sigmoid, renormalize, scale) = d_weights.device, ctx.how
        logits = _restored(logits, "logits", ctx.dtype, ctx.shape, dev)
        ids = _restored(ids, "ids", torch.int32, d_weights.shape, dev)
        d_weights = native._aligned(d_weights)
        d_logits = torch.empty_like(logits)
        E, k = logits.shape[-1], ids.shape[-1]
        with native.on_device(dev):
            rc = native.load_library().cr_choose_experts_grad(
                logits.data_ptr(), native._IN_DTYPE_CODE[logits.dtype], ids.data_ptr(), d_weights.data_ptr(), d_logits.data_ptr(),
                logits.numel() // E, E, k, sigmoid, renormalize, scale, native._stream(dev))
        if rc != 0:
            raise RuntimeError(f"cr_choose_experts_grad failed, hipError={rc}")
        return (d_logits,) + (None,) * 8


def choose_experts(logits: torch.Tensor, top_k: int, balance_bias: torch.Tensor | None = None, *, scoring: str = "softmax",
                   num_groups: int = 1, top_groups: int | None = None, group_score: str = "max", renormalize: bool = True,
                   scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """logits [..., E] -> (expert_ids int32 [..., k], weights float32 [..., k]).

    Scores are softmax(logits) or sigmoid(logits) (``scoring``).  The choice goes by
    score + ``balance_bias`` [E] (which only chooses: the weights are the scores').
    With ``num_groups`` the E experts are that many equal groups in order, ranked by
    their greatest choice (``group_score`` "max") or the sum of their two greatest
    ("sum2"), and only experts of the ``top_groups`` greatest groups are chosen (None:
    of all).  The k greatest are returned greatest first; ties, of choices that
    agree to 43 bits (or to 2^-1064: a bias of 0 and a score below exp(-737)), go to
    the lowest index, and without a bias the order is the logits' own.  The weights are the chosen scores, divided by their sum where
    ``renormalize``, times ``scale``.

    An expert whose logit (or bias) is -inf is not available.  A slot for which no
    expert is left has id -1 and weight 0, which the routing takes for an unused
    slot.  A NaN ranks with +inf, and every weight that depends on it is NaN.

    Differentiable in the logits, for a given choice; ids and the bias have no gradient."""
    if logits.is_cuda and scoring in _SCORING and group_score in _GROUP_SCORES:
        host = native.host_or_none()
        p = None if host is None else host.choose_experts(logits, top_k, balance_bias, scoring == "sigmoid", num_groups,
                                                          top_groups, group_score == "sum2", renormalize, scale)
        if p is not None:
            return p
    native.check_runs("choose_experts", logits, balance_bias)
    _check_dtype(logits, "logits")
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise ValueError(f"logits must be [..., E], got shape {tuple(logits.shape)}")
    E = logits.shape[-1]
    top_k, num_groups = operator.index(top_k), operator.index(num_groups)
    if scoring not in _SCORING:
        raise ValueError(f"scoring must be one of {_SCORING}, got {scoring!r}")
    if group_score not in _GROUP_SCORES:
        raise ValueError(f"group_score must be one of {_GROUP_SCORES}, got {group_score!r}")
    if not 1 <= num_groups or E % num_groups:
        raise ValueError(f"{E} experts are not num_groups={num_groups} equal groups")
    top_groups = num_groups if top_groups is None else operator.index(top_groups)
    if not 1 <= top_groups <= num_groups:
        raise ValueError(f"top_groups must be 1 to {num_groups}, got {top_groups}")
    if not 1 <= top_k <= E // num_groups * top_groups:
        raise ValueError(f"top_k must be 1 to {E // num_groups * top_groups}, got {top_k}")
    scale = float(scale)
    if not math.isfinite(scale) or abs(scale) > torch.finfo(torch.float32).max:
        raise ValueError(f"scale must be finite in float32, got {scale}")
    _count(logits.numel() // E * top_k, "slots")
    if balance_bias is not None:
        _check_dtype(balance_bias, "balance_bias")
        if tuple(balance_bias.shape) != (E,):
            raise ValueError(f"balance_bias of shape {tuple(balance_bias.shape)} does not fit: {(E,)} expected")
    _same_device(logits, balance_bias)
    if E > max_experts():
        raise ValueError(f"{E} experts are too many: at most {max_experts()} experts")
    _no_tangent("choose_experts", logits, balance_bias)
    how = (top_k, scoring == "sigmoid", num_groups, top_groups, group_score == "sum2", bool(renormalize), scale)
    if torch.is_grad_enabled() and logits.requires_grad:
        return _Choose.apply(logits, balance_bias, *how)
    return _choose(logits, balance_bias, *how)
