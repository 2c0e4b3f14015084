"""A mixture-of-experts feed-forward on microscaled 4-bit weights: what the
operators of ``_int4.mxfp4`` and ``_int4.experts`` are for, run together.

    moe = Mxfp4MoE.from_float(w_gate, w_up, w_down, convrot_groupsize=256)
    y = moe(x, expert_ids, weights)

``x`` is [..., D], ``expert_ids`` [..., k] the router's choice (an id outside
[0, E) leaves a slot unused), ``weights`` [..., k] what it gives each, with the
same leading sizes.  A token's output is
``sum_j weights[j] * down_e(silu(gate_e(x)) * up_e(x))``.  The experts are frozen
and run without a graph; the router's weights get their gradient, so a router
can be trained over them.

    block = RoutedMxfp4MoE(moe, router_weight, norm_weight, top_k=4)
    y, h = block(x, residual)

is a block's feed-forward whole: the residual's addition, the norm, the router and
its choice in front of the experts.
"""
from __future__ import annotations

import torch

from . import _int4


class Mxfp4MoE(torch.nn.Module):
    """Experts' weights as buffers: ``w1`` / ``s1`` [E, 2 F, D] (gate rows, then up
    rows) and ``w2`` / ``s2`` [E, D, F], codes and scales of quantize_mxfp4."""

    def __init__(self, w1, s1, w2, s2, convrot_groupsize: int | None = None):
        super().__init__()
        E, F2, D2 = w1.shape
        if F2 % 2 or w2.shape != (E, 2 * D2, F2 // 4):
            raise ValueError(f"down codes of shape {tuple(w2.shape)} do not fit gate and up codes of shape "
                             f"{tuple(w1.shape)}")
        for name, t in (("w1", w1), ("s1", s1), ("w2", w2), ("s2", s2)):
            self.register_buffer(name, t)
        self.num_experts = E
        self.convrot_groupsize = convrot_groupsize

    @classmethod
    def from_float(cls, w_gate, w_up, w_down, convrot_groupsize: int | None = None) -> "Mxfp4MoE":
        """w_gate, w_up [E, F, D] and w_down [E, D, F] in float32, bfloat16 or float16, quantized on the GPU."""
        with torch.no_grad():
            w1 = _int4.quantize_mxfp4(torch.cat((w_gate, w_up), dim=1), convrot_groupsize)
            w2 = _int4.quantize_mxfp4(w_down, convrot_groupsize)
        return cls(*w1, *w2, convrot_groupsize)

    def forward(self, x: torch.Tensor, expert_ids: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        if torch.is_grad_enabled() and x.requires_grad:
            raise RuntimeError("the experts are frozen: gradients reach the router's weights only; pass x.detach()")
        if expert_ids.dim() == 0 or weights.shape != expert_ids.shape or expert_ids.shape[:-1] != x.shape[:-1]:
            raise ValueError(f"expert_ids of shape {tuple(expert_ids.shape)} and weights of shape {tuple(weights.shape)} do not "
                             f"fit x of shape {tuple(x.shape)}")
        k = expert_ids.shape[-1]
        G = self.convrot_groupsize
        x2 = x.reshape(-1, x.shape[-1])
        plan = _int4.sort_tokens_by_expert(expert_ids.reshape(-1, k), self.num_experts)
        with torch.no_grad():
            gate, up = _int4.mxfp4_expert_linear(x2, self.w1, self.s1, plan, convrot_groupsize=G).chunk(2, dim=-1)
            h = torch.nn.functional.silu(gate) * up
            rows = _int4.mxfp4_expert_linear(h, self.w2, self.s2, plan, convrot_groupsize=G, sorted_rows=True)
        return _int4.combine_expert_rows(rows, weights.reshape(-1, k), plan).reshape(x.shape)


class RoutedMxfp4MoE(torch.nn.Module):
    """Norm, router and experts: y = moe(n, choice of n's logits), n the norm of x, or of
    the stream h = x + residual, which is returned beside y.

    ``router_weight`` [E, D] is the one parameter (its logits are taken in float32);
    the norm's weight and the ``balance_bias`` [E] are buffers.  The other arguments
    are choose_experts'.  As the experts are frozen, x is too."""

    def __init__(self, moe: Mxfp4MoE, router_weight: torch.Tensor, norm_weight: torch.Tensor | None = None, *, top_k: int,
                 balance_bias: torch.Tensor | None = None, scoring: str = "softmax", num_groups: int = 1,
                 top_groups: int | None = None, group_score: str = "max", renormalize: bool = True, scale: float = 1.0,
                 eps: float = 1e-6):
        super().__init__()
        D = 2 * moe.w1.shape[-1]
        if tuple(router_weight.shape) != (moe.num_experts, D):
            raise ValueError(f"router_weight of shape {tuple(router_weight.shape)} does not fit {moe.num_experts} experts of {D}")
        self.moe = moe
        self.router_weight = torch.nn.Parameter(router_weight.detach())
        self.register_buffer("norm_weight", norm_weight)
        self.register_buffer("balance_bias", balance_bias)
        self.top_k, self.eps = top_k, eps
        self.how = dict(scoring=scoring, num_groups=num_groups, top_groups=top_groups, group_score=group_score,
                        renormalize=renormalize, scale=scale)

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, residual)):
            raise RuntimeError("the experts are frozen: gradients reach the router's weights only; pass x.detach()")
        with torch.no_grad():
            n = _int4.rms_norm(x, self.norm_weight, residual, self.eps)
        n, h = (n, None) if residual is None else n
        with torch.autocast(n.device.type, enabled=False):
            logits = torch.nn.functional.linear(n.to(torch.float32), self.router_weight.to(torch.float32))
        ids, weights = _int4.choose_experts(logits, self.top_k, self.balance_bias, **self.how)
        y = self.moe(n, ids, weights)
        return y if residual is None else (y, h)
