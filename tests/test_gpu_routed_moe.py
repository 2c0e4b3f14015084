"""A block's feed-forward whole: residual and norm, router, choice, experts; and the router's gradient through all of it."""
import importlib

import pytest
import torch

from conftest import PKG_NAME
from test_gpu_choose import plain, weights_of

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def block_of(E, D, F, dtype, seed, **how):
    moe = importlib.import_module(PKG_NAME + ".mxfp4_moe")
    g = torch.Generator().manual_seed(seed)
    w = [(torch.randn(E, *s, generator=g) * s[-1] ** -0.5).cuda() for s in ((F, D), (F, D), (D, F))]
    experts = moe.Mxfp4MoE.from_float(*w, convrot_groupsize=16)
    router = (torch.randn(E, D, generator=g) * D ** -0.5).cuda()
    norm = (1 + 0.2 * torch.randn(D, generator=g)).to(dtype).cuda()
    bias = (torch.randint(-100, 101, (E,), generator=g) * 0.001).cuda()
    return moe.RoutedMxfp4MoE(experts, router, norm, balance_bias=bias, **how)


HOW = [dict(top_k=3), dict(top_k=4, scoring="sigmoid", num_groups=4, top_groups=2, group_score="sum2", scale=2.5),
       dict(top_k=2, renormalize=False)]


@pytest.mark.parametrize("how", HOW)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T", [1, 7, 130])
def test_block(backend, gpu, T, dtype, how):
    E, D, F = 8, 160, 224
    block = block_of(E, D, F, dtype, 3, **how)
    g = torch.Generator().manual_seed(T)
    x, r = (torch.randn(T, D, generator=g).to(dtype).cuda() for _ in range(2))
    y, h = block(x, r)
    assert torch.equal(h, (x.float() + r.float()).to(dtype))
    n, _ = backend.rms_norm(x, block.norm_weight, r)
    logits = torch.nn.functional.linear(n.float(), block.router_weight.detach())
    ids, weights = backend.choose_experts(logits, block.top_k, block.balance_bias, **block.how)
    want_ids, want = plain(logits, block.top_k, block.balance_bias, **block.how)
    assert torch.equal(ids.cpu(), want_ids) and torch.allclose(weights.cpu().double(), want, rtol=64 * U)
    assert torch.equal(y, block.moe(n, ids, weights))
    assert y.shape == x.shape and y.dtype == dtype
    y3 = block(x.reshape(1, T, D), r.reshape(1, T, D))[0]
    assert torch.equal(y3.reshape(T, D), y)
    assert torch.equal(block(h), y)                                       # the stream alone

    # the router's gradient: the experts' rows are what they give a single token with weight 1
    dy = torch.randn(T, D, generator=g).to(dtype).cuda()
    got, = torch.autograd.grad(block(x, r)[0], block.router_weight, dy)
    with torch.no_grad():
        rows = torch.stack([block.moe(n, ids[:, j:j + 1].contiguous(), torch.ones_like(weights[:, j:j + 1])) for j in range(block.top_k)], 1)
    d_w = (rows.double() * dy.double()[:, None]).sum(-1).cpu()
    W = block.router_weight.detach().cpu().double().requires_grad_(True)
    l = n.cpu().double() @ W.T
    w = weights_of(l, ids.cpu(), block.how.get("scoring", "softmax"), block.how.get("renormalize", True), block.how.get("scale", 1.0))
    want, = torch.autograd.grad(w, W, d_w)
    # 32-bit sums: of D products in each d_w and logit, T of them in the gradient; logits are below 8
    size = 8 * block.how.get("scale", 1.0) * (rows.double() * dy.double()[:, None]).abs().sum(-1).amax() * n.double().abs().sum(0).amax()
    assert bool(((got.cpu().double() - want).abs() <= (D + T + 64) * U * float(size)).all())


def test_frozen_and_captured(backend, gpu):
    block = block_of(16, 128, 96, torch.bfloat16, 5, top_k=2)
    x, r = (torch.randn(40, 128, device="cuda").to(torch.bfloat16) for _ in range(2))
    with pytest.raises(RuntimeError, match="frozen"):
        block(x.clone().requires_grad_(True), r)
    with torch.no_grad():
        block(x, r)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block(x, r)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, h = block(x, r)
        for seed in range(4):
            x.copy_(torch.randn(40, 128, device="cuda"))
            graph.replay()
            want = block(x, r)
            torch.cuda.synchronize()
            assert torch.equal(y, want[0]) and torch.equal(h, want[1])
