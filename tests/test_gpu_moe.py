"""The mixture-of-experts feed-forward on MXFP4 weights: the operators together,
against the same steps in 64 bits on the same codes, and a router trained over it."""
import importlib

import numpy as np
import pytest
import torch

import mx_format as mx
from conftest import PKG_NAME
from test_gpu_mxfp4 import np64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def moe_cls(gpu):
    return importlib.import_module(PKG_NAME + ".mxfp4_moe").Mxfp4MoE


def layer(moe_cls, E, D, F, G, seed=0):
    g = torch.Generator().manual_seed(seed)
    gate, up, down = (torch.randn(s, generator=g) * s[-1] ** -0.5 for s in ((E, F, D), (E, F, D), (E, D, F)))
    return moe_cls.from_float(gate.cuda(), up.cuda(), down.cuda(), convrot_groupsize=G)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,k,E,D,F,G", [(1, 2, 4, 256, 512, 256), (9, 3, 5, 128, 96, 16), (200, 2, 6, 320, 448, 64)])
def test_forward(backend, moe_cls, T, k, E, D, F, G, dtype):
    print("moe", T, k, E, D, F, G, dtype, flush=True)
    moe = layer(moe_cls, E, D, F, G)
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, D, generator=g).to(dtype)
    ids = torch.randint(-1, E, (T, k), generator=g)
    w = torch.rand(T, k, generator=g)
    got = np64(moe(x.cuda(), ids.cuda(), w.cuda()))
    # the quantized input and the quantized hidden rows are the library's own codes
    xq = mx.dequantize(*(t.cpu().numpy() for t in backend.quantize_mxfp4(x.cuda(), G)))
    order, position, offsets = mx.plan(ids.numpy(), E)
    w1 = mx.dequantize(moe.w1.cpu().numpy(), moe.s1.cpu().numpy())
    w2 = mx.dequantize(moe.w2.cpu().numpy(), moe.s2.cpu().numpy())
    hidden = np.zeros((T * k, 2 * F))
    for e in range(E):
        r = slice(offsets[e], offsets[e + 1])
        hidden[r] = xq[order[r] // k] @ w1[e].T
    h = torch.from_numpy(hidden).float().to(dtype).cuda()
    h = torch.nn.functional.silu(h[:, :F]) * h[:, F:]
    hq = mx.dequantize(*(t.cpu().numpy() for t in backend.quantize_mxfp4(h, G)))
    rows = np.zeros((T * k, D))
    for e in range(E):
        r = slice(offsets[e], offsets[e + 1])
        rows[r] = hq[r] @ w2[e].T
    picked = np.where((position >= 0)[..., None], rows[np.maximum(position, 0)], 0)
    want = (picked * w.double().numpy()[..., None]).sum(axis=1)
    # a hidden value that rounds to the other neighbour moves its 4-bit code by a step at most: a quarter of the block's
    # largest value in 1 of the 32; the two sums agree far closer than the 4-bit values they are made of
    assert np.linalg.norm(got - want) <= 0.05 * np.linalg.norm(want)
    assert (got[(ids.numpy() < 0).all(axis=1)] == 0).all()


def test_router_gradient_and_training(moe_cls):
    """The router's weights get <d_out, the expert's row>, and a few steps of descent lower the loss."""
    T, k, E, D, F = 64, 2, 4, 128, 256
    moe = layer(moe_cls, E, D, F, 64)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(T, D, generator=g).cuda()
    router = torch.randn(E, D, generator=g).cuda().mul_(0.02).requires_grad_()
    target = torch.randn(T, D, generator=g).cuda()
    losses = []
    for _ in range(12):
        top, ids = (x @ router.T).topk(k)
        w = torch.softmax(top, dim=-1)
        loss = (moe(x, ids, w) - target).square().mean()
        losses.append(loss.item())
        (grad,) = torch.autograd.grad(loss, router)
        assert torch.isfinite(grad).all() and grad.abs().max() > 0
        with torch.no_grad():
            router -= 0.5 * grad / grad.norm()
    assert losses[-1] < losses[0]
    # one unit vector of weights at a time: the layer is linear in them
    ids = torch.stack((torch.arange(T) % E, (torch.arange(T) + 1) % E), dim=1).cuda()
    w = torch.rand(T, k, generator=g).cuda().requires_grad_()
    d = torch.randn(T, D, generator=g).cuda()
    (got,) = torch.autograd.grad(moe(x, ids, w), w, d)
    one = [(moe(x, ids, torch.eye(k, device="cuda")[j].expand(T, k)) * d).double().sum(dim=-1) for j in range(k)]
    assert torch.allclose(got.double(), torch.stack(one, dim=1), rtol=1e-4, atol=1e-4)


def test_refusals(moe_cls):
    moe = layer(moe_cls, 2, 64, 64, 16)
    x, ids, w = torch.zeros(3, 64, device="cuda"), torch.zeros(3, 1, dtype=torch.int64, device="cuda"), torch.ones(3, 1, device="cuda")
    assert moe(x, ids, w).shape == (3, 64)
    with pytest.raises(RuntimeError, match="frozen"):
        moe(x.requires_grad_(), ids, w)
    with pytest.raises(ValueError, match="do not fit"):
        moe_cls(moe.w1, moe.s1, moe.w1, moe.s1)
