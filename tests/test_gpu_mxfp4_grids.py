"""GPU checks of calls whose workgroups are more than one launch holds (2^32 threads)."""
import pytest
import torch

from test_gpu_mxfp4 import say

pytestmark = pytest.mark.gpu


def test_more_tokens_than_a_launch(backend, gpu):
    """2^24 tokens and a few, a workgroup each: plan, gather, combine and their gradients."""
    T, D = 2 ** 24 + 37, 8
    say("tokens past a launch", T, D)
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(0, 3, (T, 1), generator=g, device="cuda", dtype=torch.int32)
    ids[::1001] = -1
    plan = backend.sort_tokens_by_expert(ids, 3)
    used = int((ids >= 0).sum())
    assert plan.offsets.tolist()[-1] == used
    order = plan.order.long()
    assert (order[used:] == -1).all() and (ids.flatten()[order[:used]].diff() >= 0).all()
    x = torch.randn(T, D, generator=g, device="cuda").to(torch.bfloat16).requires_grad_()
    w = torch.rand(T, 1, generator=g, device="cuda").requires_grad_()
    rows = backend.gather_expert_rows(x, plan)
    assert torch.equal(rows[:used], x[order[:used]]) and int(rows[used:].count_nonzero()) == 0
    held = rows.detach().requires_grad_()
    out = backend.combine_expert_rows(held, w, plan)
    there = (ids >= 0).flatten()
    want = torch.where(there[:, None], x.detach().float() * w.detach(), 0).to(torch.bfloat16)
    assert torch.equal(out, want)
    d = torch.randn(T, D, generator=g, device="cuda").to(torch.bfloat16)
    d_rows, d_w = torch.autograd.grad(out, (held, w), d)
    assert torch.equal(d_rows[:used], (d[order[:used]].float() * w.detach()[order[:used]]).to(torch.bfloat16))
    assert int(d_rows[used:].count_nonzero()) == 0
    want = torch.where(there, (x.detach().double() * d.double()).sum(dim=1), 0)
    size = (x.detach().double() * d.double()).abs().sum(dim=1)
    assert ((d_w.flatten().double() - want).abs() <= (D + 8) * 2.0 ** -24 * size).all()
    (d_x,) = torch.autograd.grad(rows, x, held.detach())
    assert torch.equal(d_x, torch.where(there[:, None], x.detach(), 0))


def test_more_rows_than_a_launch_quantizes(backend, gpu):
    """Rows of 32 values, eight a workgroup: 2^27 of them and a few through a linear, its codes' launch too long."""
    M, K, N = 2 ** 27 + 5 * 8 + 3, 32, 8
    say("rows past a launch", M, K, N)
    g = torch.Generator().manual_seed(2)
    last = torch.randn(70, K, generator=g).to(torch.bfloat16).cuda()
    wc, ws = backend.quantize_mxfp4(torch.randn(N, K, generator=g).cuda())
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    x[-70:] = last
    y = backend.mxfp4_linear(x, wc, ws)
    assert torch.equal(y[-70:], backend.mxfp4_linear(last, wc, ws)) and int(y[:-70].count_nonzero()) == 0


def test_more_tiles_than_a_launch(backend, gpu):
    """Tokens whose codes take more than 2^32 bytes, and columns enough for more than 2^23 workgroups of 512 threads."""
    T, K, N = 2 ** 21 + 37, 4096, 4128
    say("tiles past a launch", T, K, N)
    g = torch.Generator().manual_seed(1)
    last = torch.randn(50, K, generator=g).to(torch.bfloat16).cuda()
    wc, ws = backend.quantize_mxfp4(torch.randn(2, N, K, generator=g).cuda())
    x = torch.zeros(T, K, dtype=torch.bfloat16, device="cuda")
    x[-50:] = last
    ids = torch.zeros(T, 1, dtype=torch.int64, device="cuda")
    ids[-20:] = 1
    y = backend.mxfp4_expert_linear(x, wc, ws, backend.sort_tokens_by_expert(ids, 2))
    want = backend.mxfp4_expert_linear(last, wc, ws, backend.sort_tokens_by_expert(ids[-50:].contiguous(), 2))
    assert torch.equal(y[-50:], want)
    assert not any(bool(part.any()) for part in y[:-50].split(1 << 18))


def test_more_values_than_a_launch(backend, gpu):
    """2^36 values and a row: quantized and back."""
    M, K = 2 ** 21 + 1, 32768
    say("values past a launch", M, K)
    torch.cuda.empty_cache()
    last = torch.randn(1, K, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    x[-1:] = last
    codes, scales = backend.quantize_mxfp4(x)
    small = backend.quantize_mxfp4(last)
    assert torch.equal(codes[-1:], small[0]) and torch.equal(scales[-1:], small[1])
    assert not any(bool(part.any()) for part in codes[:-1].split(1 << 16))
    del x
    back = backend.dequantize_mxfp4(codes, scales, output_dtype=torch.bfloat16)
    assert torch.equal(back[-1:], backend.dequantize_mxfp4(*small, output_dtype=torch.bfloat16))
    assert not any(bool(part.any()) for part in back[:-1].split(1 << 16))
    del back, codes, scales
    torch.cuda.empty_cache()
