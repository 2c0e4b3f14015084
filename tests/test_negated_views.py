"""Lazily negated views (torch's negative bit): operands count by their values."""
import pytest
import torch


def test_operands_are_written_out(native):
    x = torch.arange(8.0).reshape(2, 4)
    y = native._aligned(torch._neg_view(x))
    assert not y.is_neg() and torch.equal(y, -x)
    assert native._aligned(x) is x


def test_a_negated_plan_is_refused(backend):
    i = torch.int32
    plan = backend.ExpertPlan(torch._neg_view(torch.zeros(2, dtype=i)), torch.zeros(2, 1, dtype=i), torch.zeros(3, dtype=i))
    with pytest.raises(ValueError, match="a plan is"):
        plan.check()


@pytest.mark.gpu
def test_products_and_gradients(backend, gpu):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(6, 64, generator=g).cuda()
    w, s = backend.quantize_mxfp4(torch.randn(32, 64, generator=g).cuda())
    assert torch.equal(backend.mxfp4_linear(torch._neg_view(x), w, s), backend.mxfp4_linear(-x, w, s))
    ids = torch.tensor([[0], [1], [2], [1], [0], [2]]).cuda()
    plan = backend.sort_tokens_by_expert(ids, 3)
    for a, b in zip(plan, backend.sort_tokens_by_expert(torch._neg_view(-ids), 3)):
        assert torch.equal(a, b)
    assert torch.equal(backend.gather_expert_rows(torch._neg_view(x), plan), backend.gather_expert_rows(-x, plan))
    rows, weights = x.clone().requires_grad_(), torch.rand(6, 1, generator=g).cuda().requires_grad_()
    out = backend.combine_expert_rows(rows, weights, plan)
    a = torch.autograd.grad(out, (rows, weights), torch._neg_view(x), retain_graph=True)
    b = torch.autograd.grad(out, (rows, weights), -x)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
