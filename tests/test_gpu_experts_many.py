"""GPU checks of plans of nearly 2^31 slots: sums of a row number and a tile, a row of slots or a grid pass 31 bits."""
import pytest
import torch

from test_gpu_mxfp4 import say

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def room(gpu):
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def many(backend, T, k, unused):
    """All slots to expert 0, but the last 40 tokens' odd ones to expert 1 and the last ``unused`` to none."""
    ids = torch.zeros((T, k), dtype=torch.int32, device="cuda")
    ids[-40:, 1::2] = 1
    if unused:
        ids.view(-1)[-unused:] = -1
    plan = backend.sort_tokens_by_expert(ids, 2)
    tail = ids[-40:].clone()
    return tail, plan


def spans(n, step=1 << 27):
    return [(i, min(i + step, n)) for i in range(0, n, step)]


def expected_order(T, k, tail):
    """Slots of the last 40 tokens in sorted order, where the sorted rows of expert 0 before them end, and the used rows."""
    slot = torch.arange(40 * k, device="cuda") + (T - 40) * k
    flat = tail.flatten()
    last = torch.cat((slot[flat == 0], slot[flat == 1]))
    return last, (T - 40) * k, (T - 40) * k + last.numel()


@pytest.mark.parametrize("T,k,unused", [(2 ** 25 - 1, 64, 0), (2 ** 28 - 1, 8, 101)])
def test_plan_and_rows(backend, gpu, T, k, unused):
    R, D = T * k, 8
    say("slots near 2^31", T, k, unused)
    tail, plan = many(backend, T, k, unused)
    last, n0, used = expected_order(T, k, tail)
    assert plan.offsets.tolist() == [0, n0 + int((tail == 0).sum()), used]
    for a, b in spans(n0):
        want = torch.arange(a, b, dtype=torch.int32, device="cuda")
        assert torch.equal(plan.order[a:b], want) and torch.equal(plan.position.view(-1)[a:b], want)
    assert torch.equal(plan.order[n0:used].long(), last) and bool((plan.order[used:] == -1).all())
    assert torch.equal(plan.position.view(-1)[last].long(), torch.arange(n0, used, device="cuda"))
    assert bool((plan.position[-40:][tail < 0] == -1).all())
    x = torch.randn(T, D, generator=torch.Generator("cuda").manual_seed(1), device="cuda", dtype=torch.bfloat16)
    rows = backend.gather_expert_rows(x, plan)
    for a, b in spans(T - 40, 1 << 20):
        assert torch.equal(rows[a * k:b * k].view(b - a, k, D), x[a:b, None].expand(b - a, k, D))
    assert torch.equal(rows[n0:used], x[last // k]) and int(rows[used:].count_nonzero()) == 0
    w = torch.zeros(T, k, device="cuda")
    w[:, 0] = 1
    w[-40:] = 0.5
    rows.requires_grad_()
    w.requires_grad_()
    out = backend.combine_expert_rows(rows, w, plan)
    assert torch.equal(out[:-40], x[:-40])
    there = (tail >= 0).sum(dim=1, keepdim=True)
    assert torch.equal(out[-40:], (x[-40:].float() * 0.5 * there).to(torch.bfloat16))
    d_rows, d_w = torch.autograd.grad(out, (rows, w), x)
    assert torch.equal(d_rows[n0:used], (x[last // k].float() * 0.5).to(torch.bfloat16))
    assert int(d_rows[used:].count_nonzero()) == 0
    square = (x.double() ** 2).sum(dim=1)
    for a, b in spans(T - 40, 1 << 20):
        near = (d_w[a:b].double() - square[a:b, None]).abs() <= 16 * 2.0 ** -24 * square[a:b, None]
        assert bool(near.all())
    got = d_w[-40:].double()
    assert bool(((got - torch.where(tail >= 0, square[-40:, None], 0)).abs() <= 16 * 2.0 ** -24 * square[-40:, None]).all())


@pytest.mark.parametrize("T,k,unused", [(2 ** 25 - 1, 64, 0), (2 ** 25 - 1, 64, 70), (2 ** 28 - 1, 8, 0), (2 ** 28 - 1, 8, 13)])
def test_products(backend, gpu, T, k, unused):
    """The staged kernel, and the one for few rows, which takes tokens whose codes pass 2^32 bytes."""
    K, N = 32, 4
    say("rows near 2^31", T, k, unused)
    tail, plan = many(backend, T, k, unused)
    last, n0, used = expected_order(T, k, tail)
    g = torch.Generator().manual_seed(2)
    wc, ws = backend.quantize_mxfp4(torch.randn(2, N, K, generator=g).cuda())
    x = torch.zeros(T, K, dtype=torch.bfloat16, device="cuda")
    x[-50:] = torch.randn(50, K, generator=g).to(torch.bfloat16).cuda()
    x[5] = 1
    y = backend.mxfp4_expert_linear(x, wc, ws, plan)
    both = [backend.mxfp4_linear(x[-50:], wc[e], ws[e]) for e in range(2)]
    e = (torch.arange(n0, used, device="cuda") >= plan.offsets[1]).long()
    want = torch.stack(both)[e, last // k - (T - 50)]
    assert torch.equal(y[n0:used], want) and int(y[used:].count_nonzero()) == 0
    assert torch.equal(y[n0 - 10 * k:n0].view(10, k, N), both[0][:10, None].expand(10, k, N))
    one = backend.mxfp4_linear(x[5:6], wc[0], ws[0])
    assert torch.equal(y[5 * k:6 * k], one.expand(k, N))
    for a, b in spans(n0 - 10 * k):
        part = y[a:b]
        assert int(part.count_nonzero()) == (int(one.count_nonzero()) * k if a <= 5 * k < b else 0)
