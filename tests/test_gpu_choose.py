"""The router's choice against a plain implementation in 64 bits: types, numbers of experts, groups, masks, ties, gradients."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24                                   # half a step of float32
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def plain(logits, k, bias=None, scoring="softmax", num_groups=1, top_groups=None, group_score="max", renormalize=True, scale=1.0):
    """ids, weights and, for the gradient, the weights as a function of the logits, one token after another."""
    l = logits.double().cpu().reshape(-1, logits.shape[-1])
    T, E = l.shape
    top_groups = top_groups or num_groups
    score = torch.sigmoid(l) if scoring == "sigmoid" else torch.softmax(l, -1)
    choice = l if bias is None else score + bias.double().cpu()
    ids = torch.full((T, k), -1, dtype=torch.int32)
    for t in range(T):
        c = [-math.inf if l[t, e] == -math.inf else float(choice[t, e]) for e in range(E)]
        rank = [float(score[t, e]) if bias is None and group_score == "sum2" and c[e] > -math.inf else c[e] for e in range(E)]
        size = E // num_groups
        value = []
        for g in range(num_groups):
            two = sorted(rank[g * size:(g + 1) * size], reverse=True)[:2]
            value.append(two[0] if group_score == "max" or len(two) < 2 or two[1] == -math.inf else two[0] + two[1])
        kept = sorted(range(num_groups), key=lambda g: (-value[g], g))[:top_groups]
        left = sorted((e for e in range(E) if e // size in kept and c[e] > -math.inf), key=lambda e: (-c[e], e))[:k]
        ids[t, :len(left)] = torch.tensor(left, dtype=torch.int32)
    return ids.reshape(*logits.shape[:-1], k), weights_of(l, ids, scoring, renormalize, scale).reshape(*logits.shape[:-1], k)


def weights_of(l, ids, scoring, renormalize, scale):
    score = torch.sigmoid(l) if scoring == "sigmoid" else torch.softmax(l, -1)
    there = ids >= 0
    w = torch.where(there, score.gather(1, ids.clamp(min=0).long()), 0.0)
    if renormalize:
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(total > 0, total, 1.0)
    return w * scale


def spread(logits):
    l = logits.double().cpu()
    l = torch.where(l.isinf(), 0.0, l)
    return float((l.amax() - l.amin()).abs())


def tolerance(logits, E):
    """Relative, of a weight: an exponent's argument is off by U of its size (the spread at most), the sums of up to E
    positive scores by their depth (a lane's 16, then 6 steps), exp by 2 steps, then a quotient and a product: 4 U for
    each of the two scores."""
    return (2 * spread(logits) + 16 + 6 + 8 + 2) * U


def logits_of(T, E, dtype, seed, shape=None):
    g = torch.Generator().manual_seed(seed)
    return (2.0 * torch.randn(T, E, generator=g) + 0.7 * torch.randn(E, generator=g)).to(dtype).cuda().reshape(shape or (T, E))


def bias_of(E, seed):
    g = torch.Generator().manual_seed(seed + 77)
    return (torch.randint(-100, 101, (E,), generator=g) * 0.001).cuda()


def compare(q, logits, k, bias=None, **how):
    ids, w = q.choose_experts(logits, k, bias, **how)
    want_ids, want_w = plain(logits, k, bias, **how)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32 and ids.shape == w.shape == want_ids.shape
    assert torch.equal(ids.cpu(), want_ids)
    bound = want_w.abs() * tolerance(logits, logits.shape[-1]) + 1e-37
    assert bool(((w.cpu().double() - want_w).abs() <= bound).all())
    return ids, w


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E,k", [(1, 1), (2, 2), (7, 3), (8, 8), (16, 1), (31, 4), (32, 4), (33, 33), (48, 6), (64, 8), (100, 6),
                                 (128, 2), (129, 9), (160, 6), (250, 8), (256, 8), (256, 16), (257, 5), (512, 10), (1000, 40),
                                 (1024, 64), (1023, 1023)])
def test_numbers_of_experts(backend, gpu, dtype, E, k):
    for T in (1, 37):
        compare(backend, logits_of(T, E, dtype, E + T), k)
        compare(backend, logits_of(T, E, dtype, E + T + 1), k, bias_of(E, E), scoring="sigmoid", scale=2.5)


@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("biased", [True, False])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("group_score", ["max", "sum2"])
@pytest.mark.parametrize("E,groups,top,k", [(256, 8, 4, 8), (64, 8, 3, 6), (96, 6, 2, 5), (100, 5, 5, 6), (60, 20, 7, 8), (16, 16, 9, 9),
                                            (1024, 32, 5, 12), (34, 2, 1, 17), (1000, 500, 4, 8)])
def test_groups(backend, gpu, E, groups, top, k, group_score, scoring, biased, renormalize):
    for dtype in (torch.float32, torch.bfloat16):
        compare(backend, logits_of(29, E, dtype, E), k, bias_of(E, E) if biased else None, scoring=scoring, num_groups=groups,
                top_groups=top, group_score=group_score, renormalize=renormalize)


@pytest.mark.parametrize("T", [1, 2, 63, 64, 65, 1000, 4097])
def test_numbers_of_tokens(backend, gpu, T):
    compare(backend, logits_of(T, 64, torch.bfloat16, T), 6, bias_of(64, 1))


def test_leading_sizes_and_strides(backend, gpu):
    l = logits_of(24, 40, torch.bfloat16, 3, (2, 3, 4, 40))
    ids, _ = compare(backend, l, 5)
    assert ids.shape == (2, 3, 4, 5)
    assert torch.equal(backend.choose_experts(l.transpose(0, 2), 5)[0], ids.transpose(0, 2))
    wide = logits_of(24, 81, torch.float16, 4)
    compare(backend, wide[:, 1:], 5)                                    # rows that do not start at 16 bytes
    compare(backend, wide[::3, ::2], 5)
    compare(backend, wide[0], 5)                                        # one token without a leading size
    compare(backend, wide[:1].expand(9, -1), 5)
    neg = torch.complex(wide.float(), -wide.float()).conj().imag       # lazily negated
    assert neg.is_neg()
    compare(backend, neg, 5)
    empty = backend.choose_experts(wide[:0], 5)
    assert empty[0].shape == empty[1].shape == (0, 5)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [True, False])
def test_masked_experts(backend, gpu, scoring, biased):
    E, k, inf = 48, 6, math.inf
    l = logits_of(40, E, torch.float32, 8)
    l[:, 5] = -inf
    for t in range(E):                                                 # t available experts in the rows, none in the first
        if t < 40:
            l[t, t:] = -inf
    bias = bias_of(E, 8) if biased else None
    for how in ({}, dict(num_groups=6, top_groups=2), dict(num_groups=6, top_groups=3, group_score="sum2"), dict(renormalize=False)):
        ids, w = compare(backend, l, k, bias, scoring=scoring, **how)
        assert bool((ids[0] == -1).all()) and bool((w[0] == 0).all())
        assert bool((ids[3, 3:] == -1).all()) and bool((w[ids < 0] == 0).all())
    if biased:
        bias[7] = -inf
        ids, _ = compare(backend, logits_of(40, E, torch.float32, 9), k, bias, scoring=scoring)
        assert not bool((ids == 7).any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_masks_of_the_lowest_value(backend, gpu, dtype, scoring):
    """Still experts, behind all others, of weight 0; where there is nothing else they share it."""
    l = logits_of(20, 32, dtype, 2)
    l[:, 8:] = torch.finfo(dtype).min
    l[7] = torch.finfo(dtype).min
    ids, w = backend.choose_experts(l, 12, scoring=scoring)
    assert bool((ids[:7, 8:] == torch.arange(8, 12, device="cuda")).all()) and bool((w[:7, 8:] == 0).all())
    assert torch.equal(ids[7].cpu(), torch.arange(12, dtype=torch.int32)) and torch.allclose(w[7], torch.full_like(w[7], 1 / 12), rtol=4 * U)
    assert not bool(w.isnan().any())
    assert torch.allclose(w.sum(-1), torch.ones(20, device="cuda"), rtol=16 * U)


def test_far_logits_keep_their_ratios(backend, gpu):
    """Renormalized weights hold where the scores themselves are below 32 bits."""
    l = torch.tensor([[-200.0, -201.0, -300.0, -1e30], [-90.0, -91.0, -92.0, -1e30]], device="cuda")
    _, w = backend.choose_experts(l, 3, scoring="sigmoid")
    e = torch.tensor([[1.0, math.exp(-1), math.exp(-100)], [1.0, math.exp(-1), math.exp(-2)]], dtype=torch.float64)
    want = e / e.sum(-1, keepdim=True)
    assert bool(((w.cpu().double() - want).abs() <= want * 260 * U + 1e-44).all())      # arguments up to 100 apart


def test_ties_go_to_the_lowest_index(backend, gpu):
    E, k = 96, 10
    flat = torch.zeros(5, E, device="cuda")
    want = torch.arange(k, dtype=torch.int32).expand(5, k)
    for how in ({}, dict(bias=torch.zeros(E, device="cuda")), dict(bias=torch.full((E,), -2.0, device="cuda")),
                dict(bias=torch.full((E,), -0.0, device="cuda"), scoring="sigmoid")):
        bias = how.pop("bias", None)
        assert torch.equal(backend.choose_experts(flat, k, bias, **how)[0].cpu(), want)
    ids, _ = backend.choose_experts(flat, k, num_groups=8, top_groups=2)
    assert torch.equal(ids.cpu(), want)
    g = torch.Generator().manual_seed(1)
    few = torch.randint(-2, 3, (300, E), generator=g).to(torch.bfloat16).cuda()       # many equal logits in a row
    zero = torch.where(few == 0, torch.where(torch.rand(300, E, generator=g).cuda() < 0.5, -0.0, 0.0).to(torch.bfloat16), few)
    for l in (few, zero):
        compare(backend, l, k)
        compare(backend, l, k, torch.zeros(E, device="cuda"), scoring="sigmoid")
        compare(backend, l, k, num_groups=8, top_groups=3, group_score="sum2")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [60, 70000])
def test_ties_of_sums(backend, gpu, T, dtype):
    """The scores of x and -x make 1, whatever x is: of such groups the lowest."""
    x = (3.0 * torch.randn(T, 4, generator=torch.Generator().manual_seed(5))).to(dtype).cuda()
    pairs = torch.stack((x, -x), -1).reshape(T, 8)
    ids, _ = backend.choose_experts(pairs, 4, scoring="sigmoid", num_groups=4, top_groups=2, group_score="sum2")
    assert bool((ids < 4).all())
    ids, _ = backend.choose_experts(pairs.flip(1), 2, torch.zeros(8, device="cuda"), scoring="sigmoid", num_groups=4, top_groups=1,
                                    group_score="sum2")
    assert bool((ids < 2).all())


def test_values_that_are_not_finite(backend, gpu):
    E, k = 40, 4
    l = logits_of(6, E, torch.float32, 5)
    clean = backend.choose_experts(l, k, renormalize=False)
    l[1, 17] = math.nan
    l[2, 9] = math.inf
    l[3, 3] = l[3, 30] = math.nan
    for scoring in ("softmax", "sigmoid"):
        for bias in (None, torch.zeros(E, device="cuda")):
            for how in ({}, dict(num_groups=4, top_groups=2), dict(num_groups=4, top_groups=2, group_score="sum2")):
                ids, w = backend.choose_experts(l, k, bias, scoring=scoring, **how)
                assert bool(((ids >= 0) & (ids < E)).all())
                assert all(len(set(r)) == k for r in ids.tolist())
                assert bool(w[1].isnan().all()) and bool(w[3].isnan().all())
                assert not bool(w[[0, 4, 5]].isnan().any())
                if bias is None or scoring == "sigmoid":
                    assert ids[1, 0] == 17 and ids[2, 0] == 9 and ids[3, :2].tolist() == [3, 30] or how
    ids, w = backend.choose_experts(l, k, renormalize=False, scoring="sigmoid")
    assert w[2, 0] == 1 and w[1].isnan().tolist() == [True, False, False, False]
    assert torch.equal(ids[[0, 4, 5]], clean[0][[0, 4, 5]])
    masked = l.clone()
    masked[:, 20:] = -math.inf                                         # not chosen beside a NaN either
    out = torch.zeros(E, device="cuda")
    out[:12] = -math.inf
    for scoring in ("softmax", "sigmoid"):
        for how in ({}, dict(num_groups=4, top_groups=2, group_score="sum2")):
            assert bool((backend.choose_experts(masked, k, torch.zeros(E, device="cuda"), scoring=scoring, **how)[0] < 20).all())
            assert bool((backend.choose_experts(masked, k, scoring=scoring, **how)[0] < 20).all())
            ids = backend.choose_experts(masked, k, out, scoring=scoring, **how)[0]
            assert bool(((ids < 20) & ((ids >= 12) | (ids == -1))).all())
    bias = torch.zeros(E, device="cuda")
    bias[11] = math.inf                                                # one that is always chosen
    bias[12] = math.nan                                                # ranks with it
    ids, w = backend.choose_experts(l[[0, 4, 5]], k, bias)
    assert bool((ids[:, 0] == 11).all()) and bool((ids[:, 1] == 12).all()) and not bool(w.isnan().any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (3, 1, 1), (70, 100, 6), (129, 256, 8), (40, 33, 33), (9, 1024, 70)])
def test_gradient(backend, gpu, T, E, k, scoring, renormalize, dtype):
    l = logits_of(T, E, dtype, 11 * T + E)
    if E > 50:
        l[:, 3::16] = -math.inf
        l[0, k // 2:] = -math.inf                                      # slots without an expert
    l.requires_grad_(True)
    g = torch.randn(T, k, generator=torch.Generator().manual_seed(T)).cuda()
    ids, w = backend.choose_experts(l, k, scoring=scoring, renormalize=renormalize, scale=1.7)
    assert not ids.requires_grad
    d, = torch.autograd.grad(w, l, g)
    assert d.dtype == dtype and d.shape == l.shape
    ref = l.detach().cpu().double().requires_grad_(True)
    weights = weights_of(ref, ids.cpu(), scoring, renormalize, 1.7)
    want, = torch.autograd.grad(weights, ref, g.cpu().double())
    # the terms are p_j (g_j - sum p g) and s_e sum p g: each as exact as the weights, their difference of rounded sums
    # of up to k products; then the output's own rounding
    size = 1.7 * weights.detach().abs().amax(-1, keepdim=True) / 1.7 * g.cpu().double().abs().amax(-1, keepdim=True)
    bound = want.abs() * torch.finfo(dtype).eps / 2 + size * (2 * tolerance(l.detach(), E) + (k + 8) * U) + torch.finfo(dtype).tiny
    assert bool(((d.cpu().double() - want).abs() <= bound).all())


def test_gradient_by_differences(backend, gpu):
    """The weights' own differences, where the choice stays."""
    l = torch.tensor([[1.0, -0.5, 2.0, 0.25, 0.0, -3.0]], device="cuda")
    g = torch.tensor([[0.7, -1.2, 0.4]], device="cuda")
    for scoring in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            f = lambda t: backend.choose_experts(t, 3, scoring=scoring, renormalize=renormalize)[1]
            x = l.clone().requires_grad_(True)
            d, = torch.autograd.grad(f(x), x, g)
            step = 2.0 ** -7                    # differences: step^2 / 6 of a third derivative below 1, 2 U / step of rounding
            for e in range(6):
                s = torch.zeros_like(l)
                s[0, e] = step
                diff = float(((f(l + s).double() - f(l - s).double()) * g.double()).sum()) / (2 * step)
                assert abs(diff - float(d[0, e])) <= 3 * (step ** 2 / 6 + 8 * U / step)


def test_gradient_forms(backend, gpu):
    l = logits_of(30, 64, torch.float32, 1, (5, 6, 64))
    leaf = l.clone().requires_grad_(True)
    g = torch.randn(5, 6, 4, device="cuda")
    ids, w = backend.choose_experts(leaf.transpose(0, 1), 4)
    d, = torch.autograd.grad(w, leaf, g.transpose(0, 1))
    ids2, w2 = backend.choose_experts(leaf, 4)
    d2, = torch.autograd.grad(w2, leaf, g)
    assert torch.equal(d, d2) and torch.equal(ids.transpose(0, 1), ids2)
    d3, = torch.autograd.grad(backend.choose_experts(leaf, 4)[1].sum(), leaf)          # a broadcast gradient
    assert d3.shape == leaf.shape
    bias = bias_of(64, 1).requires_grad_(True)
    w = backend.choose_experts(leaf, 4, bias)[1]
    assert torch.autograd.grad(w, (leaf, bias), g, allow_unused=True)[1] is None
    with torch.no_grad():
        assert not backend.choose_experts(leaf, 4)[1].requires_grad
    _, w = backend.choose_experts(leaf, 4)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        d, = torch.autograd.grad(w.sum(), leaf, create_graph=True)
        d.sum().backward()
    _, w = backend.choose_experts(leaf * 1.0, 4)
    w.sum().backward()
    _, w = backend.choose_experts(leaf, 4)
    with torch.no_grad():
        leaf.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        w.sum().backward()


def test_python_path_answers_alike(backend, native, gpu, monkeypatch):
    l, bias = logits_of(333, 160, torch.bfloat16, 2), bias_of(160, 2)
    how = dict(scoring="sigmoid", num_groups=8, top_groups=3, group_score="sum2", scale=2.5)
    g = torch.randn(333, 6, device="cuda")

    def both():
        leaf = l.clone().requires_grad_(True)
        ids, w = backend.choose_experts(leaf, 6, bias, **how)
        return ids, w.detach(), torch.autograd.grad(w, leaf, g)[0], *backend.choose_experts(l, 6, bias.half().float(), **how)

    host = both()
    monkeypatch.setattr(native, "host_or_none", lambda: None)
    assert all(torch.equal(a, b) for a, b in zip(host, both()))
    assert torch.equal(backend.choose_experts(l, 6, bias.half(), **how)[0], host[3])


def test_plan_of_the_choice(backend, gpu):
    """Slots without an expert are unused ones of the plan, and their tokens' outputs zero."""
    l = logits_of(50, 16, torch.float32, 3)
    l[4] = -math.inf
    l[5, 1:] = -math.inf
    ids, w = backend.choose_experts(l, 3)
    plan = backend.sort_tokens_by_expert(ids, 16)
    assert int(plan.offsets[-1]) == 48 * 3 + 1
    x = torch.randn(50, 64, device="cuda")
    y = backend.combine_expert_rows(backend.gather_expert_rows(x, plan), w, plan)
    assert bool((y[4] == 0).all())
    keep = [t for t in range(50) if t != 4]
    assert torch.allclose(y[keep], x[keep], rtol=16 * U, atol=1e-6)     # the weights of a token add up to 1


def test_streams_and_graphs(backend, gpu):
    l = logits_of(500, 256, torch.bfloat16, 6)
    bias = bias_of(256, 6)
    how = dict(scoring="sigmoid", num_groups=8, top_groups=4, group_score="sum2")
    want = backend.choose_experts(l, 8, bias, **how)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = backend.choose_experts(l, 8, bias, **how)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    x = l.clone()
    backend.choose_experts(x, 8, bias, **how)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = backend.choose_experts(x, 8, bias, **how)
    for seed in range(4):
        x.copy_(logits_of(500, 256, torch.bfloat16, 100 + seed))
        graph.replay()
        again = backend.choose_experts(x, 8, bias, **how)
        torch.cuda.synchronize()
        assert torch.equal(out[0], again[0]) and torch.equal(out[1], again[1])


def test_gradient_in_a_graph(backend, gpu):
    """Forward and backward captured whole, as autograd.grad runs them, replayed with other inputs."""
    x = logits_of(300, 96, torch.float32, 1).requires_grad_(True)
    g = torch.randn(300, 5, device="cuda")

    def step():
        w = backend.choose_experts(x, 5, renormalize=False)[1]
        return torch.autograd.grad(w, x, g)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        d = step()
    for seed in range(4):
        with torch.no_grad():
            x.copy_(logits_of(300, 96, torch.float32, 50 + seed))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(d, want)


def test_many_rows(backend, gpu):
    """Two million tokens, against torch's own order."""
    T, E = 1 << 21, 32
    l = torch.randn(T, E, device="cuda").to(torch.bfloat16)
    ids, w = backend.choose_experts(l, 2)
    want = torch.sort(l.float(), dim=-1, descending=True, stable=True)
    assert torch.equal(ids.long(), want.indices[:, :2])
    top = want.values[:, :2].double()
    e = torch.exp(top - top[:, :1])
    assert bool(((w.double() - e / e.sum(-1, keepdim=True)).abs() <= 64 * U).all())


def plain_many(logits, k, bias, scoring, num_groups, top_groups, group_score):
    """The choice of many tokens, in 64 bits with stable sorts."""
    l = logits.double()
    T, E = l.shape
    score = torch.sigmoid(l) if scoring == "sigmoid" else torch.softmax(l, -1)
    c = l if bias is None else score + bias.double()
    rank = score if bias is None and group_score == "sum2" else c
    c, rank = (t.masked_fill(l == -math.inf, -math.inf) for t in (c, rank))
    if num_groups > 1:
        two = rank.reshape(T, num_groups, -1).sort(dim=-1, descending=True).values[..., :2]
        value = two[..., 0] if group_score == "max" or two.shape[-1] < 2 else \
            torch.where(two[..., 1] == -math.inf, two[..., 0], two.sum(-1))
        kept = value.sort(dim=-1, descending=True, stable=True).indices[:, :top_groups]
        mask = torch.zeros_like(value, dtype=torch.bool).scatter_(1, kept, True).repeat_interleave(E // num_groups, 1)
        c = c.masked_fill(~mask, -math.inf)
    top = c.sort(dim=-1, descending=True, stable=True)
    return torch.where(top.values[:, :k] == -math.inf, -1, top.indices[:, :k]).int()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("E,k,groups,top", [(8, 2, 1, 1), (30, 4, 3, 2), (32, 8, 2, 1), (33, 3, 1, 1), (64, 6, 8, 3), (100, 6, 1, 1), (100, 8, 5, 2),
                                            (128, 4, 1, 1), (128, 8, 4, 2), (250, 10, 1, 1), (256, 8, 8, 4), (256, 12, 16, 5), (512, 8, 8, 2),
                                            (1000, 8, 10, 3), (14, 12, 1, 1), (32, 9, 1, 1), (64, 16, 4, 3), (128, 16, 1, 1), (128, 20, 1, 1),
                                            (130, 33, 10, 4), (254, 10, 2, 1), (512, 10, 1, 1), (1024, 17, 1, 1)])
def test_many_tokens(backend, gpu, E, k, groups, top, dtype):
    """Calls of 2^19 logits and more, which give a lane sixteen experts, with some rows masked, and their gradients."""
    T = (1 << 19) // E + 77
    g = torch.Generator(device="cuda").manual_seed(E + k)
    l = (2 * torch.randn(T, E, generator=g, device="cuda") + 0.7 * torch.randn(E, generator=g, device="cuda")).to(dtype)
    l[::5, ::3] = -math.inf
    l[11] = -math.inf
    bias = bias_of(E, k)
    d_w = torch.randn(T, k, generator=g, device="cuda")
    for scoring, b, group_score, renormalize in (("softmax", None, "max", True), ("sigmoid", bias, "sum2", True), ("softmax", bias, "max", False),
                                                 ("softmax", None, "sum2", False), ("sigmoid", None, "max", False)):
        leaf = l.clone().requires_grad_(True)
        ids, w = backend.choose_experts(leaf, k, b, scoring=scoring, num_groups=groups, top_groups=top, group_score=group_score,
                                        renormalize=renormalize, scale=1.5)
        assert torch.equal(ids, plain_many(l, k, b, scoring, groups, top, group_score))
        ref = l.double().requires_grad_(True)
        want = torch.nan_to_num(weights_of(ref, ids, scoring, renormalize, 1.5))           # the row without an expert
        tol = tolerance(l, E)
        assert bool(((w.double() - want).abs() <= want.abs() * tol + 1e-37).all())
        d, = torch.autograd.grad(w, leaf, d_w)
        keep = torch.ones(T, 1, device="cuda")
        keep[11] = 0
        ok = l.double().masked_fill(keep == 0, 0.0).requires_grad_(True)                    # its gradient is zero
        exact, = torch.autograd.grad(weights_of(ok, ids, scoring, renormalize, 1.5) * keep, ok, d_w.double())
        size = want.amax(-1, keepdim=True) / 1.5 * 1.5 * d_w.double().abs().amax(-1, keepdim=True)
        bound = exact.abs() * torch.finfo(dtype).eps / 2 + size * (2 * tol + (k + 8) * U) + torch.finfo(dtype).tiny
        assert bool(((d.double() - exact).abs() <= bound).all())


def test_past_32_bits(backend, gpu):
    """Logits whose numbers pass 2^31 and bytes 2^32; the last tokens are the first ones' copies."""
    T, E = (1 << 23) + 77, 264
    l = torch.empty(T, E, dtype=torch.bfloat16, device="cuda").normal_()
    l[-9:] = l[:9]
    bias = bias_of(E, 1)
    how = dict(scoring="sigmoid", num_groups=8, top_groups=3, group_score="sum2")
    few = backend.choose_experts(l[:9], 5, bias, **how)
    leaf = l.requires_grad_(True)
    ids, w = backend.choose_experts(leaf, 5, bias, **how)
    for got, want in zip((ids, w), few):
        assert torch.equal(got[:9], want) and torch.allclose(got[-9:].float(), want.float(), rtol=32 * U)
    d_w = torch.randn(9, 5, device="cuda").repeat(T // 9 + 1, 1)[:T]
    d_w[-9:] = d_w[:9]
    d, = torch.autograd.grad(w, leaf, d_w)
    assert bool(d[:9].any()) and torch.allclose(d[-9:].float(), d[:9].float(), rtol=2.0 ** -6)
