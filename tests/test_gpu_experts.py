"""GPU checks of expert routing and of the experts' MXFP4 products against their
definitions in 64 bits."""
import numpy as np
import pytest
import torch

import mx_format as mx
from test_gpu_mxfp4 import DTYPES, exact_operands, np64, rounded_once, say

pytestmark = pytest.mark.gpu


def choice(T, k, E, seed, unused=0.1, skew=1.0):
    g = np.random.RandomState(seed)
    p = np.exp(skew * g.randn(E))
    ids = np.stack([g.choice(E, k, p=p / p.sum()) for _ in range(T)]) if T else np.zeros((0, k), int)
    ids[g.rand(T, k) < unused] = -1
    return ids


PLANS = [(1, 1, 1), (1, 4, 32), (3, 2, 7), (16, 4, 32), (77, 3, 13), (100, 8, 100), (333, 6, 1000), (1030, 4, 64),
         (2500, 2, 1024), (5000, 5, 3)]


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("T,k,E", PLANS)
def test_plan(backend, gpu, T, k, E, dtype):
    say("plan", T, k, E, dtype)
    ids = choice(T, k, E, seed=T + k + E)
    ids.reshape(-1)[::17] = E + 3                             # outside: unused too
    plan = backend.sort_tokens_by_expert(torch.from_numpy(ids).to(dtype).cuda(), E)
    for got, want in zip((plan.order, plan.position, plan.offsets), mx.plan(ids, E)):
        assert got.dtype == torch.int32 and np.array_equal(got.cpu().numpy(), want)
    assert plan.num_experts == E


@pytest.mark.parametrize("ids", [np.full((500, 3), -1), np.full((3000, 3), 5), np.zeros((0, 2), int),
                                 np.array([[2 ** 40, -2 ** 40, 3]])], ids=["unused", "one expert", "no tokens", "far out"])
def test_plan_extremes(backend, gpu, ids):
    plan = backend.sort_tokens_by_expert(torch.from_numpy(ids.astype(np.int64)).cuda(), 8)
    for got, want in zip((plan.order, plan.position, plan.offsets), mx.plan(ids, 8)):
        assert np.array_equal(got.cpu().numpy(), want)


def routed(backend, T, k, E, D, dtype, seed, unused=0.1):
    g = torch.Generator().manual_seed(seed)
    ids = choice(T, k, E, seed, unused)
    if T > 2:
        ids[T // 2] = -1                                      # a token without a used slot
    plan = backend.sort_tokens_by_expert(torch.from_numpy(ids).cuda(), E)
    x = torch.randn(T, D, generator=g).to(dtype)
    rows = torch.randn(T * k, D, generator=g).to(dtype)
    w = torch.rand(T, k, generator=g)
    return ids, plan, x, rows, w


ROUTES = [(1, 1, 2, 1), (5, 3, 4, 7), (16, 4, 32, 2048), (33, 2, 5, 1001), (100, 8, 64, 264), (257, 6, 9, 96), (64, 1, 8, 4100)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,D", ROUTES)
def test_gather_and_combine(backend, gpu, T, k, E, D, dtype):
    say("route", T, k, E, D, dtype)
    ids, plan, x, rows, w = routed(backend, T, k, E, D, dtype, seed=T + D)
    order, position, _ = mx.plan(ids, E)
    got = backend.gather_expert_rows(x.cuda(), plan)
    want = np.where((order >= 0)[:, None], np64(x)[np.maximum(order, 0) // k], 0)
    assert got.dtype == dtype and np.array_equal(np64(got), want)
    picked = np.where((position >= 0)[..., None], np64(rows)[np.maximum(position, 0)], 0)
    for weights in (w, w.to(torch.bfloat16), w.to(torch.float16)):
        terms = picked * np64(weights)[..., None]
        out = backend.combine_expert_rows(rows.cuda(), weights.cuda(), plan)
        off = k * 2.0 ** -24 * np.abs(terms).sum(axis=1)       # k fused multiply-adds in fp32, then one rounding
        assert out.dtype == dtype and rounded_once(out, terms.sum(axis=1), off, dtype)
        if T > 2:
            assert (out[T // 2] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,D", ROUTES)
def test_gradients(backend, gpu, T, k, E, D, dtype):
    say("gradients", T, k, E, D, dtype)
    ids, plan, x, rows, w = routed(backend, T, k, E, D, dtype, seed=T + D + 1)
    order, position, _ = mx.plan(ids, E)
    g = torch.Generator().manual_seed(3)
    d_rows, d_out = torch.randn(T * k, D, generator=g).to(dtype), torch.randn(T, D, generator=g).to(dtype)
    xc, rc, wc = (t.cuda().requires_grad_() for t in (x, rows, w))
    backend.gather_expert_rows(xc, plan).backward(d_rows.cuda())
    backend.combine_expert_rows(rc, wc, plan).backward(d_out.cuda())
    used = (position >= 0)[..., None]
    terms = np.where(used, np64(d_rows)[np.maximum(position, 0)], 0)
    want, off = terms.sum(axis=1), k * 2.0 ** -24 * np.abs(terms).sum(axis=1)
    assert rounded_once(xc.grad, want, off, dtype)
    of_row = np.where(order >= 0, np64(w).reshape(-1)[np.maximum(order, 0)], 0)[:, None]
    want = of_row * np64(d_out)[np.maximum(order, 0) // k]
    assert rounded_once(rc.grad, want, 2.0 ** -24 * np.abs(want), dtype)      # one product in fp32
    terms = np.where(used, np64(rows)[np.maximum(position, 0)], 0) * np64(d_out)[:, None]
    want, off = terms.sum(axis=-1), (D + 8) * 2.0 ** -24 * np.abs(terms).sum(axis=-1)
    assert wc.grad.dtype == torch.float32 and (np.abs(np64(wc.grad) - want) <= off).all()
    if T > 2:
        assert (np64(wc.grad)[T // 2] == 0).all() and (np64(xc.grad)[T // 2] == 0).all()


def test_gradients_against_differences(backend, gpu):
    """<combine(rows, w), g> is linear in the rows and in the weights, <gather(x), h> in x: a difference over a step of
    1 is the derivative, to the roundings of the two sums (D k terms of size about 1, 2^-24 each)."""
    T, k, E, D = 6, 3, 4, 24
    ids, plan, x, rows, w = routed(backend, T, k, E, D, torch.float32, seed=8)
    g = torch.randn(T, D, generator=torch.Generator().manual_seed(1)).cuda()
    h = torch.randn(T * k, D, generator=torch.Generator().manual_seed(2)).cuda()
    x, rows, w = (t.cuda().requires_grad_() for t in (x, rows, w))

    def value(x, rows, w):
        out = (backend.combine_expert_rows(rows, w, plan) * g).double().sum() \
            + (backend.gather_expert_rows(x, plan) * h).double().sum()
        return out

    value(x, rows, w).backward()
    for which, t in enumerate((x, rows, w)):
        for i in range(0, t.numel(), 5):
            args = [v.detach().clone() for v in (x, rows, w)]
            args[which].view(-1)[i] += 0.5
            hi = value(*args)
            args[which].view(-1)[i] -= 1.0
            assert abs(float(hi - value(*args)) - float(t.grad.view(-1)[i])) < T * D * k * 8 * 2.0 ** -24


def test_partial_and_repeated_gradients(backend, gpu):
    """Only one side asks for its gradient; bf16 weights get a bf16 gradient; two runs give the same bits."""
    T, k, E, D = 40, 4, 6, 520
    ids, plan, x, rows, w = routed(backend, T, k, E, D, torch.bfloat16, seed=5)
    rows, w = rows.cuda(), w.cuda()
    d = torch.randn(T, D, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()

    def grads(r, v):
        return torch.autograd.grad(backend.combine_expert_rows(r, v, plan), [t for t in (r, v) if t.requires_grad], d)

    r, v = rows.clone().requires_grad_(), w.clone().requires_grad_()
    both = grads(r, v)
    assert torch.equal(grads(r, w)[0], both[0]) and torch.equal(grads(rows, v)[0], both[1])
    assert all(torch.equal(a, b) for a, b in zip(both, grads(r, v)))
    half = w.to(torch.bfloat16).requires_grad_()
    assert grads(rows, half)[0].dtype == torch.bfloat16
    strided = d.t().contiguous().t()
    assert torch.equal(torch.autograd.grad(backend.combine_expert_rows(r, w, plan), r, strided)[0], both[0])


def test_unused_rows_do_not_reach_the_sums(backend, gpu):
    """Rows past the last used one and NaN in them: zeros out, and no NaN."""
    T, k, E, D = 12, 3, 4, 64
    ids, plan, x, rows, w = routed(backend, T, k, E, D, torch.float32, seed=6, unused=0.5)
    used = int(plan.offsets[-1])
    rows[used:] = float("nan")
    w[torch.from_numpy(ids) < 0] = float("nan")
    rc, wc = rows.cuda().requires_grad_(), w.cuda().requires_grad_()
    out = backend.combine_expert_rows(rc, wc, plan)
    out.backward(torch.ones_like(out))
    assert torch.isfinite(out).all() and torch.isfinite(rc.grad).all() and torch.isfinite(wc.grad).all()
    assert (rc.grad[used:] == 0).all() and (wc.grad.cpu()[torch.from_numpy(ids) < 0] == 0).all()
    assert (backend.gather_expert_rows(x.cuda(), plan)[used:] == 0).all()


# ---- the experts' products -------------------------------------------------

EXPERTS = [(1, 1, 1, 64, 64), (1, 4, 32, 256, 512), (5, 2, 3, 33, 96), (16, 4, 8, 128, 1056), (40, 3, 70, 100, 160),
           (64, 6, 4, 260, 512), (150, 2, 5, 96, 2080), (300, 4, 6, 384, 640), (900, 3, 2, 200, 256)]


@pytest.mark.parametrize("rows", [False, True], ids=["tokens", "sorted"])
@pytest.mark.parametrize("T,k,E,N,K", EXPERTS)
def test_expert_linear_exact(backend, gpu, T, k, E, N, K, rows):
    say("experts", T, k, E, N, K, rows)
    ids = choice(T, k, E, seed=T + N)
    order, _, offsets = mx.plan(ids, E)
    x, wc, ws = exact_operands(T * k if rows else T, N, K, seed=T + K, E=E)
    bias = np.random.RandomState(2).randint(-64, 64, (E, N)) / 8.0
    want = np.zeros((T * k, N))
    for e in range(E):
        r = slice(offsets[e], offsets[e + 1])
        a = x[r] if rows else x[order[r] // k]
        want[r] = a @ mx.dequantize(wc[e], ws[e]).T + bias[e]
    plan = backend.sort_tokens_by_expert(torch.from_numpy(ids).cuda(), E)
    w, s = torch.from_numpy(wc).cuda(), torch.from_numpy(ws).cuda()
    y = backend.mxfp4_expert_linear(torch.from_numpy(x).float().cuda(), w, s, plan, torch.from_numpy(bias).float().cuda(),
                                    sorted_rows=rows)
    assert np.array_equal(np64(y), want)
    for dtype in (torch.bfloat16, torch.float16):
        y = backend.mxfp4_expert_linear(torch.from_numpy(x).to(dtype).cuda(), w, s, plan,
                                        torch.from_numpy(bias).to(dtype).cuda(), sorted_rows=rows)
        assert torch.equal(y.cpu(), torch.from_numpy(want).float().to(dtype))


@pytest.mark.parametrize("rows", [False, True], ids=["tokens", "sorted"])
@pytest.mark.parametrize("T,k,E,N,K,tile", [(7, 4, 9, 512, 320, 0), (1500, 3, 70, 1000, 544, 128), (1024, 2, 8, 4096, 2848, 256)])
def test_expert_linear_exact_by_tile(backend, native, gpu, T, k, E, N, K, tile, rows):
    assert native.load_library().cr_mxfp4_tile(T * k, N, K, E) == tile
    say("experts", T, k, E, N, K, rows)
    ids = choice(T, k, E, seed=T + N, skew=0.5)
    order, _, offsets = mx.plan(ids, E)
    x, wc, ws = exact_operands(T * k if rows else T, N, K, seed=T + K, E=E)
    plan = backend.sort_tokens_by_expert(torch.from_numpy(ids).cuda(), E)
    xt = torch.from_numpy(x).cuda()
    a = xt if rows else xt[torch.from_numpy(np.maximum(order, 0) // k).cuda().long()]
    want = torch.zeros(T * k, N, dtype=torch.float64, device="cuda")
    for e in range(E):
        r = slice(offsets[e], offsets[e + 1])
        want[r] = a[r] @ torch.from_numpy(mx.dequantize(wc[e], ws[e])).cuda().T
    w, s = torch.from_numpy(wc).cuda(), torch.from_numpy(ws).cuda()
    for dtype in DTYPES:
        y = backend.mxfp4_expert_linear(xt.to(dtype), w, s, plan, sorted_rows=rows)
        assert torch.equal(y, want.float().to(dtype))


@pytest.mark.parametrize("ids", ["unused", "one expert", "no tokens"])
def test_expert_linear_extremes(backend, gpu, ids):
    E, N, K, k = 6, 72, 96, 2
    T = 0 if ids == "no tokens" else 200
    ids = np.full((T, k), -1 if ids == "unused" else 4)
    order, _, offsets = mx.plan(ids, E)
    x, wc, ws = exact_operands(max(T, 1), N, K, seed=1, E=E)
    x = x[:T]
    plan = backend.sort_tokens_by_expert(torch.from_numpy(ids).cuda(), E)
    y = backend.mxfp4_expert_linear(torch.from_numpy(x).float().cuda(), torch.from_numpy(wc).cuda(),
                                    torch.from_numpy(ws).cuda(), plan)
    want = np.where((order >= 0)[:, None], x[np.maximum(order, 0) // k] @ mx.dequantize(wc[4], ws[4]).T, 0) if T \
        else np.zeros((0, N))
    assert np.array_equal(np64(y), want)


def test_experts_in_a_graph(backend, gpu):
    """A whole routed layer captured and replayed, other choices and tokens each time."""
    T, k, E, N, K = 20, 2, 5, 64, 128
    x, wc, ws = exact_operands(T, N, K, seed=12, E=E)
    w, s = torch.from_numpy(wc).cuda(), torch.from_numpy(ws).cuda()
    ids, xt = torch.from_numpy(choice(T, k, E, 1)).cuda(), torch.from_numpy(x).float().cuda()
    weights = torch.full((T, k), 0.5, device="cuda")

    def layer(ids, xt):
        plan = backend.sort_tokens_by_expert(ids, E)
        return backend.combine_expert_rows(backend.mxfp4_expert_linear(xt, w, s, plan), weights, plan)

    layer(ids, xt)
    torch.cuda.synchronize()
    held, held_x = ids.clone(), xt.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(held, held_x)
    for seed in range(4):
        new = torch.from_numpy(choice(T, k, E, seed)).cuda()
        held.copy_(new)
        held_x.copy_(xt.roll(seed, 0))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, layer(new, xt.roll(seed, 0)))


def test_rows_past_32_bits(backend, gpu):
    """Sorted rows of more than 2^32 bytes: gather, combine and their gradients on the last rows."""
    T, k, D = 150000, 2, 8192
    ids = torch.full((T, k), -1, dtype=torch.int64)
    ids[:, 0] = 0
    ids[-3:, 1] = 1
    plan = backend.sort_tokens_by_expert(ids.cuda(), 2)
    x = torch.zeros(T, D, dtype=torch.bfloat16, device="cuda")
    x[-3:] = torch.randn(3, D, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).cuda()
    rows = backend.gather_expert_rows(x, plan)
    assert rows.numel() * 2 > 2 ** 32 and plan.offsets.tolist() == [0, T, T + 3]
    assert torch.equal(rows[T:T + 3], x[-3:]) and torch.equal(rows[T - 3:T], x[-3:]) and int(rows[T + 3:].count_nonzero()) == 0
    w = torch.ones(T, k, device="cuda")
    out = backend.combine_expert_rows(rows, w, plan)
    assert torch.equal(out[-3:], (2 * x[-3:].float()).to(torch.bfloat16)) and int(out[:-3].count_nonzero()) == 0
    rows.requires_grad_()
    (d_rows,) = torch.autograd.grad(backend.combine_expert_rows(rows, w, plan), rows, x)
    assert torch.equal(d_rows[T:T + 3], x[-3:]) and int(d_rows[T + 3:].count_nonzero()) == 0


def test_tokens_past_32_bit_offsets(backend, native, gpu):
    """Tokens whose codes take more than 2^32 bytes: the last ones' products as a small call gives them."""
    T, K, N = 2 ** 21 + 37, 4096, 40
    g = torch.Generator().manual_seed(1)
    last = torch.randn(50, K, generator=g).to(torch.bfloat16).cuda()
    wc, ws = backend.quantize_mxfp4(torch.randn(2, N, K, generator=g).cuda())
    x = torch.zeros(T, K, dtype=torch.bfloat16, device="cuda")
    x[-50:] = last
    ids = torch.zeros(T, 1, dtype=torch.int64, device="cuda")
    ids[-20:] = 1
    y = backend.mxfp4_expert_linear(x, wc, ws, backend.sort_tokens_by_expert(ids, 2))
    want = backend.mxfp4_expert_linear(last, wc, ws, backend.sort_tokens_by_expert(ids[-50:].contiguous(), 2))
    assert torch.equal(y[-50:], want) and int(y[:-50].count_nonzero()) == 0


def test_differentiating_twice_raises(backend, gpu):
    ids, plan, x, rows, w = routed(backend, 6, 2, 3, 16, torch.float32, seed=1)
    x, rows, w = (t.cuda().requires_grad_() for t in (x, rows, w))
    for out, wrt in ((backend.gather_expert_rows(x, plan), x), (backend.combine_expert_rows(rows, w, plan), w)):
        g = torch.randn_like(out).requires_grad_()
        (first,) = torch.autograd.grad(out, wrt, g, create_graph=True)
        with pytest.raises(RuntimeError, match="twice|once_differentiable"):
            first.sum().backward()


def test_python_path_gives_the_same(backend, native, gpu, monkeypatch):
    """Without the host module the same calls run through Python: the same bits, forward and backward."""
    ids, plan, x, rows, w = routed(backend, 30, 3, 5, 264, torch.bfloat16, seed=2)
    x, rows, w = (t.cuda().requires_grad_() for t in (x, rows, w))
    wc, ws = backend.quantize_mxfp4(torch.randn(5, 40, 264 // 8 * 8 - 8, device="cuda", generator=torch.Generator("cuda").manual_seed(1)))
    a = x.detach()[:, :256].contiguous()

    def calls():
        p = backend.sort_tokens_by_expert(torch.from_numpy(ids).cuda(), 5)
        g, c = backend.gather_expert_rows(x, p), backend.combine_expert_rows(rows, w, p)
        grads = torch.autograd.grad((g, c), (x, rows, w), (torch.ones_like(g), torch.ones_like(c)))
        codes = backend.quantize_mxfp4(a, 64)
        return [*p, g, c, *grads, *codes, backend.dequantize_mxfp4(*codes, 64), backend.mxfp4_linear(a, wc[0], ws[0]),
                backend.mxfp4_expert_linear(a, wc, ws, p)]

    first = calls()
    monkeypatch.setattr(native, "host_or_none", lambda: None)
    assert all(torch.equal(p, q) for p, q in zip(first, calls()))
