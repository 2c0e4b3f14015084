"""The norm, its gradient, its 8-bit rows and their linear against plain implementations in 64 bits."""
import importlib
import math

import pytest
import torch

from conftest import PKG_NAME

pytestmark = pytest.mark.gpu

U = 2.0 ** -24                                   # half a step of float32
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
WIDTHS = [1, 2, 3, 7, 8, 9, 63, 64, 65, 511, 512, 513, 1000, 1023, 1025, 1605, 2048, 4096, 4097, 5120, 8192, 8193, 13824, 16383, 16385,
          20000, 32767, 32768]


def data(M, D, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(1000 * D + M + seed)
    x = torch.randn(M, D, generator=g) * scale
    x[:, ::97] *= 20.0
    return x.to(dtype).cuda()


def half(dtype):
    """Half a step of the type, relative."""
    return torch.finfo(dtype).eps / 2


def kept(x, r):
    return x if r is None else (x.float() + r.float()).to(x.dtype)


def exact(h, w, eps):
    h = h.double().cpu()
    rstd = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return h * rstd * (1.0 if w is None else w.double().cpu()), rstd


def check_forward(q, x, w, r, eps=1e-6):
    out = q.rms_norm(x, w, r, eps)
    y, h = out if r is not None else (out, x)
    assert y.shape == x.shape and y.dtype == x.dtype
    if r is not None:
        assert h.dtype == x.dtype and torch.equal(h, kept(x, r))        # one rounding of a 32-bit sum
    want, _ = exact(kept(x, r), w, eps)
    # rstd rounded, two products, the output
    bound = want.abs() * (half(x.dtype) + 4 * U) + torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps
    assert bool(((y.cpu().double() - want).abs() <= bound).all())
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", WIDTHS)
def test_widths(backend, gpu, D, dtype):
    for M in (1, 5):
        x, r = data(M, D, dtype, 1), data(M, D, dtype, 2, 4.0)
        w = 1 + 0.2 * data(1, D, torch.float32, 3)[0]
        check_forward(backend, x, w.to(dtype), None)
        check_forward(backend, x, w, r)
        check_forward(backend, x, None, r, eps=1e-5)


@pytest.mark.parametrize("M", [0, 1, 2, 3, 255, 256, 257, 2047, 2049, 5000])
def test_numbers_of_rows(backend, gpu, M):
    for D in (320, 2304):
        x, r, w = data(M, D, torch.bfloat16, 1), data(M, D, torch.bfloat16, 2), data(1, D, torch.bfloat16, 3)[0]
        check_forward(backend, x, w, None)
        check_forward(backend, x, w, r)


@pytest.mark.parametrize("wdtype", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_types(backend, gpu, dtype, wdtype):
    for D in (640, 641):
        check_forward(backend, data(70, D, dtype, 1), data(1, D, wdtype, 2)[0], data(70, D, dtype, 3))


def test_forms(backend, gpu):
    x, w = data(24, 80, torch.bfloat16, 1), data(1, 80, torch.bfloat16, 2)[0]
    r = data(24, 80, torch.bfloat16, 3)
    y, h = backend.rms_norm(x, w, r)
    for shape in ((2, 3, 4, 80), (24, 1, 80)):
        y2, h2 = backend.rms_norm(x.reshape(shape), w, r.reshape(shape))
        assert y2.shape == shape and torch.equal(y2.reshape(24, 80), y) and torch.equal(h2.reshape(24, 80), h)
    assert torch.equal(backend.rms_norm(x[3], w), backend.rms_norm(x, w)[3])
    wide = data(50, 201, torch.float16, 4)
    for t in (wide[:, 1:], wide[::3, ::2], wide[:1].expand(6, -1), wide.t()):
        v = data(1, t.shape[-1], torch.float16, 5)[0]
        check_forward(backend, t, v, t.flip(0))
    neg = torch.complex(wide.float(), wide.float()).conj().imag
    assert neg.is_neg()
    check_forward(backend, neg, None, neg)
    v = data(1, 402, torch.float32, 6)[0]
    check_forward(backend, wide, v[1:202], None)                          # a weight that starts off 16 bytes
    check_forward(backend, wide, v[::2], None)
    assert torch.equal(*backend.rms_norm(x, None, x.neg()))               # zeros: 0 / sqrt(eps)
    same = backend.rms_norm(x, x[0], x)                                   # the same memory three times
    assert torch.equal(same[1], x + x)


@pytest.mark.parametrize("dtype", DTYPES)
def test_range(backend, gpu, dtype):
    """Rows of very large and very small values, whose squares leave 32 bits."""
    top = float(torch.finfo(dtype).max)
    x = data(6, 300, torch.float32, 1)
    x = x / x.abs().amax()
    scales = torch.tensor([top, top / 16, 1.0, 1e-3, 1e-18 if dtype != torch.float16 else 1e-4, 1e-30 if dtype != torch.float16 else 1e-5])
    t = (x * scales.cuda()[:, None]).to(dtype)
    for eps in (1e-6, 0.0, 1e-40):
        y = backend.rms_norm(t, None, eps=eps)
        want, _ = exact(t, None, eps)
        bound = want.abs() * (half(dtype) + 4 * U) + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
        assert bool(((y.cpu().double() - want).abs() <= bound).all())


def test_values_that_are_not_finite(backend, gpu):
    x = data(6, 200, torch.bfloat16, 1)
    x[1, 5], x[2, 7], x[3] = math.nan, math.inf, 0.0
    y = backend.rms_norm(x)
    ok = [0, 4, 5]
    assert torch.equal(y[ok], backend.rms_norm(x[ok])) and bool(y[1].isnan().all())
    assert bool(y[2, 7].isnan()) and bool((y[2, :7] == 0).all()) and bool((y[3] == 0).all())      # inf / inf, x / inf
    assert bool(backend.rms_norm(x, eps=0.0)[3].isnan().all())                                    # 0 / 0


def grads(f, leaves, out_grads):
    out = f(*leaves)
    out = out if isinstance(out, tuple) else (out,)
    return torch.autograd.grad([o for o, g in zip(out, out_grads) if g is not None], leaves, [g for g in out_grads if g is not None])


def check_gradient(q, x, w, r, dy, dh, eps=1e-6):
    """Against the 64-bit gradient of the norm of the kept sum."""
    leaves = [t.clone().requires_grad_(True) for t in (x, w, r) if t is not None]

    def own(*t):
        t = list(t)
        return q.rms_norm(t.pop(0), None if w is None else t.pop(0), None if r is None else t.pop(0), eps)

    got = grads(own, leaves, (dy, dh))
    h = kept(x, r).cpu().double()
    h64, w64 = h.clone().requires_grad_(True), (torch.ones(x.shape[-1]).double() if w is None else w.cpu().double()).requires_grad_(True)
    y = h64 / torch.sqrt((h64 * h64).mean(-1, keepdim=True) + eps) * w64
    g = dy.cpu().double()
    want_h, want_w = torch.autograd.grad(y, (h64, w64), g)
    add = torch.zeros_like(h) if dh is None else dh.cpu().double()
    rstd = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    n, gw = h * rstd, (g * w64).detach()
    mean = (gw * n).mean(-1, keepdim=True)
    # t = gw - n mean: gw off by U, n by 3 U (rstd's rounding and two products), their product and difference by U each; then the
    # product with rstd by 2 U and the sum with d_h by U.  The mean adds gw n with gw rounded to 32 bits before (the rest in
    # 64): off by at most U mean|gw n|, a bound that holds where the terms cancel and U |mean| does not, and is itself rounded.
    size = rstd * (gw.abs() + n.abs() * mean.abs())
    bound = (want_h + add).abs() * half(x.dtype) + 8 * U * (size + add.abs()) + torch.finfo(x.dtype).tiny
    bound = bound + 2 * U * rstd * n.abs() * (gw * n).abs().mean(-1, keepdim=True)
    for d in (got[0],) if r is None else (got[0], got[-1]):
        assert d.dtype == x.dtype and d.shape == x.shape
        assert bool(((d.cpu().double() - (want_h + add)).abs() <= bound).all())
    if w is not None:
        M = h.numel() // h.shape[-1]
        terms = (g * n).abs().reshape(-1, h.shape[-1]).sum(0)
        depth = math.ceil(M / min(M, 512)) + math.ceil(min(M, 512) / 16) + 16 + 3
        bound = want_w.abs() * half(w.dtype) + depth * U * terms + torch.finfo(w.dtype).tiny
        assert got[1].dtype == w.dtype and bool(((got[1].cpu().double() - want_w).abs() <= bound).all())
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", WIDTHS)
def test_gradient_widths(backend, gpu, D, dtype):
    M = 6
    x, r, dy, dh = (data(M, D, dtype, s) for s in range(4))
    w = 1 + 0.2 * data(1, D, torch.float32, 9)[0]
    check_gradient(backend, x, w, r, dy, dh)
    check_gradient(backend, x, w.to(dtype), None, dy, None)


@pytest.mark.parametrize("M", [1, 2, 511, 512, 513, 3000])
def test_gradient_rows(backend, gpu, M):
    for D in (130, 1536):
        x, r, dy, dh = (data(M, D, torch.bfloat16, s) for s in range(4))
        w = data(1, D, torch.bfloat16, 9)[0]
        first = check_gradient(backend, x, w, r, dy, dh)
        again = check_gradient(backend, x, w, r, dy, dh)
        assert all(torch.equal(a, b) for a, b in zip(first, again))     # no order of sums that changes
        check_gradient(backend, x, None, r, dy, None)
        check_gradient(backend, x, w, None, dy, None)


def test_gradient_range(backend, gpu):
    x = data(4, 300, torch.float32, 1) * torch.tensor([1e18, 1e30, 1e-18, 1.0], device="cuda")[:, None]
    check_gradient(backend, x, data(1, 300, torch.float32, 2)[0], None, data(4, 300, torch.float32, 3), None)


def test_gradient_by_differences(backend, gpu):
    x, w, r = data(3, 12, torch.float32, 1), data(1, 12, torch.float32, 2)[0], data(3, 12, torch.float32, 3)
    dy, dh = data(3, 12, torch.float32, 4), data(3, 12, torch.float32, 5)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, r)]
    got = grads(lambda a, b, c: backend.rms_norm(a, b, c), leaves, (dy, dh))

    def value(a, b, c):
        y, h = backend.rms_norm(a, b, c)
        return float((y.double() * dy.double()).sum() + (h.double() * dh.double()).sum())

    size = float((backend.rms_norm(x, w, r)[0] * dy).abs().sum() + (kept(x, r) * dh).abs().sum())
    step = 2.0 ** -6
    for i, t in enumerate((x, w, r)):
        for at in [(0, 0), (1, 5), (2, 11)] if t.dim() == 2 else [(0,), (7,)]:
            ends = []
            for sign in (1, -1):
                moved = [v.clone() for v in (x, w, r)]
                moved[i][at] += sign * step
                ends.append(value(*moved))
            diff = (ends[0] - ends[1]) / (2 * step)
            # rounding of the values over the step, and step^2 / 6 of a third derivative: y's terms over the row's size squared
            assert abs(diff - float(got[i][at])) <= 8 * U * size / step + step ** 2 * size


def test_gradient_forms(backend, gpu):
    x, w = data(20, 96, torch.float32, 1).requires_grad_(True), data(1, 96, torch.float32, 2)[0].requires_grad_(True)
    r = data(20, 96, torch.float32, 3).requires_grad_(True)
    dy, dh = data(20, 96, torch.float32, 4), data(20, 96, torch.float32, 5)
    y, h = backend.rms_norm(x, w, r)
    whole = torch.autograd.grad((y, h), (x, w, r), (dy, dh), retain_graph=True)
    only_h = torch.autograd.grad(h, (x, w, r), dh, retain_graph=True, allow_unused=True)       # the stream's alone
    assert torch.equal(only_h[0], dh) and torch.equal(only_h[2], dh) and only_h[1] is None
    only_y = torch.autograd.grad(y, (x, w, r), dy, retain_graph=True)
    assert torch.equal(only_y[1], whole[1])
    for i, leaf in enumerate((x, w, r)):                                                     # one at a time
        y1, h1 = backend.rms_norm(x if i == 0 else x.detach(), w if i == 1 else w.detach(), r if i == 2 else r.detach())
        assert torch.equal(torch.autograd.grad((y1, h1) if i != 1 else y1, leaf, (dy, dh) if i != 1 else dy)[0], whole[i])
    y1, h1 = backend.rms_norm(x, None, r)
    assert len(torch.autograd.grad((y1, h1), (x, r), (dy, dh))) == 2
    y1, h1 = backend.rms_norm(x.detach(), None, r)
    assert torch.autograd.grad((y1, h1), r, (dy, dh))[0].shape == r.shape
    d = torch.autograd.grad(backend.rms_norm(x.t(), None), x, dy.t())[0]                      # strided both ways
    assert torch.equal(d, torch.autograd.grad(backend.rms_norm(x.t().contiguous(), None), x, dy.t().contiguous())[0])
    assert torch.autograd.grad(backend.rms_norm(x, w).sum(), x)[0].shape == x.shape           # a broadcast gradient
    both = x * 1.0
    y, h = backend.rms_norm(both, w, both)                                                    # one tensor twice
    d = torch.autograd.grad((y, h), x, (dy, dh))[0]
    y2, h2 = backend.rms_norm(x, w, x.detach())
    assert torch.equal(d, 2 * torch.autograd.grad((y2, h2), x, (dy, dh))[0])
    x.grad = w.grad = r.grad = None
    y, h = backend.rms_norm(x, w, r)
    ((y * dy).sum() + (h * dh).sum()).backward()
    assert all(torch.equal(t.grad, g) for t, g in zip((x, w, r), whole))
    x.grad.mul_(2)
    assert torch.equal(r.grad, whole[2])                                                      # leaves' gradients are their own
    empty = x[:0]
    assert bool((torch.autograd.grad(backend.rms_norm(empty, w).sum(), w)[0] == 0).all())
    y = backend.rms_norm(x, w)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        d, = torch.autograd.grad(y.sum(), x, create_graph=True)
        d.sum().backward()
    y = backend.rms_norm(x, w)
    with torch.no_grad():
        w.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y, h = backend.rms_norm(x.detach(), w, r)
    with torch.no_grad():
        h.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def rotation(backend, G):
    return backend._hadamard(G, "cpu", torch.float64)


def check_rows(backend, x, w, r, G, i8t=False, eps=1e-6):
    native = importlib.import_module(PKG_NAME + "._int4.native")
    out = backend.rms_norm_int8(x, w, r, eps, G, i8t=i8t)
    rows, h = out if r is not None else (out, x)
    rows.check()
    D = x.shape[-1]
    M = x.numel() // D
    assert rows.shape == tuple(x.shape) and rows.dtype == x.dtype and rows.i8t == i8t and rows.convrot_groupsize == G
    if r is not None:
        assert torch.equal(h, kept(x, r))
    codes = rows.codes
    if i8t:
        assert codes.shape[0] % 256 == 0
        whole = native.i8t_to_int8(codes, codes.shape[0])
        assert not bool(whole[M:].any())
        codes = whole[:M].contiguous()
    y, _ = exact(kept(x, r), w, eps)
    z = (y.reshape(-1, G) @ rotation(backend, G)).reshape(M, D)
    scale = z.abs().amax(-1).clamp(min=1e-10) / 127
    assert bool(((rows.scales.cpu().double() - scale).abs() <= scale * U * (1 + 2.0 ** -20)).all())
    steps = z / rows.scales.cpu().double()[:, None]
    # the nearest code; 2^-30 of a step is what two 64-bit computations may differ by at a border
    assert bool(((codes.cpu().double() - steps).abs() <= 0.5 + 2.0 ** -30).all())
    return rows


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("G,D", [(16, 16), (16, 48), (16, 1008), (16, 1040), (16, 16400), (64, 64), (64, 1600), (64, 4160), (64, 17024),
                                 (256, 256), (256, 768), (256, 1024), (256, 1280), (256, 2304), (256, 4096), (256, 5120), (256, 13824),
                                 (256, 16384), (256, 16640), (256, 32768)])
def test_int8_widths(backend, gpu, G, D, dtype):
    for M in (1, 9):
        x, r = data(M, D, dtype, 1), data(M, D, dtype, 2, 4.0)
        w = 1 + 0.2 * data(1, D, torch.float32, 3)[0]
        check_rows(backend, x, w.to(dtype), None, G)
        a = check_rows(backend, x, w, r, G)
        if D % 64 == 0:
            b = check_rows(backend, x, w, r, G, i8t=True)
            assert torch.equal(a.scales, b.scales)


@pytest.mark.parametrize("M", [0, 1, 255, 256, 257, 3000])
def test_int8_numbers_of_rows(backend, gpu, M):
    x, r = data(M, 512, torch.bfloat16, 1), data(M, 512, torch.bfloat16, 2)
    check_rows(backend, x, None, r, 256)
    check_rows(backend, x, None, None, 64, i8t=True)


def test_int8_ties_go_to_even(backend, gpu):
    """A row of 127 and halves, one element a group: its scale is 2^-1 / sqrt(mean), so steps are whole halves."""
    D, G = 256, 16
    x = torch.zeros(1, D, device="cuda")
    v = [254.0, 1.0, 3.0, 5.0, 7.0, -1.0, -3.0, -5.0, 253.0, -253.0]      # half steps: 127, .5, 1.5, 2.5, 3.5, ...
    y = torch.zeros(D, dtype=torch.float64)
    for i, t in enumerate(v):
        y[G * i] = t
    x[0] = (y.reshape(-1, G) @ rotation(backend, G)).reshape(D).float().cuda()      # quarters: exact
    rows = backend.rms_norm_int8(x, None, None, 0.0, G)
    scale = float(rows.scales[0])
    want = torch.zeros(D, dtype=torch.int8)
    for i, t in enumerate(v):
        steps = t / 2
        want[G * i] = round(steps)                                        # to even
    near = torch.tensor([t for t in v])
    # the scale is rounded to 32 bits: a border that it moves by U goes to either neighbour, all others as they are
    got = rows.codes[0].cpu()
    assert scale > 0 and bool(((got - want).abs() <= (want != 127).to(torch.int8)).all()) and got[0] == 127
    assert not bool(got[[i for i in range(D) if i % G]].any()) and len(near) == 10


def test_int8_values(backend, gpu):
    """Zeros, values that are not finite, an infinite weight; rows beside them stay as they are."""
    x = data(7, 512, torch.bfloat16, 1)
    clean = backend.rms_norm_int8(x)
    x[1, 5], x[2, 7], x[3] = math.nan, -math.inf, 0.0
    for i8t in (False, True):
        rows = backend.rms_norm_int8(x, i8t=i8t)
        assert rows.scales[1:3].isnan().all() and rows.scales[3] == torch.tensor(1e-10 / 127, dtype=torch.float64).float()
        if not i8t:
            assert not bool(rows.codes[1:4].any())
            assert torch.equal(rows.codes[[0, 4, 5, 6]], clean.codes[[0, 4, 5, 6]])
        assert torch.equal(rows.scales[[0, 4, 5, 6]], clean.scales[[0, 4, 5, 6]])
    rows = backend.rms_norm_int8(x, eps=0.0)
    assert bool(rows.scales[3].isnan()) and not bool(rows.codes[3].any())
    for bad in (math.inf, math.nan):
        w = torch.ones(512, device="cuda")
        w[100] = bad
        rows = backend.rms_norm_int8(x, w)
        assert bool(rows.scales.isnan().all()) and not bool(rows.codes.any())
    big = data(2, 512, torch.float32, 2) * 1e36
    check_rows(backend, big, None, None, 256)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(1, 256, 64), (1, 5120, 1000), (37, 1600, 2400), (300, 4096, 1024), (512, 12288, 2048), (4096, 512, 1536)])
def test_rows_linear(backend, native, gpu, M, K, N, dtype):
    """The products of the codes, bit for bit those of the int8 product on them; and of a norm with its linears, the
    8-bit grids' own distance from the products in 64 bits."""
    G = 256 if K % 256 == 0 else 64
    x, r, nw = data(M, K, dtype, 1), data(M, K, dtype, 2), (1 + 0.2 * data(1, K, torch.float32, 3)[0]).to(dtype)
    int8 = importlib.import_module(PKG_NAME + "._int4.int8_eager")
    g = torch.Generator().manual_seed(5)
    W = torch.randn(N, K, generator=g) * K ** -0.5
    qw, ws = int8.quantize_convrot_w8a8_weight(W.half().cuda(), G)
    bias = torch.randn(N, generator=g).to(dtype).cuda()
    w8t = backend.prepare_convrot_w8a8_weight_i8t(qw)
    plain, h = backend.rms_norm_int8(x, nw, r, convrot_groupsize=G)
    tiled, h2 = backend.rms_norm_int8(x, nw, r, convrot_groupsize=G, i8t=True)
    assert torch.equal(h, h2)
    for b in (None, bias):
        y = backend.convrot_w8a8_linear_rows(plain, qw, ws, b)
        assert y.dtype == dtype and y.shape == (M, N)
        want = native.int8_convrot_gemm(plain.codes, qw, plain.scales, ws, b, torch.float32).to(dtype)
        assert torch.equal(y, want)
        assert torch.equal(backend.convrot_w8a8_linear_rows(tiled, qw, ws, b, qweight_i8t=w8t), want)
        assert torch.equal(backend.convrot_w8a8_linear_rows(tiled, qw, ws, b), want)
    n, _ = exact(kept(x, r), nw, 1e-6)
    n = n.cuda()
    back = int8.dequantize_convrot_w8a8_weight(qw, ws, G, torch.float32).double()
    # rows' codes are half a step of their scale off at most, and rotated back keep that length
    far = (y.double() - (n @ back.T + bias.double())).abs()
    lengths = back.norm(dim=-1)
    bound = plain.scales.double()[:, None] * 0.5 * K ** 0.5 * lengths[None] + (y.double().abs() + 1e-3) * (half(dtype) + 8 * U)
    assert bool((far <= bound).all())


def test_rows_of_leading_sizes(backend, gpu):
    x = data(24, 256, torch.bfloat16, 1).reshape(2, 3, 4, 256)
    int8 = importlib.import_module(PKG_NAME + "._int4.int8_eager")
    qw, ws = int8.quantize_convrot_w8a8_weight(torch.randn(96, 256).half().cuda(), 256)
    for i8t in (False, True):
        rows = backend.rms_norm_int8(x, i8t=i8t)
        y = backend.convrot_w8a8_linear_rows(rows, qw, ws)
        assert y.shape == (2, 3, 4, 96)
        flat = backend.convrot_w8a8_linear_rows(backend.rms_norm_int8(x.reshape(24, 256), i8t=i8t), qw, ws)
        assert torch.equal(y.reshape(24, 96), flat)
        none = backend.rms_norm_int8(x[:0], i8t=i8t)
        assert backend.convrot_w8a8_linear_rows(none, qw, ws).shape == (0, 3, 4, 96)


def test_gradients_are_refused(backend, gpu):
    x = data(4, 256, torch.float32, 1).requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradient"):
        backend.rms_norm_int8(x)
    with torch.no_grad():
        rows = backend.rms_norm_int8(x)
    assert rows.codes.shape == (4, 256)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x))
        for f in (backend.rms_norm, backend.rms_norm_int8, lambda t: backend.choose_experts(t, 2)):
            with pytest.raises(RuntimeError, match="gradient"):
                f(dual)


def test_python_path_answers_alike(backend, native, gpu, monkeypatch):
    x, r, dy, dh = (data(65, 768, torch.bfloat16, s) for s in range(4))
    w = data(1, 768, torch.float32, 9)[0]
    int8 = importlib.import_module(PKG_NAME + "._int4.int8_eager")
    qw, ws = int8.quantize_convrot_w8a8_weight(torch.randn(96, 768).half().cuda(), 256)
    w8t = backend.prepare_convrot_w8a8_weight_i8t(qw)

    def all_of():
        out = [*backend.rms_norm(x, w, r), backend.rms_norm(x)]
        leaves = [t.clone().requires_grad_(True) for t in (x, w, r)]
        out += grads(backend.rms_norm, leaves, (dy, dh))
        out += grads(lambda a: backend.rms_norm(a, w), leaves[:1], (dy,))
        for i8t in (False, True):
            rows, h = backend.rms_norm_int8(x, w, r, i8t=i8t)
            out += [rows.codes, rows.scales, h, backend.convrot_w8a8_linear_rows(rows, qw, ws, qweight_i8t=w8t if i8t else None)]
        return out

    host = all_of()
    monkeypatch.setattr(native, "host_or_none", lambda: None)
    assert all(torch.equal(a, b) for a, b in zip(host, all_of()))


def test_streams_and_graphs(backend, gpu):
    """Norm, its rows and their linear, captured together and replayed."""
    x, r, w = data(300, 1024, torch.bfloat16, 1), data(300, 1024, torch.bfloat16, 2), data(1, 1024, torch.bfloat16, 3)[0]
    int8 = importlib.import_module(PKG_NAME + "._int4.int8_eager")
    qw, ws = int8.quantize_convrot_w8a8_weight(torch.randn(512, 1024).half().cuda(), 256)
    w8t = backend.prepare_convrot_w8a8_weight_i8t(qw)

    def step():
        y, h = backend.rms_norm(x, w, r)
        rows, h2 = backend.rms_norm_int8(h, w, y, i8t=True)
        return y, h, h2, backend.convrot_w8a8_linear_rows(rows, qw, ws, qweight_i8t=w8t)

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(4):
        x.copy_(data(300, 1024, torch.bfloat16, 10 + seed))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_gradient_in_a_graph(backend, gpu):
    """Two graphs with workspaces of their own, replayed in turn beside eager calls."""
    sets = []
    for D in (640, 1100):
        x, r, dy, dh = (data(900, D, torch.bfloat16, s) for s in range(4))
        leaves = [x.requires_grad_(True), data(1, D, torch.float32, 9)[0].requires_grad_(True), r.requires_grad_(True)]
        step = lambda leaves=leaves, dy=dy, dh=dh: grads(backend.rms_norm, leaves, (dy, dh))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        sets.append((leaves, step, graph, out))
    for seed in range(3):
        for leaves, step, graph, out in sets:
            with torch.no_grad():
                leaves[0].copy_(data(900, leaves[0].shape[1], torch.bfloat16, 20 + seed))
            graph.replay()
        for leaves, step, graph, out in sets:
            want = step()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_past_32_bits(backend, gpu):
    """Rows whose elements' numbers pass 2^31 and bytes 2^32; the last rows are the first ones' copies."""
    M, D = 140000, 16384
    x = torch.empty(M, D, dtype=torch.bfloat16, device="cuda")
    x.normal_()
    x[-5:] = x[:5]
    w = data(1, D, torch.bfloat16, 1)[0]
    y = backend.rms_norm(x, w)
    assert torch.equal(y[-5:], y[:5]) and torch.equal(y[:5], backend.rms_norm(x[:5], w))
    del y
    rows = backend.rms_norm_int8(x, w)
    few = backend.rms_norm_int8(x[:5], w)
    assert torch.equal(rows.codes[-5:], few.codes) and torch.equal(rows.scales[-5:], few.scales)
    del rows
    tiled = backend.rms_norm_int8(x, w, i8t=True)
    assert torch.equal(tiled.scales[-5:], few.scales)
    last = M % 256
    native = importlib.import_module(PKG_NAME + "._int4.native")
    assert torch.equal(native.i8t_to_int8(tiled.codes[-256:].contiguous(), 256)[last - 5:last], few.codes)
    del tiled
    leaf = x.requires_grad_(True)
    d, = torch.autograd.grad(backend.rms_norm(leaf, w), leaf, x.detach())
    head = x.detach()[:5].clone().requires_grad_(True)
    want, = torch.autograd.grad(backend.rms_norm(head, w), head, x.detach()[:5])
    assert torch.equal(d[:5], want) and torch.equal(d[-5:], want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [3, 64, 100, 200, 320, 520, 1024, 2304, 4097, 5120, 8192, 8193, 16384, 20000, 32768])
def test_many_rows(backend, gpu, D, dtype):
    """Rows enough for every way they are shared out, several to a workgroup in turn for the gradient; references in 64 bits."""
    M = 1333 if D > 1024 else 7001
    g = torch.Generator(device="cuda").manual_seed(D)
    x, r, dy, dh = (torch.randn(M, D, generator=g, device="cuda").to(dtype) for _ in range(4))
    w = 1 + 0.2 * torch.randn(D, generator=g, device="cuda")
    leaves = [t.clone().requires_grad_(True) for t in (x, w, r)]
    y, h = backend.rms_norm(leaves[0], leaves[1], leaves[2])
    assert torch.equal(h, kept(x, r))
    h64, w64 = h.detach().double(), w.double()
    rstd = 1 / torch.sqrt((h64 * h64).mean(-1, keepdim=True) + 1e-6)
    n = h64 * rstd
    tiny = torch.finfo(dtype).tiny
    assert bool(((y.double() - n * w64).abs() <= (n * w64).abs() * (half(dtype) + 4 * U) + tiny).all())
    assert torch.equal(backend.rms_norm(h.detach(), w), y)
    d_x, d_w, d_r = torch.autograd.grad((y, h), leaves, (dy, dh))
    assert torch.equal(d_x, d_r)
    gw = dy.double() * w64
    mean = (gw * n).mean(-1, keepdim=True)
    want = rstd * (gw - n * mean) + dh.double()
    size = rstd * (gw.abs() + n.abs() * mean.abs())                     # as the bound above of each gradient
    bound = want.abs() * half(dtype) + 8 * U * (size + dh.double().abs()) + tiny
    bound += 2 * U * rstd * n.abs() * (gw * n).abs().mean(-1, keepdim=True)
    assert bool(((d_x.double() - want).abs() <= bound).all())
    terms = dy.double() * n
    # each sum: a team's rows (M over 256 teams at the least), up to 32 teams, 1024 workgroups' parts in 64 strands
    depth = math.ceil(M / 256) + 32 + 16 + 2 + 16 + 3
    assert bool(((d_w.double() - terms.sum(0)).abs() <= depth * U * terms.abs().sum(0) + tiny).all())
    plain, = torch.autograd.grad(backend.rms_norm(leaves[0], None), leaves[0], dy)
    h64 = x.double()
    rstd = 1 / torch.sqrt((h64 * h64).mean(-1, keepdim=True) + 1e-6)
    n, gw = h64 * rstd, dy.double()
    mean = (gw * n).mean(-1, keepdim=True)
    want = rstd * (gw - n * mean)
    bound = want.abs() * half(dtype) + 8 * U * rstd * (gw.abs() + n.abs() * mean.abs()) + tiny
    bound += 2 * U * rstd * n.abs() * (gw * n).abs().mean(-1, keepdim=True)
    assert bool(((plain.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("G,D", [(16, 208), (16, 2064), (64, 320), (64, 4160), (256, 256), (256, 512), (256, 768), (256, 2304), (256, 5120),
                                 (256, 8192), (256, 16384), (256, 20480)])
def test_int8_many_rows(backend, gpu, G, D, dtype):
    """Rows enough for two chunks a lane, and short rows several to a wave; the codes of a row do not depend on the call's others."""
    M = 4500 if D < 1024 else 1500
    x, r = data(M, D, dtype, 1), data(M, D, dtype, 2, 4.0)
    w = 1 + 0.2 * data(1, D, torch.float32, 3)[0]
    rows = check_rows(backend, x, w, r, G)
    few, h = backend.rms_norm_int8(x[-3:], w, r[-3:], convrot_groupsize=G)
    assert torch.equal(few.codes, rows.codes[-3:]) and torch.equal(few.scales, rows.scales[-3:])
    check_rows(backend, x, w.to(dtype), None, G, i8t=D % 64 == 0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [40, 512, 1024, 2048, 4096, 5000, 8192, 13824, 16384, 32768])
def test_gradient_of_few_rows(backend, gpu, D, dtype):
    """One workgroup, of one team or several, and the few beside it: the weight's gradient is there in each."""
    w = 1 + 0.2 * data(1, D, torch.float32, 9)[0]
    for M in (1, 2, 3, 4, 7, 25):
        x, r, dy, dh = (data(M, D, dtype, s) for s in range(4))
        check_gradient(backend, x, w, r, dy, dh)
        check_gradient(backend, x, w.to(dtype), None, dy, None)
