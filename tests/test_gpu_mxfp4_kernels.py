"""GPU checks of every kernel of the MXFP4 products at depth: each instance of the staged one over numbers of stages that
wrap its ring, the one for few rows past the width that its LDS holds, rotations inside and ahead of the products."""
import numpy as np
import pytest
import torch

import mx_format as mx
from test_gpu_experts import choice
from test_gpu_mxfp4 import DTYPES, exact_operands, np64, outliers, rounded_once, say
from test_mxfp4_kernel_query import kernel

pytestmark = pytest.mark.gpu


def exact_linear(backend, M, N, K):
    x, wc, ws = exact_operands(M, N, K, seed=M + N + K)
    bias = torch.from_numpy(np.random.RandomState(1).randint(-64, 64, N) / 8.0).cuda()
    w, s = torch.from_numpy(wc).cuda(), torch.from_numpy(ws).cuda()
    xt = torch.from_numpy(x).cuda()
    want = xt @ torch.from_numpy(mx.dequantize(wc, ws)).cuda().T + bias         # float64
    for dtype in DTYPES:
        assert torch.equal(backend.mxfp4_linear(xt.to(dtype), w, s, bias.to(dtype)), want.float().to(dtype))


# K of 1 to 13 stages of 256, the last one whole and not, and of 16
DEPTHS = [256 * n - (96 if n % 2 else 0) for n in range(1, 14)] + [4000, 4096]


@pytest.mark.parametrize("K", DEPTHS)
@pytest.mark.parametrize("M,N,tile", [(200, 700, (64, 128, 4)), (500, 5000, (128, 128, 4)), (1100, 4000, (128, 128, 2))])
def test_stages(backend, native, gpu, M, N, K, tile):
    say("stages", M, N, K, tile)
    assert kernel(native, M, N, K) == (*tile, 0)
    exact_linear(backend, M, N, K)


@pytest.mark.parametrize("K", [2080, 2304, 2336, 2560, 2848, 3040, 3328, 3584, 4096])
def test_stages_of_the_large_tile(backend, native, gpu, K):
    M, N = 3000, 4100
    say("stages", M, N, K)
    assert kernel(native, M, N, K) == (256, 256, 2, 0)
    exact_linear(backend, M, N, K)


@pytest.mark.parametrize("rows", [False, True], ids=["tokens", "sorted"])
@pytest.mark.parametrize("T,k,E,N,K,tile", [(60, 3, 4, 700, 2336, (64, 128, 4)), (60, 3, 4, 700, 4096, (64, 128, 4)),
                                            (400, 4, 6, 1200, 2336, (128, 128, 4)), (400, 4, 6, 1200, 2816, (128, 128, 4)),
                                            (900, 3, 6, 1500, 2336, (128, 128, 2)), (1500, 3, 8, 900, 2560, (128, 128, 2))])
def test_stages_of_experts(backend, native, gpu, T, k, E, N, K, tile, rows):
    say("stages of experts", T, k, E, N, K, tile, rows)
    assert kernel(native, T * k, N, K, E, 0 if rows else T) == (*tile, 0)
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
        assert torch.equal(backend.mxfp4_expert_linear(xt.to(dtype), w, s, plan, sorted_rows=rows), want.float().to(dtype))


@pytest.mark.parametrize("M,N,K", [(1, 100, 32768), (1, 100, 32800), (4, 33, 32800), (5, 100, 33024), (20, 70, 32800), (32, 40, 40000)])
def test_few_wide_rows(backend, native, gpu, M, N, K):
    """Rows wider than 32768, whose scales the kernel for few rows reads from memory.  Products are multiples of 2^-8 with
    a deviation of about 12, their sums' is 12 K^(1/2) < 2^11.3: no partial sum comes near 2^16."""
    say("few wide rows", M, N, K)
    assert kernel(native, M, N, K)[2] == 0
    exact_linear(backend, M, N, K)


@pytest.mark.parametrize("T,k,E", [(1, 2, 3), (3, 2, 2), (9, 2, 4)])
def test_few_wide_rows_of_experts(backend, native, gpu, T, k, E):
    N, K = 50, 32832
    say("few wide rows of experts", T, k, E)
    assert kernel(native, T * k, N, K, E, T)[2] == 0
    ids = choice(T, k, E, seed=T, unused=0.2)
    order, _, offsets = mx.plan(ids, E)
    x, wc, ws = exact_operands(T, N, K, seed=T, E=E)
    want = np.zeros((T * k, N))
    for e in range(E):
        r = slice(offsets[e], offsets[e + 1])
        want[r] = x[order[r] // k] @ mx.dequantize(wc[e], ws[e]).T
    plan = backend.sort_tokens_by_expert(torch.from_numpy(ids).cuda(), E)
    y = backend.mxfp4_expert_linear(torch.from_numpy(x).float().cuda(), torch.from_numpy(wc).cuda(),
                                    torch.from_numpy(ws).cuda(), plan)
    assert np.array_equal(np64(y), want)


@pytest.mark.parametrize("M", [1, 6, 40])
def test_the_widest_rows(backend, gpu, M):
    """K = 2^24: zeros but for some blocks and the last, whose products fp32 adds up exactly."""
    N, K = 132, 2 ** 24
    say("widest rows", M)
    g = torch.Generator("cuda").manual_seed(M)
    w = torch.randint(0, 256, (N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    s = torch.randint(124, 128, (N, K // 32), generator=g, device="cuda", dtype=torch.uint8)
    blocks = np.append(np.sort(np.random.RandomState(M).choice(K // 32 - 1, 60, replace=False)), K // 32 - 1)
    few, _, _ = exact_operands(M, 1, 32 * len(blocks), seed=M)
    at = torch.from_numpy((blocks[:, None] * 32 + np.arange(32)).reshape(-1)).cuda()
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    x[:, at] = torch.from_numpy(few).cuda().to(torch.bfloat16)
    b = torch.from_numpy(blocks).cuda()
    wc = w.view(N, K // 32, 16)[:, b].reshape(N, -1).cpu().numpy()
    want = few @ mx.dequantize(wc, s[:, b].cpu().numpy()).T
    y = backend.mxfp4_linear(x, w, s)
    assert torch.equal(y.cpu(), torch.from_numpy(want).float().to(torch.bfloat16))


def check_rotated(y, a, b, bias, dtype):
    """As the definition in 64 bits on the quantizer's own codes; K roundings of 2^-23 of the sum of magnitudes in the fp32
    sums, then the output's."""
    K = a.shape[-1]
    off = (K + 2) * 2.0 ** -23 * (np.abs(a) @ np.abs(b).T + np.abs(bias))
    assert y.dtype == dtype and rounded_once(y, a @ b.T + bias, off, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("G", [None, 16, 64, 256])
@pytest.mark.parametrize("M,N,K", [(1, 300, 1792), (2, 300, 5120), (3, 130, 2816), (4, 9000, 512), (4, 100, 5120), (5, 70, 2304), (16, 33, 768),
                                   (32, 100, 1280)])
def test_few_rotated_rows(backend, native, gpu, M, N, K, G, dtype):
    """Few rows, quantized in the product up to four of them: each group size, with more 16-value units than threads."""
    say("few rotated rows", M, N, K, G, dtype)
    assert kernel(native, M, N, K)[2:] == (0, M <= 4)
    x = outliers(M, K, dtype, seed=M + K).cuda()
    wc, ws = backend.quantize_mxfp4(torch.randn(N, K, generator=torch.Generator().manual_seed(5)).cuda() * K ** -0.5, G)
    xc, xs = backend.quantize_mxfp4(x, G)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(6)).to(dtype)
    y = backend.mxfp4_linear(x, wc, ws, bias.cuda(), G)
    check_rotated(y, mx.dequantize(xc.cpu().numpy(), xs.cpu().numpy()), mx.dequantize(wc.cpu().numpy(), ws.cpu().numpy()),
                  np64(bias), dtype)


@pytest.mark.parametrize("rows", [False, True], ids=["tokens", "sorted"])
@pytest.mark.parametrize("G", [16, 64, 256])
@pytest.mark.parametrize("T,k,E,N,K,dtype", [(1, 3, 5, 100, 1280, torch.bfloat16), (2, 4, 5, 64, 2560, torch.float16),
                                             (4, 2, 3, 40, 4096, torch.float32), (6, 4, 3, 90, 768, torch.bfloat16),
                                             (11, 2, 2, 70, 512, torch.float32), (50, 3, 6, 130, 1280, torch.float16),
                                             (300, 2, 4, 300, 2304, torch.bfloat16)])
def test_rotated_experts(backend, native, gpu, T, k, E, N, K, dtype, G, rows):
    """Rows quantized in the product (8 at most), ahead of it for few rows, and for staged tiles."""
    R = T * k
    say("rotated experts", T, k, E, N, K, dtype, G, rows)
    assert kernel(native, R, N, K, E, 0 if rows else T)[2:] == (0 if R <= 32 else 4, R <= 8)
    ids = choice(T, k, E, seed=T + N)
    order, _, offsets = mx.plan(ids, E)
    plan = backend.sort_tokens_by_expert(torch.from_numpy(ids).cuda(), E)
    x = outliers(R if rows else T, K, dtype, seed=T + K).cuda()
    wc, ws = backend.quantize_mxfp4(torch.randn(E, N, K, generator=torch.Generator().manual_seed(5)).cuda() * K ** -0.5, G)
    xc, xs = backend.quantize_mxfp4(x, G)
    bias = torch.randn(E, N, generator=torch.Generator().manual_seed(6)).to(dtype)
    y = backend.mxfp4_expert_linear(x, wc, ws, plan, bias.cuda(), G, sorted_rows=rows).cpu()
    a, b = mx.dequantize(xc.cpu().numpy(), xs.cpu().numpy()), mx.dequantize(wc.cpu().numpy(), ws.cpu().numpy())
    for e in range(E):
        r = slice(offsets[e], offsets[e + 1])
        check_rotated(y[r], a[r] if rows else a[order[r] // k], b[e], np64(bias)[e], dtype)
    assert int(y[offsets[-1]:].count_nonzero()) == 0
