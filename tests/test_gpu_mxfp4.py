"""GPU checks of the microscaled 4-bit tier against its definition in 64 bits."""
import numpy as np
import pytest
import torch

import mx_format as mx

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def say(*a):
    print(*a, flush=True)


def np64(t):
    return t.detach().cpu().double().numpy()


def rounded_once(y, want, off, dtype) -> bool:
    """Whether every y is a value within ``off`` of ``want`` (64 bits) rounded to ``dtype``: rounding is monotone, so
    it lies between the roundings of the ends."""
    lo, hi = (np64(torch.from_numpy(np.asarray(v)).float().to(dtype)) for v in (want - off, want + off))
    return bool(((lo <= np64(y)) & (np64(y) <= hi)).all())


def outliers(M, K, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g)
    x[:, torch.randperm(K, generator=g)[:max(1, K // 100)]] *= 20
    return x.to(dtype)


# ---- quantization --------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (5, 160), (2, 3, 64), (257, 1600), (16, 5120), (70000, 32)])
def test_codes_and_scales(backend, gpu, shape, dtype):
    say("quantize", shape, dtype)
    M = int(np.prod(shape[:-1]))
    x = outliers(M, shape[-1], dtype, seed=M).reshape(shape)
    codes, scales = backend.quantize_mxfp4(x.cuda())
    ec, es = mx.quantize(np64(x))
    assert codes.shape == (*shape[:-1], shape[-1] // 2) and scales.shape == (*shape[:-1], shape[-1] // 32)
    assert np.array_equal(scales.cpu().numpy(), es)
    assert np.array_equal(codes.cpu().numpy(), ec)


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_tie_and_scale(backend, gpu, dtype):
    """Every middle between codes, its neighbours on either side, both signs, at every power of two of the type."""
    lo, hi = {torch.bfloat16: (-133, 127), torch.float16: (-24, 15), torch.float32: (-149, 127)}[dtype]
    step = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[dtype]
    base = np.concatenate([mx.MIDDLES, mx.GRID[1:], mx.MIDDLES * (1 - step), mx.MIDDLES * (1 + 2 * step), [0.0]])
    rows = []
    for e in range(lo, hi + 1):
        v = np.zeros(32)
        v[:len(base)] = base / 4 * 2.0 ** e                  # the largest (6 / 4) gives the block's scale 2^(e - 2)
        rows += [v, -v]
    with np.errstate(over="ignore"):
        x = torch.from_numpy(np.array(rows)).to(dtype)
    x = x[torch.isfinite(x).all(dim=1)]
    say("ties", dtype, tuple(x.shape))
    codes, scales = backend.quantize_mxfp4(x.cuda())
    ec, es = mx.quantize(np64(x))
    assert np.array_equal(scales.cpu().numpy(), es)
    assert np.array_equal(codes.cpu().numpy(), ec)


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_infinity_and_zero_blocks(backend, gpu, dtype):
    x = outliers(6, 128, dtype, seed=4)
    x[0, 5], x[1, 40], x[2, 127], x[3, 32:64] = float("nan"), float("inf"), float("-inf"), 0
    x[4] = 0
    x[5, 0], x[5, 31] = float("nan"), float("inf")
    codes, scales = backend.quantize_mxfp4(x.cuda())
    ec, es = mx.quantize(np64(x))
    assert es[0, 0] == es[1, 1] == es[2, 3] == es[5, 0] == 255 and es[3, 1] == 0
    assert np.array_equal(scales.cpu().numpy(), es) and np.array_equal(codes.cpu().numpy(), ec)
    back = backend.dequantize_mxfp4(codes, scales)
    assert np.array_equal(np64(back), mx.dequantize(ec, es), equal_nan=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,G", [(1, 256, 256), (3, 48 * 16, 16), (33, 1600, 64), (9, 5120, 256), (300, 64, 64)])
def test_rotated_codes(backend, gpu, M, K, G, dtype):
    """The fp32 rotation is within 16 roundings of the group's norm of the exact one (four digits of four roundings
    each, every partial sum at most the norm): codes and scales are those of a value that near."""
    say("rotate", M, K, G, dtype)
    x = outliers(M, K, dtype, seed=M + K)
    codes, scales = backend.quantize_mxfp4(x.cuda(), G)
    y = mx.rotate(np64(x), G)
    off = 16 * 2.0 ** -24 * np.linalg.norm(np64(x).reshape(-1, G), axis=1)
    off = np.repeat(off, G).reshape(M, K // 32, 32)
    y = y.reshape(M, K // 32, 32)
    s, c = scales.cpu().numpy(), mx.unpack(codes.cpu().numpy()).reshape(M, K // 32, 32)
    amax, o = np.abs(y).max(axis=-1), off[..., 0]
    assert ((s == mx.scale_byte(amax)) | (s == mx.scale_byte(amax - o)) | (s == mx.scale_byte(amax + o))).all()
    value = mx.dequantize(mx.pack(c), s.reshape(M, K // 32, 1)).reshape(c.shape)
    near = [mx.dequantize(mx.pack(mx.codes_of(v, s)), s.reshape(M, K // 32, 1)).reshape(c.shape)
            for v in (y - off, y, y + off)]
    assert ((value == near[0]) | (value == near[1]) | (value == near[2])).all()
    same = (value == near[1]).mean()
    assert same > 0.999


def test_rotated_infinity_spreads_over_its_group(backend, gpu):
    x = outliers(2, 512, torch.float32, seed=1)
    x[0, 300] = float("inf")
    s = backend.quantize_mxfp4(x.cuda(), 256)[1].cpu().numpy()
    assert (s[0, 8:] == 255).all() and (s[0, :8] != 255).all() and (s[1] != 255).all()


# ---- and back ------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
def test_every_code_at_every_scale(backend, gpu, dtype):
    codes = mx.pack(np.tile(np.arange(16, dtype=np.uint8), 2)[None].repeat(256, 0))
    scales = np.arange(256, dtype=np.uint8)[:, None]
    back = backend.dequantize_mxfp4(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), output_dtype=dtype)
    want = torch.from_numpy(mx.dequantize(codes, scales)).to(torch.float32).to(dtype)     # exact in fp32
    assert np.array_equal(np64(back), np64(want), equal_nan=True)


@pytest.mark.parametrize("G", [16, 64, 256])
@pytest.mark.parametrize("dtype", DTYPES)
def test_rotated_back(backend, gpu, G, dtype):
    M, K = 37, 768
    x = outliers(M, K, torch.float32, seed=G)
    codes, scales = backend.quantize_mxfp4(x.cuda(), G)
    back = backend.dequantize_mxfp4(codes, scales, G, output_dtype=dtype)
    v = mx.dequantize(codes.cpu().numpy(), scales.cpu().numpy())
    want = mx.rotate(v, G)
    off = 16 * 2.0 ** -24 * np.repeat(np.linalg.norm(v.reshape(-1, G), axis=1), G).reshape(M, K)
    assert back.dtype == dtype and rounded_once(back, want, off, dtype)


def test_quantize_takes_views_and_cpu_tensors(backend, gpu):
    x = outliers(40, 256, torch.bfloat16, seed=2)
    want = backend.quantize_mxfp4(x.cuda())
    for v in (x.cuda().t().contiguous().t(), torch.cat([x.new_zeros(1), x.flatten()]).cuda()[1:].view(40, 256), x):
        codes, scales = backend.quantize_mxfp4(v)
        assert codes.device == v.device
        assert torch.equal(codes.cuda(), want[0]) and torch.equal(scales.cuda(), want[1])
    c, s = backend.quantize_mxfp4(x.cuda()[:0])
    assert c.shape == (0, 128) and s.shape == (0, 8)
    assert backend.dequantize_mxfp4(c, s).shape == (0, 256)


# ---- the linear ----------------------------------------------------------

def exact_operands(M, N, K, seed, E=None):
    """Operands whose products and sums are exact in fp32: values are multiples of 1/16 and at most 12 (scales 1/8 ..
    2), so products are multiples of 2^-8, and of K <= 4096 of them with random signs no partial sum comes near 2^16
    (its deviation is below 144 * 64 = 2^13.2)."""
    g = np.random.RandomState(seed)
    shape = (N, K) if E is None else (E, N, K)
    def draw(*s):
        return mx.pack(g.randint(0, 16, s).astype(np.uint8)), g.choice([124, 126, 127, 128], s[:-1] + (s[-1] // 32,)).astype(np.uint8)
    xc, xs = draw(M, K)
    wc, ws = draw(*shape)
    x = mx.dequantize(xc, xs)
    # a block whose largest value is below 4 units has another scale when it is quantized: put a 6 in each
    b = x.reshape(M, K // 32, 32)
    b[..., 7] = 6 * np.exp2(xs.astype(float) - 127)
    return b.reshape(M, K), wc, ws


LINEAR_SHAPES = [(1, 64, 64), (1, 512, 512), (2, 33, 32), (5, 100, 160), (16, 1000, 480), (17, 130, 1600), (31, 96, 96),
                 (64, 256, 1024), (65, 257, 2080), (100, 512, 4096), (128, 384, 640), (200, 1, 256), (256, 512, 2048),
                 (333, 480, 1632), (512, 768, 512), (700, 1030, 1056), (1025, 640, 224)]


@pytest.mark.parametrize("M,N,K", LINEAR_SHAPES)
def test_linear_exact(backend, gpu, M, N, K):
    """Products and sums that fp32 holds exactly: every output equals the definition's bit for bit."""
    say("linear", M, N, K)
    x, wc, ws = exact_operands(M, N, K, seed=M + N + K)
    assert np.array_equal(mx.dequantize(*mx.quantize(x)), x)
    want = x @ mx.dequantize(wc, ws).T
    bias = np.random.RandomState(1).randint(-64, 64, N) / 8.0
    w, s = torch.from_numpy(wc).cuda(), torch.from_numpy(ws).cuda()
    xt = torch.from_numpy(x).float().cuda()
    y = backend.mxfp4_linear(xt, w, s)
    assert y.dtype == torch.float32 and np.array_equal(np64(y), want)
    y = backend.mxfp4_linear(xt, w, s, torch.from_numpy(bias).float().cuda())
    assert np.array_equal(np64(y), want + bias)
    for dtype in (torch.bfloat16, torch.float16):            # multiples of 1/16 up to 12: exact in both
        y = backend.mxfp4_linear(xt.to(dtype), w, s, torch.from_numpy(bias).to(dtype).cuda())
        assert torch.equal(y.cpu(), torch.from_numpy(want + bias).float().to(dtype))


# the kernel for few rows, 64 x 128 tiles, one round of 128 x 128 tiles, more of them, and 256 x 256 tiles; whole tiles, edges, and N
# that is no multiple of a 16-byte piece
TILES = [(20, 512, 512, 0), (200, 700, 1600, 128), (300, 2400, 1600, 128), (500, 5000, 416, 128), (2100, 2304, 608, 128), (4096, 4096, 512, 128),
         (3900, 4001, 2336, 256), (4096, 4096, 2080, 256), (3000, 4096, 3840, 256)]


@pytest.mark.parametrize("M,N,K,tile", TILES)
def test_linear_exact_by_tile(backend, native, gpu, M, N, K, tile):
    assert native.load_library().cr_mxfp4_tile(M, N, K, 0) == tile
    say("linear", M, N, K)
    x, wc, ws = exact_operands(M, N, K, seed=M + N + K)
    bias = torch.from_numpy(np.random.RandomState(1).randint(-64, 64, N) / 8.0).cuda()
    w, s = torch.from_numpy(wc).cuda(), torch.from_numpy(ws).cuda()
    xt = torch.from_numpy(x).cuda()
    want = xt @ torch.from_numpy(mx.dequantize(wc, ws)).cuda().T + bias         # float64
    for dtype in DTYPES:
        y = backend.mxfp4_linear(xt.to(dtype), w, s, bias.to(dtype))
        assert torch.equal(y, want.float().to(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K,G", [(1, 777, 5120, 256), (7, 512, 1600, 64), (48, 300, 2304, 256), (130, 512, 512, 16),
                                     (300, 640, 1088, None), (520, 1111, 1600, 64)])
def test_linear_rotated(backend, gpu, M, N, K, G, dtype):
    """Against the definition in 64 bits on the quantizer's own codes; K roundings of 2^-23 of the sum of magnitudes
    in the fp32 sums, then the output's."""
    say("linear rotated", M, N, K, G, dtype)
    x = outliers(M, K, dtype, seed=M + K).cuda()
    w = torch.randn(N, K, generator=torch.Generator().manual_seed(5)) * K ** -0.5
    wc, ws = backend.quantize_mxfp4(w.cuda(), G)
    xc, xs = backend.quantize_mxfp4(x, G)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(6)).to(dtype)
    y = backend.mxfp4_linear(x, wc, ws, bias.cuda(), G)
    a, b = mx.dequantize(xc.cpu().numpy(), xs.cpu().numpy()), mx.dequantize(wc.cpu().numpy(), ws.cpu().numpy())
    want = a @ b.T + np64(bias)
    off = (K + 2) * 2.0 ** -23 * (np.abs(a) @ np.abs(b).T + np.abs(np64(bias)))
    assert y.dtype == dtype and rounded_once(y, want, off, dtype)


@pytest.mark.parametrize("M,N,K", [(1, 64, 96), (40, 70, 512), (300, 300, 1056)])
def test_linear_nan_reaches_its_row_only(backend, gpu, M, N, K):
    x, wc, ws = exact_operands(M, N, K, seed=3)
    want = x @ mx.dequantize(wc, ws).T
    xt = torch.from_numpy(x).float()
    xt[M // 2, K - 1] = float("nan")
    y = np64(backend.mxfp4_linear(xt.cuda(), torch.from_numpy(wc).cuda(), torch.from_numpy(ws).cuda()))
    assert np.isnan(y[M // 2]).all()
    keep = np.arange(M) != M // 2
    assert np.array_equal(y[keep], want[keep])
    ws2 = ws.copy()
    ws2[N // 3, K // 32 - 1] = 255                            # a NaN block of the weight: its column
    y = np64(backend.mxfp4_linear(torch.from_numpy(x).float().cuda(), torch.from_numpy(wc).cuda(), torch.from_numpy(ws2).cuda()))
    assert np.isnan(y[:, N // 3]).all()
    keep = np.arange(N) != N // 3
    assert np.array_equal(y[:, keep], want[:, keep])


def test_linear_forms(backend, gpu):
    """Leading dimensions, strided and misaligned operands, no rows, another stream, and a replayed graph."""
    x, wc, ws = exact_operands(24, 48, 256, seed=9)
    want = torch.from_numpy(x @ mx.dequantize(wc, ws).T).float().cuda()
    xt, w, s = torch.from_numpy(x).float().cuda(), torch.from_numpy(wc).cuda(), torch.from_numpy(ws).cuda()
    assert torch.equal(backend.mxfp4_linear(xt.reshape(2, 3, 4, 256), w, s), want.reshape(2, 3, 4, 48))
    assert torch.equal(backend.mxfp4_linear(xt.t().contiguous().t(), w, s), want)
    odd = torch.cat([w.new_zeros(3), w.flatten()])[3:].view_as(w)
    assert torch.equal(backend.mxfp4_linear(xt, odd, s.t().contiguous().t()), want)
    assert backend.mxfp4_linear(xt[:0], w, s).shape == (0, 48)
    assert backend.mxfp4_linear(xt, w[:0], s[:0]).shape == (24, 0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = backend.mxfp4_linear(xt, w, s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want)
    graph, held = torch.cuda.CUDAGraph(), xt.clone()
    with torch.cuda.graph(graph):
        y = backend.mxfp4_linear(held, w, s)
    for i in range(3):
        held.copy_(xt.roll(i, 0))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want.roll(i, 0))
        assert torch.equal(backend.mxfp4_linear(xt, w, s), want)      # the eager call between replays


def test_forward_mode_is_refused(backend, gpu):
    x, wc, ws = exact_operands(4, 32, 64, seed=2)
    xt, w, s = torch.from_numpy(x).float().cuda(), torch.from_numpy(wc).cuda(), torch.from_numpy(ws).cuda()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(xt, torch.ones_like(xt))
        with pytest.raises(RuntimeError, match="no gradient"):
            backend.mxfp4_linear(dual, w, s)
        with pytest.raises(RuntimeError, match="no gradient"):
            backend.quantize_mxfp4(dual)
        assert backend.mxfp4_linear(xt, w, s).shape == (4, 32)


def test_gradients_are_refused_on_the_gpu(backend, gpu):
    x = torch.zeros(4, 64, device="cuda", requires_grad=True)
    w, s = torch.zeros(8, 32, dtype=torch.uint8, device="cuda"), torch.zeros(8, 2, dtype=torch.uint8, device="cuda")
    with pytest.raises(RuntimeError, match="no gradient"):
        backend.mxfp4_linear(x, w, s)
    with pytest.raises(RuntimeError, match="no gradient"):
        backend.quantize_mxfp4(x)
    with torch.no_grad():
        assert backend.mxfp4_linear(x, w, s).shape == (4, 8)


def test_offsets_past_32_bits(backend, gpu):
    """An input and an output of more than 2^32 bytes and 2^31 values: the last rows as a small call gives them."""
    M, K, N = 80000, 64, 27008
    x, wc, ws = exact_operands(256, N, K, seed=4)
    w, s = torch.from_numpy(wc).cuda(), torch.from_numpy(ws).cuda()
    xt = torch.from_numpy(x).to(torch.bfloat16).cuda()
    want = backend.mxfp4_linear(xt, w, s)
    y = backend.mxfp4_linear(xt.repeat(M // 256 + 1, 1)[:M], w, s)
    assert y.numel() > 2 ** 31
    for r0 in (0, 39936, M // 256 * 256 - 256):
        assert torch.equal(y[r0:r0 + 256], want)
    del y
    big = torch.zeros(70000, 32768, dtype=torch.bfloat16, device="cuda")
    big[-1] = torch.randn(32768, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    codes, scales = backend.quantize_mxfp4(big)
    small = backend.quantize_mxfp4(big[-1:])
    assert torch.equal(codes[-1:], small[0]) and torch.equal(scales[-1:], small[1])
    assert int(codes[:-1].count_nonzero()) == 0
    back = backend.dequantize_mxfp4(codes, scales, output_dtype=torch.bfloat16)
    assert torch.equal(back[-1:], backend.dequantize_mxfp4(*small, output_dtype=torch.bfloat16))
