"""GPU checks of the MXFP4 rotation at the top of the range: a rotated value is finite wherever the rotation's exact
result is, whatever its partial sums are."""
import numpy as np
import pytest
import torch

import mx_format as mx
from test_gpu_mxfp4 import np64, rounded_once, say

pytestmark = pytest.mark.gpu

MOST = float(np.finfo(np.float32).max)


def large(M, K, dtype, seed):
    """Groups of equal and opposite values up to the type's largest, single large values among small ones, and rows at
    2^120 .. 2^127: what partial sums overflow on while most exact results do not."""
    g = np.random.RandomState(seed)
    x = np.zeros((M, K))
    for r in range(M):
        kind = r % 5
        top = float(torch.finfo(dtype).max) if kind == 0 else 10.0 ** g.uniform(37, 38.5)
        if kind < 2:                                       # all of one magnitude, signs of a group of four repeated
            x[r] = np.tile(top * g.choice([-1, 1], 4), K // 4)
        elif kind == 2:                                    # four of one sign, zeros, four of both signs
            x[r, ::16] = top
            x[r, 1::32] = -top
        elif kind == 3:
            x[r] = g.randn(K)
            x[r, g.randint(0, K, 3)] = top * g.choice([-1, 1], 3)
        else:
            x[r] = g.uniform(-1, 1, K) * 2.0 ** (120 + r % 8)
    return torch.from_numpy(np.clip(x, -MOST, MOST)).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K,G", [(40, 512, 16), (40, 512, 64), (40, 512, 256), (4, 256, 256), (15, 1088, 64)])
def test_large_values_rotate(backend, gpu, M, K, G, dtype):
    """As the codes of ordinary values: within 16 roundings of the group's norm.  A block whose exact result passes
    fp32's largest value has scale byte 255, and no other has."""
    say("rotate large", M, K, G, dtype)
    x = large(M, K, dtype, seed=M + G)
    codes, scales = backend.quantize_mxfp4(x.cuda(), G)
    y = mx.rotate(np64(x), G).reshape(M, K // 32, 32)
    off = np.repeat(16 * 2.0 ** -24 * np.linalg.norm(np64(x).reshape(-1, G), axis=1), G).reshape(y.shape)
    amax, o = np.abs(y).max(axis=-1), off.max(axis=-1)
    s, c = scales.cpu().numpy(), mx.unpack(codes.cpu().numpy()).reshape(y.shape)
    over, under = amax - o > MOST, amax + o < MOST
    assert under.mean() > 0.5
    assert (s[over] == 255).all() and (s[under] != 255).all()
    assert ((s == mx.scale_byte(amax)) | (s == mx.scale_byte(amax - o)) | (s == mx.scale_byte(amax + o)))[under].all()
    value = mx.dequantize(mx.pack(c), s[..., None]).reshape(c.shape)
    near = [mx.dequantize(mx.pack(mx.codes_of(v, s)), s[..., None]).reshape(c.shape) for v in (y - off, y, y + off)]
    assert ((value == near[0]) | (value == near[1]) | (value == near[2]))[under].all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("G", [16, 64, 256])
def test_large_values_rotate_back(backend, gpu, G, dtype):
    """Codes with scale bytes up to 254, whose own values pass fp32's largest at 253, beside small ones."""
    M, K = 24, 512
    g = np.random.RandomState(G)
    codes = g.randint(0, 256, (M, K // 2)).astype(np.uint8)
    codes[::3] = codes[::3, :1] & 0x77                     # equal values: sums as large as they get
    scales = g.choice([0, 1, 127, 240, 243, 250, 252, 253, 254], (M, K // 32)).astype(np.uint8)
    scales[::3] = 252
    v = mx.dequantize(codes, scales)
    want = mx.rotate(v, G)
    off = 16 * 2.0 ** -24 * np.repeat(np.linalg.norm(v.reshape(-1, G), axis=1), G).reshape(M, K)
    say("rotate back large", G, dtype)
    back = backend.dequantize_mxfp4(torch.from_numpy(codes).cuda(), torch.from_numpy(scales).cuda(), G, output_dtype=dtype)
    assert np.isfinite(want.astype(np.float32)).mean() > 0.3
    with np.errstate(over="ignore"):
        assert rounded_once(back, want, off, dtype)


@pytest.mark.parametrize("M", [1, 4, 12, 40])
@pytest.mark.parametrize("G", [16, 256])
def test_large_rows_in_a_product(backend, gpu, M, G):
    """Every kernel that quantizes rows: the product with small weights is what the quantizer's own codes give, and a
    row is NaN only where the exact rotation passes fp32's largest value."""
    N, K = 96, 512
    x = large(5, K, torch.bfloat16, seed=G)[[4, 3, 1, 2]].repeat(10, 1)[:M].cuda()
    xc, xs = backend.quantize_mxfp4(x, G)
    g = np.random.RandomState(2)
    wc = g.randint(0, 256, (N, K // 2)).astype(np.uint8)
    ws = g.choice([60, 61, 62], (N, K // 32)).astype(np.uint8)
    y = backend.mxfp4_linear(x, torch.from_numpy(wc).cuda(), torch.from_numpy(ws).cuda(), None, G)
    a, b = mx.dequantize(xc.cpu().numpy(), xs.cpu().numpy()), mx.dequantize(wc, ws)
    finite = np.isfinite(a).all(axis=1)
    top = np.abs(mx.rotate(np64(x), G)).max(axis=1)
    assert finite[top < MOST * (1 - 2.0 ** -18)].all()      # 16 roundings of a norm of at most 16 times it
    say("large product", M, G, int(finite.sum()))
    assert finite.any() and np.isnan(np64(y)[~finite]).all()
    a = a[finite]
    off = (K + 2) * 2.0 ** -23 * (np.abs(a) @ np.abs(b).T)
    assert rounded_once(y.cpu()[torch.from_numpy(finite)], a @ b.T, off, torch.bfloat16)
