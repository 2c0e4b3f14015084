"""The norm's C entries where there are no rows, and the 8-bit form's codes at ties."""
import math

import pytest
import torch

from test_gpu_norm import rotation

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [1, 15, 16, 4097, 32768])
def test_weight_gradient_of_no_rows_is_zero(backend, native, gpu, D, dtype):
    """A sum over nothing, in the weight's type and nowhere else; no workspace is needed."""
    lib, code = native.load_library(), {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
    rows = torch.ones(4, D, device="cuda")
    weight = torch.ones(D, dtype=dtype, device="cuda")
    around = torch.full((D + 2,), 7.0, dtype=dtype, device="cuda")
    d_x = torch.full((4, D), 7.0, device="cuda")
    assert lib.cr_rms_norm_grad_workspace(0, D) == 0
    rc = lib.cr_rms_norm_grad(rows.data_ptr(), None, rows.data_ptr(), 0, weight.data_ptr(), code[dtype], d_x.data_ptr(),
                              around[1:].data_ptr(), 0, D, 1e-6, None, 0, native._stream(rows.device))
    assert rc == 0
    assert not bool(around[1:-1].any()) and around[0] == around[-1] == 7 and bool((d_x == 7).all())
    assert lib.cr_rms_norm_grad(rows.data_ptr(), None, rows.data_ptr(), 0, weight.data_ptr(), code[dtype], d_x.data_ptr(), None, 0, D,
                                1e-6, None, 0, native._stream(rows.device)) == 0


# 127 and halves: of each number of them and its negative the squares are known, and all of them add up to 2^14
HALVES = [127.0, 0.5, -0.5, 1.5, -1.5, 2.5, -2.5, 3.5, -3.5, 4.5, -4.5, 5.5, -5.5, 6.5, -6.5, 5.0, 1.5, 0.5]
assert sum(v * v for v in HALVES) == 2 ** 14


def row_of_halves(D, order):
    """Rotated values [D] of squares that add up to 2^14, or 2^15 where D is no power of 4."""
    values = HALVES + ([-v for v in HALVES] if D == 512 else [])
    z = torch.zeros(D, dtype=torch.float64)
    z[torch.randperm(D, generator=torch.Generator().manual_seed(order))[:len(values)]] = torch.tensor(values, dtype=torch.float64)
    return z


@pytest.mark.parametrize("M", [1, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("G", [16, 64, 256])
@pytest.mark.parametrize("D", [256, 512, 1024, 4096, 16384])
def test_int8_codes_of_halves_go_to_even(backend, native, gpu, D, G, dtype, M):
    """Rows of mean square 1 and eps 0: rstd is 1, and with a weight of one power of two the largest rotated value is 127 and
    the scale 1, so codes are the rotated values themselves, halves among them: 0.5 -> 0, 1.5 -> 2, 2.5 -> 2, ...  All are exact: x is
    whole parts of 2^-12, the sum of its squares D."""
    weight = math.sqrt((2 ** 15 if D == 512 else 2 ** 14) / D)
    assert weight in (1, 2, 4, 8)
    z = torch.stack([row_of_halves(D, i % 7) for i in range(M)])
    h = (z.reshape(-1, G) @ rotation(backend, G)).reshape(M, D) / weight         # the rotation is its own inverse
    x = h.to(dtype)
    assert torch.equal(x.double(), h) and bool((h.square().sum(-1) == D).all())
    x = x.cuda()
    residual = torch.full_like(x, 0.5)
    assert torch.equal((x - residual) + residual, x)
    want = torch.round(z).to(torch.int8)                                          # torch's rounds halves to even
    assert (want.double() - z).abs().max() == 0.5
    w = torch.full((D,), weight, dtype=dtype, device="cuda")
    for i8t in (False, True):
        for r in (None, residual):
            rows = backend.rms_norm_int8(x if r is None else x - r, w, r, 0.0, G, i8t=i8t)
            rows = rows if r is None else rows[0]
            codes = native.i8t_to_int8(rows.codes, rows.codes.shape[0])[:M] if i8t else rows.codes
            assert bool((rows.scales == 1.0).all())
            assert torch.equal(codes.cpu(), want)
