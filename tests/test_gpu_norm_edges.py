"""The norm's C entries where there are no rows, and the 8-bit form's codes at ties."""
import pytest
import torch

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
