"""CPU checks: sizes past what a call takes are refused by name, before they are cut to 32 bits on the way to the library.
Expanded tensors of one element stand for the large ones."""
import ctypes

import pytest
import torch


def big(*shape, dtype=torch.float32):
    return torch.zeros(1, dtype=dtype).expand(*shape)


def plan_of(q, T, k=1, E=2):
    i = torch.int32
    return q.ExpertPlan(torch.zeros(T * k, dtype=i), torch.zeros(T, k, dtype=i), torch.zeros(E + 1, dtype=i))


WIDE = 2 ** 32 + 64                                          # 64 in 32 bits


@pytest.mark.parametrize("K", [2 ** 24 + 32, WIDE])
def test_wide_rows(backend, K):
    u = torch.uint8
    with pytest.raises(ValueError, match="at most 16777216"):
        backend.quantize_mxfp4(big(1, K))
    with pytest.raises(ValueError, match="at most 16777216"):
        backend.dequantize_mxfp4(big(1, K // 2, dtype=u), big(1, K // 32, dtype=u))
    with pytest.raises(ValueError, match="at most 16777216"):
        backend.mxfp4_linear(big(1, K), big(8, K // 2, dtype=u), big(8, K // 32, dtype=u))
    with pytest.raises(ValueError, match="at most 16777216"):
        backend.mxfp4_expert_linear(big(1, K), big(2, 8, K // 2, dtype=u), big(2, 8, K // 32, dtype=u), plan_of(backend, 1))


@pytest.mark.parametrize("n", [2 ** 31, 2 ** 32 + 8])
def test_more_than_32_bits_of_columns_or_rows(backend, n):
    u = torch.uint8
    with pytest.raises(ValueError, match="more than one call takes"):
        backend.mxfp4_linear(big(1, 32), big(n, 16, dtype=u), big(n, 1, dtype=u))
    with pytest.raises(ValueError, match="more than one call takes"):
        backend.mxfp4_expert_linear(big(1, 32), big(2, n, 16, dtype=u), big(2, n, 1, dtype=u), plan_of(backend, 1))
    with pytest.raises(ValueError, match="more than one call takes"):
        backend.gather_expert_rows(big(1, n), plan_of(backend, 1))
    with pytest.raises(ValueError, match="more than one call takes"):
        backend.combine_expert_rows(big(1, n), torch.zeros(1, 1), plan_of(backend, 1))
    with pytest.raises(ValueError, match="more than one call takes"):
        backend.mxfp4_linear(big(n, 32), big(8, 16, dtype=u), big(8, 1, dtype=u))
    with pytest.raises(ValueError, match="more than one call takes"):
        backend.quantize_mxfp4(big(n, 32))
    with pytest.raises(ValueError, match="more than one call takes"):
        backend.dequantize_mxfp4(big(n, 16, dtype=u), big(n, 1, dtype=u))


def test_columns_that_a_tile_cannot_count(backend, native):
    """A tile's columns past the last one are counted in 31 bits."""
    n, u = 2 ** 31 - 255, torch.uint8
    with pytest.raises(ValueError, match="more than one call takes"):
        backend.mxfp4_linear(big(1, 32), big(n, 16, dtype=u), big(n, 1, dtype=u))
    with pytest.raises(ValueError, match="more than one call takes"):
        backend.mxfp4_expert_linear(big(1, 32), big(2, n, 16, dtype=u), big(2, n, 1, dtype=u), plan_of(backend, 1))
    lib, z = native.load_library(), ctypes.c_void_p(0)
    assert lib.cr_mxfp4_linear(z, 1, z, z, z, 0, z, 1, n, 32, 0, z, 1 << 40, z) == -1
    assert lib.cr_mxfp4_expert_linear(z, 1, z, 1, ctypes.c_void_p(16), 2, z, z, z, 0, z, 1, n, 32, 0, z, 1 << 40, z) == -1


def test_plans_past_their_limits(backend):
    q, i = backend, torch.int32

    class Large:                                             # a plan's order or position of 2^31 slots
        dtype, device = i, torch.device("cpu")

        def __init__(self, *shape):
            self.shape = torch.Size(shape)

        def is_contiguous(self):
            return True

        def is_neg(self):
            return False

        def dim(self):
            return len(self.shape)

        def numel(self):
            return self.shape.numel()

    plan = q.ExpertPlan(Large(2 ** 31), Large(2 ** 30, 2), torch.zeros(3, dtype=i))
    with pytest.raises(ValueError, match="more than one plan holds"):
        plan.check()
    many = plan_of(q, 1, E=1025)
    many.check()                                             # rows can be gathered by it
    with pytest.raises(ValueError, match="at most 1024 experts"):
        q.mxfp4_expert_linear(torch.zeros(1, 32), big(1025, 8, 16, dtype=torch.uint8), big(1025, 8, 1, dtype=torch.uint8), many)
