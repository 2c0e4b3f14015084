"""CPU checks of the query that names the kernel of an MXFP4 product."""
import ctypes

import pytest


def kernel(native, R, N, K, experts=0, tokens=0):
    """(rows, columns, stages in LDS, x quantized in it) of the product."""
    k = (ctypes.c_int * 4)()
    assert native.load_library().cr_mxfp4_kernel(R, N, K, experts, tokens, k) == 0
    return tuple(k)


@pytest.mark.parametrize("args,want", [
    ((1, 13824, 5120), (16, 32, 0, 1)), ((4, 100, 512), (16, 16, 0, 1)), ((5, 100, 512), (16, 32, 0, 0)),
    ((32, 100, 512), (32, 32, 0, 0)), ((200, 700, 2336), (64, 128, 4, 0)), ((500, 5000, 2336), (128, 128, 4, 0)),
    ((1100, 4000, 2336), (128, 128, 2, 0)), ((8192, 13824, 5120), (256, 256, 2, 0)),
    ((8, 4096, 2048, 32, 2), (16, 32, 0, 1)), ((9, 4096, 2048, 32, 3), (16, 32, 0, 0)), ((16384, 4096, 2048, 32, 4096), (128, 128, 2, 0))])
def test_instances(native, args, want):
    """Each instance by its tile, beside the older query, which has the staged tile's columns."""
    assert kernel(native, *args) == want
    R, N, K, E = (*args, 0)[:4]
    assert native.load_library().cr_mxfp4_tile(R, N, K, E) == (want[1] if want[2] else 0)


def test_routed_tokens(native):
    """Tokens whose codes pass 2^32 bytes go to the kernel for few rows; as many sorted rows do not."""
    assert kernel(native, 2 ** 21 * 4, 4096, 4096, 8, 2 ** 21)[2] == 0
    assert kernel(native, 2 ** 21 * 4, 4096, 4096, 8, 0)[2] == 2


def test_refusals(native):
    lib, k = native.load_library(), (ctypes.c_int * 4)()
    for bad in ((-1, 8, 64, 0, 0), (4, 8, 48, 0, 0), (4, 8, 64, 0, 4), (4, 8, 64, -1, 0), (4, 2 ** 31 - 1, 64, 0, 0)):
        assert lib.cr_mxfp4_kernel(*bad, k) == -1
    assert lib.cr_mxfp4_kernel(4, 8, 64, 0, 0, None) == -1
