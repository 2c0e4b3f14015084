"""CPU checks of the microscaled 4-bit tier and of expert routing: the plain
forms the GPU tests compare with, and what the functions refuse."""
import ctypes
import importlib

import numpy as np
import pytest
import torch

import mx_format as mx
from conftest import PKG_NAME


@pytest.fixture(scope="module")
def q(backend):
    return backend


def _plan(q, T=3, k=2, E=4):
    i = torch.int32
    return q.ExpertPlan(torch.zeros(T * k, dtype=i), torch.zeros(T, k, dtype=i), torch.zeros(E + 1, dtype=i))


def test_plain_quantization_by_hand():
    x = np.zeros((1, 64))
    x[0, :8] = [7.0, -5.0, 2.5, 3.5, .25, .75, 1.75, -.1]
    x[0, 32:36] = [1.0, 0.875, 0.8125, -1.9]
    packed, s = mx.quantize(x)
    assert s.tolist() == [[127, 125]]                       # 7: 2^(2 - 2); 1.9: 2^(0 - 2)
    v = mx.dequantize(packed, s)[0]
    assert v[:8].tolist() == [6, -4, 2, 4, 0, 1, 2, 0]      # ties to even, 7 past the largest
    assert v[32:36].tolist() == [1, 1, .75, -1.5]           # .875 and .8125: ties and below in steps of .25
    assert mx.scale_byte(np.array([0, 2.0 ** -140, 2.0 ** -126, np.inf, np.nan, 2.0 ** 127])).tolist() == \
        [0, 0, 0, 255, 255, 252]


def test_plain_plan_by_hand():
    order, position, offsets = mx.plan(np.array([[2, 0], [-1, 2], [0, 9]]), 3)
    assert order.tolist() == [1, 4, 0, 3, -1, -1]
    assert position.tolist() == [[2, 0], [-1, 3], [1, -1]]
    assert offsets.tolist() == [0, 2, 2, 4]


@pytest.mark.parametrize("G", [16, 64, 256])
def test_plain_rotation_is_its_own_inverse(G):
    h = mx.rotation(G)
    assert np.array_equal(h, h.T) and np.allclose(h @ h, np.eye(G), atol=1e-12)


def test_quantize_refuses(q):
    with pytest.raises(ValueError, match="multiple of 32"):
        q.quantize_mxfp4(torch.zeros(4, 48))
    with pytest.raises(ValueError, match="multiple of 32"):
        q.quantize_mxfp4(torch.zeros(4, 0))
    with pytest.raises(ValueError, match="16, 64, 256 or None"):
        q.quantize_mxfp4(torch.zeros(4, 64), 32)
    with pytest.raises(ValueError, match="not divisible by convrot_groupsize"):
        q.quantize_mxfp4(torch.zeros(4, 320), 256)
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        q.quantize_mxfp4(torch.zeros(4, 64, dtype=torch.float64))
    with pytest.raises(ValueError, match="dimension"):
        q.quantize_mxfp4(torch.zeros(()))
    with pytest.raises(RuntimeError, match="no gradient"):
        q.quantize_mxfp4(torch.zeros(4, 64, requires_grad=True))


def test_dequantize_refuses(q):
    c, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    with pytest.raises(ValueError, match="do not fit"):
        q.dequantize_mxfp4(c, s[:, :1])
    with pytest.raises(ValueError, match="uint8"):
        q.dequantize_mxfp4(c.to(torch.int8), s)
    with pytest.raises(ValueError, match="output_dtype"):
        q.dequantize_mxfp4(c, s, output_dtype=torch.float64)
    with pytest.raises(ValueError, match="whole blocks"):
        q.dequantize_mxfp4(c[:, :8], s)
    with pytest.raises(ValueError, match="not divisible"):
        q.dequantize_mxfp4(c, s, 256)


def test_linear_refuses(q):
    x, w, s = torch.zeros(4, 64), torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2, dtype=torch.uint8)
    with pytest.raises(ValueError, match="does not match qweight"):
        q.mxfp4_linear(torch.zeros(4, 96), w, s)
    with pytest.raises(ValueError, match="2-D"):
        q.mxfp4_linear(x, w[0], s)
    with pytest.raises(ValueError, match="do not fit"):
        q.mxfp4_linear(x, w, s[:4])
    with pytest.raises(ValueError, match="bias of shape"):
        q.mxfp4_linear(x, w, s, torch.zeros(7))
    with pytest.raises(ValueError, match="bias must be"):
        q.mxfp4_linear(x, w, s, torch.zeros(8, dtype=torch.int32))
    with pytest.raises(ValueError, match="x must be"):
        q.mxfp4_linear(x.double(), w, s)
    with pytest.raises(RuntimeError, match="no gradient"):
        q.mxfp4_linear(x.requires_grad_(), w, s)
    with pytest.raises(RuntimeError, match="CUDA"):
        q.mxfp4_linear(x.detach(), w, s)


def test_expert_linear_refuses(q):
    x, w = torch.zeros(3, 64), torch.zeros(4, 8, 32, dtype=torch.uint8)
    s = torch.zeros(4, 8, 2, dtype=torch.uint8)
    p = _plan(q)
    with pytest.raises(ValueError, match="3-D"):
        q.mxfp4_expert_linear(x, w[0], s[0], p)
    with pytest.raises(ValueError, match="of 4 experts, the weights are of 3"):
        q.mxfp4_expert_linear(x, w[:3], s[:3], p)
    with pytest.raises(ValueError, match="rows"):
        q.mxfp4_expert_linear(x, w, s, p, sorted_rows=True)
    with pytest.raises(ValueError, match="rows"):
        q.mxfp4_expert_linear(torch.zeros(6, 64), w, s, p)
    with pytest.raises(ValueError, match="2-D"):
        q.mxfp4_expert_linear(torch.zeros(1, 3, 64), w, s, p)
    with pytest.raises(ValueError, match="bias of shape"):
        q.mxfp4_expert_linear(x, w, s, p, torch.zeros(8))
    with pytest.raises(RuntimeError, match="no gradient"):
        q.mxfp4_expert_linear(x.requires_grad_(), w, s, p)


def test_routing_refuses(q):
    with pytest.raises(ValueError, match=r"\[T, k\]"):
        q.sort_tokens_by_expert(torch.zeros(4, dtype=torch.int64), 4)
    with pytest.raises(ValueError, match="int32 or int64"):
        q.sort_tokens_by_expert(torch.zeros(4, 2), 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        q.sort_tokens_by_expert(torch.zeros(4, 2, dtype=torch.int64), 4)
    p = _plan(q)
    with pytest.raises(ValueError, match="does not fit a plan of 3 tokens"):
        q.gather_expert_rows(torch.zeros(4, 8), p)
    with pytest.raises(ValueError, match="do not fit a plan of 6 rows"):
        q.combine_expert_rows(torch.zeros(5, 8), torch.zeros(3, 2), p)
    with pytest.raises(ValueError, match="weights of shape"):
        q.combine_expert_rows(torch.zeros(6, 8), torch.zeros(2, 3), p)
    with pytest.raises(ValueError, match="weights must be"):
        q.combine_expert_rows(torch.zeros(6, 8), torch.zeros(3, 2, dtype=torch.float64), p)
    with pytest.raises(ValueError, match="x must be"):
        q.gather_expert_rows(torch.zeros(3, 8, dtype=torch.int32), p)
    bad = q.ExpertPlan(p.order.long(), p.position, p.offsets)
    with pytest.raises(ValueError, match="a plan is"):
        q.gather_expert_rows(torch.zeros(3, 8), bad)
    assert q.max_experts() == 1024


def test_library_refuses(native):
    """Invalid arguments return -1 before any device work."""
    lib, n = native.load_library(), ctypes.c_void_p(0)
    assert lib.cr_mxfp4_quant(n, 1, n, n, 4, 48, 0, n) == -1           # K % 32
    assert lib.cr_mxfp4_quant(n, 3, n, n, 4, 64, 0, n) == -1           # type
    assert lib.cr_mxfp4_quant(n, 1, n, n, -1, 64, 0, n) == -1          # rows
    assert lib.cr_mxfp4_quant(n, 1, n, n, 4, 64, 32, n) == -1          # group
    assert lib.cr_mxfp4_quant(n, 1, n, n, 0, 64, 16, n) == 0           # nothing to do
    assert lib.cr_mxfp4_dequant(n, n, n, 1, 4, 320, 256, n) == -1      # K % G
    assert lib.cr_mxfp4_linear(n, 1, n, n, n, 0, n, 4, 8, 64, 0, n, 0, n) == -1          # no workspace
    assert lib.cr_mxfp4_linear(n, 1, n, n, n, 5, n, 4, 8, 64, 0, n, 1 << 20, n) == -1    # bias type
    assert lib.cr_mxfp4_linear(n, 1, n, n, n, 0, n, 0, 8, 64, 0, n, 0, n) == 0
    assert lib.cr_mxfp4_expert_linear(n, 1, n, 1, n, 4, n, n, n, 0, n, 4, 8, 64, 0, n, 1 << 20, n) == -1   # no offsets
    assert lib.cr_expert_sort(n, 2, n, n, n, 4, 4, n, 1 << 20, n) == -1                  # id size
    assert lib.cr_expert_sort(n, 8, n, n, n, 4, 1025, n, 1 << 20, n) == -1               # experts
    assert lib.cr_expert_sort(n, 8, n, n, n, 4, 4, n, 1 << 20, n) == -1                  # no workspace
    assert lib.cr_expert_gather(n, 1, n, n, n, 4, 0, 4, 8, n) == -1                      # k
    assert lib.cr_expert_combine(n, 1, n, n, n, 1 << 20, 1 << 12, 8, n) == -1            # slots past 2^31
    assert lib.cr_expert_combine_grad(n, 1, n, n, n, n, n, n, 4, 2, 4, 8, n) == -1       # no weights
    assert lib.cr_mxfp4_linear_workspace(3, 8, 1600, 1) >= 3 * (1664 // 2 + 1664 // 32)
    assert lib.cr_mxfp4_linear_workspace(0, 8, 64, 1) == 0


def test_names_are_public(q):
    pkg = importlib.import_module(PKG_NAME + "._int4")
    for name in ("quantize_mxfp4", "dequantize_mxfp4", "mxfp4_linear", "mxfp4_expert_linear", "ExpertPlan",
                 "sort_tokens_by_expert", "gather_expert_rows", "combine_expert_rows"):
        assert name in pkg.__all__ and getattr(pkg, name) is getattr(q, name)
