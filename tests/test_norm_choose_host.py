"""CPU checks of what the router's choice, the norm, its 8-bit rows and their linear refuse."""
import importlib

import pytest
import torch

from conftest import PKG_NAME


@pytest.mark.parametrize("shape,k,bias,how,match", [
    ((), 1, None, {}, "must be"), ((4, 0), 1, None, {}, "must be"),
    ((4, 8), 0, None, {}, "top_k"), ((4, 8), 9, None, {}, "top_k"), ((4, 8), -1, None, {}, "top_k"),
    ((4, 8), 3, None, dict(num_groups=4, top_groups=1), "top_k"),
    ((4, 8), 1, None, dict(num_groups=3), "equal groups"), ((4, 8), 1, None, dict(num_groups=0), "equal groups"),
    ((4, 8), 1, None, dict(num_groups=16), "equal groups"), ((4, 8), 1, None, dict(num_groups=-2), "equal groups"),
    ((4, 8), 1, None, dict(num_groups=2, top_groups=3), "top_groups"), ((4, 8), 1, None, dict(num_groups=2, top_groups=0), "top_groups"),
    ((4, 8), 1, None, dict(scoring="tanh"), "scoring"), ((4, 8), 1, None, dict(group_score="mean"), "group_score"),
    ((4, 8), 1, None, dict(scale=float("nan")), "scale"), ((4, 8), 1, None, dict(scale=float("inf")), "scale"),
    ((4, 8), 1, None, dict(scale=1e39), "scale"),
    ((4, 8), 1, (4,), {}, "balance_bias"), ((4, 8), 1, (1, 8), {}, "balance_bias")])
def test_choice_refusals(backend, shape, k, bias, how, match):
    with pytest.raises(ValueError, match=match):
        backend.choose_experts(torch.zeros(shape), k, None if bias is None else torch.zeros(bias), **how)


def test_choice_types_and_devices(backend):
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        backend.choose_experts(torch.zeros(4, 8, dtype=torch.float64), 1)
    with pytest.raises(ValueError, match="balance_bias"):
        backend.choose_experts(torch.zeros(4, 8), 1, torch.zeros(8, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        backend.choose_experts(torch.zeros(4, 8), 1)
    with pytest.raises(ValueError, match="slots"):
        backend.choose_experts(torch.zeros(1, 8).expand(1 << 30, 8), 2)


def norms(backend):
    return [backend.rms_norm, lambda *a, **k: backend.rms_norm_int8(*a, **k, convrot_groupsize=16)]


@pytest.mark.parametrize("which", [0, 1])
def test_norm_refusals(backend, which):
    f, x = norms(backend)[which], torch.zeros(4, 32)
    with pytest.raises(ValueError, match="must be"):
        f(torch.zeros(()))
    with pytest.raises(ValueError, match="must be"):
        f(torch.zeros(4, 0))
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        f(x.double())
    for w in (torch.zeros(16), torch.zeros(1, 32), torch.zeros(())):
        with pytest.raises(ValueError, match="weight"):
            f(x, w)
    with pytest.raises(ValueError, match="weight"):
        f(x, torch.zeros(32, dtype=torch.float64))
    for r in (torch.zeros(32), torch.zeros(1, 32), torch.zeros(4, 32, dtype=torch.bfloat16), torch.zeros(2, 2, 32)):
        with pytest.raises(ValueError, match="residual"):
            f(x, None, r)
    for eps in (-1e-6, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            f(x, eps=eps)
    with pytest.raises(RuntimeError, match="CUDA"):
        f(x)


def test_norm_limits(backend, native):
    assert backend.max_norm_width() == 32768
    lib = native.load_library()
    n = None
    assert lib.cr_rms_norm(n, 1, n, n, 0, n, n, 4, 32769, 1e-6, n) == -1
    assert lib.cr_rms_norm(n, 3, n, n, 0, n, n, 4, 64, 1e-6, n) == -1
    assert lib.cr_rms_norm(n, 1, n, n, 3, n, n, 4, 64, 1e-6, n) == -1
    assert lib.cr_rms_norm(n, 1, n, n, 0, n, n, 4, 64, -1.0, n) == -1
    assert lib.cr_rms_norm(n, 1, n, n, 0, n, n, 4, 64, float("nan"), n) == -1
    assert lib.cr_rms_norm(n, 1, 16, n, 0, n, n, 4, 64, 1e-6, n) == -1                 # a sum with nowhere to go
    assert lib.cr_rms_norm(n, 1, n, n, 0, n, n, 0, 64, 1e-6, n) == 0
    assert lib.cr_rms_norm_grad(n, n, n, 1, n, 0, n, 16, 4, 64, 1e-6, n, 0, n) == -1    # a weight's gradient without a weight
    assert lib.cr_rms_norm_grad(n, n, n, 1, 16, 0, n, 16, 4, 64, 1e-6, n, 0, n) == -1   # or a workspace
    assert lib.cr_rms_norm_int8(n, 1, n, n, 0, n, n, n, 4, 72, 16, 0, 1e-6, n) == -1    # whole groups
    assert lib.cr_rms_norm_int8(n, 1, n, n, 0, n, n, n, 4, 64, 32, 0, 1e-6, n) == -1
    assert lib.cr_rms_norm_int8(n, 1, n, n, 0, n, n, n, 4, 80, 16, 1, 1e-6, n) == -1    # I8T: multiples of 64
    assert lib.cr_choose_experts(n, 1, n, n, n, 4, 1025, 1, 0, 1, 1, 0, 1, 1.0, n) == -1
    assert lib.cr_choose_experts(n, 1, n, n, n, 4, 8, 9, 0, 1, 1, 0, 1, 1.0, n) == -1
    assert lib.cr_choose_experts(n, 1, n, n, n, 4, 8, 1, 0, 3, 1, 0, 1, 1.0, n) == -1
    assert lib.cr_choose_experts(n, 1, n, n, n, 4, 8, 5, 0, 4, 2, 0, 1, 1.0, n) == -1
    assert lib.cr_choose_experts(n, 1, n, n, n, 4, 8, 1, 0, 1, 1, 0, 1, float("inf"), n) == -1
    assert lib.cr_choose_experts(n, 1, n, n, n, 0, 8, 1, 0, 1, 1, 0, 1, 1.0, n) == 0
    assert lib.cr_choose_experts_grad(n, 1, n, n, n, 4, 8, 9, 0, 1, 1.0, n) == -1
    assert lib.cr_w8a8_rows_linear(n, n, n, n, n, 0, n, 1, 4, 4, 72, n, 0, n) == -1
    assert lib.cr_w8a8_rows_linear(n, n, n, n, n, 0, n, 1, 4, 4, 64, n, 0, n) == -1     # no workspace


def test_int8_refusals(backend):
    x = torch.zeros(4, 80)
    for G in (0, 8, 32, 1024, None):
        with pytest.raises(ValueError, match="convrot_groupsize"):
            backend.rms_norm_int8(x, convrot_groupsize=G)
    for G in (64, 256):
        with pytest.raises(ValueError, match="not divisible"):
            backend.rms_norm_int8(x, convrot_groupsize=G)
    with pytest.raises(ValueError, match="multiples of 64"):
        backend.rms_norm_int8(x, convrot_groupsize=16, i8t=True)


def rows_of(backend, M=4, K=64, i8t=False, **other):
    R = backend.Int8Rows(torch.zeros((M + 255) // 256 * 256 if i8t else M, K, dtype=torch.int8), torch.zeros(M), (M, K), torch.bfloat16,
                         64, i8t)
    return R._replace(**other)


@pytest.mark.parametrize("i8t", [True, False])
def test_rows_linear_refusals(backend, i8t):
    f, w, s, i8 = backend.convrot_w8a8_linear_rows, torch.zeros(8, 64, dtype=torch.int8), torch.zeros(8), torch.int8
    ok = rows_of(backend, i8t=i8t)
    for bad in (ok._replace(codes=torch.zeros(3, 64, dtype=i8)), ok._replace(codes=ok.codes.float()), ok._replace(scales=torch.zeros(5)),
                ok._replace(scales=torch.zeros(4, dtype=torch.float64)), ok._replace(shape=(2, 64)), ok._replace(shape=(4, 32)),
                ok._replace(i8t=not i8t), ok._replace(dtype=torch.float64)):
        with pytest.raises(ValueError, match="rows"):
            f(bad, w, s)
    with pytest.raises(ValueError, match="qweight"):
        f(ok, torch.zeros(8, 32, dtype=i8), s)
    with pytest.raises(ValueError, match="qweight"):
        f(ok, w.float(), s)
    with pytest.raises(ValueError, match="wscales"):
        f(ok, w, torch.zeros(7))
    with pytest.raises(ValueError, match="wscales"):
        f(ok, w, s.double())
    with pytest.raises(ValueError, match="bias"):
        f(ok, w, s, torch.zeros(7))
    with pytest.raises(ValueError, match="qweight_i8t"):
        f(ok, w, s, qweight_i8t=w)
    with pytest.raises(RuntimeError, match="CUDA"):
        f(ok, w, s)


def test_traces_are_refused(backend):
    x, rows, w = torch.zeros(4, 64), rows_of(backend), torch.zeros(8, 64, dtype=torch.int8)
    for f in (lambda t: backend.choose_experts(t, 2)[1], backend.rms_norm, lambda t: backend.rms_norm_int8(t).codes,
              lambda t: backend.convrot_w8a8_linear_rows(rows._replace(scales=t[:, 0]), w, torch.zeros(8))):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, x, check_trace=False)


def test_block_refusals():
    moe = importlib.import_module(PKG_NAME + ".mxfp4_moe")
    u, E, D, F = torch.uint8, 3, 64, 96
    experts = moe.Mxfp4MoE(torch.zeros(E, 2 * F, D // 2, dtype=u), torch.zeros(E, 2 * F, D // 32, dtype=u),
                           torch.zeros(E, D, F // 2, dtype=u), torch.zeros(E, D, F // 32, dtype=u))
    for shape in ((E, D + 1), (E + 1, D), (D, E)):
        with pytest.raises(ValueError, match="router_weight"):
            moe.RoutedMxfp4MoE(experts, torch.zeros(shape), top_k=2)
    block = moe.RoutedMxfp4MoE(experts, torch.zeros(E, D), top_k=2)
    assert [n for n, _ in block.named_parameters()] == ["router_weight"]
    for args in ((torch.zeros(4, D, requires_grad=True),), (torch.zeros(4, D), torch.zeros(4, D, requires_grad=True))):
        with pytest.raises(RuntimeError, match="frozen"):
            block(*args)
