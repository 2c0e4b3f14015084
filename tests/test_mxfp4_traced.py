"""A call that a trace would not see, or whose tensors have no memory, is refused before any launch."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx


def calls(q, device):
    """Each operator as a function of one tensor, and a tensor for it."""
    kw = {"device": device}
    i, u = dict(dtype=torch.int32, **kw), dict(dtype=torch.uint8, **kw)
    x, w, s = torch.zeros(3, 64, **kw), torch.zeros(8, 32, **u), torch.zeros(8, 2, **u)
    plan = q.ExpertPlan(torch.zeros(6, **i), torch.zeros(3, 2, **i), torch.zeros(5, **i))
    we, se = torch.zeros(4, 8, 32, **u), torch.zeros(4, 8, 2, **u)
    weights = torch.zeros(3, 2, **kw)
    return {
        "quantize": (lambda t: q.quantize_mxfp4(t)[0], x),
        "dequantize": (lambda t: q.dequantize_mxfp4(t, s), w),
        "linear": (lambda t: q.mxfp4_linear(t, w, s), x),
        "expert linear": (lambda t: q.mxfp4_expert_linear(t, we, se, plan), x),
        "sort": (lambda t: q.sort_tokens_by_expert(t, 4).order, torch.zeros(3, 2, dtype=torch.int64, **kw)),
        "gather": (lambda t: q.gather_expert_rows(t, plan), x),
        "combine": (lambda t: q.combine_expert_rows(t, weights, plan), torch.zeros(6, 8, **kw)),
    }


NAMES = ["quantize", "dequantize", "linear", "expert linear", "sort", "gather", "combine"]


@pytest.mark.parametrize("name", NAMES)
def test_traces_are_refused(backend, name):
    f, t = calls(backend, "cpu")[name]
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(f, t, check_trace=False)
    for mode in ("real", "fake", "symbolic"):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(f, tracing_mode=mode, _allow_non_fake_inputs=True)(t)


@pytest.mark.parametrize("name", NAMES)
def test_tensors_without_memory_are_refused(backend, name):
    """Their data pointer reads as 0."""
    with FakeTensorMode():
        f, t = calls(backend, "cuda")[name]
        with pytest.raises(RuntimeError, match="cannot be traced"):
            f(t)
    with pytest.raises(RuntimeError, match="no memory"):                 # the mode left, its tensors kept
        f(t)
    f, t = calls(backend, "cpu")[name]
    with pytest.raises(RuntimeError, match="no memory|cannot be traced"):
        torch.func.functionalize(f)(t)


def test_operands_of_every_kernel_have_memory(native):
    with FakeTensorMode():
        t = torch.empty(4, 64, device="cuda")
    with pytest.raises(RuntimeError, match="no memory"):
        native._aligned(t)
    assert native._aligned(torch.empty(0, 64)).shape == (0, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_refused_on_the_gpu(backend, gpu, name):
    """Past the host module too; the same call runs outside of a trace."""
    f, t = calls(backend, "cuda")[name]
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(f, t, check_trace=False)
    with pytest.raises(RuntimeError, match="no memory|cannot be traced"):
        torch.func.functionalize(f)(t)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(f)(t)
    assert f(t).is_cuda
