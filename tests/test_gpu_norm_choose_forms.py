"""The router's choice and the norm: what autograd hands back, threads and streams of their own, arguments of other types."""
import importlib
import threading

import numpy as np
import pytest
import torch

from conftest import PKG_NAME
from test_gpu_experts_saved import FORMS, same, shifted, strided

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "python"])
def path(request, native, gpu, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(native, "host_or_none", lambda: None)
    else:
        assert native.host_or_none() is not None
    return request.param


def tensors(dtype, T=21, E=24, D=56):
    g = torch.Generator().manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()
    return {"logits": r(T, E), "x": r(T, D), "residual": r(T, D), "weight": r(D), "d_w": torch.randn(T, 3, generator=g).cuda(),
            "d_y": r(T, D), "d_h": r(T, D)}


def grads(backend, t, pack, unpack):
    logits, x, r, w = (t[n].clone().requires_grad_() for n in ("logits", "x", "residual", "weight"))
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        weights = backend.choose_experts(logits, 3, scoring="sigmoid")[1]
        y, h = backend.rms_norm(x, w, r)
    return torch.autograd.grad((weights, y, h), (logits, x, r, w), (t["d_w"], t["d_y"], t["d_h"]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("back", [strided, shifted, torch.clone])
def test_other_layouts_count_by_their_values(backend, path, back, dtype):
    t = tensors(dtype)
    want, got = grads(backend, t, same, same), grads(backend, t, same, back)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_saved_on_the_host(backend, path):
    t = tensors(torch.bfloat16)
    got = grads(backend, t, lambda t: t.cpu(), lambda t: t.cuda())
    assert all(torch.equal(a, b) for a, b in zip(got, grads(backend, t, same, same)))


@pytest.mark.parametrize("which,form", [(w, f) for w in ("logits", "ids", "rows", "weight") for f in FORMS if (w, f) != ("weight", "flat")])
def test_other_forms_are_refused(backend, path, which, form):
    t = tensors(torch.float32)
    shape, dtype = {"logits": ((21, 24), torch.float32), "ids": ((21, 3), torch.int32), "rows": ((21, 56), torch.float32),
                    "weight": ((56,), torch.float32)}[which]

    def back(s):
        return FORMS[form](s) if tuple(s.shape) == shape and s.dtype == dtype else s

    with pytest.raises(RuntimeError, match="saved"):
        grads(backend, t, same, back)


def test_saved_ids_of_no_expert(backend, path):
    """Ids that came back changed add nothing where they are out of range, and touch nothing else."""
    t = tensors(torch.float32)

    def back(s):
        if s.dtype != torch.int32:
            return s
        s = s.clone()
        s[0] = torch.tensor([-5, 24, 1 << 30])
        return s

    got = grads(backend, t, same, back)
    want = grads(backend, t, same, same)
    assert not bool(got[0][0].any()) and torch.equal(got[0][1:], want[0][1:]) and torch.equal(got[1], want[1])


def test_arguments_of_other_types(backend, path):
    t = tensors(torch.float32)
    want = backend.choose_experts(t["logits"], 3, num_groups=4, top_groups=2, scale=2.0)
    got = backend.choose_experts(t["logits"], np.int64(3), num_groups=np.int32(4), top_groups=np.int64(2), scale=np.float32(2.0), renormalize=1)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for bad in (dict(top_k=2.0), dict(top_k="2"), dict(top_k=2, num_groups=1.0), dict(top_k=2, num_groups=2, top_groups=1.0)):
        with pytest.raises(TypeError):
            backend.choose_experts(t["logits"], **bad)
    y = backend.rms_norm(t["x"], t["weight"], eps=np.float64(0.5))
    assert torch.equal(y, backend.rms_norm(t["x"], t["weight"], eps=0.5))
    assert torch.equal(backend.rms_norm(t["x"], eps=1), backend.rms_norm(t["x"], eps=1.0))
    x = torch.randn(4, 256, device="cuda")
    assert torch.equal(backend.rms_norm_int8(x, i8t=0).codes, backend.rms_norm_int8(x).codes)
    rows = backend.rms_norm_int8(x)
    with pytest.raises(RuntimeError, match="no gradient"):
        backend.convrot_w8a8_linear_rows(rows._replace(scales=rows.scales.clone().requires_grad_()), rows.codes, rows.scales)


class _Stop(torch.autograd.Function):
    """Its input without a gradient."""
    @staticmethod
    def forward(ctx, x):
        return x.clone()

    @staticmethod
    def backward(ctx, d):
        return None


def test_outputs_without_a_gradient(backend, path):
    """A gradient that does not arrive is none, and those of the other outputs are as they were."""
    t = tensors(torch.float32)
    logits, x, r = (t[n].clone().requires_grad_() for n in ("logits", "x", "residual"))
    _Stop.apply(backend.choose_experts(logits, 3)[1]).sum().backward()
    assert logits.grad is None
    y, h = backend.rms_norm(x, None, r)
    (_Stop.apply(y).sum() + _Stop.apply(h).sum()).backward()
    assert x.grad is None and r.grad is None
    y, h = backend.rms_norm(x, None, r)
    (_Stop.apply(y).sum() + (h * t["d_h"]).sum()).backward()
    assert torch.equal(x.grad, t["d_h"]) and torch.equal(r.grad, t["d_h"])


def test_parameters_and_subclasses(backend, path):
    """Parameters count as tensors; a weight that is frozen takes no gradient."""
    t = tensors(torch.float32)
    p = torch.nn.Parameter(t["weight"].clone(), requires_grad=False)
    assert torch.equal(backend.rms_norm(t["x"], p), backend.rms_norm(t["x"], t["weight"]))
    assert not backend.rms_norm(t["x"], p).requires_grad
    w = torch.nn.Parameter(t["weight"].clone())
    y = backend.rms_norm(t["x"], w)
    y.backward(t["d_y"])
    assert w.grad.shape == w.shape and t["x"].grad is None


def test_threads_on_streams_of_their_own(backend, path):
    """Each thread's calls give the bits of the same calls made alone, gradients among them."""
    cases = []
    for i in range(6):
        t = tensors([torch.bfloat16, torch.float32, torch.float16][i % 3], T=40 + 37 * i, E=24 + 8 * i, D=256 * (i + 1))
        cases.append(t)

    def work(t):
        rows, h = backend.rms_norm_int8(t["x"], t["weight"], t["residual"])
        return [*grads(backend, t, same, same), *backend.choose_experts(t["logits"], 5, num_groups=2, top_groups=1), rows.codes, rows.scales, h]

    want = [work(t) for t in cases]
    torch.cuda.synchronize()
    outs, start = [None] * len(cases), threading.Barrier(len(cases))

    def run(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            start.wait(timeout=60)
            for _ in range(20):
                got = work(cases[i])
            stream.synchronize()
        outs[i] = got

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=90)
    for i, got in enumerate(outs):
        assert got is not None, f"thread {i} did not finish"
        assert all(torch.equal(a, b) for a, b in zip(got, want[i])), i


def test_block_under_autocast(backend, gpu):
    """The router's logits stay in 32 bits."""
    moe = importlib.import_module(PKG_NAME + ".mxfp4_moe")
    g = torch.Generator().manual_seed(1)
    E, D, F = 16, 64, 96
    w = [torch.randn(E, *s, generator=g).cuda() for s in ((F, D), (F, D), (D, F))]
    block = moe.RoutedMxfp4MoE(moe.Mxfp4MoE.from_float(*w), torch.randn(E, D, generator=g).cuda() * 0.125, top_k=4)
    x = torch.randn(200, D, generator=g).to(torch.bfloat16).cuda()
    want = block(x)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(block(x), want)
    assert block(x[:0]).shape == (0, D)
