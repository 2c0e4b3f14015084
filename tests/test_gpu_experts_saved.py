"""GPU checks of what the routing's gradients take from autograd: hooks on saved tensors may hand back tensors of another
layout, which count by their values, or of another form, which are refused; a plan changed in between is noticed."""
import pytest
import torch

from test_gpu_experts import routed

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "python"])
def path(request, native, gpu, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(native, "host_or_none", lambda: None)
    else:
        assert native.host_or_none() is not None
    return request.param


def grads(backend, plan, x, rows, w, pack, unpack):
    """Gradients of gather and combine with the hooks on what they save."""
    x, rows, w = (t.cuda().requires_grad_() for t in (x, rows, w))
    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        g, c = backend.gather_expert_rows(x, plan), backend.combine_expert_rows(rows, w, plan)
    d = torch.Generator().manual_seed(9)
    d_rows, d_out = torch.randn(g.shape, generator=d).to(g.dtype).cuda(), torch.randn(c.shape, generator=d).to(c.dtype).cuda()
    return torch.autograd.grad((g, c), (x, rows, w), (d_rows, d_out))


def strided(t):
    return torch.stack((t, torch.zeros_like(t)), dim=-1)[..., 0]


def shifted(t):
    return torch.cat((t.new_zeros(1), t.flatten()))[1:].view(t.shape)


def same(t):
    return t


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("back", [strided, shifted, torch.clone])
def test_other_layouts_count_by_their_values(backend, path, back, dtype):
    ids, plan, x, rows, w = routed(backend, 21, 3, 5, 72, dtype, seed=3)
    want = grads(backend, plan, x, rows, w, same, same)
    got = grads(backend, plan, x, rows, w, same, back)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_saved_on_the_host(backend, path):
    ids, plan, x, rows, w = routed(backend, 21, 3, 5, 72, torch.bfloat16, seed=3)
    want = grads(backend, plan, x, rows, w, same, same)
    got = grads(backend, plan, x, rows, w, lambda t: t.cpu(), lambda t: t.cuda())
    assert all(torch.equal(a, b) for a, b in zip(got, want))


FORMS = {"host": lambda t: t.cpu(), "double": lambda t: t.double(), "fewer": lambda t: t[:1], "flat": lambda t: t.flatten(),
         "twice": lambda t: torch.cat((t, t)), "a dimension more": lambda t: t.unsqueeze(0)}


@pytest.mark.parametrize("which,form", [(w, f) for w in ("offsets", "position", "rows", "weights") for f in FORMS
                                        if (w, f) != ("offsets", "flat")])
def test_other_forms_are_refused(backend, path, which, form):
    """One of the saved tensors comes back as something else."""
    ids, plan, x, rows, w = routed(backend, 21, 3, 5, 72, torch.float32, seed=3)
    picked = {"offsets": plan.offsets, "position": plan.position, "rows": rows, "weights": w}[which]

    def back(t):
        return FORMS[form](t) if t.shape == picked.shape and t.dtype == picked.dtype else t

    with pytest.raises(RuntimeError, match="saved"):
        grads(backend, plan, x, rows, w, same, back)


@pytest.mark.parametrize("what", ["position", "offsets"])
def test_a_changed_plan_is_noticed(backend, path, what):
    ids, plan, x, rows, w = routed(backend, 21, 3, 5, 72, torch.float32, seed=3)
    rows = rows.cuda().requires_grad_()
    out = backend.combine_expert_rows(rows, w.cuda(), plan)
    getattr(plan, what).add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    if what == "position":
        x = x.cuda().requires_grad_()
        g = backend.gather_expert_rows(x, plan)
        plan.position.add_(0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            g.sum().backward()
