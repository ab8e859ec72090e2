"""Routed experts and the optimizer's functions under what sees only operators of torch: forward derivatives and traces."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
import torch.nn as nn

from raydp_amd.ops.expert_ops import combine, dispatch, expert_plan, route
from raydp_amd.ops.fused_optim import FusedAdamW, clip_grad_norm_, decode_moments

pytestmark = pytest.mark.gpu


def _inputs():
    g = torch.Generator().manual_seed(0)
    z, x = torch.randn(6, 4, generator=g).cuda(), torch.randn(6, 5, generator=g).cuda()
    w, ids = route(z, 2)
    plan = expert_plan(ids, 4)
    return z, x, w, ids, plan, dispatch(x, plan)


CALLS = {
    "route": lambda z, x, w, ids, plan, rows, f: route(f(z), 2),
    "route over all": lambda z, x, w, ids, plan, rows, f: route(f(z), 2, renormalize=False),
    "dispatch": lambda z, x, w, ids, plan, rows, f: dispatch(f(x), plan),
    "combine rows": lambda z, x, w, ids, plan, rows, f: combine(f(rows), plan, w),
    "combine weights": lambda z, x, w, ids, plan, rows, f: combine(rows, plan, f(w)),
}


@pytest.mark.parametrize("grad", [True, False], ids=["grad", "no_grad"])
@pytest.mark.parametrize("leaf", [True, False], ids=["wanted", "plain"])
@pytest.mark.parametrize("name", CALLS)
def test_a_forward_derivative_is_refused(name, leaf, grad):
    args = _inputs()
    with fwAD.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(NotImplementedError, match="forward-mode"):
            CALLS[name](*args, lambda t: fwAD.make_dual(t.clone().requires_grad_(leaf), torch.ones_like(t)))
        CALLS[name](*args, lambda t: t.clone().requires_grad_(leaf))            # (a level without tangents is no matter)


@pytest.mark.parametrize("name", CALLS)
def test_a_forward_derivative_of_a_gradient_is_refused(name):
    args, leaf = _inputs(), []
    out = CALLS[name](*args, lambda t: leaf.append(t.clone().requires_grad_()) or leaf[0])
    out = out if isinstance(out, torch.Tensor) else out[0]
    with fwAD.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(out, leaf, fwAD.make_dual(torch.ones_like(out), torch.ones_like(out)))


def test_clipping_gradients_with_tangents_is_refused():
    p = nn.Parameter(torch.ones(3, device="cuda"))
    with fwAD.dual_level():
        p.grad = fwAD.make_dual(torch.ones(3, device="cuda"), torch.ones(3, device="cuda"))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            clip_grad_norm_([p], 0.1)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            FusedAdamW([p]).step()
    p.grad = None


def _traced():
    z, x, w, ids, plan, rows = _inputs()
    p = nn.Parameter(torch.ones(300, device="cuda"))
    p.grad = torch.ones(300, device="cuda")
    opt = FusedAdamW([p])
    opt.step()
    st = opt.state[p]
    return {
        "route": (lambda t: route(t, 2)[0], z),
        "plan": (lambda t: expert_plan(t, 4).position, ids),
        "dispatch": (lambda t: dispatch(t, plan), x),
        "combine": (lambda t: combine(t, plan, w), rows),
        "decode": (lambda t: decode_moments(t, st["exp_avg_sq"], st["scales"])[0], st["exp_avg"]),
        "clip": (lambda t: clip_grad_norm_([p], 1.0) + t, x),
        "step": (lambda t: (opt.step(), t + 1)[1], x),
    }


@pytest.mark.parametrize("name", ["route", "plan", "dispatch", "combine", "decode", "clip", "step"])
@pytest.mark.parametrize("how", ["jit", "fx"])
def test_a_trace_that_would_miss_the_launch_is_refused(how, name):
    f, t = _traced()[name]
    with pytest.raises(RuntimeError, match="trace"):
        if how == "jit":
            torch.jit.trace(f, (t,), check_trace=False)
        else:
            from torch.fx.experimental.proxy_tensor import make_fx
            make_fx(f)(t)
    f(t)


def test_transforms_and_wrapped_tensors_are_refused():
    from torch._subclasses.fake_tensor import FakeTensorMode
    z, x, w, ids, plan, rows = _inputs()
    with pytest.raises(TypeError, match="wrapped"):
        torch.func.vmap(lambda t: route(t, 2)[0])(torch.stack([z, z]))
    with pytest.raises(TypeError, match="wrapped"):
        torch.func.grad(lambda t: dispatch(t, plan).sum())(x)
    with pytest.raises(TypeError, match="wrapped"):
        combine(torch._neg_view(rows), plan, w)
    leaf = rows.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="wrapped"):          # (what a backward throws arrives as this)
        torch.autograd.grad(combine(leaf, plan, w), leaf, torch.ones(3, 6, 5, device="cuda"), is_grads_batched=True)
    with FakeTensorMode():
        p = nn.Parameter(torch.ones(300, device="cuda"))
        p.grad = torch.ones(300, device="cuda")
        with pytest.raises(TypeError, match="wrapped"):
            FusedAdamW([p]).step()
    p = nn.Parameter(torch.ones(300, device="cuda"))
    p.grad = torch._neg_view(torch.ones(300, device="cuda"))
    for call in (lambda: FusedAdamW([p]).step(), lambda: clip_grad_norm_([p], 1.0)):
        with pytest.raises(TypeError, match="wrapped"):
            call()
    route(z, 2)
