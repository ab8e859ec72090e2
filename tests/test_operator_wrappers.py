"""Tensors that say they are on a GPU and have no memory there never reach a launch of the expert and optimizer kernels
(no GPU needed: fake tensors of one do without it)."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from raydp_amd.ops.expert_ops import ExpertPlan, combine, dispatch, expert_plan, route
from raydp_amd.ops.fused_optim import clip_grad_norm_, decode_moments


def _fakes():
    with FakeTensorMode():
        t = {"z": torch.randn(6, 4, device="cuda"), "x": torch.randn(6, 5, device="cuda"), "w": torch.rand(6, 2, device="cuda"),
             "rows": torch.randn(12, 5, device="cuda"), "codes": torch.zeros(300, dtype=torch.uint8, device="cuda"),
             "scales": torch.zeros(2, 2, dtype=torch.uint8, device="cuda"), "p": torch.zeros(3, device="cuda"),
             "g": torch.ones(3, device="cuda")}
        t.update({n: torch.zeros(s, dtype=torch.int32, device="cuda")
                  for n, s in (("ids", (6, 2)), ("source", (12,)), ("load", (4,)), ("offsets", (5,)))})
    t["plan"] = ExpertPlan(t["ids"], t["source"], t["load"], t["offsets"], 4, None)
    return t


def _clip(t):
    t["p"].grad = t["g"]
    clip_grad_norm_([t["p"]], 1.0)


CALLS = {
    "route": lambda t: route(t["z"], 2),
    "route, wanted": lambda t: route(t["z"].requires_grad_(), 2),
    "plan": lambda t: expert_plan(t["ids"], 4),
    "dispatch": lambda t: dispatch(t["x"], t["plan"]),
    "combine": lambda t: combine(t["rows"], t["plan"], t["w"]),
    "decode": lambda t: decode_moments(t["codes"], t["codes"], t["scales"]),
    "clip": _clip,
}


@pytest.mark.parametrize("inside", [True, False], ids=["in its mode", "outside"])
@pytest.mark.parametrize("name", CALLS)
def test_fake_tensors_are_refused(name, inside):
    t = _fakes()
    with pytest.raises(TypeError, match="wrapped"):
        if inside:
            with t["z"].fake_mode:
                CALLS[name](t)
        else:
            CALLS[name](t)
