"""Routed experts on the CPU: results and gradients in 64 bits, and what is refused (no GPU needed)."""
import math

import pytest
import torch

import expert_oracle as oracle
from raydp_amd.native import loader
from raydp_amd.ops.expert_ops import combine, dispatch, expert_plan, route


@pytest.mark.parametrize("renorm", [True, False])
def test_route_and_gradient_in_64_bits(renorm):
    g = torch.Generator().manual_seed(0)
    z = torch.randn(12, 7, generator=g).double().round(decimals=1)
    z[torch.rand(12, 7, generator=g) < 0.3] = -math.inf
    z[3] = -math.inf
    dw = torch.randn(12, 3, generator=g).double()
    zr = z.clone().requires_grad_()
    w, ids = route(zr, 3, renorm)
    ew, eids, edz = oracle.route(z, 3, renorm, dw)
    assert torch.equal(ids.long(), eids)
    torch.testing.assert_close(w, ew, rtol=1e-14, atol=0)
    (dz,) = torch.autograd.grad(w, zr, dw)
    torch.testing.assert_close(dz, edz, rtol=0, atol=1e-14)
    smooth = torch.randn(4, 6, generator=g).double().requires_grad_()
    assert torch.autograd.gradcheck(lambda t: route(t, 2, renorm)[0], (smooth,))


@pytest.mark.parametrize("T,k,E,capacity", [(0, 2, 3, 2), (0, 1, 3, None), (1, 1, 1, None), (30, 2, 5, None), (30, 3, 4, 6)])
def test_plan_dispatch_combine_and_gradients(T, k, E, capacity):
    g = torch.Generator().manual_seed(T)
    ids = torch.randint(-2, E + 1, (T, k), generator=g)
    p = expert_plan(ids, E, capacity)
    position, source, load, offsets = oracle.plan(ids, E, capacity)
    assert (p.position.flatten().tolist(), p.source.tolist(), p.load.tolist(), p.offsets.tolist()) == (position, source, load, offsets)
    x = torch.randn(T, 3, generator=g).double().requires_grad_()
    h = torch.randn(p.rows, 3, generator=g).double().requires_grad_()
    w = torch.rand(T, k, generator=g).double().requires_grad_()
    torch.testing.assert_close(dispatch(x, p), oracle.dispatch(x, position, p.rows, k), rtol=0, atol=0)
    torch.testing.assert_close(combine(h, p, w), oracle.combine(h, position, T, k, w), rtol=1e-14, atol=1e-14)
    if T:
        assert torch.autograd.gradcheck(lambda a: dispatch(a, p), (x,))
        assert torch.autograd.gradcheck(lambda a, b: combine(a, p, b), (h, w))


def test_what_is_not_filled_is_not_read():
    ids = torch.tensor([[0], [-1]])
    p = expert_plan(ids, 2, 2)
    h = torch.full((4, 2), math.nan)
    h[0] = 1.0
    assert torch.equal(combine(h, p, torch.ones(2, 1)), torch.tensor([[1.0, 1.0], [0.0, 0.0]]))


def test_refusals():
    z = torch.randn(4, 6)
    for bad in (torch.zeros(4, 6, dtype=torch.int32), torch.zeros(6)):
        with pytest.raises(ValueError, match="logits"):
            route(bad, 1)
    for k in (0, 7, -1):
        with pytest.raises(ValueError, match="k must be"):
            route(z, k)
    with pytest.raises(ValueError, match="k must be"):
        route(torch.randn(2, 40), 33)
    with pytest.raises(ValueError, match="at most 1024"):
        route(torch.randn(2, 1025), 2)
    ids = torch.zeros(4, 2, dtype=torch.int32)
    for bad in (ids.float(), ids.flatten(), ids[:, :0], ids.to(torch.int16)):
        with pytest.raises(ValueError, match="experts must be"):
            expert_plan(bad, 3)
    for E in (0, 1025):
        with pytest.raises(ValueError, match="num_experts"):
            expert_plan(ids, E)
    for c in (0, -4):
        with pytest.raises(ValueError, match="capacity"):
            expert_plan(ids, 3, c)
    with pytest.raises(ValueError, match="32 bits"):
        expert_plan(ids, 1024, 1 << 22)
    p = expert_plan(ids, 3, 5)
    for bad in (torch.randn(3, 2), torch.randn(4), torch.randn(4, 0), torch.zeros(4, 2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="dispatch"):
            dispatch(bad, p)
    with pytest.raises(ValueError, match="combine"):
        combine(torch.randn(4, 2), p)                       # samples' rows where expert rows are wanted
    rows = torch.randn(15, 2)
    for bad in (torch.rand(4, 3), torch.rand(8), torch.ones(4, 2, dtype=torch.int64)):
        with pytest.raises(ValueError, match="weights"):
            combine(rows, p, bad)


def test_plan_grid_covers_every_choice():
    plan_grid = loader.load_torch().plan_grid
    for n in list(range(0, 5000, 7)) + [4096, 4097, 262144, 262145, 10 ** 6, 2 ** 31 - 1]:
        chunk, blocks = plan_grid(n)
        assert chunk % 1024 == 0 and blocks >= 1 and chunk * blocks >= n and blocks <= 256
        assert blocks == 1 or chunk * (blocks - 1) < n
