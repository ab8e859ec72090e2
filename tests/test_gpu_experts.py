"""Routed experts on the GPU (csrc/hip/experts.hip) against plain implementations in 64 bits."""
import math

import pytest
import torch
import torch.nn as nn

import expert_oracle as oracle
from raydp_amd.ops.expert_ops import combine, dispatch, expert_plan, route

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.fixture(params=[None, 0], ids=["cached", "streamed"])
def last_level(request):
    """Both sides of the bound from which kernels stream past the caches."""
    from raydp_amd.native import loader
    ext = loader.load_torch()
    old = ext.set_last_level(request.param) if request.param is not None else None
    yield
    if old is not None:
        ext.set_last_level(old)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 16, 2), (7, 3, 3), (65, 8, 1), (130, 17, 5), (33, 64, 2), (40, 65, 8),
                                   (19, 200, 4), (9, 256, 32), (11, 300, 6), (5, 1000, 7), (3, 1024, 32)])
def test_route_and_its_gradient(T, E, k, renorm, dtype):
    """Ties (values on a coarse grid), masked experts, rows with fewer than k experts left and rows with none."""
    g = torch.Generator().manual_seed(T * 1000 + E)
    z = (torch.randn(T, E, generator=g) * 16).round() / 8
    z[torch.rand(T, E, generator=g) < 0.2] = -math.inf
    if T > 4:
        z[1] = -math.inf
        z[2, 1:] = -math.inf
        z[3] = 0.5
    dw = torch.randn(T, k, generator=g)
    zg = z.to(dtype).cuda().requires_grad_()
    w, ids = route(zg, k, renormalize=renorm)
    ew, eids, edz = oracle.route(z.to(dtype).double(), k, renorm, dw.double())
    assert ids.dtype == torch.int32 and torch.equal(ids.cpu().long(), eids)
    assert w.dtype == torch.float32
    # exp to 2 ulp of an argument below 16 (an error of 2^-24 * 16 in the exponent), a sum of E terms, the quotient
    tol = (16 + 4 + E) * 2.0 ** -24
    assert ((w.detach().cpu().double() - ew).abs() <= tol * ew).all()
    (dz,) = torch.autograd.grad(w, zg, dw.cuda())
    # terms of size p * sum |w dw| that may cancel, each as exact as the weights; then one rounding
    size = (ew * dw.double().abs()).sum(1, keepdim=True) + dw.double().abs().max(1, keepdim=True).values
    bound = (2 * tol + (k + 4) * 2.0 ** -24) * size + _half_step(dtype) * edz.abs() + 2.0 ** -25
    if dtype != torch.float16:
        bound = bound - 2.0 ** -25           # (fp16 also rounds to its smallest step, 2^-24)
    assert dz.dtype == dtype and ((dz.cpu().double() - edz).abs() <= bound + 1e-38).all()


def test_route_gradient_against_differences():
    g = torch.Generator().manual_seed(0)
    z, dw = torch.randn(6, 20, generator=g).double(), torch.randn(6, 4, generator=g).double()
    for renorm in (True, False):
        zg = z.float().cuda().requires_grad_()
        w, ids = route(zg, 4, renorm)
        (dz,) = torch.autograd.grad(w, zg, dw.float().cuda())
        h = 2.0 ** -10
        for t, e in [(0, int(ids[0, 0])), (1, int(ids[1, 3])), (2, 7), (5, 0)]:
            d = torch.zeros_like(z)
            d[t, e] = h
            up, iu, _ = oracle.route(z + d, 4, renorm)
            dn, il, _ = oracle.route(z - d, 4, renorm)
            if torch.equal(iu, il):
                diff = float(((up - dn) * dw).sum() / (2 * h))
                assert abs(float(dz[t, e]) - diff) <= 4 * h * h + 1e-5     # second order, and fp32


def test_route_layouts_nan_and_infinity():
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(50, 40, generator=g).cuda()
    a = route(wide[:, 3:20], 3)                                   # rows further apart than they are long
    b = route(wide[:, 3:20].contiguous(), 3)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    t = torch.randn(17, 50, generator=g).cuda().t()               # columns first
    a, b = route(t, 3, False), route(t.contiguous(), 3, False)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    one = torch.zeros(1, 9, device="cuda").expand(6, 9)           # one row for all
    assert torch.equal(route(one, 2)[1], torch.tensor([[0, 1]] * 6, dtype=torch.int32, device="cuda"))
    z = torch.zeros(3, 5, device="cuda")
    z[1, 2] = math.nan
    for renorm in (True, False):
        w, ids = route(z, 2, renorm)
        assert torch.isnan(w[1]).all() and torch.isfinite(w[0]).all() and torch.isfinite(w[2]).all()
        assert 2 not in ids[1].tolist()
    for dtype in DTYPES:      # zeros of either sign are a tie; both ends of the type keep their order
        big = torch.finfo(dtype).max
        z = torch.tensor([[-0.0, 0.0, -0.0, 0.0], [0.0, -0.0, 1.0, -1.0], [-big, -math.inf, big, 0.0]], device="cuda").to(dtype)
        assert route(z, 4)[1].tolist() == [[0, 1, 2, 3], [2, 0, 1, 3], [2, 3, 0, -1]]
        z = torch.tensor([[big, math.inf, big, -big, -math.inf]], device="cuda").to(dtype)
        assert route(z, 5)[1].tolist() == [[1, 0, 2, 3, -1]]
        z = torch.tensor([[big, -math.nan, big / 2, math.nan, -big]], device="cuda").to(dtype)
        assert route(z, 4)[1].tolist() == [[0, 2, 4, -1]] and torch.isnan(route(z, 4)[0]).all()
        z = torch.full((1, 7), math.nan, device="cuda").to(dtype)
        w, ids = route(z, 3)
        assert ids.tolist() == [[-1, -1, -1]] and torch.isnan(w).all()
    w, ids = route(torch.empty(0, 5, device="cuda"), 2)
    assert w.shape == (0, 2) and ids.shape == (0, 2)


PLANS = [(0, 1, 4, None), (0, 2, 3, 2), (1, 1, 1, None), (1, 2, 16, None), (3, 4, 2, 1), (65, 2, 8, None), (64, 2, 1, 100),
         (511, 3, 7, 200), (1024, 4, 64, None), (1025, 4, 64, 70), (2500, 2, 1000, None), (9000, 1, 5, 1000), (3000, 7, 1024, 25)]


@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
@pytest.mark.parametrize("T,k,E,capacity", PLANS)
def test_plan(T, k, E, capacity, wide):
    """Skewed choices, the same expert twice in a sample, experts nobody wants, and numbers that are no expert."""
    g = torch.Generator().manual_seed(T + E)
    ids = (torch.rand(T, k, generator=g) ** 2 * E * 1.05).long()
    ids[torch.rand(T, k, generator=g) < 0.1] = -1
    if T > 2:
        ids[0] = 0
        ids[1, 0] = E
        ids[2, 0] = torch.iinfo(wide).min
    p = expert_plan(ids.to(wide).cuda(), E, capacity)
    position, source, load, offsets = oracle.plan(ids, E, capacity)
    assert p.position.shape == (T, k) and p.position.flatten().tolist() == position
    assert p.rows == len(source) and p.source.tolist() == source
    assert p.load.tolist() == load and p.offsets.tolist() == offsets


def test_plan_of_many_choices_is_a_stable_sort():
    ids = torch.randint(-1, 200, (300001, 3), generator=torch.Generator().manual_seed(1)).int()
    ids[1000:200000] = 17                  # one expert takes most
    p = expert_plan(ids.cuda(), 200)
    flat = ids.flatten().long()
    key = torch.where(flat >= 0, flat, 200)
    order = torch.sort(key, stable=True).indices
    live = int((flat >= 0).sum())
    src = p.source.cpu().long()
    assert torch.equal(src[:live], order[:live]) and (src[live:] == -1).all()
    assert torch.equal(p.load.cpu().long(), torch.bincount(key, minlength=201)[:200])
    pos = p.position.cpu().long().flatten()
    assert torch.equal(pos[src[:live]], torch.arange(live)) and (pos[flat < 0] == -1).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,k,E,D,capacity", [(1, 2, 16, 384, None), (5, 1, 3, 1, None), (67, 2, 8, 7, 20), (33, 3, 4, 64, None),
                                              (70, 2, 5, 383, 30), (40, 4, 64, 1030, None), (9, 32, 40, 24, 8), (0, 2, 3, 10, 4)])
def test_dispatch_combine_and_their_gradients(T, k, E, D, capacity, dtype, last_level):
    g = torch.Generator().manual_seed(T + D)
    ids = torch.randint(-1, E, (T, k), generator=g)
    if T > 1:
        ids[1] = -1                                   # a sample without an expert
    p = expert_plan(ids.int().cuda(), E, capacity)
    position = p.position.cpu().flatten().tolist()
    x, dy = torch.randn(T, D, generator=g).to(dtype), torch.randn(T, D, generator=g).to(dtype)
    h, drows = torch.randn(p.rows, D, generator=g).to(dtype), torch.randn(p.rows, D, generator=g).to(dtype)
    # what no sample fills is never read
    empty = p.source.cpu() < 0
    h[empty], drows[empty] = math.nan, math.inf
    w = torch.rand(T, k, generator=g)
    xg, hg, wg = x.cuda().requires_grad_(), h.cuda().requires_grad_(), w.cuda().requires_grad_()
    rows, y, y1 = dispatch(xg, p), combine(hg, p, wg), combine(hg, p)
    x6, h6, w6, dy6, dr6 = (t.double() for t in (x, h.masked_fill(empty[:, None], 0), w, dy, drows.masked_fill(empty[:, None], 0)))
    assert torch.equal(rows.detach().cpu().double(), oracle.dispatch(x6, position, p.rows, k))
    half = _half_step(dtype)

    def near(got, want, size, last):
        # k (or D) fp32 products and sums of this size, and one rounding to the output's type
        got = got.detach().cpu().double()
        assert ((got - want).abs() <= size * 2.0 ** -24 + last * want.abs() + 2.0 ** -25 * (dtype == torch.float16)).all()
    size = oracle.combine(h6.abs(), position, T, k, w6)
    near(y, oracle.combine(h6, position, T, k, w6), (k + 1) * size, half)
    near(y1, oracle.combine(h6, position, T, k), (k + 1) * oracle.combine(h6.abs(), position, T, k), half)
    dh, dw = torch.autograd.grad(y, (hg, wg), dy.cuda())
    (dx,) = torch.autograd.grad(rows, xg, drows.cuda())
    want_dh, want_dw, size_dw = torch.zeros(p.rows, D).double(), torch.zeros(T, k).double(), torch.zeros(T, k).double()
    for i, r in enumerate(position):
        if r >= 0:
            t, j = i // k, i % k
            want_dh[r] = w6[t, j] * dy6[t]
            want_dw[t, j], size_dw[t, j] = h6[r] @ dy6[t], h6[r].abs() @ dy6[t].abs()
    near(dh, want_dh, 2 * want_dh.abs(), half)
    assert dw.dtype == torch.float32
    got = dw.cpu().double()
    assert ((got - want_dw).abs() <= (D + 1) * 2.0 ** -24 * size_dw).all()
    near(dx, oracle.combine(dr6, position, T, k), (k + 1) * oracle.combine(dr6.abs(), position, T, k), half)
    (dh1,) = torch.autograd.grad(y1, hg, dy.cuda())
    assert torch.equal(dh1.cpu().double(), oracle.dispatch(dy6, position, p.rows, k))


def test_rows_with_strides_shared_rows_and_odd_addresses():
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(0, 6, (37, 2), generator=g).int().cuda()
    p = expert_plan(ids, 6)
    for dtype in DTYPES:
        base = torch.randn(37, 100, generator=g).to(dtype).cuda()
        for x in (base[:, 1:72], base[:, 3:4], base.t()[:37, :20], base[:1, :33].expand(37, 33)):
            x = x.requires_grad_()
            rows = dispatch(x, p)
            assert torch.equal(rows, dispatch(x.detach().contiguous(), p))
            (dx,) = torch.autograd.grad(rows.float().sum(), x)
            assert (dx == 2).all()
            h = rows.detach()
            assert torch.equal(combine(h.t().contiguous().t(), p), combine(h, p))
    w = torch.rand(2, 37, generator=g).cuda().t()                 # weights in another order, and in another type
    h = torch.randn(p.rows, 9, generator=g).cuda()
    assert torch.equal(combine(h, p, w), combine(h, p, w.contiguous()))
    assert torch.equal(combine(h, p, w.bfloat16()), combine(h, p, w.bfloat16().float()))
    for kind in (torch.bfloat16, torch.float64):                  # and their gradient comes back in that type
        wk = w.to(kind).requires_grad_()
        (dw,) = torch.autograd.grad(combine(h, p, wk).sum(), wk)
        w32 = w.to(kind).float().requires_grad_()
        (want,) = torch.autograd.grad(combine(h, p, w32).sum(), w32)
        assert dw.dtype == kind and torch.equal(dw, want.to(kind))
    hs = torch.randn(9, p.rows, generator=g).cuda().requires_grad_()      # rows in another order
    (dh,) = torch.autograd.grad(combine(hs.t(), p, w).square().sum(), hs)
    hc = hs.detach().t().contiguous().requires_grad_()
    assert torch.equal(dh, torch.autograd.grad(combine(hc, p, w).square().sum(), hc)[0].t())
    # one weight for all: the gradient is summed over what it was broadcast to
    one = torch.full((1, 1), 0.5, device="cuda", requires_grad=True)
    y = combine(h, p, one.expand(37, 2))
    y.sum().backward()
    assert abs(float(one.grad) - float(h.double().sum())) <= 1e-4 * float(h.abs().sum())


def test_positions_past_the_rows_reach_nothing():
    """A plan belongs to its rows; one that was written over is held to them."""
    p = expert_plan(torch.zeros(4, 2, dtype=torch.int32, device="cuda"), 1)
    x, h = torch.randn(4, 5, device="cuda"), torch.randn(8, 5, device="cuda")
    p.position[1, 0] = 8
    p.position[2, 1] = 2 ** 31 - 1
    p.position[3] = -7
    rows, y = dispatch(x, p), combine(h, p)
    assert torch.equal(rows[p.position[0].long()], x[:1].expand(2, 5)) and torch.equal(y[1], h[3]) and not y[3].any()


def test_offsets_past_32_bits():
    """2^31 elements and more on either side; only rows at the far end are looked at."""
    T, k, D = 140000, 2, 8200
    x = torch.zeros(T, D, dtype=torch.bfloat16, device="cuda")
    x[-1] = torch.arange(D, device="cuda").remainder(251).to(torch.bfloat16)
    ids = torch.zeros(T, k, dtype=torch.int32, device="cuda")
    ids[:, 1] = 1
    p = expert_plan(ids, 2)
    rows = dispatch(x, p)
    assert rows.numel() > 1 << 31
    assert torch.equal(rows[-1], x[-1]) and torch.equal(rows[T - 1], x[-1]) and not rows[T:T + 5].any()
    rows[-1] += 1
    y = combine(rows, p)
    assert torch.equal(y[-1].float(), (x[-1].float() * 2 + 1).to(torch.bfloat16).float())
    assert not y[:3].any() and not y[-2].any()
    del rows, y, x
    torch.cuda.empty_cache()


def test_differentiating_twice_is_refused():
    z = torch.randn(4, 5, device="cuda", requires_grad=True)
    w, ids = route(z, 2)
    p = expert_plan(ids, 5)
    y = combine(dispatch(torch.randn(4, 3, device="cuda", requires_grad=True), p), p, w)
    (dz,) = torch.autograd.grad(y.square().sum(), z, create_graph=True)
    assert torch.isfinite(dz).all()                      # the first gradient is there
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        dz.sum().backward()


def test_gradients_of_some_inputs_only():
    g = torch.Generator().manual_seed(4)
    p = expert_plan(torch.randint(0, 3, (20, 2), generator=g).int().cuda(), 3)
    h, w = torch.randn(40, 7, generator=g).cuda(), torch.rand(20, 2, generator=g).cuda()
    both = [t.clone().requires_grad_() for t in (h, w)]
    want = torch.autograd.grad(combine(both[0], p, both[1]).square().sum(), both)
    hr, wr = h.clone().requires_grad_(), w.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(combine(hr, p, w).square().sum(), hr)[0], want[0])
    assert torch.equal(torch.autograd.grad(combine(h, p, wr).square().sum(), wr)[0], want[1])
    with torch.no_grad():
        assert not combine(hr, p, wr).requires_grad and not dispatch(hr[:20], p).requires_grad
    leaf = h.clone().requires_grad_()                     # a gradient that is one value for all
    combine(leaf, p, w).sum().backward()
    assert torch.equal(leaf.grad, torch.autograd.grad(combine(hr, p, w), hr, torch.ones(20, 7, device="cuda"))[0])


def test_same_results_every_time_on_two_streams():
    g = torch.Generator().manual_seed(2)
    z, x = torch.randn(3000, 40, generator=g).cuda(), torch.randn(3000, 70, generator=g).cuda()

    def once():
        w, ids = route(z, 3)
        p = expert_plan(ids, 40, 200)
        return combine(dispatch(x, p), p, w), p.source
    first = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = [once() for _ in range(4)]
    here = [once() for _ in range(4)]
    torch.cuda.synchronize()
    for y, s in there + here:
        assert torch.equal(y, first[0]) and torch.equal(s, first[1])


class _Bf16Linear(torch.autograd.Function):
    """nn.Linear with the tower's operand rounding: bf16 operands in all three products, fp32 sums."""

    @staticmethod
    def forward(ctx, a, w, b):
        a, w = a.bfloat16().float(), w.bfloat16().float()
        ctx.save_for_backward(a, w)
        return a @ w.t() + b

    @staticmethod
    def backward(ctx, g):
        a, w = ctx.saved_tensors
        g = g.bfloat16().float()
        return g @ w, g.t() @ a, g.sum(0)


class _Routed(nn.Module):
    """A routed tower: every expert is a FusedLinearTower over its fixed-size slice of the rows."""

    def __init__(self, d, hidden, experts, k, capacity):
        super().__init__()
        from raydp_amd.ops.linear_ops import FusedLinearTower
        self.router = nn.Linear(d, experts)
        self.lins = nn.ModuleList(nn.Linear(a, b) for _ in range(experts) for a, b in ((d, hidden), (hidden, d)))
        self.out = nn.Linear(d, 1)
        self.k, self.experts, self.capacity = k, experts, capacity
        self.towers = [FusedLinearTower([self.lins[2 * e], self.lins[2 * e + 1]], [True, False]) for e in range(experts)]

    def forward(self, x, fused=True):
        z = self.router(x)
        if fused:
            w, ids = route(z, self.k)
            p = expert_plan(ids, self.experts, self.capacity)
            rows = dispatch(x, p).view(self.experts, self.capacity, -1)
            h = torch.stack([t(rows[e]) for e, t in enumerate(self.towers)]).view(p.rows, -1)
            return self.out(x + combine(h, p, w))
        top, ids = torch.topk(z, self.k, dim=1)
        w = torch.softmax(top, 1)
        y = x
        for e in range(self.experts):
            up, down = self.lins[2 * e], self.lins[2 * e + 1]
            h = _Bf16Linear.apply(torch.relu(_Bf16Linear.apply(x, up.weight, up.bias)), down.weight, down.bias)
            y = y + h * (w * (ids == e)).sum(1, keepdim=True)
        return self.out(y)


def _routed_step(model, opt, x, target):
    loss = nn.functional.binary_cross_entropy_with_logits(model(x), target)
    opt.zero_grad(set_to_none=True)
    loss.backward()
    opt.step()
    return loss.detach()


def test_a_training_step_of_a_routed_tower():
    """route -> dispatch -> expert towers -> combine -> loss -> clipped 8-bit AdamW, as a training loop runs them: gradients
    against the dense computation of all experts, then steps, eager and captured, that give the same bits."""
    from raydp_amd.ops.fused_optim import FusedAdamW
    torch.manual_seed(0)
    model = _Routed(48, 64, 4, 2, 256).cuda()
    x, target = torch.randn(256, 48, device="cuda"), torch.rand(256, 1, device="cuda").round()
    params = list(model.parameters())
    got = torch.autograd.grad(nn.functional.binary_cross_entropy_with_logits(model(x), target), params)
    want = torch.autograd.grad(nn.functional.binary_cross_entropy_with_logits(model(x, fused=False), target), params)
    for p, a, b in zip(params, got, want):
        # the same operands, rounded alike: what differs is the order of fp32 sums and, by that, a bf16 rounding here and
        # there, of one element by one step
        assert float((a - b).norm()) <= 2.0 ** -8 * float(b.norm()) + 1e-6, tuple(p.shape)
    import copy
    twin = copy.deepcopy(model)
    from raydp_amd.ops.linear_ops import FusedLinearTower
    twin.towers = [FusedLinearTower([twin.lins[2 * e], twin.lins[2 * e + 1]], [True, False]) for e in range(4)]
    oa = FusedAdamW(model.parameters(), lr=1e-3, max_grad_norm=0.05)
    ob = FusedAdamW(twin.parameters(), lr=1e-3, max_grad_norm=0.05)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _routed_step(model, oa, x, target)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):
        lb = _routed_step(twin, ob, x, target)
    oa.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        la = _routed_step(model, oa, x, target)
    for k in range(4):
        new = torch.randn(256, 48, device="cuda")
        x.copy_(new)
        graph.replay()
        lb = _routed_step(twin, ob, new, target)
        torch.cuda.synchronize()
        assert float(la) == float(lb), k
        for a, b in zip(model.parameters(), twin.parameters()):
            assert torch.equal(a, b), k
    del graph


def test_parts_of_a_plan_are_tensors_of_their_own():
    """Writing into the loads between forward and backward is no change of what backward reads."""
    x = torch.randn(20, 6, device="cuda", requires_grad=True)
    p = expert_plan(torch.arange(40, device="cuda").view(20, 2) % 3, 3, 10)
    y = combine(dispatch(x, p), p)
    p.load.clamp_(max=10)
    p.offsets.add_(1)
    (dx,) = torch.autograd.grad(y.sum(), x)
    assert torch.equal(dx, (p.position >= 0).sum(1, keepdim=True).float().expand(20, 6))
    y = combine(dispatch(x, p), p)
    p.position.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y.sum(), x)


@pytest.mark.parametrize("what", ["leaf", "result", "asked"])
def test_capturing_what_an_eager_call_made_is_refused(what):
    """Nodes of an eager call on the default stream cannot run in a capture: a leaf's gradient node that the call's result
    holds, an intermediate result's. Those of a side stream can."""
    x = torch.randn(20, 6, device="cuda", requires_grad=True)
    p = expert_plan(torch.arange(40, device="cuda").view(20, 2) % 3, 3)

    def once(leaf):
        y = combine(dispatch(leaf, p), p)
        if what == "asked":
            leaf.grad, = torch.autograd.grad(y.sum(), leaf)
        else:
            y.sum().backward()
        return y
    held = once(x)
    x.grad = None
    start = x * 1 if what == "result" else x
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(graph):
            once(start)
    assert x.grad is None
    z = x.detach().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        held = once(z)
    torch.cuda.current_stream().wait_stream(side)
    z.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = once(z)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(z.grad, torch.full_like(z, 2.0)) and torch.equal(y, held)
    del graph


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("E", [2, 4, 8, 9, 16, 32, 63, 64, 128, 256, 257, 511, 512, 513, 1024])
@pytest.mark.parametrize("most", [True, False])
def test_route_at_every_number_of_lanes(E, most, dtype):
    """Rows that fill their lanes and rows that do not, as many winners as there may be and fewer."""
    test_route_and_its_gradient(21, E, min(E, 32) if most else min(E, 5), not most, dtype)


class _PlainRouted(nn.Module):
    def __init__(self, capacity):
        super().__init__()
        self.router, self.out = nn.Linear(12, 4), nn.Linear(12, 1)
        self.experts = nn.ModuleList(nn.Linear(12, 12) for _ in range(4))
        self.capacity = capacity

    def forward(self, x):
        w, ids = route(self.router(x), 2)
        p = expert_plan(ids, 4, self.capacity)
        rows = dispatch(x, p).view(4, self.capacity, 12)
        h = torch.cat([torch.relu(e(rows[i])) for i, e in enumerate(self.experts)])
        return self.out(x + combine(h, p, w)).reshape(-1)


def test_a_routed_model_in_the_graphed_training_loop(monkeypatch):
    """TorchLoopEngine with the 8-bit optimizer: captured steps and eager ones end at the same bits."""
    from raydp_amd.ops.fused_optim import FusedAdamW
    from raydp_amd.torch.engine import TorchLoopEngine, _ShardTensors
    from raydp_amd.torch.metrics import TorchMetric
    from raydp_amd.train import session

    class Shard(_ShardTensors):
        def __init__(self, feats, labels):
            self.feats, self.labels, self.n, self.multi = [feats], labels, labels.shape[0], False
    g = torch.Generator().manual_seed(1)
    x, y = torch.randn(32 * 12 + 5, 12, generator=g).cuda(), torch.randn(32 * 12 + 5, generator=g).cuda()

    def trained(graphed):
        monkeypatch.setenv("RAYDP_TORCH_GRAPHS", "1" if graphed else "0")
        torch.manual_seed(0)
        model = _PlainRouted(48).cuda()
        opt = FusedAdamW(model.parameters(), lr=1e-2, max_grad_norm=1.0)
        session._set_session(session._Session(session.TrainContext(), {}, lambda *a: None, "/tmp"))
        try:
            e = TorchLoopEngine(model, opt, nn.MSELoss(), TorchMetric(["MeanAbsoluteError"]), torch.device("cuda:0"),
                                {"batch_size": 32, "shuffle": False, "drop_last": False}, None)
            e.train = e.eval = Shard(x, y)
            for _ in range(3):
                e.train_epoch()
        finally:
            session._set_session(None)
        assert (e.graphed is not None and e.graphed.failed is None and bool(e.graphed.graphs)) == graphed, e.graph_status
        return model
    a, b = trained(True), trained(False)
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q)


def test_a_routed_model_graphed_by_shape():
    """graph_model holds the forward and the backward in a graph; the losses that the loop keeps do not matter to it."""
    import copy
    from raydp_amd.train.gpu_policy import graph_model
    torch.manual_seed(0)
    ref = _PlainRouted(48).cuda()
    mine = copy.deepcopy(ref)
    graph_model(mine)
    g = torch.Generator().manual_seed(3)
    for i in range(8):
        x, y = torch.randn(32, 12, generator=g).cuda(), torch.randn(32, generator=g).cuda()
        kept = [nn.functional.mse_loss(m(x), y) for m in (ref, mine)]
        for loss, m in zip(kept, (ref, mine)):
            m.zero_grad()
            loss.backward()
        assert float(kept[0]) == float(kept[1])
        for p, q in zip(ref.parameters(), mine.parameters()):
            assert torch.equal(p.grad, q.grad), i
            with torch.no_grad():
                p -= 0.1 * p.grad
                q -= 0.1 * q.grad
