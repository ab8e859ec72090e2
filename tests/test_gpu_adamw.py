"""FusedAdamW (8- and 32-bit moments), clip_grad_norm_ and decode_moments on the GPU (csrc/hip/adamw.hip) against plain
implementations in 64 bits."""
import copy
import math

import pytest
import torch
import torch.nn as nn

from raydp_amd.ops.fused_optim import FusedAdamW, clip_grad_norm_, decode_moments

from adamw_oracle import Oracle, spacing

pytestmark = pytest.mark.gpu

# lengths around lanes (4), waves' scale blocks (256), workgroups (1024) and norm chunks (4096)
SHAPES = [(1,), (3,), (4,), (255,), (256,), (257,), (1023,), (1025,), (7, 11, 13), (4099,), (64, 513)]


def _make(shapes, dtype, seed, scale=1.0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    ps = [(torch.randn(s, generator=g) * 0.1).to(dtype).to(device).requires_grad_() for s in shapes]

    def grads():
        # elements of one tensor differ by orders of magnitude, some are exactly zero
        return [(torch.randn(s, generator=g) * torch.exp(2 * torch.randn(s, generator=g)) * scale *
                 (torch.rand(s, generator=g) > 0.05)).to(dtype).to(device) for s in shapes]
    return ps, grads


@pytest.fixture(params=[None, 0], ids=["cached", "streamed"])
def last_level(request):
    """Both sides of the bound from which kernels stream past the caches."""
    from raydp_amd.native import loader
    ext = loader.load_torch()
    old = ext.set_last_level(request.param) if request.param is not None else None
    yield
    if old is not None:
        ext.set_last_level(old)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cfg", [dict(lr=1e-3), dict(lr=1e-2, betas=(0.0, 0.5), eps=1e-6, weight_decay=0.1),
                                 dict(lr=3e-4, maximize=True, max_grad_norm=0.5, seed=77),
                                 dict(lr=1e-3, betas=(0.95, 0.0), weight_decay=0.0, max_grad_norm=1e9)])
def test_one_step_from_any_state_matches_the_definition(bits, dtype, cfg, last_level):
    """One step after another: the oracle takes the kernel's own state before each step, so that a rounding of one step is
    not carried into the next comparison."""
    params, grads = _make(SHAPES, dtype, 3)
    opt = FusedAdamW(params, state_bits=bits, **cfg)
    for step in range(1, 5):
        before = [p.detach().double().cpu() for p in params]
        oracle = Oracle.of(opt, params, bits)
        gs = grads()
        for p, g in zip(params, gs):
            p.grad = g
        opt.step()
        oracle.step([g.double().cpu() for g in gs], **cfg)
        if cfg.get("max_grad_norm") is not None:
            assert abs(float(opt.grad_norm) - oracle.norm) <= 2 ** -24 * oracle.norm
        for i, p in enumerate(params):
            got, want = p.detach().double().cpu(), oracle.p[i]
            if dtype == torch.float32:
                # decay, its product and the sum: three roundings of p. The update before anything cancels in it, in units
                # of 2^-24: m 8 (below), v half of its 9, square root and reciprocal 2 each (1 ulp), their two constants,
                # sum, quotient and product 5: 21.5, under 32
                tol = 3 * 2 ** -24 * (want.abs() + before[i].abs()) + 2 ** -19 * oracle.upd_terms[i]
                assert ((got - want).abs() <= tol + 1e-30).all(), (i, step)
            else:
                # dithered to bf16: one of the two neighbours; the same one but where 32 bits round over the border
                assert ((got - want).abs() <= 2 ** -7 * want.abs() + 1e-30).all(), (i, step)
                assert (got != want).sum() <= 2 + 1e-3 * got.numel()
            st = opt.state[p]
            if bits == 8:
                m, v = (t.double().cpu() for t in decode_moments(st["exp_avg"], st["exp_avg_sq"], st["scales"]))
                for a, b, emin in ((m, oracle.m[i], -14), (v, oracle.v[i], -30)):
                    # one code's spacing where 32 bits round over the dithered border (2^-24 of 2^-20: about 1e-5 an element)
                    assert ((a - b).abs() <= torch.maximum(spacing(a, emin), spacing(b, emin))).all()
                    assert (a != b).sum() <= 2 + 1e-3 * a.numel()
            else:
                # in units of 2^-24 of the larger term of m: b1 and its product 2; clip factor, its product, 1 - b1 and
                # its product 4; the sum, at most twice the larger term, 2: 8. v, of itself: clip factor and product
                # (squared) 4, square, 1 - b2 and its product 3, the sum 1, and 1 over for second order: 9
                big = oracle.m_terms[i]
                assert ((st["exp_avg"].double().cpu() - oracle.m[i]).abs() <= 8 * 2 ** -24 * big + 1e-40).all()
                v = st["exp_avg_sq"].double().cpu()
                assert ((v - oracle.v[i]).abs() <= 9 * 2 ** -24 * oracle.v[i] + 1e-40).all()
            assert float(st["step"]) == step


def test_codes_equal_those_of_the_cpu_bit_for_bit():
    """Moments are separately rounded products and sums on both sides: without clipping every code, scale and (fp32 path)
    moment of several steps is the same."""
    for dtype in (torch.float32, torch.bfloat16):
        a, grads = _make(SHAPES, dtype, 5)
        b = [p.detach().cpu().clone().requires_grad_() for p in a]
        oa, ob = FusedAdamW(a, seed=9), FusedAdamW(b, seed=9)
        for _ in range(6):
            for p, q, g in zip(a, b, grads()):
                p.grad, q.grad = g, g.cpu()
            oa.step()
            ob.step()
        for p, q in zip(a, b):
            for n in ("exp_avg", "exp_avg_sq", "scales"):
                assert torch.equal(oa.state[p][n].cpu(), ob.state[q][n]), n
            diff = (p.detach().cpu().double() - q.detach().double()).abs()
            assert (diff <= 6 * 2 ** (-22 if dtype == torch.float32 else -7) * (q.detach().double().abs() + 1e-2)).all()


def test_unaligned_parameters_and_gradients_and_what_lies_between_them():
    """Parameters and gradients that are slices of one buffer at odd offsets, as in a gradient bucket: the same bits as on
    their own, and nothing outside the slices changes."""
    for dtype, bits in ((torch.float32, 8), (torch.bfloat16, 8), (torch.float32, 32)):
        lens, at = [5, 300, 1, 1027, 9001], [1, 9, 311, 315, 1345]
        flat = torch.randn(10400, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
        gflat = torch.randn(10400, generator=torch.Generator().manual_seed(2)).to(dtype).cuda()
        params = [nn.Parameter(flat[a:a + n]) for a, n in zip(at, lens)]
        alone = [nn.Parameter(flat[a:a + n].clone()) for a, n in zip(at, lens)]
        for ps in (params, alone):
            for p, a, n in zip(ps, at, lens):
                p.grad = gflat[a:a + n] if ps is params else gflat[a:a + n].clone()
        keep = flat.clone()
        o1, o2 = FusedAdamW(params, state_bits=bits), FusedAdamW(alone, state_bits=bits)
        for _ in range(3):
            o1.step()
            o2.step()
        for p, q in zip(params, alone):
            assert torch.equal(p.detach(), q.detach())
        inside = torch.zeros(10400, dtype=torch.bool, device="cuda")
        for a, n in zip(at, lens):
            inside[a:a + n] = True
        assert torch.equal(flat[~inside], keep[~inside])
        assert not torch.equal(flat[inside], keep[inside])


@pytest.mark.parametrize("count", [1, 64, 65, 300])
def test_any_number_of_tensors(count):
    """One launch takes 64 tensors, one preparation 256; both types mixed in one group, some without gradient, one empty."""
    g = torch.Generator().manual_seed(count)
    mk = [torch.randn(1 + 37 * (i % 9), generator=g).to(torch.bfloat16 if i % 3 == 1 else torch.float32) for i in range(count)]
    many = [t.clone().cuda().requires_grad_() for t in mk]
    if count > 1:
        many[1] = torch.zeros(0, device="cuda", requires_grad=True)
    cpu = [p.detach().cpu().clone().requires_grad_() for p in many]
    om, oc = FusedAdamW(many, max_grad_norm=2.0), FusedAdamW(cpu, max_grad_norm=2.0)
    for step in range(2):
        for i, (p, q) in enumerate(zip(many, cpu)):
            if i % 7 == 3 and step == 0:
                p.grad = q.grad = None       # its own step count starts later
                continue
            gr = torch.randn(p.shape, generator=g).to(p.dtype)
            p.grad, q.grad = gr.cuda(), gr
        om.step()
        oc.step()
    assert abs(float(om.grad_norm) - float(oc.grad_norm)) <= 2 ** -23 * float(oc.grad_norm)
    for i, (p, q) in enumerate(zip(many, cpu)):
        tol = 2 ** (-21 if p.dtype == torch.float32 else -7)
        assert ((p.detach().cpu().double() - q.detach().double()).abs() <= tol * (q.detach().double().abs() + 0.01)).all(), i
        if p.numel():
            assert float(om.state[p]["step"]) == float(oc.state[q]["step"]) == (1 if i % 7 == 3 else 2)


def test_groups_with_their_own_options_share_the_norm():
    """Groups of other moments' bits, rates, betas and decay; places count on over groups; one norm for all."""
    g = torch.Generator().manual_seed(12)
    shapes = [(300,), (5, 7), (2000,), (64,)]
    gpu = [torch.randn(s, generator=g).cuda().requires_grad_() for s in shapes]
    cpu = [p.detach().cpu().clone().requires_grad_() for p in gpu]

    def make(ps):
        return FusedAdamW([dict(params=ps[:2], lr=1e-2, state_bits=32, betas=(0.8, 0.99)),
                           dict(params=ps[2:], weight_decay=0.3, eps=1e-5, maximize=True)], max_grad_norm=1.5, seed=6)
    a, b = make(gpu), make(cpu)
    for _ in range(3):
        for p, q in zip(gpu, cpu):
            q.grad = torch.randn(p.shape, generator=g)
            p.grad = q.grad.cuda()
        a.step()
        b.step()
        assert abs(float(a.grad_norm) - float(b.grad_norm)) <= 2 ** -23 * float(b.grad_norm)
    for p, q in zip(gpu, cpu):
        for n in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(a.state[p][n].cpu(), b.state[q][n]), n
        assert ((p.detach().cpu() - q.detach()).abs() <= 2 ** -21 * (q.detach().abs() + 0.1)).all()
    extra = torch.ones(9, device="cuda", requires_grad=True)
    extra.grad = torch.ones(9, device="cuda")
    a.add_param_group(dict(params=[extra], max_grad_norm=1.5, seed=6))
    a.step()
    assert float(a.state[extra]["step"]) == 1 and float(a.state[gpu[0]]["step"]) == 4


def test_gradients_made_in_inference_mode_are_clipped():
    p = nn.Parameter(torch.zeros(700, device="cuda"))
    with torch.inference_mode():
        grad = torch.ones(700, device="cuda")
    with torch.inference_mode():
        norm = clip_grad_norm_([_With(grad)], 1.0)
    assert abs(float(norm) - math.sqrt(700)) < 1e-4 and abs(float(grad.norm()) - 1) < 1e-4
    p.grad = torch.ones(700, device="cuda")
    opt = FusedAdamW([p])
    with torch.inference_mode():
        opt.step()
    assert float(opt.state[p]["step"]) == 1


class _With:
    def __init__(self, grad):
        self.grad = grad


def test_a_left_out_step_leaves_a_towers_image_right():
    from raydp_amd.ops.linear_ops import FusedLinearTower
    lin = nn.Linear(40, 24).cuda()
    tower = FusedLinearTower([lin], [False])              # no forward yet: no image
    opt = FusedAdamW(lin.parameters(), max_grad_norm=1.0)
    for p in lin.parameters():
        p.grad = torch.full_like(p, math.inf)
    opt.step()
    x = torch.randn(9, 40, device="cuda")
    assert torch.equal(tower(x), FusedLinearTower([lin], [False])(x))
    with torch.no_grad():
        lin.weight.mul_(2.0)                              # changed behind the optimizer
    opt.step()
    assert torch.equal(tower(x), FusedLinearTower([lin], [False])(x))


def test_blocks_of_zeros_tiny_and_huge_values():
    """All-zero blocks stay zero and divide by eps only; magnitudes at both ends of fp32 keep finite, sensible moments; a
    second moment that is not zero is never stored as zero."""
    n = 256 * 6
    p = torch.ones(n, device="cuda", requires_grad=True)
    g = torch.zeros(n)
    g[256:512] = 1e-18 * torch.randn(256, generator=torch.Generator().manual_seed(0))
    g[512:768] = 1e15 * torch.randn(256, generator=torch.Generator().manual_seed(1))
    g[768:1024] = torch.logspace(-12, 3, 256)
    g[1024] = 1.0
    p.grad = g.cuda()
    opt = FusedAdamW([p], lr=1e-3, weight_decay=0.0)
    opt.step()
    st = opt.state[p]
    m, v = decode_moments(st["exp_avg"], st["exp_avg_sq"], st["scales"])
    assert torch.isfinite(p).all() and torch.isfinite(m).all() and torch.isfinite(v).all()
    assert (m[:256] == 0).all() and (v[:256] == 0).all() and (p[:256] == 1).all() and (st["scales"][0] == 0).all()
    v32 = (g.cuda() * g.cuda() * (1 - 0.999))
    assert ((v > 0) == (v32 > 0)).all()
    big = v[768:1024].max()
    assert abs(float(big) / (0.001 * 1e6) - 1) <= 0.126


def test_non_finite_values_show_in_their_block_and_a_clipped_step_is_left_out():
    p = torch.ones(600, device="cuda", requires_grad=True)
    g = torch.full((600,), 0.1, device="cuda")
    g[300], g[5] = math.nan, math.inf
    p.grad = g
    opt = FusedAdamW([p])
    opt.step()
    m, v = decode_moments(opt.state[p]["exp_avg"], opt.state[p]["exp_avg_sq"], opt.state[p]["scales"])
    assert torch.isnan(m[:512]).all() and torch.isnan(v[:512]).all() and torch.isfinite(m[512:]).all()
    bad = torch.isnan(p.detach())
    assert bad[300] and bad[5] and bad.sum() == 2          # the step itself: where the gradient was not finite
    opt.step()
    assert torch.isnan(p.detach()[:512]).all() and torch.isfinite(p.detach()[512:]).all()
    for bits in (8, 32):
        for poison in (math.nan, math.inf):
            q = torch.ones(600, device="cuda", requires_grad=True)
            o = FusedAdamW([q], state_bits=bits, max_grad_norm=1.0)
            q.grad = torch.full((600,), 0.1, device="cuda")
            o.step()
            keep = q.detach().clone(), {k: t.clone() for k, t in o.state[q].items()}
            q.grad[599] = poison
            o.step()
            assert not math.isfinite(float(o.grad_norm))
            assert torch.equal(q.detach(), keep[0])
            for k, t in keep[1].items():
                assert torch.equal(o.state[q][k], t), k


def test_weights_of_a_fused_tower_get_their_image():
    from raydp_amd.ops.linear_ops import FusedLinearTower
    torch.manual_seed(0)
    lins = [nn.Linear(63, 129).cuda(), nn.Linear(129, 5).cuda()]
    tower = FusedLinearTower(lins, [True, False])
    x = torch.randn(77, 63, device="cuda")
    opt = FusedAdamW([p for lin in lins for p in lin.parameters()], lr=1e-2)
    for _ in range(2):
        opt.zero_grad()
        tower(x).square().mean().backward()
        opt.step()
    for li, lin in enumerate(lins):
        assert torch.equal(tower.images[li], lin.weight.detach().to(torch.bfloat16))
    assert torch.equal(tower(x), FusedLinearTower(lins, [True, False])(x))


def test_state_dict_round_trip_and_a_torch_adamw_state():
    p, grads = _make([(300, 3), (5,)], torch.bfloat16, 4)
    opt = FusedAdamW(p, lr=1e-2, max_grad_norm=3.0, seed=5)
    for g in (grads(), grads()):
        for a, b in zip(p, g):
            a.grad = b
        opt.step()
    q = [t.detach().clone().requires_grad_() for t in p]
    again = FusedAdamW(q, lr=1.0)
    again.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert again.param_groups[0]["max_grad_norm"] == 3.0 and again.param_groups[0]["seed"] == 5
    g = grads()
    for a, b, gr in zip(p, q, g):
        a.grad, b.grad = gr, gr.clone()
    opt.step()
    again.step()
    for a, b in zip(p, q):
        assert torch.equal(a.detach(), b.detach())
        for n, t in opt.state[a].items():
            assert again.state[b][n].dtype == t.dtype and torch.equal(again.state[b][n], t), n
    # fp32 moments of torch's AdamW are coded: within half a code's spacing (1/16), never a positive v to 0
    r = [t.detach().float().requires_grad_() for t in p]
    ref = torch.optim.AdamW(r, lr=1e-2)
    for a, gr in zip(r, g):
        a.grad = gr.float()
    ref.step()
    mine = FusedAdamW([t.detach().clone().requires_grad_() for t in r])
    mine.load_state_dict(ref.state_dict())
    for a, b in zip(r, mine.param_groups[0]["params"]):
        st = mine.state[b]
        m, v = decode_moments(st["exp_avg"], st["exp_avg_sq"], st["scales"])
        top_m, top_v = ref.state[a]["exp_avg"].abs().max(), ref.state[a]["exp_avg_sq"].max()
        assert ((m - ref.state[a]["exp_avg"]).abs() <= ref.state[a]["exp_avg"].abs() / 16 + top_m * 2 ** -17).all()
        assert ((v - ref.state[a]["exp_avg_sq"]).abs() <= ref.state[a]["exp_avg_sq"] / 16 + top_v * 2 ** -32).all()
        assert float(st["step"]) == 1


def test_captured_step_follows_eager_ones():
    """A captured step (norm, preparation, step) replayed between eager steps of a twin: the same bits every time, also with
    a learning rate that changes on the device."""
    p, grads = _make([(1000,), (3, 257)], torch.float32, 6)
    q = [t.detach().clone().requires_grad_() for t in p]
    lr = torch.tensor(1e-3, device="cuda")
    # (the twin's number is the tensor's value: 1e-3 itself is 4.7e-8 of it away from it)
    oa, ob = FusedAdamW(p, lr=lr, max_grad_norm=0.7), FusedAdamW(q, lr=float(lr), max_grad_norm=0.7)
    static = grads()
    for a, b, g in zip(p, q, static):
        a.grad, b.grad = g, g.clone()
    oa.step()
    ob.step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        oa.step()
    for k in range(4):
        new = grads()
        for s, b, g in zip(static, q, new):
            s.copy_(g)
            b.grad = g
        lr.fill_(1e-3 / (k + 1))
        ob.param_groups[0]["lr"] = float(torch.tensor(1e-3 / (k + 1), dtype=torch.float32))
        graph.replay()
        ob.step()
        torch.cuda.synchronize()
        assert float(oa.grad_norm) == float(ob.grad_norm)
        for a, b in zip(p, q):
            assert torch.equal(a.detach(), b.detach()), k
            for n, t in ob.state[b].items():
                assert torch.equal(oa.state[a][n], t), (k, n)
    del graph


def test_first_step_inside_a_capture_is_refused():
    p = torch.ones(300, device="cuda", requires_grad=True)
    p.grad = torch.ones(300, device="cuda")
    opt = FusedAdamW([p])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            opt.step()
    torch.cuda.synchronize()
    opt.step()
    assert float(opt.state[p]["step"]) == 1


def test_another_stream_and_a_gradient_in_another_order():
    p = torch.randn(64, 48, device="cuda").requires_grad_()
    q = p.detach().clone().requires_grad_()
    g = torch.randn(48, 64, device="cuda")
    q.grad = g.t().contiguous()
    p.grad = g.t()                    # not contiguous
    a, b = FusedAdamW([p], max_grad_norm=1.0), FusedAdamW([q], max_grad_norm=1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step()
    torch.cuda.current_stream().wait_stream(side)
    b.step()
    assert torch.equal(p.detach(), q.detach())


@pytest.mark.parametrize("limit", [0.0, 0.01, 1e6, math.inf])
def test_clip_grad_norm_matches_its_definition(limit, last_level):
    """Over both types, odd offsets, an order of dimensions that is not C's, and more tensors than one launch takes."""
    gen = torch.Generator().manual_seed(8)
    flat = torch.randn(40000, generator=gen).cuda()
    gs = [flat[1:4098], flat[5000:5001], flat[6001:20000], torch.randn(33, 65, generator=gen).cuda().t()]
    gs += [torch.randn(1 + 19 * (i % 50), generator=gen).to(torch.bfloat16 if i % 2 else torch.float32).cuda() for i in range(140)]
    params = []
    for g in gs:
        p = nn.Parameter(torch.empty_like(g))
        p.grad = g
        params.append(p)
    params += [params[3], nn.Parameter(torch.zeros(3, device="cuda"))]       # listed twice; without a gradient
    outside = flat.clone()
    before = [g.double().cpu() for g in gs]
    want = math.sqrt(sum(float(b.square().sum()) for b in before))
    norm = clip_grad_norm_(iter(params), limit)
    assert abs(float(norm) - want) <= 2 ** -24 * want and norm.dtype == torch.float32 and norm.dim() == 0
    f = min(1.0, limit / (want + 1e-6))
    for g, b in zip(gs, before):
        eps = 2 ** -8 if g.dtype == torch.bfloat16 else 2 ** -24
        # the factor's rounding, the product's, and for bf16 the last one
        assert ((g.double().cpu() - b * f).abs() <= (eps + 2 * 2 ** -24) * (b * f).abs()).all()
        if f == 1.0:
            assert torch.equal(g.double().cpu(), b)
    same = torch.ones(40000, dtype=torch.bool, device="cuda")
    for s in (slice(1, 4098), slice(5000, 5001), slice(6001, 20000)):
        same[s] = False
    assert torch.equal(flat[same], outside[same])


def test_clip_of_non_finite_gradients_and_in_a_graph():
    p = nn.Parameter(torch.ones(5000, device="cuda"))
    p.grad = torch.ones(5000, device="cuda")
    p.grad[17] = math.inf
    assert float(clip_grad_norm_([p], 1.0)) == math.inf
    p.grad = torch.ones(5000, device="cuda")
    p.grad[17] = math.nan
    assert math.isnan(float(clip_grad_norm_([p], 1.0))) and torch.isnan(p.grad).all()
    p.grad = torch.ones(5000, device="cuda")
    graph = torch.cuda.CUDAGraph()
    clip_grad_norm_([p], 1.0)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_([p], 1.0)
    for k in range(3):
        p.grad.fill_(k + 1.0)
        graph.replay()
        torch.cuda.synchronize()
        want = (k + 1.0) * math.sqrt(5000)
        assert abs(float(norm) - want) <= 2 ** -23 * want
        torch.testing.assert_close(p.grad, torch.full_like(p.grad, 1 / math.sqrt(5000)), rtol=1e-6, atol=0)
    del graph


def _loop(sched, graphed, bits, monkeypatch):
    """Three epochs of the torch-loop engine on a small MLP with FusedAdamW."""
    from raydp_amd.torch.engine import TorchLoopEngine, _ShardTensors
    from raydp_amd.torch.metrics import TorchMetric
    from raydp_amd.train import session

    class Shard(_ShardTensors):
        def __init__(self, feats, labels):
            self.feats, self.labels, self.n, self.multi = [feats], labels, labels.shape[0], False
    monkeypatch.setenv("RAYDP_TORCH_GRAPHS", "1" if graphed else "0")
    session._set_session(session._Session(session.TrainContext(), {}, lambda *a: None, "/tmp"))
    try:
        torch.manual_seed(0)
        dev = torch.device("cuda:0")
        model = nn.Sequential(nn.Linear(12, 64), nn.ReLU(), nn.Linear(64, 1))
        lr = torch.tensor(1e-2, device=dev) if sched else 1e-2
        opt = FusedAdamW(model.parameters(), lr=lr, state_bits=bits, max_grad_norm=0.5)
        sch = torch.optim.lr_scheduler.StepLR(opt, step_size=3, gamma=0.5) if sched else None
        e = TorchLoopEngine(model, opt, nn.MSELoss(), TorchMetric(["MeanAbsoluteError"]), dev,
                            {"batch_size": 32, "shuffle": True, "drop_last": False}, sch)
        g = torch.Generator().manual_seed(1)
        e.train = Shard(torch.randn(32 * 21 + 9, 12, generator=g).to(dev), torch.randn(32 * 21 + 9, 1, generator=g).to(dev))
        for _ in range(3):
            e.train_epoch()
        torch.cuda.synchronize()
        sd = {k: v.detach().cpu() for k, v in e.state_dict().items()}
        failed = e.graphed.failed if graphed else None
        assert (e.graphed is not None) == graphed and failed is None and (not graphed or e.graphed.graphs), (e.graph_status, failed)
        e.close()
        return sd, e.optimizer_state_dict()
    finally:
        session._set_session(None)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("sched", [False, True])
def test_the_engine_replays_it_in_its_graphs(sched, bits, monkeypatch):
    """TorchLoopEngine captures whole steps with FusedAdamW (also under a scheduler, whose rate the kernel reads on the
    device) and trains like its eager loop, bit for bit: step counts, dither and clip factor all live on the device."""
    a, oa = _loop(sched, True, bits, monkeypatch)
    b, ob = _loop(sched, False, bits, monkeypatch)
    for k in b:
        assert torch.equal(a[k], b[k]), k
    for i, st in ob["state"].items():
        for n, t in st.items():
            assert torch.equal(oa["state"][i][n], t), (i, n)


def test_it_steps_behind_the_horovod_wrapper():
    import raydp_amd.hvd as hvd
    torch.manual_seed(0)
    net = nn.Linear(20, 3).cuda()
    ref = copy.deepcopy(net)
    hvd.init()
    try:
        opt = hvd.DistributedOptimizer(FusedAdamW(net.parameters(), lr=1e-2))
        own = FusedAdamW(ref.parameters(), lr=1e-2)
        x = torch.randn(16, 20, device="cuda")
        for _ in range(3):
            for m, o in ((net, opt), (ref, own)):
                o.zero_grad()
                m(x).square().mean().backward()
                o.step()
    finally:
        hvd.shutdown()
    for a, b in zip(net.parameters(), ref.parameters()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("cls", [torch.optim.Adam, torch.optim.AdamW])
def test_a_fused_tower_sees_the_multi_tensor_adam_step(cls):
    """torch's Adam / AdamW stepped by the kernel (hvd.DistributedOptimizer, GPU train workers): the tower's next forward
    reads the updated weights, not the bf16 images of the old ones."""
    from raydp_amd.ops.fused_optim import adam_step
    from raydp_amd.ops.linear_ops import FusedLinearTower
    torch.manual_seed(0)
    lins = [nn.Linear(32, 64).cuda(), nn.Linear(64, 8).cuda()]
    tower = FusedLinearTower(lins, [True, False])
    x = torch.randn(40, 32, device="cuda")
    opt = cls([p for lin in lins for p in lin.parameters()], lr=0.1)
    tower(x).square().mean().backward()
    adam_step(opt)
    assert torch.equal(tower(x), FusedLinearTower(lins, [True, False])(x))


@pytest.mark.parametrize("views", [((0, 8), (4, 12)), ((0, 8), (0, 8)), ((3, 4), (0, 12))])
def test_shared_memory_is_refused(views):
    """Two workgroups of one launch would race there."""
    flat = torch.ones(12, device="cuda")
    p, q = (nn.Parameter(torch.ones(b - a, device="cuda")) for a, b in views)
    p.grad, q.grad = (flat[a:b] for a, b in views)
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm_([p, q], 1.0)
    assert torch.equal(flat, torch.ones_like(flat))
    FusedAdamW([p, q]).step()                            # (a step only reads them)
    p, q = (nn.Parameter(flat[a:b]) for a, b in views)
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    with pytest.raises(ValueError, match="share memory"):
        FusedAdamW([p, q]).step()
    assert torch.equal(flat, torch.ones_like(flat))


def test_neighbours_in_one_buffer_are_not_shared():
    flat = torch.ones(12, device="cuda")
    p, q = nn.Parameter(torch.ones(7, device="cuda")), nn.Parameter(torch.ones(5, device="cuda"))
    p.grad, q.grad = flat[5:], flat[:5]
    assert float(clip_grad_norm_([p, q], 1e9)) == pytest.approx(math.sqrt(12.0), rel=2 ** -23)
    p, q = nn.Parameter(flat[5:]), nn.Parameter(flat[:5])
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    FusedAdamW([p, q]).step()
    assert bool((flat < 1).all())


@pytest.mark.parametrize("count", [255, 256, 257, 600])
def test_clip_over_several_launches(count, last_level):
    """Lengths around a chunk (8192) and of one element, types in turn."""
    gen = torch.Generator().manual_seed(count)
    params = []
    for i in range(count):
        n = (1, 8191, 8192, 8193, 37, 16384, 300)[i % 7]
        p = nn.Parameter(torch.empty(n, dtype=torch.bfloat16 if i % 3 == 1 else torch.float32, device="cuda"))
        p.grad = torch.randn(n, generator=gen).to(p.dtype).cuda()
        params.append(p)
    before = [p.grad.double() for p in params]
    want = math.sqrt(sum(float(b.square().sum()) for b in before))
    norm = clip_grad_norm_(params, want / 3)
    # 64-bit sums of 32-bit squares: what is seen is the last rounding, to 32 bits
    assert abs(float(norm) - want) <= (2 ** -24 + 2 ** -40) * want
    f = want / 3 / (want + 1e-6)
    for p, b in zip(params, before):
        eps = 2 ** -8 if p.dtype == torch.bfloat16 else 2 ** -24
        # the factor's rounding, the product's, and for bf16 the last one
        assert ((p.grad.double() - b * f).abs() <= (eps + 2 * 2 ** -24) * (b * f).abs()).all()
