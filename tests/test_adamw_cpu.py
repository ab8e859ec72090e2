"""FusedAdamW on the CPU against the oracle, its rounding in expectation, and what is refused (no GPU needed)."""
import math

import pytest
import torch
import torch.nn as nn

from adamw_oracle import Oracle, spacing
from raydp_amd.ops.fused_optim import FusedAdamW, clip_grad_norm_, decode_moments


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps_match_the_definition(bits, dtype):
    g = torch.Generator().manual_seed(1)
    params = [(torch.randn(s, generator=g) * 0.1).to(dtype).requires_grad_() for s in [(3,), (257,), (20, 31)]]
    cfg = dict(lr=1e-2, weight_decay=0.1, max_grad_norm=0.3, seed=4)
    opt = FusedAdamW(params, state_bits=bits, **cfg)
    for _ in range(3):
        oracle = Oracle.of(opt, params, bits)
        for p in params:
            p.grad = torch.randn(p.shape, generator=g).to(dtype)
        opt.step()
        oracle.step([p.grad.double() for p in params], **cfg)
        for i, p in enumerate(params):
            st = opt.state[p]
            m, v = decode_moments(st["exp_avg"], st["exp_avg_sq"], st["scales"]) if bits == 8 else (st["exp_avg"], st["exp_avg_sq"])
            for a, b, emin in ((m, oracle.m[i], -14), (v, oracle.v[i], -30)):
                if bits == 8:       # one code's spacing where 32 bits round over the dithered border
                    assert ((a.double() - b).abs() <= torch.maximum(spacing(a.double(), emin), spacing(b, emin))).all()
                    assert (a.double() != b).sum() <= 1 + 1e-3 * a.numel()
                else:               # 2^-24 each: clip factor, constants, products and the sum, 9 at most
                    assert ((a.double() - b).abs() <= 9 * 2.0 ** -24 * torch.maximum(b.abs(), oracle.m_terms[i])).all()
            tol = 2.0 ** -7 * oracle.p[i].abs() if dtype == torch.bfloat16 else \
                4 * 2.0 ** -24 * (oracle.p[i].abs() + 0.1) + 2.0 ** -19 * oracle.upd_terms[i]
            assert ((p.detach().double() - oracle.p[i]).abs() <= tol).all()


def test_the_stored_second_moment_moves_as_the_exact_one_does():
    """With 1 - b2 = 1e-3 a step changes v by far less than a code's spacing. Over 400 equal gradients from 0 the exact v
    grows to (1 - 0.999^400) g^2 = 0.3298 g^2; the mean of 4096 stored values has to follow. One rounding adds at most
    (spacing / 2)^2 = (v / 16)^2 of variance, 400 of them at most 400 / 256 v^2 for one element: 1.25 v / 64 = 2 % for the
    mean, taken four times."""
    p = torch.zeros(4096, requires_grad=True)
    p.grad = torch.full((4096,), 0.5)
    opt = FusedAdamW([p], lr=0.0)
    for _ in range(400):
        opt.step()
    st = opt.state[p]
    m, v = decode_moments(st["exp_avg"], st["exp_avg_sq"], st["scales"])
    want = (1 - 0.999 ** 400) * 0.25
    assert abs(float(v.mean()) / want - 1) <= 0.08
    assert abs(float(m.mean()) / 0.5 - 1) <= 0.08
    assert len(v.unique()) > 1


def test_a_step_whose_norm_is_not_finite_is_left_out():
    p = torch.ones(300, requires_grad=True)
    opt = FusedAdamW([p], max_grad_norm=1.0)
    p.grad = torch.ones(300)
    opt.step()
    keep, step = p.detach().clone(), float(opt.state[p]["step"])
    p.grad[7] = math.nan
    opt.step()
    assert torch.equal(p.detach(), keep) and float(opt.state[p]["step"]) == step


def test_clip_on_the_cpu():
    p, q = nn.Parameter(torch.zeros(3)), nn.Parameter(torch.zeros(2, dtype=torch.bfloat16))
    p.grad, q.grad = torch.tensor([3.0, 0.0, 0.0]), torch.tensor([0.0, 4.0], dtype=torch.bfloat16)
    assert float(clip_grad_norm_([p, q, p], 1.0)) == 5.0
    torch.testing.assert_close(p.grad, torch.tensor([0.6, 0.0, 0.0]))
    torch.testing.assert_close(q.grad.float(), torch.tensor([0.0, 0.8]), rtol=2 ** -8, atol=0)
    assert float(clip_grad_norm_([nn.Parameter(torch.zeros(3))], 1.0)) == 0.0


def test_state_dict_keeps_codes_and_options():
    p = torch.randn(300, dtype=torch.bfloat16, requires_grad=True)
    p.grad = torch.randn(300).to(torch.bfloat16)
    opt = FusedAdamW([p], lr=3e-3, max_grad_norm=2.0, seed=3)
    opt.step()
    q = p.detach().clone().requires_grad_()
    again = type(opt)([q], lr=0.1)            # as an estimator's worker does it
    again.load_state_dict(opt.state_dict())
    q.grad = p.grad.clone()
    opt.step()
    again.step()
    assert torch.equal(p.detach(), q.detach())
    for n, t in opt.state[p].items():
        assert again.state[q][n].dtype == t.dtype and torch.equal(again.state[q][n], t)
    import copy
    import pickle
    copy.deepcopy(again).step()
    pickle.loads(pickle.dumps(again)).step()


def test_refusals():
    p = torch.ones(4, requires_grad=True)
    for kw in (dict(lr=-1.0), dict(eps=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9,)), dict(weight_decay=-1.0),
               dict(state_bits=4), dict(max_grad_norm=-1.0), dict(seed=-1), dict(seed=1 << 32), dict(lr=torch.ones(2))):
        with pytest.raises(ValueError):
            FusedAdamW([p], **kw)
    with pytest.raises(TypeError, match="dtype"):
        FusedAdamW([torch.ones(4, dtype=torch.float64, requires_grad=True)])
    with pytest.raises(ValueError, match="twice"):
        FusedAdamW([p, p])
    e = nn.Embedding(4, 2, sparse=True)
    e(torch.tensor([1])).sum().backward()
    with pytest.raises(RuntimeError, match="sparse"):
        FusedAdamW(e.parameters()).step()
    with pytest.raises(ValueError, match="sparse"):
        clip_grad_norm_(e.parameters(), 1.0)
    t = torch.ones(4, 3).t().requires_grad_()
    t.grad = torch.ones(3, 4)
    with pytest.raises(ValueError, match="contiguous"):
        FusedAdamW([t]).step()
    a, b = torch.ones(4, requires_grad=True), torch.ones(4, requires_grad=True)
    a.grad, b.grad = torch.ones(4), torch.ones(4)
    with pytest.raises(ValueError, match="optimizer's"):
        FusedAdamW([dict(params=[a], max_grad_norm=1.0), dict(params=[b])]).step()
    opt = FusedAdamW([a])
    opt.step()
    opt.param_groups[0]["state_bits"] = 32
    with pytest.raises(ValueError, match="state_bits"):
        opt.step()
    for bad in (math.nan, -1.0):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm_([a], bad)
    d = nn.Parameter(torch.ones(4, dtype=torch.float64))
    d.grad = torch.ones(4, dtype=torch.float64)
    with pytest.raises(TypeError, match="dtype"):
        clip_grad_norm_([d], 1.0)
    x = nn.Parameter(torch.ones(4, 4))
    x.grad = torch.ones(4, 1).expand(4, 4)
    with pytest.raises(ValueError, match="dense"):
        clip_grad_norm_([x], 1.0)
    c = torch.zeros(300, dtype=torch.uint8)
    s = torch.zeros(2, 2, dtype=torch.uint8)
    for bad in ((c.float(), c, s), (c, c[:299], s), (c, c, s[:1]), (c[::2], c[::2], s[:1])):
        with pytest.raises(ValueError, match="decode_moments"):
            decode_moments(*bad)
    with pytest.raises(TypeError):
        decode_moments(c, c, s, torch.float16)


@pytest.mark.parametrize("views", [((0, 8), (4, 12)), ((0, 8), (0, 8)), ((3, 4), (0, 12))])
def test_shared_memory_is_refused(views):
    flat, (p, q) = torch.ones(12), (nn.Parameter(torch.ones(b - a)) for a, b in views)
    p.grad, q.grad = (flat[a:b] for a, b in views)
    with pytest.raises(ValueError, match="share memory"):
        clip_grad_norm_([p, q], 1.0)
    assert torch.equal(flat, torch.ones(12))
    FusedAdamW([p, q]).step()                            # (a step only reads them)
    p, q = (nn.Parameter(flat[a:b]) for a, b in views)
    p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    with pytest.raises(ValueError, match="share memory"):
        FusedAdamW([p, q]).step()
    assert torch.equal(flat, torch.ones(12))


def test_neighbours_in_one_buffer_are_not_shared():
    flat, p, q = torch.ones(12), nn.Parameter(torch.ones(7)), nn.Parameter(torch.ones(5))
    p.grad, q.grad = flat[5:], flat[:5]
    assert float(clip_grad_norm_([p, q], 1e9)) == pytest.approx(math.sqrt(12.0), rel=2 ** -23)
    p, q = nn.Parameter(flat[5:]), nn.Parameter(flat[:5])
    p.grad, q.grad = torch.ones(7), torch.ones(5)
    FusedAdamW([p, q]).step()
