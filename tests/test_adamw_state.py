"""FusedAdamW's coded state where values are not numbers, the states it loads, its options, and its norm (no GPU needed)."""
import math

import pytest
import torch
import torch.nn as nn

from raydp_amd.ops.fused_optim import FusedAdamW, decode_moments

# quiet NaNs of either sign: the plain ones, all bits set, and what a bf16 NaN of all bits widens to
NANS = [0x7FC00000, 0xFFC00000, 0x7FFFFFFF, 0xFFFFFFFF, 0x7FFF0000, 0xFFFF0000]


def _bits(word):
    return torch.tensor([word - (1 << 32) if word >> 31 else word], dtype=torch.int32).view(torch.float32)


@pytest.mark.parametrize("word", NANS, ids=hex)
def test_any_nan_in_a_gradient_shows_in_both_moments_of_its_block(word):
    p = torch.ones(600, requires_grad=True)
    p.grad = torch.full((600,), 0.1)
    opt = FusedAdamW([p])
    opt.step()
    p.grad[300:301] = _bits(word)
    assert torch.isnan(p.grad[300])
    opt.step()
    st = opt.state[p]
    for t in decode_moments(st["exp_avg"], st["exp_avg_sq"], st["scales"]):
        assert torch.isnan(t[256:512]).all() and torch.isfinite(t[:256]).all() and torch.isfinite(t[512:]).all()


@pytest.mark.parametrize("word", NANS, ids=hex)
def test_a_loaded_state_with_a_nan_in_either_moment(word):
    for name, which in (("exp_avg", 0), ("exp_avg_sq", 1)):
        p, q = (torch.ones(600, requires_grad=True) for _ in range(2))
        p.grad = torch.full((600,), 0.1)
        src, dst = torch.optim.AdamW([p]), FusedAdamW([q])
        src.step()
        src.state[p][name][300:301] = _bits(word)
        dst.load_state_dict(src.state_dict())
        st = dst.state[q]
        got = decode_moments(st["exp_avg"], st["exp_avg_sq"], st["scales"])
        assert torch.isnan(got[which][256:512]).all() and torch.isfinite(got[which][:256]).all()
        assert torch.isfinite(got[1 - which]).all()


def _state(cls, **kw):
    p = torch.ones(300, requires_grad=True)
    p.grad = torch.full((300,), 0.1)
    opt = cls([p], **kw)
    opt.step()
    return opt.state_dict()


@pytest.mark.parametrize("make,match", [
    (lambda: _state(torch.optim.AdamW, amsgrad=True), "amsgrad"),
    (lambda: _state(torch.optim.Adam, amsgrad=True), "amsgrad"),
    (lambda: _state(torch.optim.Adam, weight_decay=0.1), "weight_decay"), (lambda: _state(torch.optim.AdamW, eps=1e-40), "eps")])
def test_a_state_that_means_something_else_is_refused_and_changes_nothing(make, match):
    q = torch.ones(300, requires_grad=True)
    q.grad = torch.full((300,), 0.1)
    opt = FusedAdamW([q], lr=0.25)
    opt.step()
    before = {n: t.clone() for n, t in opt.state[q].items()}
    with pytest.raises(ValueError, match=match):
        opt.load_state_dict(make())
    assert opt.param_groups[0]["lr"] == 0.25 and all(torch.equal(opt.state[q][n], t) for n, t in before.items())


def test_an_adam_state_without_decay_is_taken():
    opt = FusedAdamW([torch.ones(300, requires_grad=True)], state_bits=32)
    want = _state(torch.optim.Adam, lr=0.5)
    opt.load_state_dict(want)
    (st,) = opt.state.values()
    assert opt.param_groups[0]["lr"] == 0.5 and torch.equal(st["exp_avg"], want["state"][0]["exp_avg"])


def test_an_incomplete_coded_state_is_refused():
    for name in ("scales", "step", "exp_avg", "exp_avg_sq"):
        sd = _state(FusedAdamW)
        del sd["state"][0][name]
        with pytest.raises(ValueError, match="FusedAdamW"):
            FusedAdamW([torch.ones(300, requires_grad=True)]).load_state_dict(sd)


def test_the_norm_of_a_step_without_gradients_is_not_the_last_ones():
    p = torch.ones(3, requires_grad=True)
    opt = FusedAdamW([dict(params=[]), dict(params=[p])], max_grad_norm=1.0)
    p.grad = torch.ones(3)
    opt.step()
    assert float(opt.grad_norm) == pytest.approx(math.sqrt(3.0), rel=2 ** -23)
    p.grad = None
    opt.step()
    assert float(opt.grad_norm) == 0.0


BAD = [dict(lr=-1.0), dict(lr=torch.ones(2)), dict(eps=-1.0), dict(eps=1e-40), dict(betas=(1.0, 0.9)), dict(betas=(0.9,)),
       dict(weight_decay=-1.0), dict(state_bits=16), dict(max_grad_norm=-1.0), dict(seed=-1)]


@pytest.mark.parametrize("bad", BAD, ids=lambda d: next(iter(d)))
def test_a_groups_own_options_are_checked_like_the_optimizers(bad):
    """(A denominator under 2^-126 has no quotient on the GPU: with eps = 1e-40 a gradient of 0 would give 0 * inf.)"""
    a, b = (torch.ones(4, requires_grad=True) for _ in range(2))
    with pytest.raises(ValueError, match="FusedAdamW"):
        FusedAdamW([a], **bad)
    with pytest.raises(ValueError, match="FusedAdamW"):
        FusedAdamW([dict(params=[a], **bad)])
    opt = FusedAdamW([a])
    with pytest.raises(ValueError, match="FusedAdamW"):
        opt.add_param_group(dict(params=[b], **bad))
    assert len(opt.param_groups) == 1


def test_state_bits_set_to_nothing_there_is():
    p = torch.ones(4, requires_grad=True)
    p.grad = torch.ones(4)
    opt = FusedAdamW([p])
    opt.param_groups[0]["state_bits"] = 16
    with pytest.raises(ValueError, match="state_bits"):
        opt.step()
    assert not opt.state[p] and (p == 1).all()
