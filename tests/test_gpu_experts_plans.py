"""Plans whose tensors were put in by hand: what the row kernels read by address is looked at first."""
import pytest
import torch

from raydp_amd.ops.expert_ops import ExpertPlan, combine, dispatch, expert_plan

pytestmark = pytest.mark.gpu


def _with(**parts):
    p = expert_plan(torch.tensor([[0, 1], [1, 2], [2, 0]], dtype=torch.int32, device="cuda"), 3)
    for n, f in parts.items():
        setattr(p, n, f(getattr(p, n)))
    return p


@pytest.mark.parametrize("parts", [
    dict(position=lambda t: t.long()), dict(position=lambda t: t.t().contiguous().t()), dict(position=lambda t: t[:, :1].expand(3, 2)),
    dict(position=lambda t: t.repeat(2, 1)), dict(position=lambda t: t.flatten()), dict(position=lambda t: t.cpu()),
    dict(position=lambda t: t[:2]), dict(source=lambda t: t.long()), dict(source=lambda t: t[:1].expand(6)),
    dict(source=lambda t: t.repeat(2)), dict(source=lambda t: t[:3]), dict(source=lambda t: t.cpu()),
    dict(source=lambda t: t.view(3, 2))])
def test_a_plan_with_other_tensors_is_refused(parts):
    x, rows = torch.ones(3, 4, device="cuda"), torch.ones(6, 4, device="cuda")
    refused = 0
    for call in (lambda p: dispatch(x, p), lambda p: combine(rows, p), lambda p: combine(rows, p, torch.ones(3, 2, device="cuda"))):
        try:
            out = call(_with(**parts))
        except ValueError:
            refused += 1
        else:                    # what does not fit one of them may be another's own business
            assert out.shape[1] == 4
    assert refused >= 1
    assert dispatch(x, _with()).shape == (6, 4) and combine(rows, _with()).shape == (3, 4)


def test_a_plan_made_by_hand_is_taken():
    position = torch.tensor([[1], [0]], dtype=torch.int32, device="cuda")
    source = torch.tensor([1, 0, -1], dtype=torch.int32, device="cuda")
    load = torch.tensor([2], dtype=torch.int32, device="cuda")
    x = torch.arange(8.0, device="cuda").view(2, 4)
    rows = dispatch(x, ExpertPlan(position, source, load, load, 1, 3))
    assert torch.equal(rows, torch.stack([x[1], x[0], torch.zeros(4, device="cuda")]))
