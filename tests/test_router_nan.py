"""The router where logits are not numbers, on the CPU and the GPU."""
import math

import pytest
import torch

from raydp_amd.ops.expert_ops import route


def _nan_rows(device):
    z = torch.tensor([[1.0, math.nan, 2.0, 0.5, -math.inf], [1.0, 2.0, 3.0, 4.0, 0.0], [-math.inf, math.nan, 1.0, -math.inf, 0.0]])
    return z.to(device).requires_grad_()


@pytest.mark.parametrize("renorm", [True, False])
def test_a_rows_nan_shows_in_its_gradient(renorm):
    z = _nan_rows("cpu")
    w, ids = route(z, 3, renorm)
    (dz,) = torch.autograd.grad(w, z, torch.tensor([[1.0, 2.0, -1.0]] * 3))
    assert torch.isnan(w[0]).all() and torch.isnan(w[2]).all() and torch.isfinite(w[1]).all() and torch.isfinite(dz[1]).all()
    want = torch.zeros(3, 5, dtype=torch.bool)
    want[0], want[2] = True, True
    if renorm:                                # only what was chosen has a gradient
        want[0, 1] = want[0, 4] = want[2, 0] = want[2, 1] = want[2, 3] = False
    assert torch.equal(torch.isnan(dz), want)


@pytest.mark.gpu
@pytest.mark.parametrize("renorm", [True, False])
def test_the_kernels_say_the_same(renorm):
    """In units of 2^-24, with logits at most 4 apart: a weight is off by 8 (exponent's product and constant), 2 (exponential,
    1 ulp), 2 (sum) and 2 (quotient): 14. Its gradient p dw - p s has |dw|, |s| <= 2 and p <= 1: 2 (14 + 1) and 2 (14 + 17 + 1),
    under 100 a side, 200 between two."""
    out = []
    for device in ("cpu", "cuda"):
        z = _nan_rows(device)
        w, ids = route(z, 3, renorm)
        (dz,) = torch.autograd.grad(w, z, torch.tensor([[1.0, 2.0, -1.0]] * 3, device=device))
        out.append((w.detach().cpu(), ids.cpu(), dz.cpu()))
    assert torch.equal(out[0][1], out[1][1])
    for a, b in ((out[0][0], out[1][0]), (out[0][2], out[1][2])):
        torch.testing.assert_close(a, b, rtol=0, atol=200 * 2 ** -24, equal_nan=True)
