"""Gradients of the token log-probabilities where the logits are masked and the gradients that come in are large or no numbers."""
import pytest
import torch

import sten_b200 as sten
from gpu_util import cuda
from test_gpu_token_log_probs import DTYPES, INF, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [INF, -INF, float("nan")])
@pytest.mark.parametrize("which", ["log_prob", "entropy", "lse", "top_log_prob"])
def test_a_row_without_a_token_has_no_gradient_whatever_comes_in(which, value, dtype):
    x = logits(3, 1003, dtype, 1)
    x[1] = -INF
    t = torch.tensor([5, 6, 7], device="cuda")
    x.requires_grad_(True)
    out = getattr(sten.token_log_probs(x, t, top=3), which)
    g = torch.ones_like(out)
    g[1] = value
    [d] = torch.autograd.grad(out, x, g)
    assert not d[1].any() and bool(torch.isfinite(d).all()) and bool(d[0].any()) and bool(d[2].any())


def test_no_such_token_in_a_row_without_a_token():
    x = torch.full((2, 1003), -INF, device="cuda", requires_grad=True)
    o = sten.token_log_probs(x, torch.tensor([1003, 4], device="cuda"))
    [d] = torch.autograd.grad(o.log_prob, x, torch.ones(2, device="cuda"))
    assert bool(torch.isnan(d[0]).all()) and not d[1].any()
