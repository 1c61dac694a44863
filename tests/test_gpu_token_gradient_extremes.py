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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1.0, 0.01])
@pytest.mark.parametrize("far", [False, True])
def test_large_entropy_gradients_beside_masked_logits(far, temperature, dtype):
    """As a loss scale makes them.  The gradient is linear in what comes in, and scaling by a power of two is exact but for what becomes
    subnormal: it is 2^34 times that of a gradient of 1, to the last bits of probabilities below 2^-100."""
    x = logits(4, 1003, dtype, 3)
    x[1, 500:] = -INF
    x[2, ::2] = torch.finfo(dtype).min
    x[3, 7:] = -INF
    if far:
        x = x + 2.0 ** 26  # beyond what the exponents take in one instruction; 16-bit and fp32 logits are then equal or masked
    x.requires_grad_(True)
    scale = 2.0 ** 34
    out = sten.token_log_probs(x, temperature=temperature).entropy
    [one] = torch.autograd.grad(out, x, torch.ones_like(out), retain_graph=True)
    [many] = torch.autograd.grad(out, x, torch.full_like(out, scale))
    assert bool(torch.isfinite(one).all()) and bool(torch.isfinite(many).all())
    assert float((many.double() - one.double() * scale).abs().max()) <= scale * 2.0 ** -90
    assert not many[1, 500:].any() and not many[2, ::2].any() and not many[3, 7:].any()
