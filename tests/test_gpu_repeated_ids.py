"""Teacher ids that occur more than once in a row: one token to the gradient and to the remainder, a term each in the loss."""
import math

import pytest
import torch

import sten_b200 as sten
from gpu_util import cuda

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("remainder", [False, True])
def test_repeated_ids_beside_their_sum(remainder):
    """Splitting a token's q in two halves changes neither the gradient nor what the loss depends on the logits by: the loss is lower by
    the entropy of the split, q ln 2.  Allowed: what two losses and two gradients may be off by (1e-4, and 1.4e-5 of S p plus the
    remainder's 1.2e-6)."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(6, 900, device="cuda", generator=g) * 2
    q = torch.tensor([0.5, 0.2, 0.1], device="cuda").repeat(6, 1)
    ids = torch.tensor([3, 10, 899], device="cuda").repeat(6, 1)
    halves = torch.cat([q[:, :1] / 2, q[:, 1:], q[:, :1] / 2], 1).log()
    twice = torch.cat([ids, ids[:, :1]], 1)
    total = 1.0 if remainder else 0.8
    got = {}
    for name, i, lp in (("once", ids, q.log()), ("twice", twice, halves)):
        y = x.clone().requires_grad_(True)
        loss = sten.distillation_loss(y, i, lp, remainder=remainder, reduction="none")
        got[name] = loss.detach().double(), torch.autograd.grad(loss.sum(), y)[0].double()
    assert float((got["once"][0] - got["twice"][0] - 0.5 / total * math.log(2)).abs().max()) <= 2e-4
    assert float((got["once"][1] - got["twice"][1]).abs().max()) <= 2 * (1.4e-5 + 1.2e-6)


def test_a_loss_below_zero():
    """Two entries of the only token that the student gives anything: -ln 2 in the loss, no gradient."""
    x = torch.full((1, 40), -float("inf"), device="cuda")
    x[0, 5] = 1.0
    x.requires_grad_(True)
    loss = sten.distillation_loss(x, torch.tensor([[5, 5]], device="cuda"), torch.zeros(1, 2, device="cuda"))
    [d] = torch.autograd.grad(loss, x)
    assert abs(float(loss.detach()) + math.log(2)) <= 1e-4 and float(d.abs().max()) <= 1.4e-5
