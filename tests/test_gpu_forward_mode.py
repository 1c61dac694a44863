"""The vocabulary operators have no forward-mode derivatives, and say so instead of leaving a tangent out."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import sten_b200 as sten
from gpu_util import cuda

pytestmark = pytest.mark.gpu


def operands():
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(3, 50, device="cuda", generator=g)
    return x, torch.tensor([[4, 7]] * 3, device="cuda"), torch.log_softmax(x, -1)[:, :2].contiguous(), torch.ones(3, device="cuda")


@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("grad_mode", [False, True])
def test_dual_tensors_are_refused(recorded, grad_mode):
    x, ids, lp, w = operands()
    x.requires_grad_(recorded)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="token_log_probs has no forward-mode derivative"):
            sten.token_log_probs(dual, ids[:, 0], top=2)
        for reduction in ("mean", "none"):
            with pytest.raises(NotImplementedError, match="distillation_loss has no forward-mode derivative"):
                sten.distillation_loss(dual, ids, lp, reduction=reduction)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            sten.distillation_loss(x, ids, forward_ad.make_dual(lp, lp))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            sten.distillation_loss(x, ids, lp, weight=forward_ad.make_dual(w, w))


def test_tangents_of_upstream_gradients_are_refused():
    x, ids, lp, _ = operands()
    x.requires_grad_(True)
    for loss in (sten.token_log_probs(x).entropy.sum(), sten.distillation_loss(x, ids, lp), sten.distillation_loss(x, ids, lp, reduction="none").sum()):
        with forward_ad.dual_level():
            scale = forward_ad.make_dual(torch.ones((), device="cuda"), torch.ones((), device="cuda"))
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                torch.autograd.grad(loss * scale, x)


def test_plain_tensors_are_served_beside_dual_ones():
    x, ids, lp, w = operands()
    want = sten.token_log_probs(x, ids[:, 0]), sten.distillation_loss(x, ids, lp, weight=w)
    with forward_ad.dual_level():
        forward_ad.make_dual(x.clone(), torch.ones_like(x))
        got = sten.token_log_probs(x, ids[:, 0]), sten.distillation_loss(x, ids, lp, weight=w)
        assert torch.equal(got[0].log_prob, want[0].log_prob) and torch.equal(got[1], want[1])
        primal = forward_ad.unpack_dual(forward_ad.make_dual(x, torch.ones_like(x))).primal
        assert torch.equal(sten.token_log_probs(primal, ids[:, 0]).log_prob, want[0].log_prob)
