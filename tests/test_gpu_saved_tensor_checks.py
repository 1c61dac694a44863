"""The backward passes look at what came back of the saved tensors before the kernels get an address of it."""
import pytest
import torch
from torch.autograd.graph import saved_tensors_hooks

import sten_b200 as sten
from gpu_util import cuda

pytestmark = pytest.mark.gpu
CHANGES = {"on the host": lambda t: t.cpu(), "64 bits": lambda t: t.to(torch.int16 if t.dtype in (torch.int64, torch.int32) else torch.float64),
           "another shape": lambda t: torch.cat([t.reshape(-1), t.reshape(-1)[:1]])}


def losses():
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(3, 50, device="cuda", generator=g, requires_grad=True)
    lp, ids = torch.log_softmax(x.detach(), -1).topk(4, -1)
    w, t = torch.rand(3, device="cuda", generator=g) + 0.5, torch.arange(3, device="cuda")

    def token():
        o = sten.token_log_probs(x, t, top=3)
        return (o.log_prob + o.entropy + o.lse + o.top_log_prob.sum(-1)).sum()

    return x, {"token": (token, 5), "mean": (lambda: sten.distillation_loss(x, ids, lp, weight=w), 6),
               "none": (lambda: sten.distillation_loss(x, ids, lp, weight=w, reduction="none").sum(), 5)}


@pytest.mark.parametrize("change", CHANGES)
@pytest.mark.parametrize("name", ["token", "mean", "none"])
def test_changed_saved_tensors_are_refused(name, change):
    x, calls = losses()
    call, saved = calls[name]
    for which in range(saved):
        seen = []

        def pack(t):
            seen.append(t)
            return len(seen) - 1

        with saved_tensors_hooks(pack, lambda i: CHANGES[change](seen[i]) if i == which else seen[i]):
            loss = call()
        assert len(seen) >= saved
        with pytest.raises(RuntimeError, match="saved for the backward pass"):
            torch.autograd.grad(loss, x)


@pytest.mark.parametrize("name", ["token", "mean", "none"])
def test_logits_whose_data_was_replaced(name):
    x, calls = losses()
    loss = calls[name][0]()
    with torch.no_grad():
        held, x.data = x.data, x.data.cpu()
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, x)
    x.data = held
    assert bool(torch.isfinite(torch.autograd.grad(calls[name][0](), x)[0]).all())


def test_batched_gradients_are_refused():
    x, _ = losses()
    out = sten.token_log_probs(x).entropy
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, x, torch.eye(3, device="cuda"), is_grads_batched=True)
