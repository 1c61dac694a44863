"""Gradients when the saved tensors come back from hooks (offloading to the host, a copy in another layout)."""
import pytest
import torch
from torch.autograd.graph import save_on_cpu, saved_tensors_hooks

import sten_b200 as sten
from gpu_util import cuda
from test_gpu_distillation import check, problem
from test_gpu_token_log_probs import DTYPES, check_backward, drawn_targets, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("remainder", [False, True])
@pytest.mark.parametrize("reduction,up", [("mean", 0.5), ("sum", 3.0), ("mean", 1.0), ("none", None)])
def test_distillation_offloaded(reduction, up, remainder, dtype):
    x, ids, lp, w = problem(36, 2051, 7, dtype, 5, weighted=True)
    full, ids, lp, w = x.view(4, 9, 2051), (ids % 1998).view(4, 9, 7), lp.view(4, 9, 7), w.view(4, 9)
    upstream = None if up is None else torch.tensor(up, device="cuda")
    with save_on_cpu():
        for y, i, l, v in ((full, ids, lp, w), (full[:, :-1], ids[:, 1:], lp[:, 1:], w[:, 1:]), (full[1:, 2:7, 5:2003], ids[1:, 2:7], lp[1:, 2:7], w[1:, 2:7]),
                           (full.transpose(0, 1), ids.transpose(0, 1), lp.transpose(0, 1), w.t())):
            check(y, i, l, remainder, v, 2.0, reduction, upstream)


def test_next_token_rows_offloaded():
    """Eight sequences of 512 without their last position: the rows of the gradient and of the logits that come back differ in pitch."""
    x, ids, lp, _ = problem(8 * 512, 500, 5, torch.bfloat16, 6)
    with save_on_cpu():
        check(x.view(8, 512, 500)[:, :-1], ids.view(8, 512, 5)[:, 1:], lp.view(8, 512, 5)[:, 1:], True, upstream=torch.tensor(0.5, device="cuda"))


@pytest.mark.parametrize("remainder", [False, True])
@pytest.mark.parametrize("up", [0.5, 1.0])
def test_logits_that_come_back_with_other_levels(up, remainder):
    """Three leading dimensions of which the last two are one level in one layout and the first two in the other."""
    x, ids, lp, _ = problem(2 * 3 * 5, 1003, 7, torch.float32, 5)
    y, ids, lp = x.view(2, 3, 5, 1003)[:, :, :4], ids.view(2, 3, 5, 7)[:, :, :4], lp.view(2, 3, 5, 7)[:, :, :4]

    def other(t):
        if t.shape != y.shape or t.dtype != y.dtype:
            return t
        z = torch.zeros(2, 4, 4, 1003, device="cuda")[:, :3]
        return z.copy_(t)

    with saved_tensors_hooks(lambda t: t, other):
        check(y, ids, lp, remainder, upstream=torch.tensor(up, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES)
def test_token_log_probs_offloaded(dtype):
    full = logits(36, 2051, dtype, 5).view(4, 9, 2051)
    tokens = drawn_targets(full)
    with save_on_cpu():
        for x, t in ((full[:, :-1], tokens[:, 1:]), (full[1:, 2:7, 5:2003], tokens[1:, 2:7] % 1998), (full.transpose(0, 1), tokens.t())):
            check_backward(x, t.clamp(max=x.shape[-1] - 1), top=6)


def test_checkpointed():
    from torch.utils.checkpoint import checkpoint
    x, ids, lp, _ = problem(36, 2051, 7, torch.float32, 5)
    full, ids, lp = x.view(4, 9, 2051), ids.view(4, 9, 7), lp.view(4, 9, 7)
    grads = []
    for run in (lambda f, y: f(y), lambda f, y: checkpoint(f, y, use_reentrant=False)):
        y = full.clone().requires_grad_(True)
        loss = run(lambda z: sten.distillation_loss((z * 1.0)[:, :-1], ids[:, :-1], lp[:, :-1], remainder=True), y) * 0.25
        grads.append(torch.autograd.grad(loss, y)[0])
    assert torch.equal(*grads)
