"""The example that scores, prunes and distils a small model, and the operators' edges towards autograd."""
import os
import sys

import pytest
import torch

import sten_b200 as sten
from conftest import ROOT

pytestmark = pytest.mark.gpu


def test_distillation_recovers_what_pruning_cost():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import recover_sparse_model as example
    r = example.main(["--steps", "60", "--vocab", "2003", "--hidden", "128"])
    dense, sparse, distilled = (r[k][0] for k in ("dense", "sparse", "distilled"))
    assert dense > sparse and distilled > sparse  # pruning costs, distillation gives some of it back


def test_the_operators_are_differentiable_once():
    x = torch.randn(3, 50, device="cuda", requires_grad=True)
    ids, lp = torch.zeros(3, 1, dtype=torch.int64, device="cuda"), torch.zeros(3, 1, device="cuda")
    for loss in (sten.token_log_probs(x).entropy.sum(), sten.distillation_loss(x, ids, lp), sten.distillation_loss(x, ids, lp, reduction="none").sum()):
        [g] = torch.autograd.grad(loss, x, create_graph=True)  # the gradient itself can be had
        with pytest.raises(RuntimeError, match="once"):
            g.sum().backward()


def test_a_changed_input_is_noticed():
    x = torch.randn(3, 50, device="cuda", requires_grad=True)
    y = x * 1.0
    loss = sten.token_log_probs(y).entropy.sum()
    with torch.no_grad():
        y.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_gradients_reach_a_sparse_head():
    """Logits of a grouped n:m linear: the gradient of the loss through the sparse weight, against the dense weight's."""
    torch.manual_seed(1)
    lin = torch.nn.Linear(96, 1000).cuda()
    sb = sten.SparsityBuilder()
    sb.set_weight("weight", initial_sparsifier=sten.GroupedNMSparsifier(2, 4, 4), out_format=sten.GroupedNMTensor)
    sparse = sb.get_sparse_model(lin)
    x = torch.randn(4, 7, 96, device="cuda", requires_grad=True)
    teacher = sten.token_log_probs(torch.randn(4, 7, 1000, device="cuda"), top=5)
    [dx] = torch.autograd.grad(sten.distillation_loss(sparse(x), teacher.top_ids, teacher.top_log_prob), x)
    w = sparse.weight.wrapped_tensor.to_dense().double()
    x64 = x.detach().double().requires_grad_(True)
    logp = torch.log_softmax(x64 @ w.t() + sparse.bias.detach().double(), -1).gather(-1, teacher.top_ids)
    logq = torch.log_softmax(teacher.top_log_prob.double(), -1)
    [want] = torch.autograd.grad((logq.exp() * (logq - logp)).sum(-1).mean(), x64)
    assert float((dx.double() - want).norm() / want.norm()) < 2e-5  # two fp32 products of 96 and 1000 terms and the loss's own 1.4e-5
