"""Tensors that have no memory of their own (those of torch.func's transforms, sparse ones) are refused by every operator of the host
extension, on whose way to the library the interpreter is released."""
import pytest
import torch

import sten_b200 as sten
from gpu_util import cuda
from sten_b200 import _native as nat
from sten_b200 import ops

pytestmark = pytest.mark.gpu


def operators():
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn(64, 96, device="cuda", generator=g)
    t = sten.GroupedNMTensor.from_dense(w, 2, 4, sparse_dim=0, group_size=4, group_dim=1)
    geo = (64, 96, 2, 4, 4)
    ids, lp = torch.tensor([[4, 7]] * 3, device="cuda"), torch.full((3, 2), -1.0, device="cuda")
    return {
        "token_log_probs": (lambda x: sten.token_log_probs(x, ids[:, 0], top=2).entropy, (3, 50)),
        "distillation_loss": (lambda x: sten.distillation_loss(x, ids, lp, reduction="none"), (3, 50)),
        "spmm": (lambda x: ops.spmm(t.val, t.idx, *geo, x), (3, 96)),
        "spmm_t": (lambda x: ops.spmm_t(t.val, t.idx, *geo, x), (3, 64)),
        "column_sum": (lambda x: nat.host().column_sum(x), (3, 64)),
        "sparsify": (lambda x: ops.sparsify(x, 2, 4, 4)[0], (1, 64, 96)),
        "gather": (lambda x: ops.gather_layout(x, t.idx, 2, 4, 4), (1, 64, 96)),
        "densify": (lambda x: ops.densify(x, t.idx, 1, *geo), tuple(t.val.shape)),
    }


NAMES = ["token_log_probs", "distillation_loss", "spmm", "spmm_t", "column_sum", "sparsify", "gather", "densify"]


@pytest.mark.parametrize("name", NAMES)
def test_function_transforms(name):
    call, shape = operators()[name]
    x = torch.randn(shape, device="cuda")
    want = call(x)
    for transformed in (lambda: torch.func.jvp(call, (x,), (x,)), lambda: torch.func.grad(lambda y: call(y).sum())(x), lambda: torch.func.vmap(call)(x[None])):
        with pytest.raises(RuntimeError):
            transformed()
    assert torch.equal(call(x), want)  # the interpreter and the library are as before


@pytest.mark.parametrize("name", NAMES)
def test_sparse_tensors(name):
    call, shape = operators()[name]
    for x in (torch.randn(shape, device="cuda").to_sparse(), torch.randn(shape[-2:], device="cuda").to_sparse_csr()):
        with pytest.raises((RuntimeError, ValueError)):
            call(x)
