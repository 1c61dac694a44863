"""Layer norm of more rows than are read directly (CTAs that stay, rows through rings in shared memory), at every cut and alignment; and the
operators between the products beside tensors that have no memory of their own."""
import pytest
import torch

import sten_b200 as sten
from gpu_util import cuda
from test_gpu_layer_norm import BF16, F16, F32, check, operands

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,param_dtype", [(F32, F32), (F16, F32), (F16, F16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("rows,width", [(6001, 33), (5003, 520), (5000, 1023), (2600, 1024), (1300, 2047), (700, 4100), (601, 8192), (601, 8191), (450, 10000)])
def test_many_rows(dtype, param_dtype, rows, width):
    check(*operands((rows, width), dtype, param_dtype, rows % 2 == 1, seed=width))


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("offset", [1, 3, 8])
def test_many_rows_at_other_addresses(dtype, offset):
    x, r, w, b, g, gs = operands((3000, 1040), dtype, F32, True)
    part = slice(offset, offset + 1016)
    check(x[:, part], r[:, 8:1024], w[part], b[:1016], g[:, :1016], gs[:, part])


def test_many_rows_of_odd_values():
    x, _, w, b, g, _ = operands((4000, 600), F32, F32, False)
    with torch.no_grad():
        x[100, 5], x[3999, 0], x[2000] = float("nan"), -float("inf"), 7.0
        y = sten.layer_norm(x, w, b)
    bad = torch.isnan(y).all(1)
    assert bad.nonzero().flatten().tolist() == [100, 3999] and torch.isfinite(y[~bad]).all() and torch.equal(y[2000], b)


def test_the_sum_that_is_returned_is_an_output_of_its_own():
    """Written to in place, it is missed by the backward pass, which says so."""
    x, r, w, b, g, gs = operands((10, 64), F32, F32, True)
    x.requires_grad_(True)
    y, h = sten.layer_norm(x, w, b, residual=r)
    with torch.no_grad():
        h.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, g)


def test_sparse_tensors_and_wrappers_are_refused():
    ids, x, u = torch.zeros(4, dtype=torch.int64, device="cuda"), torch.randn(4, 16, device="cuda"), torch.rand(4, device="cuda")
    for call in (lambda t: sten.layer_norm(t), lambda t: sten.embedding(ids, t), lambda t: sten.sample_tokens(t, u)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call(x.to_sparse())
    gnm = sten.GroupedNMTensor.from_dense(torch.randn(16, 16, device="cuda"), n=2, m=4, sparse_dim=0, group_size=2, group_dim=1)
    wrapped = sten.SparseTensorWrapper.wrapped_from_dense(gnm, torch.randn(16, 16, device="cuda"), None)
    for call in (lambda t: sten.layer_norm(t), lambda t: sten.embedding(ids, t), lambda t: sten.sample_tokens(t, u)):
        with pytest.raises(TypeError, match="dense"):
            call(wrapped)


def test_batched_calls_are_refused():
    x = torch.randn(3, 4, 16, device="cuda")
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: sten.layer_norm(t))(x)
    out = sten.layer_norm(x[0].requires_grad_(True))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out.sum(1), x[0], torch.eye(4, device="cuda"), is_grads_batched=True)
    again = sten.layer_norm(torch.randn(2, 8, device="cuda"))  # the interpreter is as it was
    assert bool(torch.isfinite(again).all())


def test_calls_on_two_streams_at_once():
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = [torch.randn(4000, 1024, device="cuda", generator=gen).half() for _ in range(2)]
    ids = [torch.randint(0, 3000, (9000,), device="cuda", generator=gen) for _ in range(2)]
    w = torch.randn(3000, 1024, device="cuda", generator=gen).half().requires_grad_(True)
    g = [torch.randn(9000, 1024, device="cuda", generator=gen).half() for _ in range(2)]
    u = torch.rand(4000, device="cuda", generator=gen)

    def work(i):
        [d] = torch.autograd.grad(sten.embedding(ids[i], w), w, g[i])
        return [sten.layer_norm(x[i]), d, sten.sample_tokens(x[i], u, top_p=0.9).tokens]
    want = [work(0), work(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = work(i)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))
