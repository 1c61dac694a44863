"""Distillation from kept log-probabilities against a plain implementation in 64 bits; its gradient against automatic
differentiation of that, and against differences.

Tolerances, per row and in units of tau^2 * weight.  log p and log q come from 32-bit sums of a relative error below 6e-6 and two
roundings of values below 64 each (1.4e-5 in all, as for the token log-probabilities); they are weighed with q, whose sum is 1, and
the sum over at most 256 kept tokens rounds 13 times (13 * 2^-24 * 40): below 5e-5.  The remainder 1 - sum q is off by at most 20
roundings of values up to 1 (1.2e-6) and is multiplied with logarithms of at most 40: 5e-5 more.  In the gradient probabilities have a
relative error of 1.4e-5, p_0 and r of twice that, and the remainder the absolute one above."""
import pytest
import torch

import sten_b200 as sten
from gpu_util import cuda

pytestmark = pytest.mark.gpu
INF = float("inf")
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF_ULP = {torch.float32: (2.0 ** -22, 2.0 ** -126), torch.float16: (2.0 ** -11 * 1.01, 2.0 ** -25), torch.bfloat16: (2.0 ** -8 * 1.01, 2.0 ** -126)}
LOSS = 1e-4


def problem(rows, vocab, kept, dtype, seed, scale=2.5, pad=False, weighted=False, temperature=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, vocab, device="cuda", generator=g) * scale).to(dtype)
    t = (x.float() * 0.8 + torch.randn(rows, vocab, device="cuda", generator=g)) / temperature
    lp, ids = torch.log_softmax(t, 1).topk(kept, 1)
    if pad:
        ids = ids.clone()
        ids[torch.rand(rows, kept, device="cuda", generator=g) < 0.3] = -1
    w = None
    if weighted:
        w = torch.rand(rows, device="cuda", generator=g) + 0.2
        w[::3] = 0
    return x, ids, lp, w


def parts(x, ids, lp, remainder, w, tau):
    """Row losses in 64 bits (differentiable), and the terms that the errors of the gradient are made of."""
    z = x / tau
    valid = ids >= 0
    at = ids.clamp(min=0).long()
    logq = lp.double().masked_fill(~valid, -INF)
    empty = (x == -INF).all(-1)
    z = torch.where(empty[..., None], 0.0, z)
    z = z - z.detach().amax(-1, keepdim=True)  # beside the lowest fp32 value even 64 bits have no room for a log-sum-exp
    lse = torch.logsumexp(z, -1, keepdim=True)
    hidden = torch.zeros(z.shape, dtype=torch.int32, device=z.device).scatter_add_(-1, at, valid.int()) > 0
    if remainder:
        some = torch.ones_like(empty)
        anything = ((z > -INF) & ~hidden).any(-1)
        log_p0 = torch.where(anything, torch.logsumexp(torch.where(hidden | ~anything[..., None], torch.where(anything[..., None], -INF, 0.0), z), -1) - lse[..., 0], 0.0)
        q0 = torch.where(anything, (1 - logq.exp().sum(-1)).clamp(min=0), 0.0)
        tail = torch.special.xlogy(q0, q0) - q0 * log_p0
    else:
        some = (logq > -INF).any(-1)
        logq = logq - torch.where(some, torch.logsumexp(logq, -1), 0.0)[..., None]
        log_p0, q0, tail = None, torch.zeros_like(lse[..., 0]), 0.0
    q = logq.exp()
    logp = z.gather(-1, at) - lse
    term = torch.where(q > 0, q * (logq.masked_fill(q == 0, 0.0) - logp.masked_fill(q == 0, 0.0)), 0.0)
    weight = torch.ones_like(lse[..., 0]) if w is None else w.double()
    counts = some & ~empty & (weight != 0)
    loss = torch.where(counts, tau * tau * weight * (term.sum(-1) + tail), 0.0)
    with torch.no_grad():
        p = (z - lse).exp()
        qj = torch.zeros_like(z).scatter_add_(-1, at, q)
        size = p + qj
        if remainder:
            r = torch.where(hidden, 0.0, (z - lse - log_p0[..., None]).exp()).nan_to_num(0.0)
            size = size + r * (log_p0.exp() + q0 + 0.05)[..., None]
    return loss, weight, counts, size


def check(x, ids, lp, remainder=False, w=None, tau=1.0, reduction="mean", upstream=None):
    xr = x.detach().requires_grad_(True)
    x64 = x.detach().double().requires_grad_(True)
    got = sten.distillation_loss(xr, ids, lp, remainder=remainder, weight=w, temperature=tau, reduction=reduction)
    rows, weight, counts, size = parts(x64, ids, lp, remainder, w, tau)
    total = float(weight.sum()) if reduction == "mean" else 1.0
    unit = tau * tau * weight * counts
    if reduction == "none":
        want, allowed = rows, LOSS * unit
        upstream = torch.linspace(-1, 2, rows.numel(), device="cuda").view(rows.shape) if upstream is None else upstream
    else:
        want, allowed = rows.sum() / total if total else rows.sum() * 0, LOSS * unit.sum() / (total or 1.0)
    assert got.shape == want.shape and got.dtype == torch.float32
    plain = sten.distillation_loss(x, ids, lp, remainder=remainder, weight=w, temperature=tau, reduction=reduction)
    finite = torch.isfinite(want.detach())
    assert torch.equal(got.detach().double()[~finite], want.detach()[~finite]) and torch.equal(plain.double()[~finite], want.detach()[~finite])
    for value in (got.detach(), plain):  # with and without a gradient rows may be cut and added differently
        assert float(((value.double() - want.detach())[finite].abs() - allowed.expand_as(want)[finite] - 2.0 ** -22 * want.detach()[finite].abs()).max() if finite.any() else -1) <= 0
    [d] = torch.autograd.grad(got, xr, upstream)
    up = (torch.ones((), device="cuda") if upstream is None else upstream).double()
    [want_d] = torch.autograd.grad(want, x64, up)
    want_d = torch.where((counts & bool(total))[..., None], want_d, 0.0)
    rel, tiny = HALF_ULP[x.dtype]
    scale = (tau * weight / (total or 1.0) * (up if reduction == "none" else up.expand_as(weight))).abs() * counts
    off = (d.double() - want_d).abs() - rel * want_d.abs() - tiny - 6e-5 * scale[..., None] * size
    assert float(off.max()) <= 0, f"gradient off by {float(off.max())} more than allowed"
    assert d.dtype == x.dtype
    return got, d


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("remainder", [False, True])
@pytest.mark.parametrize("rows,vocab,kept", [(1, 2, 1), (3, 9, 2), (2, 40, 33), (5, 33, 8), (33, 511, 16), (1, 4099, 32), (300, 4107, 5), (700, 1023, 64), (2, 30522, 8),
                                             (1, 131072, 256), (40, 70001, 100), (310, 33333, 17)])
def test_loss_and_gradient(rows, vocab, kept, remainder, dtype):
    x, ids, lp, w = problem(rows, vocab, kept, dtype, rows + vocab + kept)
    check(x, ids, lp, remainder)


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("remainder", [False, True])
@pytest.mark.parametrize("tau", [0.5, 1.0, 3.0])
def test_reductions_weights_padding(reduction, remainder, tau):
    for rows, vocab in ((7, 2003), (400, 1500)):
        x, ids, lp, w = problem(rows, vocab, 13, torch.float32, rows, pad=True, weighted=True, temperature=tau)
        check(x, ids, lp, remainder, w, tau, reduction)
        check(x, ids.int(), lp.half(), remainder, None, tau, reduction)
        check(x, ids, lp.bfloat16(), remainder, torch.zeros_like(w), tau, reduction)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("remainder", [False, True])
def test_upstream_other_than_one(remainder, dtype):
    x, ids, lp, w = problem(20, 3001, 9, dtype, 3, weighted=True)
    for up in (1.0, 0.25, -3.0, 1024.0, 0.0):
        check(x, ids, lp, remainder, w, 2.0, "mean", torch.tensor(up, device="cuda"))


def test_gradients_of_scaled_losses_are_rounded_once():
    x, ids, lp, _ = problem(512, 4099, 9, torch.float16, 3)
    xr = x.requires_grad_(True)
    [d] = torch.autograd.grad(sten.distillation_loss(xr, ids, lp) * 65536.0, xr)
    x64 = x.detach().double().requires_grad_(True)
    [want] = torch.autograd.grad(parts(x64, ids, lp, False, None, 1.0)[0].mean() * 65536.0, x64)
    assert float((d.double() - want).norm() / want.norm()) < 2.0 ** -11  # scaled after rounding most would be lost as subnormals


@pytest.mark.parametrize("remainder", [False, True])
def test_two_backward_passes(remainder):
    x, ids, lp, _ = problem(20, 3001, 9, torch.bfloat16, 3)
    x.requires_grad_(True)
    loss = sten.distillation_loss(x, ids, lp, remainder=remainder)
    [a] = torch.autograd.grad(loss, x, retain_graph=True)
    first = a.clone()
    a.zero_()  # the caller's to change
    [b] = torch.autograd.grad(loss, x, torch.tensor(2.0, device="cuda"), retain_graph=True)
    [c] = torch.autograd.grad(loss, x)
    assert torch.equal(c, first) and torch.equal(b.float(), first.float() * 2)
    d = torch.autograd.grad(sten.distillation_loss(x, ids, lp, remainder=remainder, reduction="none").sum() / 20, x)[0]
    assert float((d.double() - first.double()).norm() / first.double().norm()) < 2.0 ** -8


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("remainder", [False, True])
def test_masks_and_extremes(remainder, dtype):
    low = torch.finfo(dtype).min
    x, ids, lp, _ = problem(9, 5003, 6, dtype, 8)
    x[0] = -INF                              # no student
    x[1, :] = low                            # a uniform one
    x[2, ids[2, 0]] = 80.0                   # sure of the teacher's first token: all others together have e^-70
    x[3].masked_fill_(torch.zeros(5003, dtype=torch.bool, device="cuda").scatter_(0, ids[3], True).logical_not(), -INF)  # nothing but the kept
    x[4, ids[4]] = low                       # gives the kept tokens nothing
    x[5, 2500:] = -INF
    ids[5] = torch.arange(6, device="cuda") * 7
    ids[6] = -1                              # no teacher
    lp[7, 1:] = -INF
    ids[8, 5] = -1
    check(x, ids, lp, remainder, reduction="none")
    got, d = check(x[[0, 2, 3, 5, 6, 7, 8]], ids[[0, 2, 3, 5, 6, 7, 8]], lp[[0, 2, 3, 5, 6, 7, 8]], remainder)
    assert bool(torch.isfinite(got)) and bool(torch.isfinite(d).all()) and not d[0].any()


def test_masked_kept_token_is_an_infinite_loss_with_a_finite_gradient():
    x, ids, lp, _ = problem(3, 900, 4, torch.float32, 8)
    x[1, ids[1, 2]] = -INF
    for remainder in (False, True):
        y = x.clone().requires_grad_(True)
        loss = sten.distillation_loss(y, ids, lp, remainder=remainder, reduction="none")
        assert torch.isinf(loss).tolist() == [False, True, False]
        [d] = torch.autograd.grad(loss, y, torch.ones_like(loss))
        assert bool(torch.isfinite(d).all())


@pytest.mark.parametrize("remainder", [False, True])
def test_nan_and_unread_rows(remainder):
    x, ids, lp, _ = problem(5, 3000, 4, torch.bfloat16, 8)
    x[1, 2999] = float("nan")
    x[2, 5] = INF
    x[3, 1] = float("nan")
    w = torch.tensor([1.0, 1.0, 1.0, 0.0, 1.0], device="cuda")
    ids[4, 1] = 3000  # no such token
    y = x.requires_grad_(True)
    loss = sten.distillation_loss(y, ids, lp, remainder=remainder, weight=w, reduction="none")
    assert torch.isnan(loss).tolist() == [False, True, True, False, True] and float(loss[3]) == 0
    [d] = torch.autograd.grad(loss, y, torch.ones_like(loss))
    assert bool(torch.isfinite(d[0]).all()) and not d[3].any() and all(bool(torch.isnan(d[i]).all()) for i in (1, 2, 4))


@pytest.mark.parametrize("remainder", [False, True])
@pytest.mark.parametrize("vocab", [700, 131072])
def test_an_id_that_occurs_twice_is_one_token(remainder, vocab):
    x, ids, lp, _ = problem(6, vocab, 9, torch.float32, 8)
    lp = lp - 1.0
    ids[1, 4] = ids[1, 0]
    ids[2, :] = ids[2, 3]
    ids[3, 8] = ids[3, 7] = ids[3, 2]
    ids[4, 0] = (ids[4, 1] + 65536) % vocab  # another token with the same low bits
    check(x, ids, lp, remainder, reduction="none")
    check(x, ids, lp, remainder)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("remainder", [False, True])
def test_strided_rows(remainder, dtype):
    x, ids, lp, _ = problem(36, 2051, 7, dtype, 5)
    full, ids, lp = x.view(4, 9, 2051), (ids % 1998).view(4, 9, 7), lp.view(4, 9, 7)
    for y, i, l in ((full[:, :-1], ids[:, 1:], lp[:, 1:]), (full[:, 1:], ids[:, 1:], lp[:, 1:]), (full[1:, 2:7, 5:2003], ids[1:, 2:7], lp[1:, 2:7]),
                    (full[..., ::2], ids % 1026, lp), (full.transpose(0, 1), ids.transpose(0, 1), lp.transpose(0, 1)), (full[:1, :1].expand(3, 5, 2051), ids[:3, :5], lp[:3, :5])):
        for reduction in ("mean", "none"):
            check(y, i, l, remainder, reduction=reduction)
            check(y, i, l, remainder, reduction=reduction, upstream=torch.tensor(0.5, device="cuda").expand(y.shape[:-1] if reduction == "none" else ()))


@pytest.mark.parametrize("remainder", [False, True])
def test_clusters_that_take_several_rows(remainder):
    """Rows of 1 MB are shared by four CTAs each, and there are more of them than clusters; some are not read."""
    x, ids, lp, w = problem(300, 262144, 40, torch.float32, 5, weighted=True)
    check(x, ids, lp, remainder, w)
    check(x, ids, lp, remainder, w, 2.0, "none")


def test_offsets_past_32_bits():
    pitch = 1_200_000_003
    store = torch.empty(2 * pitch + 40000, dtype=torch.bfloat16, device="cuda")
    x, ids, lp, _ = problem(3, 33333, 7, torch.bfloat16, 6)
    y = store.as_strided((3, 33333), (pitch, 1))
    y.copy_(x)
    check(y, ids, lp, True)


@pytest.mark.parametrize("remainder", [False, True])
def test_differences(remainder):
    gen = torch.Generator(device="cuda").manual_seed(11)
    x, ids, lp, w = problem(3, 61, 5, torch.float32, 12, scale=1.5, weighted=True)
    v = torch.randn(3, 61, device="cuda", generator=gen) / 8

    def value(y):
        return sten.distillation_loss(y, ids, lp, remainder=remainder, weight=w, temperature=1.3)

    x.requires_grad_(True)
    [g] = torch.autograd.grad(value(x), x)
    eps = 0.02
    with torch.no_grad():
        slope = float(value(x + eps * v) - value(x - eps * v)) / (2 * eps)
    assert abs(slope - float((g * v).sum())) < 2e-3  # third derivative along v below 1, values off by less than 3e-5


@pytest.mark.parametrize("remainder", [False, True])
@pytest.mark.parametrize("tau", [1.0, 1.5])
def test_no_part_of_the_error_is_the_same_in_every_row(remainder, tau):
    """A student near its teacher: the loss is a small difference, and a bias of the exponentials (ex2.approx has one of half a unit
    in the last place, 6e-8) would be a large part of it.  Allowed on the average of 2000 rows, in units of tau^2: that bias once, and
    four standard errors of single errors of 6e-7."""
    x, ids, lp, _ = problem(2000, 20011, 17, torch.float32, 4, temperature=tau)
    got = sten.distillation_loss(x, ids, lp, remainder=remainder, temperature=tau, reduction="none")
    want = parts(x.double(), ids, lp, remainder, None, tau)[0]
    assert abs(float((got.double() - want).mean())) <= tau * tau * (6e-8 + 4 * 6e-7 / 2000 ** 0.5)


def test_no_rows_streams_and_graphs():
    e = torch.empty(0, 100, device="cuda", requires_grad=True)
    none = torch.empty(0, 4, device="cuda")
    for reduction in ("none", "sum", "mean"):
        loss = sten.distillation_loss(e, none.long(), none, reduction=reduction)
        assert loss.shape == ((0,) if reduction == "none" else ()) and float(loss.sum()) == 0
        assert torch.autograd.grad(loss.sum(), e)[0].shape == (0, 100)
    x, ids, lp, w = problem(37, 40001, 20, torch.bfloat16, 8, weighted=True)

    def step():
        y = x.detach().requires_grad_(True)
        loss = sten.distillation_loss(y, ids, lp, remainder=True, weight=w)
        return loss.detach(), torch.autograd.grad(loss, y)[0]

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = step()
    graph.replay()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_teacher_kept_by_token_log_probs():
    """The two operators together: the top of a teacher, and a student held against it."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    t = torch.randn(16, 5000, device="cuda", generator=gen) * 3
    kept = sten.token_log_probs(t, top=128, temperature=2.0)
    same = sten.distillation_loss(t, kept.top_ids, kept.top_log_prob, temperature=2.0, remainder=True)
    other = sten.distillation_loss(t.roll(1, 0), kept.top_ids, kept.top_log_prob, temperature=2.0, remainder=True)
    assert abs(float(same)) < 4 * LOSS < float(other)


def test_refusals():
    x, ids, lp, w = problem(4, 100, 5, torch.float32, 1, weighted=True)
    for args, error in (((x.double(), ids, lp), TypeError), ((x, ids.short(), lp), TypeError), ((x, ids, lp.double()), TypeError), ((x, ids[:3], lp), ValueError),
                        ((x, ids, lp[:, :4]), ValueError), ((x, ids[:, :0], lp[:, :0]), ValueError), ((x.cpu(), ids, lp), RuntimeError), ((x, ids.cpu(), lp), RuntimeError),
                        ((x, ids[0], lp[0]), ValueError)):
        with pytest.raises(error):
            sten.distillation_loss(*args)
    for kw, error in (({"reduction": "batchmean"}, ValueError), ({"weight": w.double()}, TypeError), ({"weight": w[:3]}, ValueError), ({"temperature": 0.0}, RuntimeError),
                      ({"weight": w.requires_grad_(True)}, ValueError)):
        with pytest.raises(error):
            sten.distillation_loss(x, ids, lp, **kw)
    with pytest.raises(ValueError, match="teacher_log_probs"):
        sten.distillation_loss(x, ids, lp.requires_grad_(True))
    x, ids, lp, w = problem(4, 400, 257, torch.float32, 1)
    with pytest.raises(RuntimeError, match="256"):
        sten.distillation_loss(x, ids, lp)
    x = torch.zeros(1, (1 << 20) + 1, device="cuda")
    with pytest.raises(RuntimeError, match="1048576"):
        sten.distillation_loss(x, ids[:1, :4], lp[:1, :4], remainder=True)
    check(x, ids[:1, :4].contiguous(), lp[:1, :4].contiguous())  # without a remainder it is served
    check(x[:, 1:], ids[:1, :4].contiguous(), lp[:1, :4].contiguous(), True)
