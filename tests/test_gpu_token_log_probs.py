"""Token log-probabilities, entropy and top alternatives against plain implementations in 64 bits, and their gradients against the
formula's and against differences.

Tolerances.  A 32-bit sum over a row of up to 2^17 logits goes through at most 16 + 8 + 9 roundings (a group, a thread's groups, the
merging of threads and CTAs) and its terms are exponentials whose argument, at most 30 here, is rounded twice: their relative error
is below 40 * 2^-24 + 30 * 2^-23 < 6e-6.  That is the error of s and so the absolute one of ln s; log-probabilities and log-sum-exp add
two roundings of values below 64 (8e-6), or of whatever size the log-sum-exp has.  The entropy weighs the same errors with the distance from the maximum (at most 30):
30 * 6e-6.  A probability has the relative error of its exponential, 6e-6 + 8e-6; 16-bit gradients add half a unit in their last place."""
import pytest
import torch

import sten_b200 as sten
from gpu_util import cuda

pytestmark = pytest.mark.gpu
INF = float("inf")
ABS, ABS_H, REL_P = 1.4e-5, 1.8e-4, 1.4e-5
HALF_ULP = {torch.float32: (0.0, 0.0), torch.float16: (2.0 ** -11, 2.0 ** -25), torch.bfloat16: (2.0 ** -8, 0.0)}
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def logits(rows, vocab, dtype, seed, scale=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(rows, vocab, device="cuda", generator=g) * scale).to(dtype)


def reference(x, targets=None, temperature=1.0, top=0, ignore=-100):
    x64 = x.double()
    z = x64 / temperature
    empty = (x64 == -INF).all(-1)
    top_z = torch.where(empty, 0.0, z.amax(-1))[..., None]  # apart: beside the lowest fp32 value even 64 bits have no room for the rest
    rest = torch.logsumexp(z - top_z, -1)
    lse = rest + top_z[..., 0]
    logp = torch.where(empty[..., None], -INF, z - top_z - rest[..., None])
    p = logp.exp()
    out = {"lse": lse, "entropy": -torch.where(p == 0, 0.0, p * logp).sum(-1)}
    if targets is not None:
        ok = targets != ignore
        out["log_prob"] = torch.where(ok, logp.gather(-1, targets.clamp(min=0)[..., None])[..., 0], 0.0)
    if top:
        out["top_ids"] = torch.sort(x.float(), dim=-1, descending=True, stable=True).indices[..., :top]
        out["top_log_prob"] = logp.gather(-1, out["top_ids"])
    return out


def close(got, want, absolute, relative=0.0):
    got = got.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    infinite = torch.isinf(want)
    assert torch.equal(got[infinite], want[infinite])
    fine = torch.isfinite(want)
    d = (got - want)[fine].abs() - absolute - relative * want[fine].abs()
    assert d.numel() == 0 or float(d.max()) <= 0, f"off by {float(d.max())} more than allowed"


def check_forward(x, targets=None, temperature=1.0, top=0):
    got, want = sten.token_log_probs(x, targets, temperature=temperature, top=top), reference(x, targets, temperature, top)
    close(got.lse, want["lse"], ABS, 2.0 ** -22)
    close(got.entropy, want["entropy"], ABS_H)
    assert (got.log_prob is None) == (targets is None) and (got.top_ids is None) == (top == 0)
    if targets is not None:
        close(got.log_prob, want["log_prob"], ABS)
    if top:
        assert torch.equal(got.top_ids, want["top_ids"])
        close(got.top_log_prob, want["top_log_prob"], ABS)
    return got


def formula(x, targets, temperature, top_ids, g_log_prob, g_entropy, g_lse, g_top, ignore=-100):
    """Gradient of the logits in 64 bits."""
    z = x.double() / temperature
    empty = (x == -INF).all(-1, keepdim=True)
    z = z - torch.where(empty, 0.0, z.amax(-1, keepdim=True))
    logp = torch.where(empty, -INF, z - torch.logsumexp(z, -1, keepdim=True))
    p = logp.exp()
    plogp = torch.where(p == 0, 0.0, p * logp)
    d = torch.zeros_like(z)
    if g_entropy is not None:
        d -= g_entropy.double()[..., None] * (plogp - p * plogp.sum(-1, keepdim=True))
    if g_lse is not None:
        d += g_lse.double()[..., None] * p
    if g_log_prob is not None:
        g = torch.where(targets != ignore, g_log_prob.double(), 0.0)[..., None]
        d -= g * p
        d.scatter_add_(-1, targets.clamp(min=0)[..., None], g)
    if g_top is not None:
        d -= g_top.double().sum(-1, keepdim=True) * p
        d.scatter_add_(-1, top_ids, g_top.double())
    return torch.where(empty, 0.0, d / temperature)


def check_backward(x, targets, temperature=1.0, top=0, which="peot", seed=3):
    x = x.detach().requires_grad_(True)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = sten.token_log_probs(x, targets, temperature=temperature, top=top)
    lead = x.shape[:-1]
    g = {k: torch.randn(*lead, *([top] if k == "t" else []), device="cuda", generator=gen) if k in which and (k != "t" or top) else None for k in "peot"}
    pairs = [(o, g[k]) for k, o in zip("peot", (out.log_prob, out.entropy, out.lse, out.top_log_prob)) if g[k] is not None and o is not None]
    [got] = torch.autograd.grad([o for o, _ in pairs], x, [v for _, v in pairs])
    want = formula(x.detach(), targets, temperature, out.top_ids, g["p"], g["e"], g["o"], g["t"])
    assert got.dtype == x.dtype
    # what a probability's error can amount to: its factor A + B log p has terms of the gradients' sizes, log p down to -30
    size = sum(v.abs().sum(-1) if v.dim() > len(lead) else v.abs() * (31 if k == "e" else 1) for k, v in g.items() if v is not None)
    rel, tiny = HALF_ULP[x.dtype]
    p = torch.softmax(x.detach().double() / temperature, -1).nan_to_num(0.0)
    allowed = REL_P * (p + 1e-30) * size.double()[..., None] / temperature * 2 + (rel * 1.01 + 1e-6) * want.abs() + tiny + 1e-30
    worst = float(((got.double() - want).abs() - allowed).max())
    assert worst <= 0, f"off by {worst} more than allowed"
    return got


def drawn_targets(x, seed=9, ignored=False):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randint(0, x.shape[-1], x.shape[:-1], device="cuda", generator=gen)
    if ignored:
        t[torch.rand(t.shape, device="cuda", generator=gen) < 0.3] = -100
    return t


SHAPES = [(1, 1), (3, 2), (5, 7), (2, 8), (4, 33), (33, 511), (1, 4096), (9, 4099), (300, 4107), (700, 1023), (2, 30522), (1, 131072), (40, 70001), (310, 33333)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_forward(rows, vocab, dtype):
    x = logits(rows, vocab, dtype, rows + vocab)
    check_forward(x, drawn_targets(x, ignored=True), top=min(vocab, 5))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_backward(rows, vocab, dtype):
    x = logits(rows, vocab, dtype, rows + vocab)
    check_backward(x, drawn_targets(x, ignored=True), top=min(vocab, 5))


@pytest.mark.parametrize("which", ["p", "e", "o", "t", "pe", "pt"])
@pytest.mark.parametrize("temperature", [0.5, 1.0, 3.0])
def test_backward_of_each_output(which, temperature):
    x = logits(6, 3001, torch.float32, 4)
    check_backward(x, drawn_targets(x), temperature, 4, which)
    t = sten.token_log_probs(x, top=4).top_ids[:, 2].contiguous()  # targets among the alternatives: one entry with both gradients
    check_backward(x, t, temperature, 4, which if which != "e" else "pet")


@pytest.mark.parametrize("top", [1, 2, 31, 64, 127, 128])
@pytest.mark.parametrize("rows,vocab,dtype", [(3, 128, torch.float32), (2, 513, torch.float16), (5, 9001, torch.bfloat16), (400, 2050, torch.float32),
                                              (2, 131071, torch.bfloat16), (320, 50001, torch.bfloat16)])
def test_top_sizes(rows, vocab, dtype, top):
    check_forward(logits(rows, vocab, dtype, top), top=top, temperature=0.7)


@pytest.mark.parametrize("rows,vocab", [(2, 5000), (400, 6001), (1, 131072)])
@pytest.mark.parametrize("kind", ["constant", "two values", "integers", "ascending", "descending", "one thread's columns", "signed zeros", "mostly masked", "steps"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_top_of_rows_that_tie_or_crowd(rows, vocab, kind, dtype):
    gen = torch.Generator(device="cuda").manual_seed(7)
    col = torch.arange(vocab, device="cuda").expand(rows, vocab)
    r = torch.rand(rows, vocab, device="cuda", generator=gen)
    x = {"constant": lambda: torch.full((rows, vocab), -1.25, device="cuda"), "two values": lambda: (r > 0.5).float(), "integers": lambda: (r * 9).floor() - 4,
         "ascending": lambda: col * 1e-4, "descending": lambda: col * -1e-4, "signed zeros": lambda: torch.where(r > 0.5, 0.0, -0.0),
         "one thread's columns": lambda: torch.where(col // 8 % 512 == 3, r + 9, r), "mostly masked": lambda: torch.where(r < 12 / vocab, r, -INF),
         "steps": lambda: torch.where(col // 8 % 512 < 130, (r * 4096).floor() / 512 + 9, r)}[kind]()
    check_forward(x.to(dtype).contiguous(), top=50)
    check_forward(x.to(dtype).contiguous()[:, 3:], top=128)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_masks_and_extremes(dtype, temperature):
    low = torch.finfo(dtype).min
    x = logits(8, 5003, dtype, 1)
    x[0] = -INF                # nothing left
    x[1, 7:] = -INF            # a few tokens left
    x[2] = low                 # the lowest value everywhere is a uniform row
    x[3, 1:] = low             # ... and next to one ordinary logit a mask
    x[4] = -INF
    x[4, 4999] = -3.0          # one token left, in the tail
    x[5, ::2] = -INF
    x[6, :] = torch.finfo(dtype).max if dtype != torch.float16 else 60000.0
    t = torch.tensor([5, 9, 100, 0, 4999, 1, 17, -100], device="cuda")
    got = check_forward(x, t, temperature, top=9)
    assert float(got.log_prob[0]) == -INF and float(got.entropy[0]) == 0 and float(got.log_prob[4]) == 0
    d = check_backward(x, t, temperature, 9, which="pet")
    assert not d[0].any() and bool(torch.isfinite(d).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [float("nan"), INF])
@pytest.mark.parametrize("at", [0, 1, 700, 4101])
def test_nan_and_infinity_stay_in_their_row(dtype, value, at):
    x = logits(3, 4102, dtype, 2)
    x[1, at] = value
    t = drawn_targets(x)
    got = sten.token_log_probs(x, t, top=3)
    for v in (got.log_prob, got.entropy, got.lse, got.top_log_prob):
        assert bool(torch.isnan(v[1]).all()) and bool(torch.isfinite(v[0]).all()) and bool(torch.isfinite(v[2]).all())
    assert int(got.top_ids[1, 0]) == at  # NaN counts as the largest, +inf is
    x.requires_grad_(True)
    [d] = torch.autograd.grad(sten.token_log_probs(x, t).log_prob.sum(), x)
    assert bool(torch.isnan(d[1]).all()) and bool(torch.isfinite(d[0]).all()) and bool(torch.isfinite(d[2]).all())


def test_nan_among_the_top_alternatives_is_ordered_by_column():
    x = logits(1, 9000, torch.float32, 2)
    x[0, 8000] = x[0, 17] = x[0, 4001] = float("nan")
    x[0, 300] = INF
    assert sten.token_log_probs(x, top=5).top_ids[0, :4].tolist() == [17, 4001, 8000, 300]


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_rows(dtype):
    full = logits(4 * 9, 2051, dtype, 5).view(4, 9, 2051)
    tokens = drawn_targets(full)
    for x, t in ((full[:, :-1], tokens[:, 1:]), (full[:, 1:], tokens[:, :-1]), (full[1:, 2:7, 5:2003], tokens[1:, 2:7] % 1998), (full[..., ::2], tokens % 1026),
                 (full.transpose(0, 1), tokens.t()), (full[:1, :1].expand(3, 5, 2051), tokens[:3, :5]), (full.view(2, 2, 9, 2051)[:, :1, ::3], tokens.view(2, 2, 9)[:, :1, ::3])):
        t = t.clamp(max=x.shape[-1] - 1)
        check_forward(x, t, top=6)
        got = check_backward(x, t, top=6)
        assert got.shape == x.shape


def test_gradient_reaches_the_base_of_a_view():
    full = logits(2 * 5, 777, torch.float32, 5).view(2, 5, 777).requires_grad_(True)
    t = drawn_targets(full[:, 1:])
    sten.token_log_probs(full[:, :-1], t).log_prob.mean().backward()
    want = formula(full.detach()[:, :-1], t, 1.0, None, torch.full(t.shape, 1 / 8, device="cuda"), None, None, None)
    close(full.grad[:, :-1], want, 1e-6)
    assert not full.grad[:, -1].any()


def test_offsets_past_32_bits():
    pitch = 1_200_000_003  # elements: the third row begins past 2^31 elements and 4 GB
    store = torch.empty(2 * pitch + 40000, dtype=torch.bfloat16, device="cuda")
    x = store.as_strided((3, 33333), (pitch, 1))
    x.copy_(logits(3, 33333, torch.bfloat16, 6))
    check_forward(x, drawn_targets(x), top=4)
    check_backward(x, drawn_targets(x), top=4)


def test_differences():
    gen = torch.Generator(device="cuda").manual_seed(11)
    x, v = logits(1, 61, torch.float32, 12, 1.5), torch.randn(1, 61, device="cuda", generator=gen) / 8
    t = torch.tensor([4], device="cuda")

    def value(y):
        o = sten.token_log_probs(y, t, temperature=1.3, top=3)
        return (o.log_prob * 0.7 + o.entropy * 1.1 - o.lse * 0.4 + o.top_log_prob.sum(-1) * 0.2).sum()

    x.requires_grad_(True)
    [g] = torch.autograd.grad(value(x), x)
    eps = 0.02  # the third derivative along v is below 1, an output's error below 3e-5: eps^2 / 6 + 3e-5 / eps < 2e-3
    with torch.no_grad():
        slope = float(value(x + eps * v) - value(x - eps * v)) / (2 * eps)
    assert abs(slope - float((g * v).sum())) < 2e-3


def test_no_rows_and_outputs_without_gradient():
    x = torch.empty(0, 100, device="cuda", requires_grad=True)
    o = sten.token_log_probs(x, torch.empty(0, dtype=torch.int64, device="cuda"), top=2)
    assert o.entropy.shape == (0,) and o.top_ids.shape == (0, 2)
    assert torch.autograd.grad(o.log_prob.sum(), x)[0].shape == (0, 100)
    y = logits(4, 100, torch.float32, 1)
    assert sten.token_log_probs(y).log_prob is None
    o = sten.token_log_probs(y.requires_grad_(True), top=2)
    assert not o.top_ids.requires_grad and o.entropy.requires_grad
    assert sten.token_log_probs(y[0], torch.tensor(3, device="cuda")).log_prob.shape == ()  # one row, no leading dimension


def test_no_such_token():
    x = logits(4, 100, torch.float32, 1).requires_grad_(True)
    o = sten.token_log_probs(x, torch.tensor([5, 100, -7, -100], device="cuda"))
    assert torch.isnan(o.log_prob).tolist() == [False, True, True, False] and float(o.log_prob[3]) == 0
    [d] = torch.autograd.grad(o.log_prob.nansum(), x)
    assert bool(torch.isfinite(d[0]).all()) and not d[3].any()
    assert float(sten.token_log_probs(x, torch.tensor([5, 6, 7, -7], device="cuda"), ignore_index=-7).log_prob[3]) == 0


def test_repeated_calls_streams_and_graphs_agree():
    x = logits(37, 40001, torch.bfloat16, 8)
    t = drawn_targets(x)
    first = sten.token_log_probs(x, t, top=20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = x.clone()
        second = sten.token_log_probs(y, t, top=20)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = sten.token_log_probs(x, t, top=20)
    x.copy_(x.flip(0))
    graph.replay()
    for a, b, c, d in zip(first, second, third, sten.token_log_probs(x, t, top=20)):
        assert torch.equal(a, b) and torch.equal(c, d) and not torch.equal(a, c)


def test_refusals():
    x, t = logits(4, 100, torch.float32, 1), torch.zeros(4, dtype=torch.int64, device="cuda")
    for bad, error in (((x.double(), t), TypeError), ((x, t.int()), TypeError), ((x, t[:3]), ValueError), ((x, t.cpu()), RuntimeError), ((x.cpu(), None), RuntimeError),
                       ((x[:, :0], t), ValueError), ((torch.zeros((), device="cuda"), None), ValueError), (([1.0], None), TypeError)):
        with pytest.raises(error):
            sten.token_log_probs(*bad)
    for args, error in (({"top": 101}, ValueError), ({"top": -1}, ValueError), ({"temperature": 0.0}, RuntimeError), ({"temperature": -1.0}, RuntimeError),
                        ({"temperature": float("nan")}, RuntimeError), ({"temperature": INF}, RuntimeError)):
        with pytest.raises(error):
            sten.token_log_probs(x, t, **args)
    with pytest.raises(RuntimeError, match="128"):
        sten.token_log_probs(logits(2, 300, torch.float32, 1), top=129)
    sparse = sten.SparseTensorWrapper.wrapped_from_dense(sten.GroupedNMTensor.from_dense(torch.randn(8, 16, device="cuda"), 2, 4, sparse_dim=0, group_size=2, group_dim=1),
                                                         torch.empty(8, 16, device="cuda"), None)
    with pytest.raises(TypeError, match="dense"):
        sten.token_log_probs(sparse)
