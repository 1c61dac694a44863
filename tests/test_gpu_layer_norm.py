"""Layer norm and its gradients against the definition in 64 bits.

Bounds, with u = 2^-24, n columns and S additions in a row for a sum (32 elements of a thread or width / 512, 5 steps in a warp, 5 over warps,
and a rounding or two of the division): a sum is off by at most S u times the sum of magnitudes.  They are followed through the formulas to
first order, and the last rounding adds half a step of the result's type.
"""
import pytest
import torch

import sten_b200 as sten
from gpu_util import cuda

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def half_step(t, values):
    return torch.finfo(t).eps / 2 * values.abs() + torch.finfo(t).smallest_normal * torch.finfo(t).eps  # below the normal numbers steps are of one size


def additions(width):
    return max(32, -(-width // 512)) + 14


def definition(x, residual, weight, bias, eps):
    """(h, y, and bounds of y) in 64 bits; h is the sum as it is returned."""
    h = x.double()
    if residual is not None:
        h = (h + residual.double()).to(x.dtype).double()
    n, s = h.shape[-1], additions(h.shape[-1])
    mean = h.mean(-1, keepdim=True)
    d = h - mean
    var = (d * d).mean(-1, keepdim=True)
    rstd = (var + eps).rsqrt()
    k = d * rstd
    e_mean = s * U * h.abs().mean(-1, keepdim=True)
    e_d = e_mean + U * (d.abs() + e_mean)
    e_rstd = ((s + 4) * U * var + e_mean ** 2 + 2 * U * (d.abs() * e_d).mean(-1, keepdim=True)) / (var + eps) / 2 + 3 * U  # relative
    e_k = rstd * e_d + k.abs() * (e_rstd + U)
    w = torch.ones(n, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    y = k * w + (0.0 if bias is None else bias.double())
    e_y = w.abs() * e_k + U * ((k * w).abs() + y.abs())
    return dict(h=h, mean=mean, rstd=rstd, k=k, y=y, e_k=e_k, e_rstd=e_rstd, e_y=e_y + half_step(x.dtype, y.abs() + e_y), w=w)


def gradients(f, g_y, g_sum, dtype, param_dtype):
    """d_x, d_weight, d_bias and their bounds."""
    k, w, rstd, e_k = f["k"], f["w"], f["rstd"], f["e_k"]
    g = g_y.double()
    a, s = g * w, additions(k.shape[-1]) + 2
    m1, m2 = a.mean(-1, keepdim=True), (a * k).mean(-1, keepdim=True)
    e1 = s * U * a.abs().mean(-1, keepdim=True)
    e2 = (s + 2) * U * (a * k).abs().mean(-1, keepdim=True) + (a.abs() * e_k).mean(-1, keepdim=True)
    inner = a - m1 - k * m2
    gs = torch.zeros_like(a) if g_sum is None else g_sum.double()
    dx = rstd * inner + gs
    size = a.abs() + m1.abs() + (k * m2).abs()
    e = rstd * (U * a.abs() + e1 + k.abs() * e2 + e_k * m2.abs() + 3 * U * size + inner.abs() * (f["e_rstd"] + U)) + U * (dx.abs() + gs.abs())
    rows = g.reshape(-1, g.shape[-1])
    kr, ek = k.reshape(rows.shape), e_k.reshape(rows.shape)
    steps = len(rows) + 24
    dw, db = (rows * kr).sum(0), rows.sum(0)
    e_w = steps * U * (rows * kr).abs().sum(0) + (rows.abs() * ek).sum(0)
    e_b = steps * U * rows.abs().sum(0)
    return [(dx, e + half_step(dtype, dx.abs() + e)), (dw, e_w + half_step(param_dtype, dw.abs() + e_w)), (db, e_b + half_step(param_dtype, db.abs() + e_b))]


def within(got, want, bound, what):
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"{what}: off by {float(off.max()):.3g}, {float((off / bound).max()):.3g} of what is allowed"


def operands(shape, dtype, param_dtype, residual, seed=0, weight=True, bias=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*size, scale=1.0, shift=0.0):
        return torch.randn(*size, device="cuda", generator=gen) * scale + shift
    x = normal(*shape, scale=1.5, shift=0.5)
    x[..., shape[-1] // 3] += 20
    return (x.to(dtype), normal(*shape).to(dtype) if residual else None, normal(shape[-1], scale=0.2, shift=1.0).to(param_dtype) if weight else None,
            normal(shape[-1]).to(param_dtype) if bias else None, normal(*shape).to(dtype), normal(*shape).to(dtype) if residual else None)


def check(x, residual, weight, bias, g_y, g_sum, eps=1e-5):
    leaves = [t for t in (x, residual, weight, bias) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    o = sten.layer_norm(x, weight, bias, eps=eps, residual=residual)
    outputs, ups = ([o], [g_y]) if residual is None else (list(o), [g_y, g_sum])
    grads = dict(zip(map(id, leaves), torch.autograd.grad(outputs, leaves, ups)))
    with torch.no_grad():
        f = definition(x, residual, weight, bias, eps)
        if residual is not None:
            assert torch.equal(outputs[1].double(), f["h"])
        assert outputs[0].dtype == x.dtype and outputs[0].shape == x.shape
        within(outputs[0], f["y"], f["e_y"], "y")
        params = [t for t in (weight, bias) if t is not None]
        want = gradients(f, g_y, g_sum, x.dtype, params[0].dtype if params else x.dtype)
        within(grads[id(x)], *want[0], "d_x")
        if residual is not None:
            assert torch.equal(grads[id(residual)], grads[id(x)])
        for t, (d, e), what in ((weight, want[1], "d_weight"), (bias, want[2], "d_bias")):
            if t is not None:
                assert grads[id(t)].dtype == t.dtype
                within(grads[id(t)], d, e, what)
    again = sten.layer_norm(x, weight, bias, eps=eps, residual=residual)
    assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad([again] if residual is None else list(again), leaves, ups), grads.values()))
    with torch.no_grad():
        bare = sten.layer_norm(x, weight, bias, eps=eps, residual=residual)
    assert torch.equal(bare if residual is None else bare[0], outputs[0])


@pytest.mark.parametrize("dtype,param_dtype", [(F32, F32), (F16, F32), (F16, F16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 7), (5, 64), (37, 255), (16, 1024), (300, 1000), (333, 1023), (9, 4104), (70, 8192), (3, 8200), (2, 16384), (5, 40001)])
def test_sizes(dtype, param_dtype, rows, width):
    check(*operands((rows, width), dtype, param_dtype, rows % 2 == 1, seed=width))


@pytest.mark.parametrize("rows", [1, 2, 147, 149, 297, 5000])
@pytest.mark.parametrize("width", [96, 2048])
def test_rows(rows, width):
    check(*operands((rows, width), BF16, F32, rows % 2 == 0, seed=rows))


@pytest.mark.parametrize("weight", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("width", [512, 9000])
def test_parameters_that_are_not_there(weight, bias, width):
    check(*operands((20, width), F16, F32, True, weight=weight, bias=bias))


@pytest.mark.parametrize("dtype", [F32, F16])
def test_strides_and_alignment(dtype):
    x, r, w, b, g, gs = operands((6, 10, 264), dtype, F32, True)
    check(x[:, :-1], r[:, 1:], w, b, g[:, :-1], gs[:, :-1])          # sequences without an end: copied
    check(x[..., 1:257], r[..., 8:264], w[4:260], b[1:257], g[..., :256], gs[..., 3:259])
    check(x[0, :, 8:], r[0, :, 8:], w[8:], b[8:], g[0, :, 8:], gs[0, :, 8:])  # a row pitch above the width
    check(x.transpose(0, 2), r.transpose(0, 2), w[:6], b[:6], g.transpose(0, 2), gs.transpose(0, 2))
    check(x[0], r[0], w, b, g[0, :1].expand(10, -1), gs[0, :, :1].expand(-1, 264))
    check(x[0, 0], None, w, b, g[0, 0], None)


@pytest.mark.parametrize("width", [768, 9999])
def test_which_gradients_are_wanted(width):
    x, r, w, b, g, gs = operands((50, width), BF16, F32, True)
    x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True), r.requires_grad_(True)
    leaves = [x, r, w, b]
    y, h = sten.layer_norm(x, w, b, residual=r)
    full = torch.autograd.grad([y, h], leaves, [g, gs], retain_graph=True)
    for i in range(4):
        assert torch.equal(torch.autograd.grad([y, h], leaves[i], [g, gs], retain_graph=True)[0], full[i])
    # one output alone: the norm's gradient is that with a zero for the sum, the sum's goes straight through
    only = torch.autograd.grad(y, leaves, g, retain_graph=True)
    zero = torch.autograd.grad([y, h], leaves, [g, torch.zeros_like(gs)], retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(only, zero))
    through = torch.autograd.grad(h, leaves, gs, allow_unused=True)
    assert torch.equal(through[0], gs) and torch.equal(through[1], gs) and through[2] is None and through[3] is None
    w2 = w.detach()
    y = sten.layer_norm(x.detach(), w2, b)
    assert y.requires_grad
    assert torch.equal(torch.autograd.grad(y, b, g)[0], full[3])
    same = sten.layer_norm(x, w, b, residual=x)
    [d] = torch.autograd.grad(list(same), x, [g, gs])
    two = sten.layer_norm(x, w, b, residual=x.detach().clone().requires_grad_(True))
    assert torch.equal(d, 2 * torch.autograd.grad(list(two), x, [g, gs])[0])


@pytest.mark.parametrize("residual", [False, True])
def test_against_differences(residual):
    """The derivative along a direction, from differences of the definition in 64 bits."""
    x, r, w, b, g, gs = operands((17, 200), F32, F32, residual)
    leaves = [t.requires_grad_(True) for t in (x, r, w, b) if t is not None]
    o = sten.layer_norm(x, w, b, residual=r)
    grads = torch.autograd.grad([o] if r is None else list(o), leaves, [g] if r is None else [g, gs])
    gen = torch.Generator(device="cuda").manual_seed(9)
    with torch.no_grad():
        f = definition(x, r, w, b, 1e-5)
        bounds = dict(zip(("x", "w", "b"), (e for _, e in gradients(f, g, gs, F32, F32))))
        bounds["r"] = bounds["x"]
        for leaf, d, name in zip(leaves, grads, ("x", "r", "w", "b") if residual else ("x", "w", "b")):
            v = torch.randn(leaf.shape, device="cuda", generator=gen).double()

            def loss(step):
                t = {"x": x, "r": r, "w": w, "b": b}
                t = {k: None if q is None else q.double() + (step * v if k == name else 0) for k, q in t.items()}
                h = t["x"] if r is None else t["x"] + t["r"]
                y = torch.nn.functional.layer_norm(h, (200,), t["w"], t["b"], 1e-5)
                return float((y * g.double()).sum() + (0 if r is None else (h * gs.double()).sum()))
            step = 1e-5
            slope = (loss(step) - loss(-step)) / (2 * step)
            # the kernel normalises the rounded sum: another point, 2^-24 of the sum away, where the slope is another by as much relatively
            moved = 2.0 ** -22 * float((d.double() * v).abs().sum()) * 50 if residual else 0.0
            allowed = float((bounds[name] * v.abs()).sum()) + 1e-7 * float((d.double() * v).abs().sum()) + moved
            assert abs(float((d.double() * v).sum()) - slope) <= allowed


def test_odd_values():
    x, _, w, b, g, _ = operands((8, 300), F32, F32, False)
    with torch.no_grad():
        x[1, 7], x[3, 0], x[5] = float("nan"), float("inf"), 2.5
    x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)
    y = sten.layer_norm(x, w, b)
    assert torch.isnan(y[1]).all() and torch.isnan(y[3]).all() and torch.isfinite(y[[0, 2, 4, 5, 6, 7]]).all()
    assert torch.equal(y[5], b)  # a constant row: its differences from the mean are 0
    d, dw, db = torch.autograd.grad(y, [x, w, b], g)
    assert torch.isnan(d[1]).all() and torch.isnan(d[3]).all() and torch.isfinite(d[[0, 2, 4, 5, 6, 7]]).all()
    assert torch.isnan(dw).all() and torch.isfinite(db).all()
    # a mean far above the spread: the differences are what counts
    far = (torch.randn(4, 1024, device="cuda") + 4096).requires_grad_(True)
    check(far.detach().clone(), None, None, None, torch.randn(4, 1024, device="cuda"), None)


def test_no_rows():
    x = torch.empty(0, 3, 20, device="cuda", requires_grad=True)
    w, b = (torch.ones(20, device="cuda", requires_grad=True) for _ in range(2))
    y, h = sten.layer_norm(x, w, b, residual=x.detach())
    d, dw, db = torch.autograd.grad([y, h], [x, w, b], [torch.empty_like(y), torch.empty_like(h)])
    assert y.shape == x.shape == d.shape and not dw.any() and not db.any()


def test_streams_and_graphs():
    x, r, w, b, g, gs = operands((100, 1024), F16, F32, True)
    for t in (x, r, w, b):
        t.requires_grad_(True)

    def step():
        y, h = sten.layer_norm(x, w, b, residual=r)
        return [y, h, *torch.autograd.grad([y, h], [x, r, w, b], [g, gs])]
    want = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    del got
    graphs = []
    for _ in range(2):  # two graphs with memory of their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, step()))
    for _ in range(3):
        with torch.no_grad():
            x.add_(0.25)
            b.mul_(1.5)
        for graph, _ in graphs:
            graph.replay()
        want = step()
        for _, got in graphs:
            assert all(torch.equal(p, q) for p, q in zip(got, want))
        del want


def test_a_graph_outside_of_the_capture_is_told():
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    held = sten.layer_norm(x)  # keeps the node that accumulates x's gradient
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    told = []
    with torch.cuda.graph(graph, stream=side):
        try:
            sten.layer_norm(x)
        except RuntimeError as e:
            told.append(str(e))
        with torch.no_grad():
            y = sten.layer_norm(x)
    assert len(told) == 1 and "before capturing" in told[0]
    graph.replay()
    assert torch.equal(y, held)


def test_refusals():
    x, r, w, b, g, gs = operands((4, 32), F16, F32, True)
    for call, kind, text in (
            (lambda: sten.layer_norm(x.double()), TypeError, "float32"), (lambda: sten.layer_norm(x, w.to(BF16)), TypeError, "weight"), (lambda: sten.layer_norm(x, w[:31]), ValueError, "weight"),
            (lambda: sten.layer_norm(x, w, b.half()), TypeError, "one type"), (lambda: sten.layer_norm(x, residual=r.float()), TypeError, "residual"),
            (lambda: sten.layer_norm(x, residual=r[:1]), ValueError, "residual"), (lambda: sten.layer_norm(x, w.cpu()), RuntimeError, "CUDA"), (lambda: sten.layer_norm(x[..., :0]), ValueError, "feature"),
            (lambda: sten.layer_norm(x, eps=-1.0), RuntimeError, "eps"), (lambda: sten.layer_norm(torch.zeros((), device="cuda")), ValueError, "feature")):
        with pytest.raises(kind, match=text):
            call()
    import torch.autograd.forward_ad as forward_ad
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="layer_norm has no forward-mode"):
        sten.layer_norm(forward_ad.make_dual(x, x))
    x.requires_grad_(True)
    y = sten.layer_norm(x, w)
    [d] = torch.autograd.grad(y, x, g, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        d.sum().backward()


@pytest.mark.parametrize("which", range(3))
@pytest.mark.parametrize("change", [lambda t: t.cpu(), lambda t: t.double(), lambda t: torch.cat([t.reshape(-1), t.reshape(-1)[:1]])])
def test_changed_saved_tensors_are_refused(which, change):
    x, _, w, b, g, _ = operands((4, 32), F16, F32, False)
    x.requires_grad_(True)
    seen = []

    def pack(t):
        seen.append(t)
        return len(seen) - 1
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda i: change(seen[i]) if i == which else seen[i]):
        y = sten.layer_norm(x, w, b)
    assert len(seen) == 3
    with pytest.raises(RuntimeError, match="saved for the backward pass"):
        torch.autograd.grad(y, x, g)


def test_more_than_2_to_the_32_elements():
    rows, width = 65600, 65537
    x = torch.zeros(rows, width, dtype=F16, device="cuda")
    x[-1] = torch.randn(width, device="cuda").half()
    with torch.no_grad():
        y = sten.layer_norm(x, eps=1e-5)
        last = sten.layer_norm(x[-1:], eps=1e-5)
    assert torch.equal(y[-1:], last) and float(last.float().std()) > 0.9 and not y[-2].any()
