"""Embedding and the gradient of its matrix against the definition in 64 bits.

A row of the gradient that has c positions is off by at most c + 1 roundings (its additions and the scaling) of u = 2^-24 of the sum of
magnitudes, and half a step of its type; a looked-up row by one rounding and half a step.
"""
import pytest
import torch

import sten_b200 as sten
from gpu_util import cuda

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def half_step(t, values):
    return torch.finfo(t).eps / 2 * values.abs() + torch.finfo(t).smallest_normal * torch.finfo(t).eps


def ids_of(kind, tokens, vocab, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if kind == "one":
        return torch.full((tokens,), vocab // 2, device="cuda")
    if kind == "even":
        return torch.randint(0, vocab, (tokens,), device="cuda", generator=gen)
    if kind == "runs":  # ids that fill pieces of the sorted list to their ends
        return torch.arange(tokens, device="cuda") // 32 % vocab
    if kind == "wrong":
        return torch.randint(-vocab, 2 * vocab, (tokens,), device="cuda", generator=gen)
    return torch.exp(torch.rand(tokens, device="cuda", generator=gen) * torch.log(torch.tensor(float(vocab)))).long().clamp(0, vocab - 1)


def check(ids, weight, g, scale=1.0, padding=None):
    weight.requires_grad_(True)
    vocab, width = weight.shape
    out = sten.embedding(ids, weight, scale=scale, padding_idx=padding)
    [d] = torch.autograd.grad(out, weight, g)
    assert out.shape == (*ids.shape, width) and out.dtype == weight.dtype == d.dtype and d.shape == weight.shape
    with torch.no_grad():
        flat, rows, up = ids.reshape(-1).long(), out.reshape(-1, width), g.reshape(-1, width)
        there = (flat >= 0) & (flat < vocab)
        assert torch.isnan(rows[~there]).all()
        want = weight[flat[there]].double() * scale
        assert bool(((rows[there].double() - want).abs() <= U * want.abs() + half_step(weight.dtype, want)).all())
        counted = there if padding is None else there & (flat != padding % vocab)
        at, up = flat[counted], up[counted].double()
        total = torch.zeros(vocab, width, dtype=torch.float64, device="cuda").index_add_(0, at, up) * scale
        size = torch.zeros(vocab, width, dtype=torch.float64, device="cuda").index_add_(0, at, up.abs()) * abs(scale)
        c = torch.bincount(at, minlength=vocab)[:, None]
        off = (d.double() - total).abs()
        assert bool((off <= (c + 1) * U * size + half_step(d.dtype, total.abs() + (c + 1) * U * size)).all()), f"off by {float(off.max())}"
        assert not d[c[:, 0] == 0].any()
    [again] = torch.autograd.grad(sten.embedding(ids, weight, scale=scale, padding_idx=padding), weight, g)
    assert torch.equal(d, again)
    return d


def case(kind, tokens, vocab, width, dtype, scale=1.0, padding=None, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    w = torch.randn(vocab, width, device="cuda", generator=gen).to(dtype)
    return check(ids_of(kind, tokens, vocab, seed), w, torch.randn(tokens, width, device="cuda", generator=gen).to(dtype), scale, padding)


@pytest.mark.parametrize("kind", ["one", "even", "runs", "wrong", "words"])
@pytest.mark.parametrize("tokens", [1, 31, 33, 1000, 1025, 2500, 9000, 40001])
def test_lists(kind, tokens):
    case(kind, tokens, 700, 72, BF16, seed=tokens)


@pytest.mark.parametrize("vocab", [1, 2, 511, 512, 70000, 300000])  # one, two and three passes of the sort
@pytest.mark.parametrize("kind", ["words", "even"])
def test_vocabularies(kind, vocab):
    case(kind, 5000, vocab, 48, F32, scale=3.0, padding=-1, seed=vocab)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("width", [1, 8, 100, 255, 256, 257, 1023, 1024, 4104])
def test_widths(dtype, width):
    case("words", 777, 333, width, dtype, scale=width ** 0.5, padding=0, seed=width)


@pytest.mark.parametrize("dtype,vocab,width", [(F32, 9333, 7641), (F16, 5000, 20003), (BF16, 70001, 1001), (F32, 40, 900000), (F16, 90, 700008)])
def test_large_matrices_with_few_tokens(dtype, vocab, width):
    stale = [torch.full((vocab, width), float("nan"), dtype=dtype, device="cuda") for _ in range(3)]  # what the gradient's memory may hold before
    del stale
    case("even", 7, vocab, width, dtype)


def test_pieces_longer_than_the_shortest():
    case("words", 120000, 3000, 1024, BF16)   # pieces of 96 positions and more
    case("one", 70000, 3, 2048, F32)


def test_a_hot_row_is_added_in_the_order_of_positions():
    g = torch.zeros(6000, 8, device="cuda")
    g[::1000] = torch.tensor([1e8, 1.0, -1e8, 1.0, 3e-8, 1.0], device="cuda")[:, None]
    w = torch.zeros(4, 8, device="cuda")
    a = check(torch.zeros(6000, dtype=torch.int64, device="cuda"), w, g)
    order = torch.randperm(5000, device="cuda")  # other ids between them, and other zeros: the same sum
    ids = torch.cat([torch.zeros(6000, dtype=torch.int64, device="cuda"), 1 + order % 3])
    b = check(ids, w, torch.cat([g, torch.zeros(5000, 8, device="cuda")]))
    assert torch.equal(a[0], b[0])


def test_shapes_strides_and_types_of_ids():
    gen = torch.Generator(device="cuda").manual_seed(1)
    wide = torch.randn(90, 144, device="cuda", generator=gen, dtype=F32).to(F16)
    ids = torch.randint(0, 90, (7, 12), device="cuda", generator=gen)
    g = torch.randn(7, 12, 144, device="cuda", generator=gen).half()
    a = check(ids, wide.detach().clone(), g, 2.0, 5)
    b = check(ids.int(), wide.detach().clone(), g, 2.0, 5 - 90)
    assert torch.equal(a, b)
    for w in (wide.detach()[:, 8:72], wide.detach()[:, 1:65], wide.detach().t()[:64].t()):
        check(ids[:, ::2], w, g[:, ::2, 40:104])
    check(ids, wide.detach().clone(), g[:1, :1].expand(7, 12, 144))
    check(ids[0, 0], wide.detach().clone(), g[0, 0])
    [d] = torch.autograd.grad(sten.embedding(ids, wide.requires_grad_(True)).sum(), wide)
    assert torch.equal(d, torch.bincount(ids.reshape(-1), minlength=90)[:, None].half().expand(90, 144))


def test_no_tokens():
    w = torch.randn(5, 6, device="cuda", requires_grad=True)
    out = sten.embedding(torch.empty(0, 3, dtype=torch.int64, device="cuda"), w)
    [d] = torch.autograd.grad(out, w, torch.empty_like(out))
    assert out.shape == (0, 3, 6) and not d.any()


def test_a_matrix_of_more_than_2_to_the_31_elements():
    vocab, width = 530000, 4104
    w = torch.zeros(vocab, width, dtype=BF16, device="cuda", requires_grad=True)
    ids = torch.tensor([0, vocab - 1, vocab - 2, vocab - 1], device="cuda")
    with torch.no_grad():
        w[-1] = 3.0
    out = sten.embedding(ids, w)
    assert bool((out[1] == 3).all()) and bool((out[3] == 3).all()) and not out[[0, 2]].any()
    g = torch.randn(4, width, device="cuda").to(BF16)
    [d] = torch.autograd.grad(out, w, g)
    assert torch.equal(d[0], g[0]) and torch.equal(d[-2], g[2]) and torch.equal(d[-1], (g[1].float() + g[3].float()).to(BF16)) and not d[1:-2].any()


def test_streams_and_graphs():
    gen = torch.Generator(device="cuda").manual_seed(3)
    ids, w = ids_of("words", 3000, 5000), torch.randn(5000, 256, device="cuda", generator=gen, requires_grad=True)
    g = torch.randn(3000, 256, device="cuda", generator=gen)

    def step():
        out = sten.embedding(ids, w, scale=2.0, padding_idx=0)
        return [out, *torch.autograd.grad(out, w, g)]
    want = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    del got
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, step()))
    for turn in range(3):
        ids.copy_(ids_of("words", 3000, 5000, seed=turn + 10))
        for graph, _ in graphs:
            graph.replay()
        want = step()
        for _, got in graphs:
            assert all(torch.equal(p, q) for p, q in zip(got, want))
        del want


def test_refusals():
    w, ids = torch.randn(5, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for call, kind, text in (
            (lambda: sten.embedding(ids.short(), w), TypeError, "ids"), (lambda: sten.embedding(ids, w.double()), TypeError, "weight"), (lambda: sten.embedding(ids, w[0]), ValueError, "matrix"),
            (lambda: sten.embedding(ids, w, padding_idx=5), ValueError, "padding_idx"), (lambda: sten.embedding(ids, w, padding_idx=-6), ValueError, "padding_idx"),
            (lambda: sten.embedding(ids.cpu(), w), RuntimeError, "CUDA"), (lambda: sten.embedding(ids, w, scale=float("nan")), RuntimeError, "scale"), (lambda: sten.embedding(ids, w[:0]), ValueError, "matrix")):
        with pytest.raises(kind, match=text):
            call()
    import torch.autograd.forward_ad as forward_ad
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="embedding has no forward-mode"):
        sten.embedding(ids, forward_ad.make_dual(w, w))
    w.requires_grad_(True)
    [d] = torch.autograd.grad(sten.embedding(ids, w).sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        d.sum().backward()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.cpu()):
        out = sten.embedding(ids, w)
    with pytest.raises(RuntimeError, match="saved for the backward pass"):
        torch.autograd.grad(out.sum(), w)
