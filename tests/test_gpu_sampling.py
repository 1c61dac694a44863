"""Sampled tokens against the definition, row by row in 64 bits.

A token is the definition's unless the row's number is within the weights' rounding of the border between two tokens, or a run's end as near
to top_p: weights are rounded to 2^-46 of the largest (2^-(62 - log2 vocab) for larger vocabularies) and known to 2^-42, so sums of n of them
are within n 2^-46 + 2^-42 of the total; `EDGE` (2^-28) is above that for every size here.  Numbers that near a border are compared with both of its
sides.  The log-probability is one rounding (2^-24) of its value, and 2^-38 for what the sums and the logarithm are off by.
"""
import math

import numpy as np
import pytest
import torch

import sten_b200 as sten
from gpu_util import cuda

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
EDGE = 2.0 ** -28


def definition(x, u, temperature, top_k, top_p, min_p):
    """Tokens that the row's number may fall to (one, or two where it is at a border), and {token: log-probability}s."""
    x = x.astype(np.float64)
    if not x.max() < math.inf or np.isnan(x).any() or x.max() == -math.inf:
        return [({-1: math.nan})]
    if temperature == 0:
        return [{int(x.argmax()): 0.0}]
    z = (x - x.max()) / temperature
    w = np.exp(z)
    order = np.argsort(-x, kind="stable")
    if 0 < top_k < len(x):
        order = order[:top_k]
    results = []
    ends = [len(order)]
    if top_p < 1:
        share = np.cumsum(w[order]) / w[order].sum()
        ends = [1 + int((share[:-1] < top_p + e).sum()) for e in (-EDGE, 0.0, EDGE)]
    for end in sorted(set(ends)):
        keep = order[:end]
        if min_p > 0:
            keep = keep[z[keep] >= math.log(min(min_p, 1.0))]
        keep = np.sort(keep)
        upto = np.cumsum(w[keep])
        total = upto[-1]
        for e in (-EDGE, 0.0, EDGE):
            i = min(int((upto <= (u + e) * total).sum()), len(keep) - 1)
            results.append({int(keep[i]): z[keep[i]] - math.log(total)})
    return results


def check(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, edges=0.02):
    o = sten.sample_tokens(x, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    lead = x.shape[:-1]
    assert o.tokens.shape == o.log_prob.shape == lead and o.tokens.dtype == torch.int64 and o.log_prob.dtype == F32
    rows = x.double().reshape(-1, x.shape[-1]).cpu().numpy()
    of = [v.reshape(-1).double().tolist() if isinstance(v, torch.Tensor) else [v] * len(rows) for v in (u, temperature, top_k, top_p, min_p)]
    at_edge = 0
    for r, (token, lp) in enumerate(zip(o.tokens.reshape(-1).tolist(), o.log_prob.reshape(-1).tolist())):
        allowed = definition(rows[r], of[0][r], of[1][r], int(of[2][r]), of[3][r], of[4][r])
        at_edge += len({t for d in allowed for t in d}) > 1
        fits = [d[token] for d in allowed if token in d]
        assert fits, f"row {r}: {token}, not among {allowed}"
        if token >= 0:
            assert any(abs(lp - want) <= 2.0 ** -24 * abs(want) + 2.0 ** -28 for want in fits), (r, lp, fits)
        else:
            assert math.isnan(lp)
    assert at_edge <= edges * len(rows) + 1  # the numbers are not all at borders
    return o


def logits(rows, vocab, dtype, seed=0, scale=2.5, ahead=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, vocab, device="cuda", generator=gen) * scale
    if ahead:
        x[1::2].scatter_add_(1, torch.randint(0, vocab, (rows // 2, 2), device="cuda", generator=gen), 12 * torch.rand(rows // 2, 2, device="cuda", generator=gen))
    return x.to(dtype), torch.rand(rows, device="cuda", generator=gen)


SETTINGS = {"plain": {}, "cold": dict(temperature=0.3), "hot": dict(temperature=4.0), "greedy": dict(temperature=0.0), "k1": dict(top_k=1), "k50": dict(top_k=50), "k": dict(top_k=777, temperature=3.0),
            "p": dict(top_p=0.9), "p small": dict(top_p=1e-6), "p0": dict(top_p=0.0), "p near 1": dict(top_p=0.999), "min": dict(min_p=0.05), "min 1": dict(min_p=1.0),
            "all": dict(temperature=1.3, top_k=200, top_p=0.95, min_p=0.01), "k over all": dict(top_k=1 << 40, top_p=0.5)}


@pytest.mark.parametrize("name", SETTINGS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (5, 64), (40, 1000), (9, 4099), (4, 30522), (2, 131072)])
def test_settings(name, dtype, rows, vocab):
    x, u = logits(rows, vocab, dtype, seed=vocab)
    check(x, u, **SETTINGS[name])


@pytest.mark.parametrize("rows", [1, 17, 74, 149, 296, 300, 700])
@pytest.mark.parametrize("setting", [{}, dict(top_p=0.9), dict(top_k=30, top_p=0.8, min_p=0.02)])
def test_rows_and_clusters(rows, setting):
    x, u = logits(rows, 20011, BF16, seed=rows)
    o = check(x, u, **setting)
    for a, b in ((0, 1), (rows // 2, rows), (rows - 1, rows)):  # the same rows cut in other ways
        part = sten.sample_tokens(x[a:b], u[a:b], **setting)
        assert torch.equal(part.tokens, o.tokens[a:b]) and torch.equal(part.log_prob, o.log_prob[a:b])


@pytest.mark.parametrize("scale", [0.3, 1.0, 2.5])  # the narrower, the more logits there are beside the border
@pytest.mark.parametrize("setting", [dict(top_p=0.9), dict(top_k=2048), dict(top_k=50000), dict(top_k=9000, top_p=0.7)])
def test_long_rows_with_borders_far_down(setting, scale):
    x, u = logits(600, 90001, BF16, seed=3, scale=scale, ahead=False)
    o = sten.sample_tokens(x, u, **setting)  # by the CTAs that many rows get
    some = torch.arange(0, 600, 40, device="cuda")
    few = check(x[some], u[some], **setting)
    assert torch.equal(few.tokens, o.tokens[some]) and torch.equal(few.log_prob, o.log_prob[some])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_settings_of_every_row(dtype):
    x, u = logits(60, 5003, dtype)
    gen = torch.Generator().manual_seed(3)

    def pick(values, t):
        return torch.tensor(values, dtype=t)[torch.randint(0, len(values), (60,), generator=gen)].cuda()
    s = dict(temperature=pick((0.0, 0.5, 1.0, 1.7), F32), top_k=pick((0, 1, 3, 100, 9999), torch.int64), top_p=pick((0.0, 0.3, 0.9, 1.0), F32), min_p=pick((0.0, 0.1, 1.0), F32))
    o = check(x, u, **s)
    for r in range(0, 60, 7):
        one = sten.sample_tokens(x[r], u[r], **{k: v[r].item() for k, v in s.items()})
        assert one.tokens.item() == o.tokens[r].item() and one.log_prob.item() == o.log_prob[r].item()
    beyond = sten.sample_tokens(x, u, top_k=torch.full((60,), -3, device="cuda"), top_p=torch.full((60,), 7.0, device="cuda"), min_p=torch.full((60,), -1.0, device="cuda"))
    plain = sten.sample_tokens(x, u)
    assert torch.equal(beyond.tokens, plain.tokens) and torch.equal(beyond.log_prob, plain.log_prob)


def test_ties():
    for dtype in (F32, F16, BF16):
        u = (torch.arange(64, device="cuda") + 0.5) / 64
        flat = torch.full((64, 6400), 1.5, dtype=dtype, device="cuda")
        assert torch.equal(sten.sample_tokens(flat, u).tokens, torch.arange(64, device="cuda") * 100 + 50)
        assert torch.equal(sten.sample_tokens(flat, u, top_k=64).tokens, torch.arange(64, device="cuda"))
        assert torch.equal(sten.sample_tokens(flat, u, top_p=0.5).tokens, torch.arange(64, device="cuda") * 50 + 25)
        assert torch.equal(sten.sample_tokens(flat, u, top_k=128, top_p=0.5).tokens, torch.arange(64, device="cuda"))
        check(flat, u, top_k=50, top_p=0.61, edges=1)
        few = torch.randint(0, 5, (64, 3001), device="cuda").to(dtype)  # five values, six hundred tokens of each
        few[:, ::7] *= -0.0                                            # 0 and -0 are equal
        for setting in ({}, dict(top_k=700), dict(top_p=0.7), dict(top_k=900, top_p=0.93), dict(min_p=0.1), dict(temperature=0.0), dict(top_k=400, min_p=0.5)):
            check(few, torch.rand(64, device="cuda"), edges=0.2, **setting)


def test_masks_and_odd_values():
    x, u = logits(12, 999, F32)
    x[0, 5], x[1, 998], x[2] = float("nan"), float("inf"), -float("inf")
    x[3, 1:] = -float("inf")
    x[4, :] = torch.finfo(F32).min
    x[5, :500] = torch.finfo(F32).min
    x[6, 100:] = -float("inf")
    x[7] *= 1e30
    x[8] *= 1e-30
    x[9, :] = -float("inf")
    x[9, 3] = torch.finfo(F32).min
    x[10, 3] = torch.finfo(F32).max
    x[11, 0] = -float("nan")
    for setting in SETTINGS.values():
        o = check(x, u, edges=1, **setting)
        assert o.tokens[[0, 1, 2, 11]].tolist() == [-1] * 4 and o.tokens[3] == 0 and o.tokens[9] == 3 and o.tokens[10] == 3
        h = x.clamp(-60000, 60000) if setting else x
        check(h.to(F16), u, edges=1, **setting)
        check(x.to(BF16), u, edges=1, **setting)


def test_numbers_at_the_ends_and_settings_without_meaning():
    x, _ = logits(1, 1000, BF16)
    x = x.expand(9, -1)
    u = torch.tensor([0.0, 1.0, 2.0, -1.0, float("nan"), 1 - 2.0 ** -24, 2.0 ** -149, 1e-30, 0.5], device="cuda")
    for setting in ({}, dict(top_k=20), dict(top_p=0.6), dict(min_p=0.1)):
        o = sten.sample_tokens(x, u, **setting)
        t = o.tokens.tolist()
        assert t[4] == -1 and math.isnan(o.log_prob[4]) and t[0] == t[3] == t[6] == t[7] and t[1] == t[2] and t[0] < t[8] < t[1]
        everywhere = sten.sample_tokens(x[:1].expand(4096, -1), torch.arange(4096, device="cuda") / 4096, **setting).tokens
        assert everywhere.min() == t[0] and bool((everywhere.diff() >= 0).all())
    nan = torch.tensor([float("nan"), -1.0, 1e31, 1.0], device="cuda")
    assert sten.sample_tokens(x[:4], u[:4].clamp(0, 1), temperature=nan).tokens[:3].tolist() == [-1] * 3
    assert sten.sample_tokens(x[:2], u[:2], top_p=nan[[0, 3]]).tokens[0] == -1 and sten.sample_tokens(x[:2], u[:2], min_p=nan[[0, 3]]).tokens[0] == -1


def test_frequencies():
    """Evenly spaced numbers hit every token as often as its probability says: n p of n, to within one."""
    x, _ = logits(1, 300, F32, ahead=False)
    n = 1 << 15
    for setting in ({}, dict(top_k=40), dict(top_p=0.8), dict(min_p=0.03, temperature=1.5)):
        o = sten.sample_tokens(x.expand(n, -1), torch.arange(n, device="cuda") / n, **setting)
        counts = torch.bincount(o.tokens, minlength=300).double()
        p = torch.zeros(300, dtype=torch.float64, device="cuda").scatter_(0, o.tokens, o.log_prob.double().exp())
        assert bool(((counts - n * p).abs() <= 1 + n * 2.0 ** -22).all()) and abs(float(p.sum()) - 1) < 300 * 2.0 ** -22 + float((p < 2 / n).sum()) / n + 1e-3


def test_shapes_strides_and_alignment():
    x, u = logits(60, 1201, F16)
    x3, u3 = x.view(5, 12, 1201), u.view(5, 12)
    for setting in ({}, dict(top_k=9, top_p=0.9)):
        a = check(x3[:, :-1], u3[:, :-1], **setting)
        b = sten.sample_tokens(x3[:, :-1].contiguous(), u3[:, :-1].contiguous(), **setting)
        assert torch.equal(a.tokens, b.tokens)
        check(x3[..., 1:], u3, **setting)
        check(x3[..., 3:1000], u3, **setting)
        check(x3[..., ::2], u3, **setting)
        check(x3.transpose(0, 1), u3.t(), **setting)
        check(x3[0, 0], u3[0, 0], **setting)
    assert sten.sample_tokens(x[:0], u[:0]).tokens.shape == (0,)


def test_more_than_2_to_the_31_elements():
    rows, vocab = 16500, 131073
    x = torch.zeros(rows, vocab, dtype=BF16, device="cuda")
    x[-1, 77] = 50
    x[-2, vocab - 1] = 50
    u = torch.full((rows,), 0.5, device="cuda")
    for setting in ({}, dict(top_k=1)):
        o = sten.sample_tokens(x, u, **setting)
        assert o.tokens[-2:].tolist() == [vocab - 1, 77] and bool((o.tokens[:-2] == (vocab // 2 if not setting else 0)).all())


def test_streams_and_graphs():
    x, u = logits(33, 9000, BF16)
    for setting in ({}, dict(top_k=10), dict(top_p=0.9)):
        want = sten.sample_tokens(x, u, **setting)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = sten.sample_tokens(x, u, **setting)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got.tokens, want.tokens)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = sten.sample_tokens(x, u, **setting)
        for seed in (5, 6):
            u.copy_(torch.rand(33, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
            graph.replay()
            want = sten.sample_tokens(x, u, **setting)
            assert torch.equal(out.tokens, want.tokens) and torch.equal(out.log_prob, want.log_prob)


def test_with_the_scores_of_tokens():
    """What is drawn, scored: without filters both operators say the same."""
    x, u = logits(50, 30522, BF16)
    o = sten.sample_tokens(x, u, temperature=0.8)
    lp = sten.token_log_probs(x, o.tokens, temperature=0.8).log_prob
    # token_log_probs sums some 30 terms in a row in 32 bits: 40 roundings of the logarithm's argument
    assert bool(((o.log_prob - lp).abs() <= 2.0 ** -23 * lp.abs() + 40 * 2.0 ** -24).all())


def test_refusals():
    x, u = logits(4, 100, F16)
    for call, kind, text in (
            (lambda: sten.sample_tokens(x, u.double()), TypeError, "uniform"), (lambda: sten.sample_tokens(x, u[:3]), ValueError, "uniform"), (lambda: sten.sample_tokens(x.double(), u), TypeError, "logits"),
            (lambda: sten.sample_tokens(x, u, temperature=-1.0), RuntimeError, "temperature"), (lambda: sten.sample_tokens(x, u, temperature=float("nan")), RuntimeError, "temperature"),
            (lambda: sten.sample_tokens(x, u, top_p=1.5), RuntimeError, "top_p"), (lambda: sten.sample_tokens(x, u, min_p=-0.1), RuntimeError, "min_p"), (lambda: sten.sample_tokens(x, u, top_k=-1), RuntimeError, "top_k"),
            (lambda: sten.sample_tokens(x, u, top_k=2.5), TypeError, "int"), (lambda: sten.sample_tokens(x, u, top_k=u), TypeError, "top_k"), (lambda: sten.sample_tokens(x, u, top_p=u[:2]), ValueError, "top_p"),
            (lambda: sten.sample_tokens(x, u.cpu()), RuntimeError, "CUDA"), (lambda: sten.sample_tokens(x, u, min_p=u.cpu()), RuntimeError, "device"), (lambda: sten.sample_tokens(x[:, :0], u), ValueError, "last dimension")):
        with pytest.raises(kind, match=text):
            call()
