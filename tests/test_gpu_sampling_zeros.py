"""Sampling where the logit that ends what is kept is 0: rows with thousands of equal zeros (0 and -0), which the lists beside a border do not hold, so that
the search goes over the row, by one CTA and by several.  Against the definition, and against the same rows in a larger batch.

The definition and its tolerances are those of the other sampling tests; `edges` says how many rows may lie at a border at all.
"""
import pytest
import torch

import sten_b200 as sten
from gpu_util import cuda
from test_gpu_sampling import BF16, F16, F32, check

pytestmark = pytest.mark.gpu
# the last value of the type below 2: its integer ends in ones
BELOW_2 = {F32: 2 - 2.0 ** -23, F16: 2 - 2.0 ** -10, BF16: 2 - 2.0 ** -7}


def rectified(rows, vocab, dtype, seed, scale=0.4, sign=1.0):
    """Half of a row is 0, a third of that -0; the largest logits are those whose integers end in ones, and random ones."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, vocab, device="cuda", generator=gen) * scale).clamp_(min=0).to(dtype)
    x[:, ::3] *= torch.where(x[:, ::3] == 0, -1.0, 1.0).to(dtype)
    top = torch.tensor([BELOW_2[dtype], 2.0, 2.5, 3.0 * BELOW_2[dtype] / 2, 4 * BELOW_2[dtype]], device="cuda").to(dtype)
    at = torch.randint(0, vocab, (rows, 1), device="cuda", generator=gen)
    x.scatter_(1, at, top[torch.arange(rows, device="cuda") % 6 % 5][:, None])
    x[5::6].scatter_(1, at[5::6], 0)  # every sixth row keeps its own
    return (x * sign).to(dtype), torch.rand(rows, device="cuda", generator=gen)


SETTINGS = {"count": lambda n: dict(top_k=int(0.6 * n)), "weight": lambda n: dict(top_p=0.8), "both": lambda n: dict(top_k=int(0.9 * n), top_p=0.85), "cold": lambda n: dict(top_k=int(0.55 * n), temperature=0.7),
            "count and share": lambda n: dict(top_k=int(0.7 * n), top_p=0.999, min_p=0.01)}


@pytest.mark.parametrize("name", SETTINGS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab", [(1, 20011), (13, 20011), (64, 20011), (12, 131072), (40, 5003)])
def test_borders_at_zero(name, dtype, rows, vocab):
    x, u = rectified(rows, vocab, dtype, seed=rows + vocab)
    setting = SETTINGS[name](vocab)
    o = check(x, u, edges=0.2, **setting)
    many = -(-1500 // rows)  # more rows than the device has CTAs: each gets fewer
    again = sten.sample_tokens(x.repeat(many, 1), u.repeat(many), **setting)
    assert torch.equal(again.tokens, o.tokens.repeat(many)) and torch.equal(again.log_prob, o.log_prob.repeat(many))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,vocab", [(1, 20011), (12, 131072), (700, 9001)])
def test_zeros_are_the_largest(dtype, rows, vocab):
    x, u = rectified(rows, vocab, dtype, seed=vocab, sign=-1.0)
    some = slice(0, 24)
    for setting in (dict(top_k=int(0.3 * vocab)), dict(top_k=int(0.7 * vocab)), dict(top_p=0.3), dict(top_k=vocab // 2, top_p=0.9)):
        # rows of 9001: 0.9 of the weight of 4500 equal logits is that of exactly 4050, so the run may end on either side of a token
        o = check(x[some], u[some], edges=1 if setting.get("top_k") == 4500 else 0.2, **setting)
        assert torch.equal(sten.sample_tokens(x, u, **setting).tokens[some], o.tokens)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_zeros_beside_the_smallest_numbers(dtype):
    """0 between numbers of both signs whose integers are next to its own."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    step = 2.0 ** -149 if dtype == F32 else 2.0 ** -133
    x = (torch.randint(-4, 5, (9, 30011), device="cuda", generator=gen).double() * step).to(dtype)
    x[::2, 77] = BELOW_2[dtype]
    u = torch.rand(9, device="cuda", generator=gen)
    for k in (3000, 13000, 14500, 16000, 20000, 29000):
        o = check(x, u, top_k=k, edges=1)
        again = sten.sample_tokens(x.repeat(170, 1), u.repeat(170), top_k=k)
        assert torch.equal(again.tokens, o.tokens.repeat(170))
