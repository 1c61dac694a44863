"""Logits that another stream writes to while tokens are drawn from them: a token that the settings leave in every version of the row, or -1 with NaN.

60001 of 131072 logits are 10 or 20 (one of them always 30), the others at most 1, and top_k is 30000: whenever each of them is looked at, every logit that can be
among the k largest is one of the 60001.  Their number keeps the border out of the lists, so that the search goes over the row several times.
"""
import pytest
import torch

import sten_b200 as sten
from gpu_util import cuda

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 8, 600])
def test_lost_borders_are_told(dtype, rows):
    vocab, many = 131072, 60001
    gen = torch.Generator(device="cuda").manual_seed(rows)
    x = (torch.rand(rows, vocab, device="cuda", generator=gen) * 2 - 1).to(dtype)
    at = torch.randperm(vocab, device="cuda", generator=gen)[:many]
    among = torch.zeros(vocab, dtype=torch.bool, device="cuda").index_fill_(0, at, True)
    versions = [torch.where(among, torch.tensor(v, dtype=dtype, device="cuda"), x) for v in (10.0, 20.0)]
    for v in versions:
        v[:, at[0]] = 30
    u = torch.rand(rows, device="cuda", generator=gen)
    settings = [dict(top_k=30000), dict(top_k=30000, top_p=0.9)]
    for s in settings:
        sten.sample_tokens(versions[0], u, temperature=50.0, **s)
    x.copy_(versions[0])
    writes = torch.cuda.CUDAGraph()
    with torch.cuda.graph(writes):
        for i in range(40):
            x.copy_(versions[(i + 1) % 2])
    torch.cuda.synchronize()
    side, drawn = torch.cuda.Stream(), []
    for i in range(60):
        with torch.cuda.stream(side):
            writes.replay()
        drawn += [sten.sample_tokens(x, u, temperature=50.0, **s) for s in settings]
    torch.cuda.synchronize()
    tokens, log_prob = torch.stack([d.tokens for d in drawn]), torch.stack([d.log_prob for d in drawn])
    none = tokens == -1
    assert bool((none | ((tokens >= 0) & among[tokens.clamp(0, vocab - 1)])).all())
    assert bool(torch.isnan(log_prob[none]).all())
    for s in settings:  # and after the writes everything is as before
        a, b = sten.sample_tokens(x, u, temperature=50.0, **s), sten.sample_tokens(versions[0], u, temperature=50.0, **s)
        assert torch.equal(a.tokens, b.tokens) and torch.equal(a.log_prob, b.log_prob) and bool(among[a.tokens].all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 8, 600])
def test_a_largest_logit_that_is_gone(dtype, rows):
    """Temperature 0: one of the columns that are the largest in some version, or -1 with NaN."""
    vocab, columns = 131072, (77, 130000)
    x = torch.zeros(rows, vocab, dtype=dtype, device="cuda")
    versions = [x.clone(), x.clone()]
    for v, c, top in zip(versions, columns, (50.0, 60.0)):
        v[:, c] = top
    u = torch.full((rows,), 0.5, device="cuda")
    x.copy_(versions[0])
    sten.sample_tokens(x, u, temperature=0.0)
    writes = torch.cuda.CUDAGraph()
    with torch.cuda.graph(writes):
        for i in range(40):
            x.copy_(versions[(i + 1) % 2])
    torch.cuda.synchronize()
    side, drawn = torch.cuda.Stream(), []
    for i in range(100):
        with torch.cuda.stream(side):
            writes.replay()
        drawn.append(sten.sample_tokens(x, u, temperature=0.0))
    torch.cuda.synchronize()
    tokens, log_prob = torch.stack([d.tokens for d in drawn]), torch.stack([d.log_prob for d in drawn])
    none = tokens == -1
    # where a version is half written, neither of the two may be there: the first of the zeros
    assert bool((none | (tokens == columns[0]) | (tokens == columns[1]) | (tokens == 0)).all())
    assert bool(torch.isnan(log_prob[none]).all()) and bool((log_prob[~none] == 0).all())
