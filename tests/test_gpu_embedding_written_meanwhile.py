"""Ids that another stream writes to while the embedding's gradient is computed from them: every position is added to one of the rows that it may belong to.

The gradients that come in are small whole numbers, so that sums are exact in any order, and all versions of the ids are rows of the matrix: the rows' gradients
together are the sum over all positions, whichever version a position was read in.
"""
import pytest
import torch

import sten_b200 as sten
from gpu_util import cuda

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,vocab,width,id_type", [(1, 70000, 8, torch.int64), (33, 5, 1, torch.int64), (3000, 300, 64, torch.int32), (3000, 300000, 64, torch.int64), (60001, 40000, 72, torch.int64)])
def test_every_position_is_added_once(tokens, vocab, width, id_type):
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    versions = [torch.randint(a, b, (tokens,), device="cuda", generator=gen).to(id_type) for a, b in ((0, (vocab + 1) // 2), (vocab // 2, vocab))]
    ids = versions[0].clone()
    w = torch.zeros(vocab, width, device="cuda", requires_grad=True)
    g = torch.randint(-8, 9, (tokens, width), device="cuda", generator=gen).float()
    total = g.double().sum(0)
    assert tokens * 8 < 2 ** 24  # exact in 32 bits
    out = sten.embedding(ids, w)
    alias = ids.data  # written to without autograd's knowledge, as a loader that does not wait would
    writes = torch.cuda.CUDAGraph()
    with torch.cuda.graph(writes):
        for i in range(40):
            alias.copy_(versions[(i + 1) % 2])
    torch.cuda.synchronize()
    side, sums = torch.cuda.Stream(), []
    for i in range(30):
        with torch.cuda.stream(side):
            writes.replay()
        [d] = torch.autograd.grad(out, w, g, retain_graph=True)
        sums.append(d.double().sum(0))
    torch.cuda.synchronize()
    assert bool((torch.stack(sums) == total).all())
    [d] = torch.autograd.grad(out, w, g)
    assert torch.equal(d, torch.zeros_like(w).index_add_(0, ids.long(), g))
