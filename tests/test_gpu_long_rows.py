"""Long rows that few threads take: 64 threads add up 131072 logits each row, in chains of up to 143 roundings.

Tolerances.  A row's terms go through a group's sum (8 fp32 or 16 16-bit additions and one of its two halves), a thread's groups (128 or 64) and
the merging of 64 threads (6): 143 or 87 roundings of 2^-24, their relative error below 8.6e-6.  The terms are exponentials whose
argument, at most 30 here, is rounded twice and once more where threads are merged (4e-6).  So s is off by less than 1.3e-5 of itself, its
logarithm by as much; log-probabilities add two roundings of values below 64 (8e-6), the entropy weighs the error with the distance
from the maximum (30).  A probability has the error of s and of its own exponential."""
import pytest
import torch

import sten_b200 as sten
from gpu_util import cuda
from test_gpu_token_log_probs import close, drawn_targets, formula, logits, reference

pytestmark = pytest.mark.gpu
ABS, ABS_H, REL_P = 2.1e-5, 4e-4, 2.1e-5
HALF_ULP = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}


@pytest.mark.parametrize("dtype,rows", [(torch.float32, 2368), (torch.bfloat16, 2048)])
def test_rows_of_131072_by_64_threads(dtype, rows):
    x = logits(rows, 131072, dtype, 7)
    t = drawn_targets(x)
    x.requires_grad_(True)
    got = sten.token_log_probs(x, t)
    gen = torch.Generator(device="cuda").manual_seed(3)
    g = [torch.randn(rows, device="cuda", generator=gen) for _ in range(2)]
    [d] = torch.autograd.grad([got.log_prob, got.entropy], x, g)
    x = x.detach()
    for a in range(0, rows, 148):
        b = min(rows, a + 148)
        want = reference(x[a:b], t[a:b])
        close(got.lse[a:b].detach(), want["lse"], ABS, 2.0 ** -22)
        close(got.log_prob[a:b].detach(), want["log_prob"], ABS)
        close(got.entropy[a:b].detach(), want["entropy"], ABS_H)
        grad = formula(x[a:b], t[a:b], 1.0, None, g[0][a:b], g[1][a:b], None, None)
        size = g[0][a:b].abs() + g[1][a:b].abs() * 31
        allowed = REL_P * torch.softmax(x[a:b].double(), -1) * size.double()[:, None] * 2 + (HALF_ULP[dtype] * 1.01 + 1e-6) * grad.abs() + 1e-30
        assert float(((d[a:b].double() - grad).abs() - allowed).max()) <= 0
