"""Gradients of up to 128 alternatives, at sizes whose rows go to CTAs of 64, 128, 256 and 512 threads and to clusters of four."""
import pytest
import torch

import sten_b200 as sten
from gpu_util import cuda
from test_gpu_token_log_probs import DTYPES, check_backward, drawn_targets, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("top", [63, 64, 65, 127, 128])
@pytest.mark.parametrize("rows,vocab", [(3, 128), (1000, 2000), (300, 4107), (9, 4099), (5, 9001), (1, 131072), (320, 50001)])
def test_every_alternative_has_its_gradient(rows, vocab, top, dtype):
    x = logits(rows, vocab, dtype, top)
    check_backward(x, drawn_targets(x, ignored=True), top=top)
    check_backward(x, drawn_targets(x), 0.7, top, which="t")
    last = sten.token_log_probs(x, top=top).top_ids[:, -1].contiguous()  # targets that are an alternative too
    check_backward(x, last, top=top, which="pt")


@pytest.mark.parametrize("top", [64, 65, 128])
def test_a_row_of_gradients_adds_up_to_zero(top):
    """Log-probabilities do not change when a constant is added to the logits.  Allowed: the row's 2000 elements, below 1 in size and
    rounded to 2^-24 of themselves, and probabilities that are off by 1.4e-5 of themselves beside factors of at most sum |g|."""
    x = logits(1000, 2000, torch.float32, 5).requires_grad_(True)
    out = sten.token_log_probs(x, top=top).top_log_prob
    g = torch.randn(out.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    [d] = torch.autograd.grad(out, x, g)
    assert float((d.double().sum(1).abs() - (1.4e-5 + 2.0 ** -24) * 2 * g.double().abs().sum(1)).max()) <= 0
