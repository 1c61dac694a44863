"""Scoring and distilling a model whose weights were made sparse: operators over the rows of its logits.

``token_log_probs`` reads logits once for the log-probabilities of given tokens, the entropy and the top alternatives of every
row; ``distillation_loss`` holds a student against the top log-probabilities that ``token_log_probs`` kept of its teacher.  Both
take fp32, fp16 and bf16 logits of any row length and alignment, compute in 32 bits, and differentiate with respect to the
logits (once, in reverse mode; dual tensors are refused).  The reference has no counterpart: it leaves every loss to the model code.

    with torch.no_grad():                                               # the dense model, once per batch
        kept = sten.token_log_probs(teacher(x), top=64, temperature=2.0)
    loss = sten.distillation_loss(student(x), kept.top_ids, kept.top_log_prob, temperature=2.0, remainder=True)
    loss.backward()                                                     # through the sparse weights
    score = sten.token_log_probs(student(x)[:, :-1], x[:, 1:])          # log-probability of every next token
"""
from typing import NamedTuple, Optional

import torch

from . import _native as nat
from .dispatch import SparseTensorWrapper


class TokenLogProbs(NamedTuple):
    """What ``token_log_probs`` finds in every row: float32 tensors of the logits' leading shape (``top_*``: and ``top``)."""

    log_prob: Optional[torch.Tensor]
    entropy: torch.Tensor
    lse: torch.Tensor
    top_log_prob: Optional[torch.Tensor]
    top_ids: Optional[torch.Tensor]


def _dense(logits):
    if isinstance(logits, SparseTensorWrapper):
        raise TypeError("logits must be a dense tensor")
    return logits


def token_log_probs(logits, targets=None, *, temperature=1.0, top=0, ignore_index=-100):
    """Log-probabilities under ``softmax(logits / temperature)`` along the last dimension.

    ``logits``: ``[..., vocab]``; leading dimensions may be strided (``logits[:, :-1]`` is not copied).  ``targets``: int64 tokens of
    the leading shape, or None; where one is ``ignore_index`` its log-probability is 0 and has no gradient, where it is no token of
    the vocabulary the log-probability and the row's gradient are NaN.  ``top`` (at most 128): how many of the largest logits to
    return, largest first, equal ones in the order of their ids.

    A row that is -inf throughout has log-probabilities and log-sum-exp -inf, entropy 0 and no gradient; a row that holds NaN or +inf
    gives NaN."""
    return TokenLogProbs(*nat.host().token_log_probs(_dense(logits), targets, ignore_index, temperature, top))


class SampledTokens(NamedTuple):
    """What ``sample_tokens`` draws from every row: int64 and float32 tensors of the logits' leading shape."""

    tokens: torch.Tensor
    log_prob: torch.Tensor


def sample_tokens(logits, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One token of every row of ``logits [..., vocab]`` by the row's number in ``uniform`` (float32 in [0, 1), the leading shape).

    ``top_k`` keeps the k largest logits of a row (0: all; equal ones in the order of their ids), ``top_p`` of these the shortest run, largest first,
    whose probabilities under ``softmax(logits / temperature)`` reach p of their sum (at least one token), ``min_p`` of these the ones of at
    least min_p times the largest probability.  The token is the first, in the order of ids, where the probabilities of what is left
    exceed ``uniform`` times their sum; ``log_prob`` is its log-probability among what is left.  Each setting is a number or a tensor with
    one for each row (float32; ``top_k`` int64).  ``temperature`` 0 takes the first of the largest logits.

    A row that holds NaN or +inf, or is -inf throughout, gives token -1 and log-probability NaN (so may one that is written to meanwhile).  The same logits, number and settings give
    the same token in every call, whatever else is in the batch.  Not differentiable: ``token_log_probs`` is."""
    return SampledTokens(*nat.host().sample_tokens(_dense(logits), uniform, temperature, top_k, top_p, min_p))


_REDUCTIONS = {"none": nat.NMG_REDUCE_NONE, "sum": nat.NMG_REDUCE_SUM, "mean": nat.NMG_REDUCE_MEAN}


def distillation_loss(logits, teacher_ids, teacher_log_probs, *, remainder=False, weight=None, temperature=1.0, reduction="mean"):
    """Divergence ``temperature**2 * KL(teacher || softmax(logits / temperature))`` of every row from a teacher of whom the top
    log-probabilities were kept.

    ``teacher_ids`` (int64 or int32, negative: padding) and ``teacher_log_probs`` (float): ``[..., kept]``, at most 256 a row, as
    ``token_log_probs(..., top=kept, temperature=temperature)`` returns them.  Without ``remainder`` the teacher's distribution is the
    softmax of the kept values (so any logits divided by the temperature will do); with it the kept values are log-probabilities,
    and the mass they leave over is held against the student's probability of all other tokens together.  ``weight``: float32 of
    the leading shape; rows of weight 0 are not read.  ``reduction``: "none", "sum", or "mean" over the rows' weights.

    A reduced loss of logits that require a gradient keeps, beside them, a tensor of their size with their gradient until its backward
    pass.  That tensor is not among the saved ones: hooks on those (``save_on_cpu``, checkpointing) leave it on the device.

    A token that occurs more than once among a row's ids has a term of its own in the loss for each occurrence, which lowers the loss by
    a constant and may take it below 0; the gradient and the remainder are those of one token with the summed probability.

    Gradients go to the logits only.  Rows of which the mask (or the padding) leaves nothing have loss 0 and gradient 0."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'none', 'sum' or 'mean', got {reduction!r}")
    return nat.host().distill(_dense(logits), teacher_ids, teacher_log_probs, weight, remainder, temperature, _REDUCTIONS[reduction])
