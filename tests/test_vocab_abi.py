"""The vocabulary operators' C entry points answer bad arguments with a status, before any CUDA call, and the package refuses what it
has no kernel for."""
import ctypes

import pytest
import torch

import sten_b200 as sten
from sten_b200 import _native as nat

one = ctypes.c_void_p(16)  # never dereferenced: validation fails first


def token(**change):
    a = dict(logits=one, rows=2, inner=2, ld=8, ld_outer=16, vocab=8, dtype=nat.NMG_F32, targets=one, ignore=-100, temperature=1.0, top=2, log_prob=one, entropy=one,
             lse=one, top_log_prob=one, top_ids=one, norm=None, stream=None)
    return nat.lib().nmg_token_log_probs(*{**a, **change}.values())


def distill(**change):
    a = dict(logits=one, rows=2, inner=2, ld=8, ld_outer=16, vocab=8, dtype=nat.NMG_F32, ids=one, id_bytes=8, log_probs=one, teacher=nat.NMG_F32, kept=2, remainder=0,
             temperature=1.0, weight=None, reduction=nat.NMG_REDUCE_MEAN, row_loss=one, norm=one, total=None, loss=one, d_logits=None, ld_d=8, ld_d_outer=16, stream=None)
    return nat.lib().nmg_distill(*{**a, **change}.values())


@pytest.mark.parametrize("change,status,text", [
    ({"logits": None}, 1, b"logits"), ({"rows": 0}, 1, b"rows"), ({"vocab": 0}, 1, b"vocab"), ({"vocab": 1 << 31}, 1, b"vocab"), ({"dtype": 3}, 1, b"dtype"),
    ({"temperature": 0.0}, 1, b"temperature"), ({"temperature": float("nan")}, 1, b"temperature"), ({"top": 9}, 1, b"top"), ({"top": -1}, 1, b"top"),
    ({"top": 129, "vocab": 1000}, 2, b"top"), ({"entropy": None}, 1, b"entropy"), ({"log_prob": None}, 1, b"log_prob"), ({"top_ids": None}, 1, b"top_ids"),
    ({"logits": ctypes.c_void_p(18)}, 1, b"aligned"), ({"norm": ctypes.c_void_p(20)}, 1, b"norm")])
def test_token_arguments(change, status, text):
    assert token(**change) == status and text in nat.lib().nmg_last_error()


def test_token_backward_arguments():
    f = nat.lib().nmg_token_log_probs_backward
    head = (one, 2, 2, 8, 16, 8, nat.NMG_F32)
    assert f(*head, None, -100, 1.0, 0, None, one, None, one, None, None, None, one, 8, 16, None) == 1  # g_log_prob without targets
    assert f(*head, None, -100, 1.0, 0, None, one, None, None, one, None, None, one, 8, 16, None) == 1  # g_entropy without entropy
    assert f(*head, None, -100, 1.0, 2, None, one, None, None, None, None, one, one, 8, 16, None) == 1  # g_top without top_ids
    assert f(*head, None, -100, 1.0, 0, None, None, None, None, None, one, None, one, 8, 16, None) == 1  # no norm


@pytest.mark.parametrize("change,status,text", [
    ({"kept": 0}, 1, b"kept"), ({"kept": 257}, 2, b"kept"), ({"id_bytes": 2}, 1, b"ids"), ({"teacher": 5}, 1, b"teacher"), ({"ids": None}, 1, b"NULL"),
    ({"remainder": 1, "vocab": (1 << 20) + 1}, 2, b"remainder"), ({"reduction": 3}, 1, b"reduction"), ({"loss": None}, 1, b"loss"), ({"weight": one}, 1, b"total"),
    ({"reduction": nat.NMG_REDUCE_NONE, "d_logits": one}, 1, b"nmg_distill_backward"), ({"norm": ctypes.c_void_p(20)}, 1, b"norm"), ({"temperature": -2.0}, 1, b"temperature")])
def test_distill_arguments(change, status, text):
    assert distill(**change) == status and text in nat.lib().nmg_last_error()


def test_tensors_on_the_cpu_are_refused():
    x, t = torch.randn(2, 9), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA"):
        sten.token_log_probs(x, t)
    with pytest.raises(RuntimeError, match="CUDA"):
        sten.distillation_loss(x.requires_grad_(True), t[:, None], torch.zeros(2, 1))
    with pytest.raises(ValueError, match="reduction"):
        sten.distillation_loss(x, t[:, None], torch.zeros(2, 1), reduction="batch")
