"""nmg_sample_tokens answers bad arguments with a status, before any CUDA call, and the package refuses what it has no kernel for."""
import ctypes

import pytest
import torch

import sten_b200 as sten
from sten_b200 import _native as nat

one = ctypes.c_void_p(16)  # never dereferenced: validation fails first


def sample(**change):
    a = dict(logits=one, rows=2, inner=2, ld=8, ld_outer=16, vocab=8, dtype=nat.NMG_F32, uniform=one, temperatures=None, temperature=1.0, top_ks=None, top_k=0, top_ps=None, top_p=1.0,
             min_ps=None, min_p=0.0, tokens=one, log_prob=one, stream=None)
    return nat.lib().nmg_sample_tokens(*{**a, **change}.values())


@pytest.mark.parametrize("change,text", [
    ({"logits": None}, b"logits"), ({"rows": 0}, b"rows"), ({"vocab": 0}, b"vocab"), ({"vocab": 1 << 31}, b"vocab"), ({"dtype": 3}, b"dtype"), ({"uniform": None}, b"uniform"),
    ({"tokens": None}, b"tokens"), ({"log_prob": None}, b"log_prob"), ({"temperature": -1.0}, b"temperature"), ({"temperature": float("nan")}, b"temperature"), ({"temperature": 1e40}, b"temperature"),
    ({"top_k": -1}, b"top_k"), ({"top_p": -0.1}, b"top_p"), ({"top_p": 1.1}, b"top_p"), ({"top_p": float("nan")}, b"top_p"), ({"min_p": 2.0}, b"min_p"), ({"logits": ctypes.c_void_p(18)}, b"aligned")])
def test_arguments(change, text):
    assert sample(**change) == 1 and text in nat.lib().nmg_last_error()


def test_tensors_on_the_cpu_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        sten.sample_tokens(torch.randn(2, 9), torch.rand(2))
