"""Layer norm and embedding: bad arguments are answered with a status before any CUDA call, and the package refuses what it has no kernel for."""
import ctypes

import pytest
import torch

import sten_b200 as sten
from sten_b200 import _native as nat

one = ctypes.c_void_p(16)  # never dereferenced: validation fails first


def at(address):
    return ctypes.c_void_p(address)


def norm(**change):
    a = dict(x=one, ld_x=8, residual=None, ld_residual=0, rows=2, width=8, dtype=nat.NMG_F16, weight=one, bias=one, param_dtype=nat.NMG_F32, eps=1e-5, y=one, sum=None,
             stats=None, stream=None)
    return nat.lib().nmg_layer_norm(*{**a, **change}.values())


def norm_backward(**change):
    a = dict(h=one, ld_h=8, rows=2, width=8, dtype=nat.NMG_F16, weight=one, param_dtype=nat.NMG_F32, stats=one, g_y=one, ld_g_y=8, g_sum=None, ld_g_sum=0, d_x=one, d_weight=None,
             d_bias=None, workspace=None, workspace_bytes=0, stream=None)
    return nat.lib().nmg_layer_norm_backward(*{**a, **change}.values())


def embed(**change):
    a = dict(weight=one, vocab=5, width=8, ld=8, dtype=nat.NMG_F32, ids=one, id_bytes=8, tokens=3, scale=1.0, out=one, stream=None)
    return nat.lib().nmg_embedding(*{**a, **change}.values())


def embed_backward(**change):
    a = dict(g=one, ld_g=8, tokens=3, width=8, dtype=nat.NMG_F32, ids=one, id_bytes=8, vocab=5, padding=-1, scale=1.0, d_weight=one, workspace=one, workspace_bytes=1 << 20, stream=None)
    return nat.lib().nmg_embedding_backward(*{**a, **change}.values())


@pytest.mark.parametrize("change,text", [
    ({"x": None}, b"x must"), ({"y": None}, b"y must"), ({"rows": 0}, b"rows"), ({"rows": 1 << 31}, b"rows"), ({"width": 0}, b"width"), ({"dtype": 3}, b"dtype"), ({"param_dtype": nat.NMG_BF16}, b"param_dtype"),
    ({"ld_x": 7}, b"overlap"), ({"residual": one, "ld_residual": 8}, b"together"), ({"sum": one}, b"together"), ({"residual": one, "ld_residual": 7, "sum": one}, b"overlap"), ({"eps": -1.0}, b"eps"),
    ({"eps": float("nan")}, b"eps"), ({"x": at(17)}, b"aligned"), ({"weight": at(18)}, b"weight"), ({"stats": at(20)}, b"stats")])
def test_norm_arguments(change, text):
    assert norm(**change) == 1 and text in nat.lib().nmg_last_error()


@pytest.mark.parametrize("change,text", [
    ({"h": None}, b"h must"), ({"g_y": None}, b"g_y"), ({"stats": None}, b"stats"), ({"stats": at(12)}, b"stats"), ({"d_x": None}, b"NULL"), ({"ld_g_y": 4}, b"overlap"), ({"g_sum": at(17)}, b"g_sum"),
    ({"g_sum": one, "ld_g_sum": 7}, b"overlap"), ({"width": 0}, b"width"), ({"dtype": 9}, b"dtype"), ({"d_weight": at(18)}, b"d_weight")])
def test_norm_backward_arguments(change, text):
    assert norm_backward(**change) == 1 and text in nat.lib().nmg_last_error()


@pytest.mark.parametrize("change,text", [
    ({"weight": None}, b"weight"), ({"out": None}, b"out"), ({"vocab": 0}, b"vocab"), ({"width": 0}, b"width"), ({"tokens": 0}, b"tokens"), ({"id_bytes": 2}, b"bytes"), ({"ids": at(20)}, b"ids"), ({"ids": None}, b"ids"),
    ({"scale": float("inf")}, b"scale"), ({"scale": float("nan")}, b"scale"), ({"dtype": 3}, b"dtype"), ({"ld": -1}, b"ld"), ({"weight": at(18)}, b"aligned")])
def test_embedding_arguments(change, text):
    assert embed(**change) == 1 and text in nat.lib().nmg_last_error()


@pytest.mark.parametrize("change,status,text", [
    ({"g": None}, 1, b"g must"), ({"d_weight": None}, 1, b"d_weight"), ({"d_weight": at(24)}, 1, b"16-byte"), ({"padding": 5}, 1, b"padding"), ({"padding": -2}, 1, b"padding"), ({"ld_g": 4}, 1, b"overlap"),
    ({"workspace": None}, 4, b"workspace"), ({"workspace_bytes": 64}, 4, b"workspace"), ({"workspace": at(8)}, 1, b"16-byte"), ({"tokens": 1 << 31}, 1, b"tokens")])
def test_embedding_backward_arguments(change, status, text):
    assert embed_backward(**change) == status and text in nat.lib().nmg_last_error()


def test_embedding_workspace_covers_the_list_and_the_pieces():
    f = nat.lib().nmg_embedding_backward_workspace_bytes
    assert f(0, 8) == 0 and f(5, 0) == 0
    for tokens in (1, 32, 33, 5000, 1 << 20):
        length = min(512, max(32, tokens // 4096 // 32 * 32))
        assert f(tokens, 100) >= 16 * tokens + -(-tokens // length) * 2 * 100 * 4


def test_tensors_on_the_cpu_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        sten.layer_norm(torch.randn(2, 9))
    with pytest.raises(RuntimeError, match="CUDA"):
        sten.embedding(torch.zeros(2, dtype=torch.int64), torch.randn(5, 4))
    with pytest.raises(ValueError, match="padding_idx"):
        sten.embedding(torch.zeros(2, dtype=torch.int64), torch.randn(5, 4), padding_idx=5)
