"""Fused epilogues for grouped n:m linears inside transformer blocks (inference).

The reference runs ``F.linear`` and leaves bias, activation and residual to separate passes over the output
(src/sten/grouped_nm/sten_impls.py:170-173 adds the bias itself, the model code does the rest).  ``nmg_spmm_fused`` does
``activation(x W^T + b) + residual`` in the matmul's epilogue, so the intermediate is written once.  ``fuse_linear_epilogues``
rewires the two module shapes every BERT-style encoder is made of:

* ``dense`` + ``intermediate_act_fn`` (exact GELU)            -> one call with ``activation="gelu"``
* ``dense`` + ``dropout`` + ``LayerNorm(hidden + input)``     -> one call with ``residual=input`` followed by the LayerNorm, which
  ``layer_norms=True`` makes a call of ``layer_norm``

Only modules whose ``dense.weight`` is a grouped n:m parameter are touched, and only while gradients are disabled and
dropout is inactive; otherwise the module's own forward runs.
"""
import types

import torch
from torch.nn.modules import module as _module

from . import ops
from .dispatch import SparseTensorWrapper
from .grouped_nm_tensor import GroupedNMTensor
from .hidden import layer_norm


def _nmg_weight(linear):
    w = getattr(linear, "weight", None)
    if isinstance(w, SparseTensorWrapper) and isinstance(w.wrapped_tensor, GroupedNMTensor):
        s = w.wrapped_tensor.nm_strides
        if len(s["dense_shape"]) == 2 and s["sparse_dim"] == 0 and s["group_dim"] == 1:
            return w.wrapped_tensor
    return None


def sparse_linear_fused(x, gnm, bias=None, activation=None, residual=None):
    """``activation(x W^T + bias) + residual`` for a grouped n:m weight in one library call (no autograd)."""
    if activation not in ops._ACTIVATIONS:
        raise ValueError("activation must be None or 'gelu'")
    if gnm.nm_strides.get("kernel") == "sm100-expanded":
        from .nmg_impls import _wants_expanded
        M, K = (int(v) for v in gnm.nm_strides["dense_shape"])
        x2d = x.reshape(-1, K)
        if x2d.stride(-1) != 1:
            x2d = x2d.contiguous()
        if _wants_expanded(gnm, x2d, x2d.shape[0]):
            res2d = residual.reshape(-1, M) if residual is not None else None
            return ops.spmm_expanded(gnm.expanded(), M, K, x2d, bias=bias, activation=activation, residual=res2d).reshape(*x.shape[:-1], M)
    return gnm.native().linear(gnm, x, bias, ops._ACTIVATIONS[activation], residual)


def _is_exact_gelu(fn):
    name = type(fn).__name__ if not isinstance(fn, types.FunctionType) else fn.__name__
    return name in ("GELUActivation", "GELU", "gelu") and not getattr(fn, "approximate", "none") == "tanh"


def _fused_intermediate_forward(self, hidden_states):
    gnm = _nmg_weight(self.dense)
    if gnm is None or torch.is_grad_enabled() or not hidden_states.is_cuda:
        return self._sten_unfused_forward(hidden_states)
    return sparse_linear_fused(hidden_states, gnm, self.dense.bias, activation="gelu")


def _fused_output_forward(self, hidden_states, input_tensor):
    gnm = _nmg_weight(self.dense)
    dropout_off = (not self.training) or getattr(self.dropout, "p", 0.0) == 0.0
    if gnm is None or torch.is_grad_enabled() or not dropout_off or not hidden_states.is_cuda:
        return self._sten_unfused_forward(hidden_states, input_tensor)
    h, norm = sparse_linear_fused(hidden_states, gnm, self.dense.bias, residual=input_tensor), self.LayerNorm
    if self._sten_layer_norm and _is_plain_layer_norm(norm, h):
        return layer_norm(h, norm.weight, norm.bias, eps=norm.eps)
    return norm(h)


def _is_plain_layer_norm(norm, x):
    """Whether ``norm(x)`` is layer_norm of its parameters and nothing else.  Under autocast torch's norm returns fp32."""
    return (type(norm) is torch.nn.LayerNorm and not torch.is_autocast_enabled("cuda") and norm.normalized_shape == x.shape[-1:] and "forward" not in norm.__dict__
            and not norm._forward_hooks and not norm._forward_pre_hooks and not _module._global_forward_hooks and not _module._global_forward_pre_hooks
            and all(p is None or (type(p) in (torch.Tensor, torch.nn.Parameter) and p.is_cuda and p.dtype in (x.dtype, torch.float32)) for p in (norm.weight, norm.bias))
            and (norm.weight is None or norm.bias is None or norm.weight.dtype == norm.bias.dtype))


def fuse_linear_epilogues(model, layer_norms=False):
    """Rewire ``dense`` + GELU and ``dense`` + residual + LayerNorm modules of ``model`` whose dense weight is grouped n:m.
    ``layer_norms``: the norm behind the residual runs as ``layer_norm`` too where it is a plain ``torch.nn.LayerNorm`` of the last
    dimension; its results differ from torch's by roundings.  The module itself still runs under autocast (its result is fp32 there), and where it
    has a ``forward`` of its own, hooks (its own or those of all modules) or sparse parameters.  Returns the number of modules rewired.  Idempotent; modules that are
    rewired already take the new choice of ``layer_norms``."""
    count = 0
    for mod in model.modules():
        if hasattr(mod, "_sten_layer_norm"):
            mod._sten_layer_norm = bool(layer_norms)
        dense = getattr(mod, "dense", None)
        if not isinstance(dense, torch.nn.Linear) or _nmg_weight(dense) is None or hasattr(mod, "_sten_unfused_forward"):
            continue
        if hasattr(mod, "intermediate_act_fn") and _is_exact_gelu(mod.intermediate_act_fn):
            mod._sten_unfused_forward = mod.forward
            mod.forward = types.MethodType(_fused_intermediate_forward, mod)
            count += 1
        elif hasattr(mod, "LayerNorm") and hasattr(mod, "dropout"):
            mod._sten_unfused_forward = mod.forward
            mod._sten_layer_norm = bool(layer_norms)
            mod.forward = types.MethodType(_fused_output_forward, mod)
            count += 1
    return count
