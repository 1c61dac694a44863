"""What a sparse model computes between its products: from tokens to hidden states, and the layer norm behind a residual.

``embedding`` looks up scaled rows of a matrix, ``layer_norm`` normalises a tensor or its sum with a residual.  Both take fp32, fp16 and
bf16, any width and row pitch, compute in 32 bits and round once, and differentiate in reverse mode (once; dual tensors are refused):
the gradients of a matrix's row and of the norm's parameters are sums in a fixed order, the same in every run.  The reference has no
counterpart: it leaves both to the model code.

    h = sten.embedding(tokens, model.token.weight, scale=8.0, padding_idx=0)
    y, h = sten.layer_norm(sparse_linear(h), norm.weight, norm.bias, eps=norm.eps, residual=h)   # y goes on, h is the next residual
"""
from . import _native as nat
from .dispatch import SparseTensorWrapper


def _dense(t, what):
    if isinstance(t, SparseTensorWrapper):
        raise TypeError(f"{what} must be a dense tensor")
    return t


def embedding(ids, weight, *, scale=1.0, padding_idx=None):
    """``scale * weight[ids]``: ``[*ids.shape, width]`` of the matrix's type.

    ``ids``: int64 or int32 of any shape; one that is no row of ``weight [vocab, width]`` gives a row of NaN and adds to no gradient.
    ``padding_idx`` (negative: from the end): a row that is looked up like the others and gets no gradient."""
    padding = -1
    if padding_idx is not None:
        rows = weight.shape[0] if weight.dim() else 0
        if not -rows <= padding_idx < rows:
            raise ValueError(f"padding_idx must be a row of the matrix of {rows} rows, got {padding_idx}")
        padding = padding_idx % rows
    return nat.host().embedding(ids, _dense(weight, "weight"), scale, padding)


def layer_norm(x, weight=None, bias=None, *, eps=1e-5, residual=None):
    """Layer norm along the last dimension: ``(h - mean) / sqrt(var + eps) * weight + bias``.

    Without ``residual`` h is ``x`` and the norm is returned.  With it (a tensor like ``x``) h is ``x + residual`` rounded to their type,
    and ``(norm, h)`` is returned: the norm is that of the sum as it is returned.  ``weight`` and ``bias``: one element per feature, of
    x's type or both float32 (which their gradients then are too); None stands for ones and zeros."""
    for t, what in ((x, "x"), (weight, "weight"), (bias, "bias"), (residual, "residual")):
        _dense(t, what)
    return nat.host().layer_norm(x, weight, bias, eps, residual)
