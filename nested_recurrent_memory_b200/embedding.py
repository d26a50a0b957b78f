"""Scaled embedding lookup and its gradient, by the kernels behind
``ngdn2_embed`` and ``ngdn2_embed_bwd`` (include/ngdn2.h).

    y[..., :] = scale * weight[ids[...], :]
    dweight[v] = scale * sum over the tokens of v of d_out

The gradient sums in fp32 in an order that follows from the tokens alone, so
the same inputs give the same bits, and writes every row of ``dweight`` once.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ops import (_code, _differentiated, _launch, _raise_for, _require_same_device, _scratch,
                  _set_workspace, _status_ptr)

__all__ = ["embed_tokens", "embed_tokens_fwd", "embed_tokens_bwd"]


def _ids(ids):
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"ids must be int64 or int32, got {ids.dtype}")
    return ids if ids.is_contiguous() else ids.contiguous()


def _padding(padding_idx, V):
    """The padding row as a row number, negative ones counted from the end
    (as torch.nn.Embedding does); -1 for none."""
    if padding_idx is None:
        return -1
    if not -V <= padding_idx < V:
        raise ValueError(f"padding_idx must lie within the {V} rows, got {padding_idx}")
    return padding_idx % V


def embed_tokens_fwd(ids, weight, scale=1.0):
    """``scale * weight[ids]``: ids of any shape, int64 or int32; weight
    [V, D] in float32, bfloat16 or float16. Returns [*ids.shape, D] in
    weight's dtype; the product is taken in fp32 and rounded once.

    A token outside [0, V) is not read: its row is NaN, and ``check_status()``
    raises ``KernelStatusError``.
    """
    if weight.dim() != 2:
        raise ValueError(f"weight must be [V, D], got {tuple(weight.shape)}")
    dev = _require_same_device(weight, ids)
    ids = _ids(ids)
    if weight.stride(1) != 1:
        weight = weight.contiguous()
    V, D = weight.shape
    out = weight.new_empty((*ids.shape, D))
    if out.numel() == 0:
        return out
    a = _lib.EmbedArgs()
    a.abi_version = _lib.ABI_VERSION
    a.dtype = _code(weight)
    a.ids_i32 = ids.dtype == torch.int32
    a.scale = scale
    a.N, a.V, a.D = ids.numel(), V, D
    a.ids, a.weight, a.weight_stride = ids.data_ptr(), weight.data_ptr(), weight.stride(0)
    a.out, a.status = out.data_ptr(), _status_ptr(dev)
    _launch(_lib.load().ngdn2_embed, a, dev, "ngdn2_embed")
    return out


def embed_tokens_bwd(ids, d_out, num_embeddings, scale=1.0, padding_idx=None, dtype=None,
                     workspace=None):
    """The gradient of ``sum(embed_tokens(ids, weight, scale) * d_out)`` with
    respect to weight: [num_embeddings, D] in ``dtype`` (default d_out's).

    Tokens equal to ``padding_idx`` add nothing, nor do tokens outside
    [0, num_embeddings) (reported as in ``embed_tokens_fwd``). ``workspace``
    is an optional contiguous CUDA tensor used instead of new memory where it
    is large enough.
    """
    if d_out.shape[:-1] != ids.shape:
        raise ValueError(f"d_out must be [*ids.shape, D], got {tuple(d_out.shape)} for ids "
                         f"{tuple(ids.shape)}")
    dev = _require_same_device(d_out, ids)
    V, D = int(num_embeddings), d_out.shape[-1]
    pad = _padding(padding_idx, V)
    ids = _ids(ids)
    if d_out.dim() != 2:
        d_out = d_out.reshape(ids.numel(), D)
    if d_out.stride(1) != 1:
        d_out = d_out.contiguous()
    dweight = d_out.new_empty((V, D), dtype=dtype)
    if dweight.numel() == 0:
        return dweight
    a = _lib.EmbedBwdArgs()
    a.abi_version = _lib.ABI_VERSION
    a.dtype, a.out_dtype = _code(d_out), _code(dweight)
    a.ids_i32 = ids.dtype == torch.int32
    a.scale = scale
    a.N, a.V, a.D, a.padding_idx = ids.numel(), V, D, pad
    a.ids, a.d_out, a.d_stride = ids.data_ptr(), d_out.data_ptr(), d_out.stride(0)
    a.dweight, a.status = dweight.data_ptr(), _status_ptr(dev)
    lib = _lib.load()
    need = ctypes.c_size_t(0)
    _raise_for(lib.ngdn2_embed_bwd_workspace_size(ctypes.byref(a), ctypes.byref(need)),
               "ngdn2_embed_bwd")
    workspace = _scratch(need.value, workspace, dev)
    _set_workspace(a, workspace)
    _launch(lib.ngdn2_embed_bwd, a, dev, "ngdn2_embed_bwd")
    return dweight


class EmbedTokensFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.save_for_forward(ids)
        ctx.meta = (weight.shape[0], scale, padding_idx, weight.dtype)
        return embed_tokens_fwd(ids, weight, scale)

    @staticmethod
    def backward(ctx, d_out):
        (ids,) = ctx.saved_tensors
        gradient = EmbedTokensBwdFunction.apply if _differentiated(d_out) else embed_tokens_bwd
        return None, gradient(ids, d_out, *ctx.meta), None, None

    @staticmethod
    def jvp(ctx, _ids, d_weight, _scale, _padding_idx):
        (ids,) = ctx.saved_tensors
        return embed_tokens(ids, d_weight, ctx.meta[1], ctx.meta[2])


class EmbedTokensBwdFunction(torch.autograd.Function):
    """The gradient as a function of d_out: linear, so its own derivative is
    the lookup, zero for padding."""

    @staticmethod
    def forward(ctx, ids, d_out, V, scale, padding_idx, dtype):
        ctx.save_for_backward(ids)
        ctx.save_for_forward(ids)
        ctx.meta = (V, scale, padding_idx, dtype)
        ctx.d_type = d_out.dtype
        return embed_tokens_bwd(ids, d_out, V, scale, padding_idx, dtype)

    @staticmethod
    def backward(ctx, d_weight):
        (ids,) = ctx.saved_tensors
        V, scale, padding_idx, _ = ctx.meta
        d = embed_tokens(ids, d_weight, scale, padding_idx).to(ctx.d_type)
        if padding_idx is not None:
            d = d.masked_fill((ids == padding_idx % V).unsqueeze(-1), 0.0)
        return None, d, None, None, None, None

    @staticmethod
    def jvp(ctx, _ids, d_out, *_):
        (ids,) = ctx.saved_tensors
        return EmbedTokensBwdFunction.apply(ids, d_out, *ctx.meta)


def embed_tokens(ids, weight, scale=1.0, padding_idx=None):
    """``embed_tokens_fwd`` with its gradient (``embed_tokens_bwd``) in
    autograd, to any order and in forward mode. ``padding_idx``'s row is looked
    up like any other and gets no gradient."""
    _padding(padding_idx, weight.shape[0])
    if not _differentiated(weight):
        return embed_tokens_fwd(ids, weight, scale)
    return EmbedTokensFunction.apply(ids, weight, float(scale), padding_idx)
