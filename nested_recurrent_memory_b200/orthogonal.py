"""Orthogonalising weight updates by Newton-Schulz products, by the kernels
behind ``ngdn2_orth`` (include/ngdn2.h), as the Muon optimiser does.

    X_0 = G / (|G|_F + eps);   X <- a X + (b A + c A A) X,  A = X X^T

with the products taken over the smaller side of G. After a few steps the
singular values of X lie around 1 and its singular vectors are G's.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ops import (_code, _launch, _raise_for, _require_same_device, _scratch, _set_workspace,
                  _status_ptr)

__all__ = ["orthogonalize"]


def orthogonalize(update, steps=5, coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7, dtype=None,
                  workspace=None):
    """The orthogonalised update. update [..., rows, cols] in float32,
    bfloat16 or float16; leading dimensions are a batch of matrices treated
    each on its own (layers stacked, or promotion parameters
    [L - 1, H, rows, cols]). Returns the same shape in ``dtype`` (default
    update's). Operands hold 22 bits and sums are fp32 whatever the types: a
    16-bit result is the fp32 one rounded once.

    ``coefficients`` (a, b, c) must keep every singular value that starts in
    [0, 1] within [0, 4] over ``steps`` steps, else ValueError. A zero update
    gives zeros. ``workspace`` is an optional contiguous CUDA tensor used
    instead of new memory where it is large enough.
    """
    if update.dim() < 2:
        raise ValueError(f"update must be [..., rows, cols], got {tuple(update.shape)}")
    dev = _require_same_device(update)
    rows, cols = update.shape[-2:]
    out = update.new_empty(update.shape, dtype=dtype)
    if out.numel() == 0:
        return out
    flat = update if update.dim() == 3 else update.reshape(-1, rows, cols)
    a = _lib.OrthArgs()
    a.abi_version = _lib.ABI_VERSION
    a.dtype, a.out_dtype = _code(flat), _code(out)
    a.steps = int(steps)
    a.coef[0], a.coef[1], a.coef[2] = coefficients
    a.eps = eps
    a.batch, a.rows, a.cols = flat.shape[0], rows, cols
    a.update, a.out, a.status = flat.data_ptr(), out.data_ptr(), _status_ptr(dev)
    a.update_stride = flat.stride()
    lib = _lib.load()
    need = ctypes.c_size_t(0)
    rc = lib.ngdn2_orth_workspace_size(ctypes.byref(a), ctypes.byref(need))
    if rc == _lib.ERR_COEFFICIENTS:
        raise ValueError(f"coefficients {tuple(coefficients)} do not keep singular values in "
                         f"[0, 1] within [0, 4] over {steps} steps")
    _raise_for(rc, "ngdn2_orth")
    workspace = _scratch(need.value, workspace, dev)
    _set_workspace(a, workspace)
    _launch(lib.ngdn2_orth, a, dev, "ngdn2_orth")
    return out
