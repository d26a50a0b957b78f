"""Gated linear recurrence, by the kernels behind ``ngdn2_scan``,
``ngdn2_scan_bwd`` and ``ngdn2_scan_step`` (include/ngdn2.h).

    h_t = e^{g_t} h_{t-1} + x_t        for every channel, t = 1 .. T

The state is fp32 throughout. ``g`` are log-decays, as in the nested op
(``<= 0`` for a decay); ``g = -inf`` drops a finite state, so packed sequences of
different lengths are one call with -inf at each sequence's first token. ``g`` may
be positive as long as the factors of 128 consecutive steps multiply to less
than fp32's largest number.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .ops import (_code, _differentiated, _launch, _raise_for, _require_same_device, _scratch,
                  _set_workspace, _status_ptr)

__all__ = ["gated_scan", "gated_scan_fwd", "gated_scan_bwd", "step_gated_scan"]


def _check_state(state, B, D, name):
    if state is None:
        return None
    if state.shape != (B, D):
        raise ValueError(f"{name} must be [{B}, {D}], got {tuple(state.shape)}")
    if state.dtype == torch.float32 and state.is_contiguous():
        return state
    return state.to(torch.float32).contiguous()


def _scan_args(x, g, init):
    B, T, D = x.shape
    a = _lib.ScanArgs()
    a.abi_version = _lib.ABI_VERSION
    a.B, a.T, a.D = B, T, D
    a.x, a.x_dtype, a.x_stride = x.data_ptr(), _code(x), x.stride()
    a.g, a.g_dtype, a.g_stride = g.data_ptr(), _code(g), g.stride()
    a.initial_state = init.data_ptr() if init is not None else None
    return a


def _check_inputs(x, g, *others):
    if x.dim() != 3 or x.shape != g.shape:
        raise ValueError(f"x and g must both be [B, T, D], got {tuple(x.shape)} and "
                         f"{tuple(g.shape)}")
    return _require_same_device(x, g, *others)


def _workspace(a, workspace, dev):
    need = ctypes.c_size_t(0)
    _raise_for(_lib.load().ngdn2_scan_workspace_size(ctypes.byref(a), ctypes.byref(need)),
               "ngdn2_scan")
    return _scratch(need.value, workspace, dev)


def gated_scan_fwd(x, g, initial_state=None, output_final_state=False, return_aux=False,
                   workspace=None):
    """The recurrence forward. x, g [B, T, D] in float32, bfloat16 or float16
    (any strides, broadcast views included); initial_state [B, D] or None.
    Returns ``(h, final_state)``: h [B, T, D] in x's dtype, final_state
    [B, D] float32 (None unless ``output_final_state``); with ``return_aux``
    also the dict that ``gated_scan_bwd`` takes (the states entering every
    128 steps). ``workspace`` is an optional contiguous CUDA tensor used
    instead of new memory where it is large enough."""
    dev = _check_inputs(x, g, initial_state)
    B, T, D = x.shape
    init = _check_state(initial_state, B, D, "initial_state")
    h = x.new_empty((B, T, D))
    final = x.new_empty((B, D), dtype=torch.float32) if output_final_state else None
    carries = None
    if return_aux:
        carries = x.new_empty((B, -(-T // _lib.SCAN_CHUNK), D), dtype=torch.float32)
    if h.numel() == 0:
        if final is not None:
            final.zero_() if init is None else final.copy_(init)
    else:
        a = _scan_args(x, g, init)
        a.h = h.data_ptr()
        a.final_state = final.data_ptr() if final is not None else None
        a.carries = carries.data_ptr() if carries is not None else None
        ws = _workspace(a, workspace, dev)
        _set_workspace(a, ws)
        a.status = _status_ptr(dev)
        _launch(_lib.load().ngdn2_scan, a, dev, "ngdn2_scan")
    return (h, final, dict(carries=carries)) if return_aux else (h, final)


def gated_scan_bwd(x, g, dh, d_final=None, initial_state=None, aux=None, workspace=None):
    """Gradients of ``sum(h * dh) + sum(final_state * d_final)``: returns
    ``(dx, dg, d_initial)`` in the dtypes of x, g and initial_state
    (``d_initial`` is None without an initial state). ``aux`` is the
    forward's; without it the forward runs again."""
    dev = _check_inputs(x, g, dh, d_final, initial_state)
    B, T, D = x.shape
    if dh.shape != x.shape:
        raise ValueError(f"dh must be {tuple(x.shape)}, got {tuple(dh.shape)}")
    init = _check_state(initial_state, B, D, "initial_state")
    dfin = _check_state(d_final, B, D, "d_final")
    dx, dg = x.new_empty((B, T, D)), g.new_empty((B, T, D))
    dinit = x.new_empty((B, D), dtype=torch.float32) if init is not None else None
    if dx.numel() == 0:
        if dinit is not None:
            dinit.zero_() if dfin is None else dinit.copy_(dfin)
    else:
        carries = aux["carries"] if aux is not None else None
        if carries is None:
            carries = gated_scan_fwd(x, g, init, return_aux=True, workspace=workspace)[2]["carries"]
        if (tuple(carries.shape) != (B, -(-T // _lib.SCAN_CHUNK), D) or carries.device != dev
                or carries.dtype != torch.float32 or not carries.is_contiguous()):
            raise ValueError(f"aux is not that of a forward of these shapes on {dev}")
        if dh.dtype != x.dtype:
            dh = dh.to(x.dtype)
        a = _lib.ScanBwdArgs()
        a.abi_version = _lib.ABI_VERSION
        fwd = _scan_args(x, g, init)
        fwd.carries = carries.data_ptr()
        ws = _workspace(fwd, workspace, dev)
        _set_workspace(a, ws)
        a.fwd = fwd
        a.d_h, a.d_h_dtype, a.d_h_stride = dh.data_ptr(), _code(dh), dh.stride()
        a.d_final = dfin.data_ptr() if dfin is not None else None
        a.dx, a.dg = dx.data_ptr(), dg.data_ptr()
        a.d_initial = dinit.data_ptr() if dinit is not None else None
        a.status = _status_ptr(dev)
        _launch(_lib.load().ngdn2_scan_bwd, a, dev, "ngdn2_scan_bwd")
    if dinit is not None and initial_state.dtype != torch.float32:
        dinit = dinit.to(initial_state.dtype)
    return dx, dg, dinit


class GatedScanFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, g, initial_state, output_final_state):
        h, final, aux = gated_scan_fwd(x, g, initial_state, output_final_state, return_aux=True)
        ctx.save_for_backward(x, g, initial_state, aux["carries"])
        return h, final

    @staticmethod
    def backward(ctx, dh, d_final):
        x, g, init, carries = ctx.saved_tensors
        if _differentiated(x, g, init, dh, d_final):
            return *GatedScanBwdFunction.apply(x, g, dh, d_final, init, carries), None
        return *gated_scan_bwd(x, g, dh, d_final, init, dict(carries=carries)), None


class GatedScanBwdFunction(torch.autograd.Function):
    """The gradients, tied to what they depend on: asking for their derivative
    raises, however it is asked for (once_differentiable's error is passed by
    where only some inputs' gradients are asked for)."""

    @staticmethod
    def forward(ctx, x, g, dh, d_final, initial_state, carries):
        return gated_scan_bwd(x, g, dh, d_final, initial_state, dict(carries=carries))

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("gated_scan has no second derivatives")


def gated_scan(x, g, initial_state=None, output_final_state=False):
    """``gated_scan_fwd`` with its gradient (``gated_scan_bwd``) in autograd:
    returns ``(h, final_state)``. Second derivatives and forward mode raise."""
    if not _differentiated(x, g, initial_state):
        return gated_scan_fwd(x, g, initial_state, output_final_state)
    return GatedScanFunction.apply(x, g, initial_state, output_final_state)


def step_gated_scan(x, g, state, *, out_state=None):
    """One decode token: x, g [B, D], state [B, D]. Returns ``(h, state)``,
    h [B, D] in x's dtype and the new state float32; ``out_state`` may be
    ``state`` itself to update in place. Not differentiable: raises where
    autograd would follow an input (``gated_scan`` has gradients)."""
    if x.dim() != 2 or x.shape != g.shape:
        raise ValueError(f"x and g must both be [B, D], got {tuple(x.shape)} and {tuple(g.shape)}")
    if _differentiated(x, g, state):
        raise RuntimeError("step_gated_scan is not differentiable: call it under torch.no_grad(), "
                           "or gated_scan for gradients")
    dev = _require_same_device(x, g, state, out_state)
    B, D = x.shape
    state = _check_state(state, B, D, "state")
    new = torch.empty_like(state) if out_state is None else out_state
    if out_state is not None and (new.shape != (B, D) or new.dtype != torch.float32
                                  or not new.is_contiguous()):
        raise ValueError(f"out_state must be a contiguous float32 [{B}, {D}]")
    h = x.new_empty((B, D))
    if h.numel() == 0:
        return h, new
    a = _lib.ScanStepArgs()
    a.abi_version = _lib.ABI_VERSION
    a.B, a.D = B, D
    a.x, a.x_dtype, a.x_stride = x.data_ptr(), _code(x), x.stride()
    a.g, a.g_dtype, a.g_stride = g.data_ptr(), _code(g), g.stride()
    a.state_in, a.state_out, a.h = state.data_ptr(), new.data_ptr(), h.data_ptr()
    _launch(_lib.load().ngdn2_scan_step, a, dev, "ngdn2_scan_step")
    return h, new
