"""Launch wrappers of the gated linear recurrence (csrc/fla_recurrence.cu):
``h_t = exp(log_decay_t) h_{t-1} + x_t`` for every channel, over [batch, heads, seq, dim] tensors with an fp32
state before and behind them. The reference has no counterpart.
"""
from __future__ import annotations

import ctypes
import os
from typing import Optional, Tuple

import torch

from . import _lib, ops
from ._lib import FlaRecurrenceArgs
from .ops import _desc, untraced

_DTYPES = {
    torch.bfloat16: _lib.FLA_DTYPE_BF16,
    torch.float16: _lib.FLA_DTYPE_F16,
    torch.float32: _lib.FLA_DTYPE_F32,
}

MAX_SIZE = 2**30  # tokens, channels of a head, heads of all sequences


def _check_state(s: Optional[torch.Tensor], name: str, x: torch.Tensor) -> None:
    if s is None:
        return
    want = (x.shape[0], x.shape[1], x.shape[3])
    if tuple(s.shape) != want:
        raise ValueError(f"flashlinear: {name} must have shape {want}, got {tuple(s.shape)}")
    if s.device != x.device:
        raise RuntimeError("flashlinear: all tensors must be on the same device")
    if not s.is_floating_point():
        raise TypeError(f"flashlinear: {name} must be a floating-point tensor, got {s.dtype}")


def check_inputs(x: torch.Tensor, log_decay: torch.Tensor, s_init: Optional[torch.Tensor] = None) -> None:
    """Device, type and shape rules of the recurrence."""
    for t in (x, log_decay):
        if not t.is_cuda:
            raise RuntimeError("flashlinear: tensors must be CUDA tensors on an sm_100 GPU (no CPU fallback exists)")
    if x.device != log_decay.device:
        raise RuntimeError("flashlinear: all tensors must be on the same device")
    if x.dtype not in _DTYPES:
        raise TypeError(f"flashlinear: expected bfloat16, float16 or float32 tensors, got {x.dtype}")
    if log_decay.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"flashlinear: log_decay must be {x.dtype} as x is, or torch.float32, got {log_decay.dtype}")
    if x.dim() != 4:
        raise ValueError("flashlinear: expected [batch, heads, seq, dim] tensors")
    if log_decay.shape != x.shape:
        raise ValueError(f"flashlinear: x and log_decay must have the same shape, got {tuple(x.shape)} and "
                         f"{tuple(log_decay.shape)} (expand a gate that channels, heads or tokens share)")
    B, H, N, D = x.shape
    if x.numel() and max(B * H, N, D) > MAX_SIZE:
        raise ValueError(f"flashlinear: the recurrence takes up to 2^30 tokens, 2^30 channels a head and 2^30 heads of all "
                         f"sequences, got {tuple(x.shape)}")
    _check_state(s_init, "s_init", x)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` as the kernels read it: neighbouring columns next to each other in memory, no lazy sign."""
    t = t.resolve_neg()
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _state(s: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if s is None else s.resolve_neg().to(torch.float32).contiguous()


def _out_like(t: torch.Tensor) -> torch.Tensor:
    out = torch.empty_like(t)
    return out if out.stride(3) == 1 or t.shape[3] == 1 else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _args(x: torch.Tensor, g: torch.Tensor) -> FlaRecurrenceArgs:
    a = FlaRecurrenceArgs()
    a.batch, a.heads, a.seqlen, a.dim = x.shape
    a.dtype, a.g_dtype = _DTYPES[x.dtype], _DTYPES[g.dtype]
    a.x, a.g = _desc(x), _desc(g)
    return a


def _call(name: str, a: FlaRecurrenceArgs, device: torch.device) -> None:
    with torch.cuda.device(device):
        a.stream = torch.cuda.current_stream(device).cuda_stream
        a.status, a.debug_flags = ops._status_word(device).data_ptr(), ops._debug_flags
        rc = getattr(_lib.load(), name)(ctypes.byref(a))
    if rc != 0:
        raise RuntimeError(f"flashlinear: {name} returned {rc}: {_lib.strerror(rc)}")
    _debug_check(device)


def _debug_check(device: torch.device) -> None:
    if os.environ.get("FLA_DEBUG", "0") == "1":
        ops.check_status(device)


@untraced
def recurrence_fwd(
    x: torch.Tensor, log_decay: torch.Tensor, s_init: Optional[torch.Tensor] = None, keep_states: bool = False
) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """(out, s_final, states): h_t for every token in x's type, the fp32 [batch, heads, dim] state behind the last
    token, and, with keep_states, what recurrence_bwd needs of the pass (a byte buffer private to the library)."""
    native = _lib.host() if x.is_cuda else None
    if native is not None:
        res = native.recurrence_forward(x, log_decay, s_init, keep_states, ops._debug_flags, ops._status_ptr(x))
        if res is not None:
            _debug_check(x.device)
            return res
    check_inputs(x, log_decay, s_init)
    B, H, N, D = x.shape
    s_init = _state(s_init)
    x, g = _rows(x), _rows(log_decay)
    out = _out_like(x)
    if x.numel() == 0:
        s_final = torch.zeros(B, H, D, dtype=torch.float32, device=x.device) if s_init is None else s_init.clone()
        return out, s_final, None
    s_final = torch.empty(B, H, D, dtype=torch.float32, device=x.device)
    a = _args(x, g)
    a.o = _desc(out)
    a.s_init, a.s_final = None if s_init is None else s_init.data_ptr(), s_final.data_ptr()
    states = None
    if keep_states:
        a.states_bytes = _lib.load().fla_sm100_recurrence_states_bytes(ctypes.byref(a))
        states = torch.empty(a.states_bytes, dtype=torch.uint8, device=x.device)
        a.states = states.data_ptr()
    _call("fla_sm100_recurrence_fwd", a, x.device)
    return out, s_final, states


@untraced
def recurrence_bwd(
    grad_out: Optional[torch.Tensor],
    x: torch.Tensor,
    log_decay: torch.Tensor,
    states: Optional[torch.Tensor],
    grad_s_final: Optional[torch.Tensor] = None,
    needs: Tuple[bool, bool, bool] = (True, True, True),
):
    """(d_x, d_log_decay, d_s_init) of recurrence_fwd(x, log_decay, ..., keep_states=True), whose `states` are handed
    back here. None for a gradient of the outputs is zero; `needs` says which results are wanted (the others are None)."""
    native = _lib.host() if x.is_cuda else None
    if native is not None:
        res = native.recurrence_backward(grad_out, x, log_decay, states, grad_s_final, *needs, ops._debug_flags, ops._status_ptr(x))
        if res is not None:
            _debug_check(x.device)
            return res
    check_inputs(x, log_decay, grad_s_final)
    B, H, N, D = x.shape
    r_init = _state(grad_s_final)
    x, g = _rows(x), _rows(log_decay)
    dx = _out_like(x) if needs[0] else None
    dg = _out_like(g) if needs[1] else None
    ds = torch.empty(B, H, D, dtype=torch.float32, device=x.device) if needs[2] else None
    if x.numel() == 0:
        if ds is not None:
            ds = torch.zeros_like(ds) if r_init is None else r_init.clone()
        return dx, dg, ds
    if not any(needs):
        return None, None, None
    if states is None:
        raise ValueError("flashlinear: the backward needs the states of a forward with keep_states=True")
    if not states.is_cuda or states.device != x.device or not states.is_contiguous():
        raise ValueError("flashlinear: the states of the forward must be contiguous and on the device of x")
    a = _args(x, g)
    if grad_out is not None:
        if grad_out.shape != x.shape or grad_out.dtype != x.dtype or grad_out.device != x.device:
            raise ValueError("flashlinear: the gradient of the output must have its shape, type and device")
        grad_out = _rows(grad_out)
    a.d_o, a.d_x, a.d_g = _desc(grad_out), _desc(dx), _desc(dg)
    a.r_init = None if r_init is None else r_init.data_ptr()
    a.r_final = None if ds is None else ds.data_ptr()
    a.states, a.states_bytes = states.data_ptr(), states.numel() * states.element_size()
    _call("fla_sm100_recurrence_bwd", a, x.device)
    return dx, dg, ds
