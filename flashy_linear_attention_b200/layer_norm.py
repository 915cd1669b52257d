"""Launch wrappers of layer norm (csrc/fla_layer_norm.cu), with or without a residual that is added first. The
reference has no counterpart.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import FlaLayerNormArgs
from .ops import _desc, untraced
from .recurrence import _DTYPES

MAX_DIM = 32768  # columns of a row


def check_inputs(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float,
                 residual: Optional[torch.Tensor] = None) -> None:
    """Device, type and shape rules of layer norm."""
    for t in (x, weight, bias, residual):
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("flashlinear: tensors must be CUDA tensors on an sm_100 GPU (no CPU fallback exists)")
        if t.device != x.device:
            raise RuntimeError("flashlinear: all tensors must be on the same device")
    if x.dtype not in _DTYPES:
        raise TypeError(f"flashlinear: expected bfloat16, float16 or float32 tensors, got {x.dtype}")
    if x.dim() < 1:
        raise ValueError("flashlinear: layer norm needs at least one dimension")
    dim = x.shape[-1]
    if dim > MAX_DIM:
        raise ValueError(f"flashlinear: layer norm takes rows of up to {MAX_DIM} columns, got {dim}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError("flashlinear: the residual must have x's shape and type")
    shapes = [(dim,)] + ([(x.shape[1], dim)] if x.dim() == 4 else [])
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if tuple(t.shape) not in shapes:
            raise ValueError(f"flashlinear: {name} must have shape " + " or ".join(str(s) for s in shapes)
                             + f" for x of shape {tuple(x.shape)}, got {tuple(t.shape)}")
        if t.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"flashlinear: {name} must be {x.dtype} as x is, or torch.float32, got {t.dtype}")
    if weight is not None and bias is not None and (weight.shape != bias.shape or weight.dtype != bias.dtype):
        raise ValueError("flashlinear: weight and bias must have the same shape and type")
    if not eps >= 0.0:
        raise ValueError(f"flashlinear: eps must not be negative, got {eps}")
    if dim and x.numel() // dim > 2**31 - 1:
        raise ValueError("flashlinear: layer norm takes up to 2^31 - 1 rows")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` as [batch, heads, tokens, dim] with neighbouring columns next to each other, which the kernels read."""
    t = t.resolve_neg()
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        t = t.contiguous()
    if t.dim() > 4:
        return t.reshape(-1, *t.shape[-3:])
    if t.dim() == 3:
        return t.unsqueeze(1)
    return t[(None,) * (4 - t.dim())]


def _out_like(t: torch.Tensor) -> torch.Tensor:
    out = torch.empty_like(t)
    if (out.stride(-1) != 1 and t.shape[-1] != 1) or t.dim() > 4:
        return torch.empty(t.shape, dtype=t.dtype, device=t.device)
    return out


def _args(x: torch.Tensor, weight, bias, eps: float) -> FlaLayerNormArgs:
    """`x` in the form of _rows()."""
    a = FlaLayerNormArgs()
    a.batch, a.heads, a.tokens, a.dim = x.shape
    params = weight if weight is not None else bias
    a.dtype = _DTYPES[x.dtype]
    a.w_dtype = a.dtype if params is None else _DTYPES[params.dtype]
    a.per_head = int(params is not None and params.dim() == 2)
    a.eps = eps
    a.x = _desc(x)
    a.weight = None if weight is None else weight.data_ptr()
    a.bias = None if bias is None else bias.data_ptr()
    return a


def _call(name: str, a: FlaLayerNormArgs, device: torch.device) -> None:
    with torch.cuda.device(device):
        a.stream = torch.cuda.current_stream(device).cuda_stream
        rc = getattr(_lib.load(), name)(ctypes.byref(a))
    if rc != 0:
        raise RuntimeError(f"flashlinear: {name} returned {rc}: {_lib.strerror(rc)}")


def _contiguous(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if t is None else t.resolve_neg().contiguous()


@untraced
def layer_norm_fwd(
    x: torch.Tensor,
    weight: Optional[torch.Tensor],
    bias: Optional[torch.Tensor],
    eps: float = 1e-5,
    residual: Optional[torch.Tensor] = None,
    keep_stats: bool = False,
) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(out, sum, stats): the normalised rows; x + residual as it was normalised, or None; and, with keep_stats, the
    fp32 mean and reciprocal deviation of every row, for layer_norm_bwd."""
    native = _lib.host() if x.is_cuda else None
    if native is not None:
        res = native.layer_norm_forward(x, weight, bias, eps, residual, keep_stats)
        if res is not None:
            return res
    check_inputs(x, weight, bias, eps, residual)
    weight, bias = _contiguous(weight), _contiguous(bias)
    like = x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()
    out, total = _out_like(like), None if residual is None else _out_like(like)
    rows = x.numel() // x.shape[-1] if x.shape[-1] else 0
    stats = torch.empty(rows, 2, dtype=torch.float32, device=x.device) if keep_stats else None
    if x.numel() == 0:
        return out, total, stats
    rx = _rows(x)
    a = _args(rx, weight, bias, eps)
    a.y = _desc(_rows(out))
    if residual is not None:
        rz = _rows(residual)
        a.residual, a.sum = _desc(rz), _desc(_rows(total))
    a.stats = None if stats is None else stats.data_ptr()
    _call("fla_sm100_layer_norm_fwd", a, x.device)
    return out, total, stats


@untraced
def layer_norm_bwd(
    grad_out: torch.Tensor,
    x: torch.Tensor,
    weight: Optional[torch.Tensor],
    bias: Optional[torch.Tensor],
    stats: torch.Tensor,
    grad_sum: Optional[torch.Tensor] = None,
    needs: Tuple[bool, bool, bool] = (True, True, True),
):
    """(d_x, d_weight, d_bias) for what layer_norm_fwd normalised: `x`, or the sum where there was a residual, to
    which d_x belongs as well, grad_sum included. `needs` says which results are wanted (the others are None); of bias only
    shape and type matter."""
    needs = (needs[0], needs[1] and weight is not None, needs[2] and bias is not None)
    native = _lib.host() if x.is_cuda else None
    if native is not None:
        res = native.layer_norm_backward(grad_out, x, weight, bias, stats, grad_sum, *needs)
        if res is not None:
            return res
    check_inputs(x, weight, bias, 0.0)
    weight = _contiguous(weight)
    like = x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()
    dx = _out_like(like) if needs[0] else None
    dw, db = (torch.empty(t.shape, dtype=t.dtype, device=t.device) if n else None
              for t, n in ((weight, needs[1]), (bias, needs[2])))
    if x.numel() == 0:
        return dx, *(None if t is None else t.zero_() for t in (dw, db))
    if not any(needs):
        return None, None, None
    if (not stats.is_cuda or stats.device != x.device or stats.dtype != torch.float32 or not stats.is_contiguous()
            or stats.numel() != 2 * (x.numel() // x.shape[-1])):
        raise ValueError("flashlinear: the backward needs the statistics of a forward over these rows with keep_stats=True")
    for g in (grad_out, grad_sum):
        if g is not None and (g.shape != x.shape or g.dtype != x.dtype or g.device != x.device):
            raise ValueError("flashlinear: gradients of the outputs must have their shape, type and device")
    rx, rg = _rows(x), _rows(grad_out)
    rs = None if grad_sum is None else _rows(grad_sum)
    a = _args(rx, weight, bias, 0.0)
    a.d_y, a.d_sum = _desc(rg), _desc(rs)
    a.d_x = _desc(None if dx is None else _rows(dx))
    a.d_weight = None if dw is None else dw.data_ptr()
    a.d_bias = None if db is None else db.data_ptr()
    a.stats = stats.data_ptr()
    with torch.cuda.device(x.device):
        need = _lib.load().fla_sm100_layer_norm_workspace_bytes(ctypes.byref(a))
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=x.device)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
    _call("fla_sm100_layer_norm_bwd", a, x.device)
    return dx, dw, db
