"""Layer norm over rows, with the residual add before it, and its backward: the
norm in front of an MoE block.  Arguments are checked in Python, each call is
one library call on torch's current stream (include/etmoe_block.h has the
formulas); there is no CPU fallback."""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from ._lib import ET_MAX_NORM_WIDTH, lib
from .expert_threshold import (_ACT_DTYPES, _act_dtype, _call, _out_or_new, _require, _require_device,
                               _require_workspace, _vp)


def _require_rows(t, name: str, dtype=None, shape=None, device=None) -> int:
    """A 2-D tensor of rows: dense ones, any row stride.  Returns the stride."""
    _require_device(t, name)
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D [rows, d], got shape {tuple(t.shape)}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    rows, d = t.shape
    along, inner = t.stride()
    if (inner != 1 and d > 1) or (along < d and rows > 1):
        raise ValueError(f"the rows of {name} must be contiguous and must not overlap, got strides {t.stride()}")
    return max(along, d)


def _dense_rows(t, dtype, shape, device) -> bool:
    return (isinstance(t, torch.Tensor) and t.is_cuda and t.dim() == 2 and t.dtype == dtype and t.shape == shape
            and t.device == device and t.is_contiguous())


def _stat(t, h) -> bool:
    return (isinstance(t, torch.Tensor) and t.dtype == torch.float32 and t.device == h.device and t.is_contiguous()
            and t.shape == h.shape[:1])


def _new_rows(out, x, name: str):
    """`out` checked, or new dense rows like x."""
    if out is None:
        return torch.empty_like(x, memory_format=torch.contiguous_format)
    return _out_or_new(out, tuple(x.shape), x.dtype, x.device, name)


def _check_width(d: int) -> None:
    if not 1 <= d <= ET_MAX_NORM_WIDTH:
        raise ValueError(f"d must be in [1, {ET_MAX_NORM_WIDTH}], got {d}")


def _require_weight(w, name: str, d: int, dtype, device) -> int:
    _require_device(w, name)
    if w.dtype != torch.float32 and w.dtype != dtype:
        raise TypeError(f"{name} must be float32 or {dtype}, got {w.dtype}")
    _require(w, name, w.dtype, 1, device)
    if w.shape[0] != d:
        raise ValueError(f"{name} has {w.shape[0]} entries, the rows have {d}")
    return _act_dtype(w, name)


def layer_norm(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, eps: float = 1e-5,
               residual: Optional[torch.Tensor] = None, stats: bool = False, out: Optional[torch.Tensor] = None,
               out_sum: Optional[torch.Tensor] = None):
    """y = (h - mean) * rstd * weight + bias over the rows of h = x (+ residual).

    x [rows, d] f32 or bf16, rows contiguous at any stride; weight and bias [d]
    of x's type or float32.  With ``residual`` (x's type) the sum is rounded to
    x's type and returned behind y; with ``stats`` so are mean and rstd (f32
    [rows]), for :func:`layer_norm_backward`:
        y | (y, sum) | (y, mean, rstd) | (y, sum, mean, rstd)
    Binary32 arithmetic, one rounding of y, identical bits on repeated calls.
    """
    if not isinstance(x, torch.Tensor) or not isinstance(weight, torch.Tensor):
        raise TypeError("x and weight must be torch.Tensors")
    dev, dtype = x.device, x.dtype
    # (a call on a few rows takes 4 us on the device: dense tensors pass one test)
    if (x.is_cuda and x.dim() == 2 and x.is_contiguous() and dtype in _ACT_DTYPES and weight.dim() == 1
            and weight.is_contiguous() and weight.device == dev and weight.shape[0] == x.shape[1] <= ET_MAX_NORM_WIDTH
            and (weight.dtype == dtype or weight.dtype == torch.float32)
            and (bias is None or (bias.dtype == weight.dtype and bias.device == dev and bias.is_contiguous()
                                  and bias.shape == weight.shape)) and x.shape[1]):
        rows, d = x.shape
        ldx, dt, wdt = d, _ACT_DTYPES[dtype], _ACT_DTYPES[weight.dtype]
    else:
        ldx = _require_rows(x, "x")
        dt = _act_dtype(x, "x")
        rows, d = x.shape
        _check_width(d)
        wdt = _require_weight(weight, "weight", d, dtype, dev)
        if bias is not None and _require_weight(bias, "bias", d, dtype, dev) != wdt:
            raise TypeError("weight and bias must have the same dtype")
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"eps must be finite and >= 0, got {eps}")
    ldr = 0
    if residual is not None:
        if residual.dtype == dtype and residual.shape == x.shape and residual.device == dev and residual.is_contiguous():
            ldr = d
        else:
            ldr = _require_rows(residual, "residual", dtype, x.shape, dev)
        out_sum = _new_rows(out_sum, x, "out_sum")
    elif out_sum is not None:
        raise ValueError("out_sum needs a residual")
    y = _new_rows(out, x, "out")
    if stats:
        mean, rstd = (torch.empty(rows, dtype=torch.float32, device=dev) for _ in range(2))
    else:
        mean = rstd = None
    _call("et_layer_norm_fwd", dev, x.data_ptr(), ldx, None if residual is None else residual.data_ptr(), ldr,
          weight.data_ptr(), None if bias is None else bias.data_ptr(), rows, d, dt, wdt, eps, y.data_ptr(),
          None if residual is None else out_sum.data_ptr(), _vp(mean), _vp(rstd))
    if residual is None:
        return (y, mean, rstd) if stats else y
    return (y, out_sum, mean, rstd) if stats else (y, out_sum)


def layer_norm_backward_workspace_bytes(rows: int, d: int) -> int:
    return int(lib().et_layer_norm_bwd_workspace_bytes(rows, d))


def layer_norm_backward(dy: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, mean: torch.Tensor,
                        rstd: torch.Tensor, *, dsum: Optional[torch.Tensor] = None, need_dbias: bool = True,
                        out_dx: Optional[torch.Tensor] = None, out_dweight: Optional[torch.Tensor] = None,
                        out_dbias: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None):
    """(dx, dweight, dbias) of :func:`layer_norm`, h being its x, or the sum it
    returned; dx is then the gradient of x and of the residual alike.

    ``dsum`` (h's type) is added to dx: the gradient that reaches the sum past
    the norm.  dx has h's type, dweight and dbias are f32 [d] (dbias None
    without ``need_dbias``).
    """
    dev, dtype = h.device, h.dtype
    if not (_dense_rows(h, dtype, h.shape, dev) and dtype in _ACT_DTYPES and weight.is_contiguous()
            and weight.device == dev and weight.shape == h.shape[1:] and 0 < h.shape[1] <= ET_MAX_NORM_WIDTH
            and (weight.dtype == dtype or weight.dtype == torch.float32) and _stat(mean, h) and _stat(rstd, h)):
        _require_rows(h, "h")
        _act_dtype(h, "h")
        _check_width(h.shape[1])
        _require_weight(weight, "weight", h.shape[1], dtype, dev)
        for t, name in ((mean, "mean"), (rstd, "rstd")):
            _require(t, name, torch.float32, 1, dev)
            if t.shape[0] != h.shape[0]:
                raise ValueError(f"{name} has {t.shape[0]} entries, h has {h.shape[0]} rows")
    rows, d = h.shape
    ldh = d if h.is_contiguous() else _require_rows(h, "h")
    lddy = d if _dense_rows(dy, dtype, h.shape, dev) else _require_rows(dy, "dy", dtype, h.shape, dev)
    ldds = 0
    if dsum is not None:
        ldds = d if _dense_rows(dsum, dtype, h.shape, dev) else _require_rows(dsum, "dsum", dtype, h.shape, dev)
    dx = _new_rows(out_dx, h, "out_dx")
    dweight = mean.new_empty(d) if out_dweight is None else _out_or_new(out_dweight, (d,), torch.float32, dev,
                                                                        "out_dweight")
    dbias = None
    if out_dbias is not None:
        dbias = _out_or_new(out_dbias, (d,), torch.float32, dev, "out_dbias")
    elif need_dbias:
        dbias = mean.new_empty(d)
    wsb = layer_norm_backward_workspace_bytes(rows, d)
    if workspace is None:
        workspace = mean.new_empty(wsb // 4)
    else:
        _require_workspace(workspace, wsb, dev, "workspace")
    _call("et_layer_norm_bwd", dev, dy.data_ptr(), lddy, h.data_ptr(), ldh, _vp(dsum), ldds, weight.data_ptr(),
          mean.data_ptr(), rstd.data_ptr(), rows, d, _ACT_DTYPES[dtype], _ACT_DTYPES[weight.dtype], dx.data_ptr(),
          dweight.data_ptr(), _vp(dbias), workspace.data_ptr(), wsb)
    return dx, dweight, dbias


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, residual):
        r = layer_norm(x, weight, bias, eps=eps, residual=residual, stats=True)
        y, mean, rstd = r[0], r[-2], r[-1]
        h = x if residual is None else r[1]
        ctx.save_for_backward(h, weight, mean, rstd)
        ctx.has = bias is not None, residual is not None
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dsum=None):
        h, weight, mean, rstd = ctx.saved_tensors
        has_bias, has_residual = ctx.has
        if dy is None:          # only the sum was used
            return dsum, None, None, None, dsum if has_residual else None
        dx, dw, db = layer_norm_backward(dy.contiguous(), h, weight, mean, rstd,
                                         dsum=None if dsum is None else dsum.contiguous(), need_dbias=has_bias)
        return (dx, dw.to(weight.dtype), db.to(weight.dtype) if has_bias else None, None,
                dx if has_residual else None)


def layer_norm_autograd(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                        eps: float = 1e-5, residual: Optional[torch.Tensor] = None):
    """:func:`layer_norm` (y, or (y, sum) with a residual) with a backward that
    runs :func:`layer_norm_backward`.  A second derivative raises."""
    return _LayerNormFn.apply(x, weight, bias, eps, residual)
