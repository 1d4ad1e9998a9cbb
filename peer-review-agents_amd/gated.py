"""The gated projection of a dense expert -- a shared expert, that every token
takes beside its routed ones -- and its backward.  Arguments are checked in
Python, each call is one library call on torch's current stream
(include/etmoe_dense.h has the formulas); there is no CPU fallback."""
from __future__ import annotations

from functools import lru_cache
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from ._lib import ET_DTYPE_BF16, ET_DTYPE_F32, ET_GATED_GELU, ET_GATED_SILU, lib
from .expert_threshold import _call, _out_or_new, _require, _require_workspace
from .norm import _require_rows

_ACTIVATIONS = {"silu": ET_GATED_SILU, "gelu": ET_GATED_GELU}


def _check(x: torch.Tensor, w: torch.Tensor, activation: str):
    """(activation, rows, K, F, row stride of x) of checked operands."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    if isinstance(x, torch.Tensor) and x.is_cuda and x.dtype == torch.bfloat16 and x.dim() == 2 and x.is_contiguous():
        stride = x.shape[1]
    else:
        stride = _require_rows(x, "x", torch.bfloat16)
    _require(w, "w", torch.bfloat16, 2, x.device)
    rows, K = x.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise ValueError(f"x has row length {K}, w has {w.shape[1]}")
    if K < 8 or K % 8 or K >= 1 << 21:
        raise ValueError(f"K must be a positive multiple of 8 below 2^21, got {K}")
    if N < 16 or N % 16 or N >= 1 << 21:
        raise ValueError(f"w must have a positive multiple of 16 rows (gate rows, then up rows) below 2^21, got {N}")
    if N * K * 2 >= 1 << 31:
        raise ValueError("w must be below 2 GiB")
    if stride % 8 or stride >= 1 << 22 or x.data_ptr() % 16 or w.data_ptr() % 16:
        raise ValueError("x and w must be 16-byte aligned, and the rows of x a multiple of 8 elements (below 2^22) apart")
    return _ACTIVATIONS[activation], rows, K, N // 2, stride


def _aligned(t: torch.Tensor, name: str) -> int:
    at = t.data_ptr()
    if at % 16:
        raise ValueError(f"{name} must be 16-byte aligned")
    return at


def gated_linear(x: torch.Tensor, w: torch.Tensor, *, activation: str = "silu",
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """h = act(x Wg^T) * (x Wu^T), bf16 [T, F], in one kernel.

    x bf16 [T, K], rows contiguous, a multiple of 8 elements apart; w bf16
    [2F, K], the gate rows and then the up rows (an expert's layout in
    :func:`expert_gemm`).  ``activation`` "silu" or "gelu" (g Phi(g)).  Binary32
    sums, one rounding, identical bits on repeated calls.
    """
    act, rows, K, F, stride = _check(x, w, activation)
    h = x.new_empty((rows, F)) if out is None else _out_or_new(out, (rows, F), torch.bfloat16, x.device, "out")
    _call("et_gated_linear", x.device, x.data_ptr(), stride, w.data_ptr(), rows, K, F, act, _aligned(h, "out"))
    return h


def _own_place(dh: torch.Tensor) -> torch.Tensor:
    """A gradient as the library reads it: autograd may hand over a view of another tensor, from
    any element on."""
    dh = dh.contiguous()
    return dh if dh.data_ptr() % 16 == 0 else dh.clone()


@lru_cache(maxsize=1024)
def _workspace_bytes(rows: int, K: int, F: int, device: int) -> int:
    # (the splits that it has room for go by the device's CUs)
    with torch.cuda.device(device):
        return int(lib().et_gated_linear_bwd_workspace_bytes(rows, K, F))


def gated_linear_backward_workspace_bytes(rows: int, K: int, F: int, device=None) -> int:
    """Bytes that :func:`gated_linear_backward` works in on ``device`` (the current one by default)."""
    if device is None:
        return int(lib().et_gated_linear_bwd_workspace_bytes(rows, K, F))
    index = torch.device(device).index
    if index is None:
        raise ValueError(f"device must name one of the devices, got {device!r}")
    return _workspace_bytes(rows, K, F, index)


def gated_linear_backward(dh: torch.Tensor, x: torch.Tensor, w: torch.Tensor, *, activation: str = "silu",
                          need_dx: bool = True, need_dw: bool = True, out_dx: Optional[torch.Tensor] = None,
                          out_dw: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None):
    """(dx, dw) of :func:`gated_linear` from dh [T, F] and the forward's x and w
    alone: the projections are computed again, so nothing of size [T, F] has to
    be kept for it.

    dx bf16 [T, K]; dw bf16 [2F, K], or float32 in a float32 ``out_dw``.  The
    projections' gradient is rounded to bf16 once, between the products.  None
    for a gradient that is not needed.
    """
    act, rows, K, F, stride = _check(x, w, activation)
    dev = x.device
    _require(dh, "dh", torch.bfloat16, 2, dev)
    if tuple(dh.shape) != (rows, F):
        raise ValueError(f"dh must have shape {(rows, F)}, got {tuple(dh.shape)}")
    dx = dw = None
    if need_dx or out_dx is not None:
        dx = _out_or_new(out_dx, (rows, K), torch.bfloat16, dev, "out_dx")
    if need_dw or out_dw is not None:
        kind = torch.float32 if isinstance(out_dw, torch.Tensor) and out_dw.dtype == torch.float32 else torch.bfloat16
        dw = _out_or_new(out_dw, (2 * F, K), kind, dev, "out_dw")
    wsb = _workspace_bytes(rows, K, F, x.get_device())
    if workspace is None:
        workspace = torch.empty(wsb, dtype=torch.uint8, device=dev)
    else:
        _require_workspace(workspace, wsb, dev, "workspace")
    _call("et_gated_linear_bwd", dev, _aligned(dh, "dh"), x.data_ptr(), stride, w.data_ptr(), rows, K, F, act,
          None if dx is None else _aligned(dx, "out_dx"), None if dw is None else _aligned(dw, "out_dw"),
          ET_DTYPE_F32 if dw is not None and dw.dtype == torch.float32 else ET_DTYPE_BF16,
          _aligned(workspace, "workspace"), workspace.numel() * workspace.element_size())
    return dx, dw


class _GatedLinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, activation):
        ctx.save_for_backward(x, w)
        ctx.activation = activation
        return gated_linear(x, w, activation=activation)

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x, w = ctx.saved_tensors
        need_dx, need_dw, _ = ctx.needs_input_grad
        dx, dw = gated_linear_backward(_own_place(dh), x, w, activation=ctx.activation, need_dx=need_dx, need_dw=need_dw)
        return dx, dw, None


def gated_linear_autograd(x: torch.Tensor, w: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """:func:`gated_linear` with a backward that runs :func:`gated_linear_backward`.
    A second derivative raises."""
    return _GatedLinearFn.apply(x, w, activation)
