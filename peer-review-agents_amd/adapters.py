"""Low-rank adapters of many requests beside a shared projection, for serving:
every token of a batch adds its own request's adapter to the output of a
projection that all share (:func:`linear_w4`, or any other).  Formulas:
include/etmoe_dense.h; there is no CPU fallback."""
from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache
from typing import Optional

import torch

from ._lib import ET_MAX_ADAPTER_RANK, ET_MAX_ADAPTERS, lib
from .expert_threshold import _call, _require, _require_workspace
from .norm import _require_rows


@dataclass(frozen=True)
class AdapterBank:
    """The adapters of one projection: a bf16 [n, rank, K], b bf16 [n, N, rank] and
    a float32 scale [n] (alpha / rank); adapter i adds scale[i] * b[i] @ (a[i] @ x).
    rank is a multiple of 8, at most 128; adapters of lower rank have rows of a (and
    columns of b) of zeros.  The tensors are the caller's: a server writes an
    adapter into its place while others are in use."""

    a: torch.Tensor
    b: torch.Tensor
    scale: torch.Tensor

    def __post_init__(self) -> None:
        _require(self.a, "a", torch.bfloat16, 3)
        _require(self.b, "b", torch.bfloat16, 3, self.a.device)
        _require(self.scale, "scale", torch.float32, 1, self.a.device)
        n, rank, K = self.a.shape
        if self.b.shape[0] != n or self.b.shape[2] != rank:
            raise ValueError(f"b must have shape [{n}, N, {rank}], got {tuple(self.b.shape)}")
        if self.scale.shape[0] != n:
            raise ValueError(f"scale has {self.scale.shape[0]} entries, a has {n} adapters")
        if not 1 <= n <= ET_MAX_ADAPTERS:
            raise ValueError(f"there must be 1 to {ET_MAX_ADAPTERS} adapters, got {n}")
        if rank < 8 or rank % 8 or rank > ET_MAX_ADAPTER_RANK:
            raise ValueError(f"rank must be a positive multiple of 8, at most {ET_MAX_ADAPTER_RANK}, got {rank}")
        for name, size in (("K", K), ("N", self.b.shape[1])):
            if size < 8 or size % 8 or size >= 1 << 22:
                raise ValueError(f"{name} must be a positive multiple of 8 below 2^22, got {size}")
        if self.a.data_ptr() % 16 or self.b.data_ptr() % 16:
            raise ValueError("a and b must be 16-byte aligned")

    @property
    def num_adapters(self) -> int:
        return self.a.shape[0]

    @property
    def device(self) -> torch.device:
        return self.a.device


@dataclass(frozen=True)
class AdapterPlan:
    """A batch's tokens sorted by adapter (:func:`adapter_plan`): ``order`` [T], and
    ``items``, of which the first ``num_items`` [1] are valid."""

    order: torch.Tensor
    items: torch.Tensor
    num_items: torch.Tensor
    num_tokens: int
    num_adapters: int

    def __post_init__(self) -> None:
        most = int(lib().et_adapter_plan_items(self.num_tokens, self.num_adapters))
        if most < 0:
            raise ValueError(f"no plan of {self.num_tokens} tokens and {self.num_adapters} adapters")
        _require(self.order, "order", torch.int32, 1)
        _require(self.items, "items", torch.int32, 2, self.order.device)
        _require(self.num_items, "num_items", torch.int32, 1, self.order.device)
        if (self.order.shape[0] != self.num_tokens or self.items.shape[0] < most or self.items.shape[1] != 4
                or self.num_items.shape[0] != 1 or self.items.data_ptr() % 16):
            raise ValueError(f"a plan of {self.num_tokens} tokens and {self.num_adapters} adapters needs order "
                             f"[{self.num_tokens}], 16-byte aligned items [{most}, 4] and num_items [1]")

    @property
    def device(self) -> torch.device:
        return self.order.device


def adapter_plan(index: torch.Tensor, num_adapters: int) -> AdapterPlan:
    """Sorts a batch's tokens by adapter, once for all projections of a step.

    index int32 [T]: each token's adapter, 0 .. num_adapters - 1; any other value
    (-1) is none.  No host synchronisation.
    """
    _require(index, "index", torch.int32, 1)
    T, dev = index.shape[0], index.device
    if not 1 <= num_adapters <= ET_MAX_ADAPTERS:
        raise ValueError(f"num_adapters must be in [1, {ET_MAX_ADAPTERS}], got {num_adapters}")
    most = int(lib().et_adapter_plan_items(T, num_adapters))
    if most < 0:
        raise ValueError(f"index must have fewer than 2^30 entries, got {T}")
    # (one allocation: items, then order and their number)
    flat = torch.empty(4 * most + T + 1, dtype=torch.int32, device=dev)
    items, order, count = flat[:4 * most].view(most, 4), flat[4 * most:4 * most + T], flat[4 * most + T:]
    _call("et_adapter_plan", dev, index.data_ptr(), T, num_adapters, order.data_ptr(), items.data_ptr(), count.data_ptr())
    return AdapterPlan(order, items, count, T, num_adapters)


@lru_cache(maxsize=1024)
def _workspace_bytes(num_tokens: int, n: int, K: int, rank: int, device: int) -> int:
    # (the splits that it has room for go by the device's CUs)
    with torch.cuda.device(device):
        return int(lib().et_adapter_add_workspace_bytes(num_tokens, n, K, rank))


def adapter_add_workspace_bytes(num_tokens: int, bank: AdapterBank) -> int:
    n, rank, K = bank.a.shape
    return _workspace_bytes(num_tokens, n, K, rank, bank.a.get_device())


def _rows(t: torch.Tensor, name: str, rows: int, width: int, dev) -> int:
    """The row stride of a checked bf16 [rows, width]."""
    if (isinstance(t, torch.Tensor) and t.dtype == torch.bfloat16 and t.device == dev and t.shape == (rows, width)
            and t.is_contiguous()):
        stride = width
    else:
        stride = _require_rows(t, name, torch.bfloat16, torch.Size((rows, width)), dev)
    if stride % 8 or t.data_ptr() % 16:
        raise ValueError(f"{name} must be 16-byte aligned and its rows a multiple of 8 elements apart")
    return stride


def adapter_add(y: torch.Tensor, x: torch.Tensor, bank: AdapterBank, plan: AdapterPlan, *,
                out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[t] = y[t] + scale[i] * b[i] @ (a[i] @ x[t]), i token t's adapter; out[t] =
    y[t] for a token without one.

    y bf16 [T, N] (the shared projection of x), x bf16 [T, K]: rows contiguous,
    multiples of 8 elements apart.  ``out`` may be y (in place); a new tensor
    by default.  Binary32 sums (the inner one kept to 16 bits), one rounding,
    identical bits on repeated calls.
    """
    if not isinstance(bank, AdapterBank) or not isinstance(plan, AdapterPlan):
        raise TypeError("bank must be an AdapterBank and plan an AdapterPlan")
    a, b, order = bank.a, bank.b, plan.order
    n, rank, K = a.shape
    N, T, dev = b.shape[1], plan.num_tokens, a.device
    if plan.num_adapters != n:
        raise ValueError(f"the plan is of {plan.num_adapters} adapters, the bank has {n}")
    if order.device != dev:
        raise ValueError(f"the plan is on {order.device}, the bank on {dev}")
    ldy, ldx = _rows(y, "y", T, N, dev), _rows(x, "x", T, K, dev)
    if out is None:
        out, ldo = y.new_empty((T, N)), N
    else:
        ldo = _rows(out, "out", T, N, dev)
    wsb = _workspace_bytes(T, n, K, rank, a.get_device())
    if workspace is None:
        workspace = y.new_empty(wsb >> 1)       # (bf16 elements)
    else:
        _require_workspace(workspace, wsb, dev, "workspace")
    _call("et_adapter_add", dev, y.data_ptr(), ldy, x.data_ptr(), ldx, a.data_ptr(), b.data_ptr(), bank.scale.data_ptr(),
          order.data_ptr(), plan.items.data_ptr(), plan.num_items.data_ptr(), T, n, K, N, rank, out.data_ptr(), ldo,
          workspace.data_ptr(), wsb)
    return out
