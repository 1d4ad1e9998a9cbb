"""Products with 4-bit weights and group scales, for serving: the experts'
projections over a routing plan and a dense layer's, where a few tokens at a
time make the reading of the weights the work.  Formulas and layout:
include/etmoe_block.h; there is no CPU fallback."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from ._lib import ET_MAX_EXPERTS, lib
from .expert_threshold import (_EPILOGUES, RoutingPlan, _act_dtype, _call, _check_plan, _known_counts, _out_or_new,
                               _require, _require_device, _vp)

_SCALE_TYPES = {torch.bfloat16: 0, torch.float16: 1}
_GROUPS = (32, 64, 128)


@dataclass
class W4Weight:
    """A 4-bit weight as the products read it: w = (q - 8) * scale of E experts
    (1: a dense layer), N rows, K columns, ``group`` columns to a scale.  Made by
    :func:`pack_w4`; ``packed`` and ``scales`` are its layout, not for indexing, and
    that of one version of the library (a pickle of another version's raises)."""

    packed: torch.Tensor
    scales: torch.Tensor
    num_experts: int
    N: int
    K: int
    group: int
    parts: int

    def __getstate__(self) -> dict:
        return {**self.__dict__, "layout": lib().et_block_abi_version()}

    def __setstate__(self, state: dict) -> None:
        state = dict(state)
        if state.pop("layout", None) != lib().et_block_abi_version():
            raise ValueError("the weight was packed by another version of the library: pack its values and scales again")
        self.__dict__.update(state)

    def __post_init__(self) -> None:
        # (the products read as much as these sizes say)
        _check_sizes(self.num_experts, self.N, self.K, self.group, self.parts)
        L = lib()
        for t, name, dtypes, n in (
                (self.packed, "packed", (torch.uint8,), L.et_w4_packed_bytes(self.num_experts, self.N, self.K, self.parts)),
                (self.scales, "scales", tuple(_SCALE_TYPES),
                 L.et_w4_packed_scales(self.num_experts, self.N, self.K, self.group, self.parts))):
            if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
                raise TypeError(f"{name} must be a tensor of {' or '.join(map(str, dtypes))}")
            if not t.is_contiguous() or t.numel() != n:
                raise ValueError(f"{name} must be contiguous with {n} elements, got shape {tuple(t.shape)}")
            if t.data_ptr() % 16:
                raise ValueError(f"{name} must be 16-byte aligned")
        if self.scales.device != self.packed.device:
            raise ValueError(f"scales are on {self.scales.device}, packed is on {self.packed.device}")

    @property
    def device(self) -> torch.device:
        return self.packed.device


def _check_sizes(E: int, N: int, K: int, group: int, parts: int) -> None:
    if not 1 <= E <= ET_MAX_EXPERTS:
        raise ValueError(f"num_experts must be in [1, {ET_MAX_EXPERTS}], got {E}")
    if parts not in (1, 2):
        raise ValueError(f"parts must be 1 or 2, got {parts}")
    if N < 8 * parts or N % (8 * parts):
        raise ValueError(f"N must be a positive multiple of 8 for each of {parts} parts, got {N}")
    if K < 8 or K % 8 or K >= 1 << 22:
        raise ValueError(f"K must be a positive multiple of 8 below 2^22, got {K}")
    if group not in _GROUPS:
        raise ValueError(f"group must be one of {_GROUPS}, got {group}")
    if N * K >= 1 << 31 or N >= 1 << 22:
        raise ValueError("N * K must be below 2^31 and N below 2^22")


def quantize_w4(w: torch.Tensor, *, group: int = 128,
                scale_dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """(q, scales) of a weight w [E, N, K] or [N, K] (f32 or bf16): for each group
    of a row scale = max(largest / 7, -smallest / 8) in ``scale_dtype`` and
    q = 8 + w / scale rounded to nearest, held to 0..15.  q uint8 [..., N, K / 2],
    the even column in the low half; scales [..., N, ceil(K / group)]."""
    _require_device(w, "w")
    dt = _act_dtype(w, "w")
    if w.dim() not in (2, 3) or not w.is_contiguous():
        raise ValueError("w must be a contiguous [E, N, K] or [N, K] tensor")
    if scale_dtype not in _SCALE_TYPES:
        raise TypeError(f"scale_dtype must be bfloat16 or float16, got {scale_dtype}")
    *lead, N, K = w.shape
    E = lead[0] if lead else 1
    _check_sizes(E, N, K, group, 1)
    q = torch.empty(*lead, N, K // 2, dtype=torch.uint8, device=w.device)
    scales = torch.empty(*lead, N, -(-K // group), dtype=scale_dtype, device=w.device)
    _call("et_w4_quantize", w.device, _vp(w), dt, E, N, K, group, _SCALE_TYPES[scale_dtype], _vp(q), _vp(scales))
    return q, scales


def pack_w4(q: torch.Tensor, scales: torch.Tensor, *, group: int = 128, parts: int = 1) -> W4Weight:
    """Lays a 4-bit weight out for the products, once.  q uint8 [E, N, K / 2] (or
    [N, K / 2], a dense layer), two values of 0..15 to a byte, the even column in
    the low half; scales bf16 or f16 [..., N, ceil(K / group)].  ``parts=2`` for a weight
    of gate rows and up rows that is to run with ``epilogue="swiglu"``."""
    _require_device(q, "q")
    if q.dtype != torch.uint8:
        raise TypeError(f"q must be uint8, got {q.dtype}")
    if q.dim() not in (2, 3):
        raise ValueError(f"q must be [E, N, K / 2] or [N, K / 2], got shape {tuple(q.shape)}")
    dev = q.device
    if scales.dtype not in _SCALE_TYPES:
        raise TypeError(f"scales must be bfloat16 or float16, got {scales.dtype}")
    _require(q, "q", torch.uint8, q.dim(), dev)
    _require(scales, "scales", scales.dtype, q.dim(), dev)
    *lead, N, half = q.shape
    E, K = (lead[0] if lead else 1), 2 * half
    _check_sizes(E, N, K, group, parts)
    if tuple(scales.shape) != (*lead, N, -(-K // group)):
        raise ValueError(f"scales must have shape {(*lead, N, -(-K // group))}, got {tuple(scales.shape)}")
    L = lib()
    packed = torch.empty(int(L.et_w4_packed_bytes(E, N, K, parts)), dtype=torch.uint8, device=dev)
    laid = torch.empty(int(L.et_w4_packed_scales(E, N, K, group, parts)), dtype=scales.dtype, device=dev)
    _call("et_w4_pack", dev, _vp(q), _vp(scales), E, N, K, group, parts, _vp(packed), _vp(laid))
    return W4Weight(packed, laid, E, N, K, group, parts)


def _check_weight(w: W4Weight, dev) -> None:
    if not isinstance(w, W4Weight):
        raise TypeError("the weight must be a W4Weight (pack_w4)")
    if w.device != dev:
        raise ValueError(f"the weight is on {w.device}, expected {dev}")


def unpack_w4(w: W4Weight, plan: Optional[RoutingPlan] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The weight as bf16 [E, N, K], each value rounded once; with a plan only
    the experts with slots (the others' blocks of ``out`` are left as they were)."""
    _check_weight(w, w.packed.device)
    dev = w.device
    if plan is not None:
        _check_plan(plan, dev)
        if plan.num_experts != w.num_experts:
            raise ValueError(f"w has {w.num_experts} experts, plan has {plan.num_experts}")
    out = _out_or_new(out, (w.num_experts, w.N, w.K), torch.bfloat16, dev, "out")
    _call("et_w4_unpack", dev, _vp(w.packed), _vp(w.scales), _SCALE_TYPES[w.scales.dtype],
          None if plan is None else _vp(plan.expert_offsets), w.num_experts, w.N, w.K, w.group, w.parts,
          0 if plan is None else plan.rows, _vp(out))
    return out


def _gemm(a, w: W4Weight, rows: int, sorted_token, offsets, epilogue: str, row_scale, out, max_slots: int,
          route: int = -1, known: int = 1):
    dev = a.device
    if epilogue not in _EPILOGUES:
        raise ValueError(f"epilogue must be one of {sorted(_EPILOGUES)}, got {epilogue!r}")
    if a.shape[1] != w.K:
        raise ValueError(f"a has row length {a.shape[1]}, w has K = {w.K}")
    swiglu = epilogue == "swiglu"
    if swiglu and w.parts != 2:
        raise ValueError("the swiglu epilogue needs a weight packed with parts=2")
    if epilogue == "row_scale":
        if row_scale is None:
            raise ValueError("the row_scale epilogue needs row_scale")
        _require(row_scale, "row_scale", torch.float32, 1, dev)
        if row_scale.shape[0] < rows:
            raise ValueError(f"row_scale has {row_scale.shape[0]} entries, out has {rows} rows")
    shape = (rows, w.N // 2 if swiglu else w.N)
    c = a.new_empty(shape) if out is None else _out_or_new(out, shape, torch.bfloat16, dev, "out")
    at, to = a.data_ptr(), c.data_ptr()
    if at % 16 or to % 16:
        raise ValueError("a and out must be 16-byte aligned")
    _call("et_expert_gemm_w4_impl", dev, at, a.shape[0], sorted_token, w.packed.data_ptr(), w.scales.data_ptr(),
          _SCALE_TYPES[w.scales.dtype], offsets, w.num_experts, w.K, w.N, w.group, w.parts, rows, _EPILOGUES[epilogue],
          row_scale.data_ptr() if epilogue == "row_scale" else None, to, max_slots, route, known)
    return c


def linear_w4(x: torch.Tensor, w: W4Weight, *, epilogue: str = "none", row_scale: Optional[torch.Tensor] = None,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x @ w^T of bf16 rows x [T, K] and a dense 4-bit weight, bf16 [T, N] (or
    [T, N / 2] with ``epilogue="swiglu"``); epilogues as in :func:`expert_gemm_w4`."""
    _require(x, "x", torch.bfloat16, 2)
    _check_weight(w, x.device)
    if w.num_experts != 1:
        raise ValueError(f"w has {w.num_experts} experts: use expert_gemm_w4")
    return _gemm(x, w, x.shape[0], None, None, epilogue, row_scale, out, x.shape[0])


def expert_gemm_w4(a: torch.Tensor, w: W4Weight, plan: RoutingPlan, *, gather: bool = True, epilogue: str = "none",
                   row_scale: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`expert_gemm` on 4-bit weights: p[s] = A[row(s)] @ W[e(s)]^T for every
    routed slot, then the epilogue ("none", "row_scale", "swiglu"), rounded once
    to bf16.  a is the token matrix [T, K] (gather=True) or slot-major
    [rows, K].  Rows of ``out`` past the routed slots are left as they were."""
    _require(a, "a", torch.bfloat16, 2)
    _check_weight(w, a.device)
    _check_plan(plan, a.device)
    if w.num_experts != plan.num_experts:
        raise ValueError(f"w has {w.num_experts} experts, plan has {plan.num_experts}")
    if gather:
        if a.shape[0] != plan.num_tokens:
            raise ValueError(f"a has {a.shape[0]} rows, plan has {plan.num_tokens} tokens")
        if a.shape[0] * a.shape[1] * 2 >= 1 << 31:
            raise ValueError("in gather mode the token matrix must be below 2 GiB")
    elif a.shape[0] != plan.rows:
        raise ValueError(f"a has {a.shape[0]} rows, plan has {plan.rows} slots")
    most, known = _known_counts(plan)
    return _gemm(a, w, plan.rows, _vp(plan.sorted_token) if gather else None, _vp(plan.expert_offsets), epilogue,
                 row_scale, out, most, known=known)
