"""The optimizer step of weights that are matrices -- an expert's or a shared
expert's projections, routers -- along the orthogonalised momentum: batched
Newton-Schulz steps on the matrix cores, over many tensors at once.  Beside
:class:`AdamW`, which the other parameters (norms, biases, embeddings) keep.

Every function validates its arguments in Python and makes one library call for
all tensors of a kind (include/etmoe_dense.h has the formulas); there is no CPU
fallback."""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence

import torch

from ._lib import MuonScalars, lib
from .expert_threshold import _call, _require_device, _require_workspace, _vp
from .optimizer import (_DTYPES, _changed, _check_apart, _check_list, _check_masters, _check_params, _check_scale, _kinds,
                        _pointers)

# The coefficients of Newton-Schulz steps that bring singular values of a
# momentum, down to a thousandth of the largest, near 1 in five steps.
MUON_COEFFICIENTS = (3.4445, -4.7750, 2.0315)

_MOST_SIDE = 1 << 16


def _matrices(shape, name: str):
    """(E, m, n) of a tensor of matrices in its last two dimensions."""
    if len(shape) < 2:
        raise ValueError(f"{name} must have two dimensions at least, got shape {tuple(shape)}")
    m, n = int(shape[-2]), int(shape[-1])
    if max(m, n) >= _MOST_SIDE:
        raise ValueError(f"the sides of {name}'s matrices must be below {_MOST_SIDE}, got {(m, n)}")
    return math.prod(shape[:-2]), m, n


_dims = torch.Tensor.size


def _check_matrices(ts, name: str, shapes, dims=None) -> None:
    """The tensors (or None) hold the matrices of `shapes`, as tensors of dimensions `dims` do.  A list's
    number of elements is not enough here: the step depends on the rows that it is read in."""
    if dims is not None and list(map(_dims, ts)) == dims:       # (160 ns a tensor, the loop 410)
        return
    for i, (t, (_, m, n)) in enumerate(zip(ts, shapes)):
        if t is not None and t.shape[-2:] != (m, n):
            raise ValueError(f"{name}[{i}] must hold matrices of {(m, n)}, got shape {tuple(t.shape)}")


def _shape_array(shapes):
    return (ctypes.c_int64 * (3 * len(shapes)))(*[v for s in shapes for v in s])


def _coefficients(coefficients, steps: int, eps: float):
    if len(coefficients) != 3 or not all(math.isfinite(c) for c in coefficients):
        raise ValueError("coefficients must be three finite numbers")
    if not 1 <= steps <= 64:
        raise ValueError(f"steps must be in [1, 64], got {steps}")
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"eps must be finite and >= 0, got {eps}")
    a, b, c = map(float, coefficients)
    # (as the library checks it: f16 holds the numbers in between)
    most, fine = 1.0, 0.0 < a < 16.0 and abs(b) < 64.0 and abs(c) < 64.0
    for _ in range(steps if fine else 0):
        values = [most * k / 256.0 for k in range(257)]
        slopes = [abs(a + b * s * s + c * s ** 4) for s in values]
        before, most = most, max(most, 1.01 * max(s * f for s, f in zip(values, slopes)))
        fine = max(slopes) <= 1.01 * a and most < 1.9
        if not fine or most == before:      # (refused, or all further steps are alike)
            break
    if not fine:
        raise ValueError("coefficients must keep singular values from [0, 1] below 1.9 and |a + b s^2 + c s^4| at most a "
                         f"(below 16), got {tuple(coefficients)}")
    return a, b, c


_checked = {}


def _check_coefficients(coefficients, steps: int, eps: float):
    """The coefficients as floats, looked over once for each choice."""
    key = (*coefficients, steps, eps)
    if key not in _checked:
        if len(_checked) > 64:
            _checked.clear()
        _checked[key] = _coefficients(coefficients, steps, eps)
    return _checked[key]


def _workspace_bytes(shapes) -> int:
    return int(lib().et_orthogonalize_workspace_bytes(_shape_array(shapes), len(shapes)))


def _workspace(shapes, workspace, dev):
    nbytes = _workspace_bytes(shapes)
    if workspace is None:
        return torch.empty(max(nbytes, 256), dtype=torch.uint8, device=dev)
    _require_workspace(workspace, nbytes, dev, "workspace")
    if workspace.data_ptr() % 256:
        raise ValueError("workspace must be 256-byte aligned")
    return workspace


def orthogonalize_workspace_bytes(shapes: Sequence[Sequence[int]]) -> int:
    """Bytes that :func:`orthogonalize` and :func:`muon_step_` work in, for tensors of these shapes or some of them."""
    return _workspace_bytes([_matrices(s, "shape") for s in shapes])


def orthogonalize(g: torch.Tensor, *, steps: int = 5, coefficients=MUON_COEFFICIENTS, eps: float = 1e-7,
                  out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Newton-Schulz steps on every matrix [m, n] of g [..., m, n] (f32 or bf16,
    contiguous): with (a, b, c) the coefficients,

        X = g / (|g| + eps);  ``steps`` times  A = X X^T,  X = (a + b A + c A A) X

    (over the shorter side), which leaves g's singular vectors and brings its
    singular values near 1.  bf16, of g's shape; ``out`` may be a bf16 g itself.  Held in f16 between the
    products, with binary32 sums: 0.1 to 0.2% off in norm.  A zero matrix gives
    zero, a matrix with a value that is not finite NaN.
    """
    _require_device(g, "g")
    if g.dtype not in _DTYPES:
        raise TypeError(f"g must be float32 or bfloat16, got {g.dtype}")
    if not g.is_contiguous():
        raise ValueError("g must be contiguous")
    shapes = [_matrices(g.shape, "g")]
    a, b, c = _check_coefficients(coefficients, steps, eps)
    dev = g.device
    if out is None:
        out = torch.empty(g.shape, dtype=torch.bfloat16, device=dev)
    else:
        _require_device(out, "out")
        if out.dtype != torch.bfloat16:
            raise TypeError(f"out must be {torch.bfloat16}, got {out.dtype}")
        if out.shape != g.shape or out.device != dev or not out.is_contiguous():
            raise ValueError(f"out must be contiguous, of shape {tuple(g.shape)} on {dev}")
    ws = _workspace(shapes, workspace, dev)
    _call("et_orthogonalize", dev, _pointers([g]), _pointers([out]), _shape_array(shapes), 1, _DTYPES[g.dtype], steps,
          (ctypes.c_float * 3)(a, b, c), eps, _vp(ws), ws.numel() * ws.element_size())
    return out


def _scalars(lr: float, momentum: float, weight_decay: float, nesterov: bool, steps: int, coefficients, eps: float):
    if not 0.0 <= momentum < 1.0:
        raise ValueError(f"momentum must be in [0, 1), got {momentum}")
    if not (lr >= 0.0 and weight_decay >= 0.0 and max(lr, weight_decay) < math.inf):
        raise ValueError("lr and weight_decay must be finite and >= 0")
    a, b, c = _check_coefficients(coefficients, steps, eps)
    return MuonScalars(momentum, 1.0 - momentum, 1.0 - lr * weight_decay, eps, a, b, c, steps, int(bool(nesterov)))


def _size(shape, update_rms: Optional[float]) -> float:
    """What an orthogonal matrix of this shape is multiplied by: its entries' root
    mean square is 1 / sqrt(max(m, n))."""
    _, m, n = shape
    if update_rms is None:
        return math.sqrt(max(1.0, m / n)) if n else 0.0
    return update_rms * math.sqrt(max(m, n))


def _check_update(update_rms) -> None:
    if update_rms is not None and not 0.0 < update_rms < math.inf:
        raise ValueError(f"update_rms must be None or a number above 0, got {update_rms}")


def _step(dev, params, grads, momenta, masters, shapes, step_sizes, scalars, grad_scale, workspace) -> None:
    """The library calls of one step, its lists checked."""
    kinds = list(_kinds(params, grads))

    def take(ts, at):
        return ts if at is None else [ts[i] for i in at]

    # (the calls, one behind the other, share a workspace: what the largest needs, and refused before the first
    # call, which a later refusal would leave half a step behind)
    if len(kinds) == 1:
        ws = _workspace(shapes, workspace, dev)
    else:
        most = max((take(shapes, at) for at in kinds), key=_workspace_bytes)
        ws = _workspace(most, workspace, dev)
    for at in kinds:
        p, g, sh = take(params, at), take(grads, at), take(shapes, at)
        low = p[0].dtype == torch.bfloat16
        _call("et_muon", dev, _pointers(p), _pointers(g), _pointers(take(momenta, at)), _pointers(take(masters, at)) if low else None,
              (ctypes.c_float * len(p))(*take(step_sizes, at)), _shape_array(sh), len(p), _DTYPES[p[0].dtype],
              _DTYPES[g[0].dtype], scalars, _vp(grad_scale), _vp(ws), ws.numel() * ws.element_size())


def muon_step_(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], momentum_buffers: Sequence[torch.Tensor], *,
               lr: float, momentum: float = 0.95, weight_decay: float = 0.0, nesterov: bool = True,
               update_rms: Optional[float] = 0.2, steps: int = 5, coefficients=MUON_COEFFICIENTS, eps: float = 1e-7,
               masters: Optional[Sequence[Optional[torch.Tensor]]] = None, grad_scale: Optional[torch.Tensor] = None,
               workspace: Optional[torch.Tensor] = None) -> None:
    """One step, in place, over all tensors of matrices [..., m, n]: with
    g = grad * grad_scale,

        m = momentum m + (1 - momentum) g
        U = (1 - momentum) g + momentum m   (``nesterov``), or m
        w = (1 - lr weight_decay) w - lr s X,   X of :func:`orthogonalize`, of U

    s = update_rms sqrt(max(m, n)), so that a step's entries have a root mean
    square of lr * update_rms in every matrix (0.2 is about AdamW's); with
    ``update_rms=None`` s = sqrt(max(1, m / n)).  A float32 parameter is w
    itself; a bfloat16 one is w rounded, w being its float32 master.  The
    momenta are float32; grads float32 or bfloat16; both, and the masters, hold the parameters'
    matrices (their last two dimensions).  Skipped, every bit kept,
    where ``grad_scale`` (one float32 value on the device) is not finite.  No
    two tensors may share memory.
    """
    index, sizes = _check_params(params)
    dev = params[0].device
    shapes = [_matrices(p.shape, f"params[{i}]") for i, p in enumerate(params)]
    _check_list(grads, "grads", _DTYPES.keys(), index, sizes)
    _check_list(momentum_buffers, "momentum_buffers", {torch.float32}, index, sizes)
    _check_masters(params, masters, index, sizes)
    dims = list(map(_dims, params))
    _check_matrices(grads, "grads", shapes, dims)
    _check_matrices(momentum_buffers, "momentum_buffers", shapes, dims)
    _check_matrices(masters or (), "masters", shapes)
    _check_scale(grad_scale, dev)
    _check_update(update_rms)
    scalars = _scalars(lr, momentum, weight_decay, nesterov, steps, coefficients, eps)
    _step(dev, params, grads, momentum_buffers, masters, shapes, [lr * _size(s, update_rms) for s in shapes], scalars,
          grad_scale, workspace)
    _changed(params)


class Muon:
    """:func:`muon_step_` with its momenta held, for a fixed list of parameters,
    each a matrix or a tensor of matrices [..., m, n].

    The momenta (and the masters of bfloat16 parameters, unless given) are views
    of one allocation for each kind, ``flat[name]``, each tensor from a multiple
    of 256 elements on.  ``step(grads)`` takes one gradient for each parameter,
    or None for one that has none this time: it and its momentum stay as they
    are.  The workspace is allocated for each step: for the up to 20 tensors that run at a time
    about four bytes an element, and four for an element of a matrix's shorter side squared; none
    for matrices that one block takes (a shorter side of at most 64, some 75000 elements).
    """

    def __init__(self, params: Sequence[torch.Tensor], *, lr: float = 1e-3, momentum: float = 0.95,
                 weight_decay: float = 0.0, nesterov: bool = True, update_rms: Optional[float] = 0.2, steps: int = 5,
                 coefficients=MUON_COEFFICIENTS, eps: float = 1e-7,
                 masters: Optional[Sequence[Optional[torch.Tensor]]] = None):
        self.params = list(params)
        self._index, self._sizes = _check_params(self.params)
        self._shapes = [_matrices(p.shape, f"params[{i}]") for i, p in enumerate(self.params)]
        self._dims = list(map(_dims, self.params))
        self._dtypes = [p.dtype for p in self.params]
        dev = self.params[0].device
        _scalars(lr, momentum, weight_decay, nesterov, steps, coefficients, eps)
        _check_update(update_rms)
        self.lr, self.momentum, self.weight_decay, self.nesterov = lr, momentum, weight_decay, bool(nesterov)
        self.update_rms, self.iterations, self.coefficients, self.eps = update_rms, steps, tuple(coefficients), eps
        self._starts, n = [], 0
        for size in self._sizes:
            self._starts.append(n)
            n += -(-size // 256) * 256
        if masters is not None:
            _check_masters(self.params, masters, self._index, self._sizes)
            _check_matrices(masters, "masters", self._shapes)
        _check_apart(self.params + list(masters or ()), "parameters and masters")
        self.masters = list(masters) if masters is not None and torch.bfloat16 in self._dtypes else None
        self.flat = dict(momentum_buffers=torch.zeros(n, dtype=torch.float32, device=dev))
        own = masters is None and torch.bfloat16 in self._dtypes
        if own:
            self.flat["masters"] = torch.zeros(n, dtype=torch.float32, device=dev)
        self._lay_out()
        if own:
            for v, p in zip(self.masters, self.params):
                if v is not None:
                    v.copy_(p.detach())

    def _views(self, name: str) -> list:
        flat = self.flat[name]
        return [flat[a:a + s].view(p.shape) for a, s, p in zip(self._starts, self._sizes, self.params)]

    def _lay_out(self) -> None:
        self.momentum_buffers = self._views("momentum_buffers")
        if "masters" in self.flat:
            self.masters = [v if t == torch.bfloat16 else None for v, t in zip(self._views("masters"), self._dtypes)]

    def __getstate__(self) -> dict:
        """What a copy or a pickle holds: all but the views."""
        state = dict(self.__dict__)
        del state["momentum_buffers"]
        if "masters" in self.flat:
            del state["masters"]
        return state

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state)
        self._index, _ = _check_params(self.params)     # (on another device, perhaps; never on the host)
        self._dims = list(map(_dims, self.params))
        self._lay_out()

    def step(self, grads: Sequence[Optional[torch.Tensor]], *, grad_scale: Optional[torch.Tensor] = None,
             lr: Optional[float] = None, workspace: Optional[torch.Tensor] = None) -> None:
        """One step; ``lr`` for this step only."""
        params, sizes, shapes, masters, momenta = self.params, self._sizes, self._shapes, self.masters, self.momentum_buffers
        dims = self._dims
        if not isinstance(grads, (list, tuple)):
            raise TypeError("grads must be a list or a tuple of tensors")
        if len(grads) != len(params):
            raise ValueError(f"grads has {len(grads)} tensors, params has {len(params)}")
        _check_list(params, "params", _DTYPES.keys(), self._index, sizes)
        if [p.dtype for p in params] != self._dtypes:
            raise TypeError("a parameter changed its type")
        _check_matrices(params, "params", shapes, dims)
        if any(g is None for g in grads):
            some = [i for i, g in enumerate(grads) if g is not None]
            params, grads, sizes, shapes, dims, momenta = (
                [ts[i] for i in some] for ts in (params, grads, sizes, shapes, dims, momenta))
            masters = None if masters is None else [masters[i] for i in some]
        dev = self.params[0].device
        _check_list(grads, "grads", _DTYPES.keys(), self._index, sizes)
        _check_matrices(grads, "grads", shapes, dims)
        _check_scale(grad_scale, dev)
        lr = self.lr if lr is None else lr
        scalars = _scalars(lr, self.momentum, self.weight_decay, self.nesterov, self.iterations, self.coefficients, self.eps)
        if params:
            _step(dev, params, grads, momenta, masters, shapes, [lr * _size(s, self.update_rms) for s in shapes], scalars,
                  grad_scale, workspace)
            _changed(params)

    def state_dict(self) -> dict:
        """Copies of the momenta and masters (flat)."""
        held = {k: v.clone() for k, v in self.flat.items()}
        if self.masters is not None and "masters" not in held:
            held["masters"] = [None if m is None else m.clone() for m in self.masters]
        return held

    def load_state_dict(self, held: dict) -> None:
        """Takes over :meth:`state_dict`'s values; the parameters are the caller's.
        A state that does not fit changes nothing."""
        names = set(self.flat) | ({"masters"} if self.masters is not None else set())
        if set(held) != names:
            raise ValueError(f"state has {sorted(held)}, expected {sorted(names)}")
        pairs = [(v, held[k], k) for k, v in self.flat.items()]
        if "masters" in held and "masters" not in self.flat:
            if not isinstance(held["masters"], (list, tuple)) or len(held["masters"]) != len(self.masters):
                raise ValueError("masters must be a list of one entry for each parameter")
            pairs += [(m, o, f"masters[{i}]") for i, (m, o) in enumerate(zip(self.masters, held["masters"])) if m is not None]
        for mine, other, name in pairs:
            if not isinstance(other, torch.Tensor) or other.dtype != mine.dtype or other.shape != mine.shape:
                raise ValueError(f"{name} must be {mine.dtype} of shape {tuple(mine.shape)}")
        for mine, other, _ in pairs:
            mine.copy_(other)
