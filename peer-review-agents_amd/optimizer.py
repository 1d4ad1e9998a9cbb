"""The optimizer step of the weights around the expert path: AdamW over many
tensors at once, with states in 32 or in 8 bits, and the global gradient norm
that clips it.

The gradients of this package's expert projections and router are float32
(:func:`expert_gemm_weight_grad`, :func:`router_weight_grad`) and their weights
bfloat16, so a parameter is either a float32 tensor or a bfloat16 one with a
float32 master that the step works on.  Every function validates its arguments
in Python and makes one library call for all tensors of a kind (include/
etmoe_block.h has the formulas); there is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence

import torch

from ._lib import ET_DTYPE_BF16, ET_DTYPE_F32, AdamWScalars, lib
from .expert_threshold import _call, _require, _require_device, _require_workspace, _vp

# Elements that share one scale of the 8-bit states.
ADAMW8_BLOCK = 256

_DTYPES = {torch.float32: ET_DTYPE_F32, torch.bfloat16: ET_DTYPE_BF16}

# A step over many small tensors takes some 20 us on the device, so the checks
# of a list run as C calls mapped over it: 50 ns for each tensor and check.
_data_ptr = torch.Tensor.data_ptr
_numel = torch.Tensor.numel
_get_device = torch.Tensor.get_device
_is_contiguous = torch.Tensor.is_contiguous


def _array(ptrs):
    """A host array of pointers, as ctypes passes it."""
    return (ctypes.c_void_p * len(ptrs))(*ptrs)


def _pointers(ts):
    return _array(list(map(_data_ptr, ts)))


def _numel_array(sizes):
    return (ctypes.c_int64 * len(sizes))(*sizes)


def _check_list(ts, name: str, dtypes, device: int, sizes) -> set:
    """Every tensor of `ts` contiguous, on HIP device `device`, of one of
    `dtypes` and of as many elements as `sizes` says.  Returns their dtypes."""
    if not isinstance(ts, (list, tuple)):
        raise TypeError(f"{name} must be a list or a tuple of tensors")
    if len(ts) != len(sizes):
        raise ValueError(f"{name} has {len(ts)} tensors, params has {len(sizes)}")
    try:        # (the unbound methods refuse what is no tensor)
        if list(map(_numel, ts)) == sizes and all(map(_is_contiguous, ts)) and set(map(_get_device, ts)) <= {device}:
            found = {t.dtype for t in ts}
            if found <= dtypes:
                return found
    except TypeError:
        raise TypeError(f"{name} must hold torch.Tensors") from None
    for i, t in enumerate(ts):
        _require_device(t, f"{name}[{i}]")
        if t.dtype not in dtypes:
            raise TypeError(f"{name}[{i}] must be {' or '.join(map(str, dtypes))}, got {t.dtype}")
        if not t.is_contiguous():
            raise ValueError(f"{name}[{i}] must be contiguous")
        if t.numel() != sizes[i]:
            raise ValueError(f"{name}[{i}] has {t.numel()} elements, expected {sizes[i]}")
        if t.get_device() != device:
            raise ValueError(f"{name}[{i}] is on {t.device}, expected cuda:{device}")
    return {t.dtype for t in ts}


def _check_params(params) -> tuple:
    """(device index, sizes) of a checked, non-empty list of parameters."""
    if not isinstance(params, (list, tuple)):
        raise TypeError("params must be a list or a tuple of tensors")
    if not params:
        raise ValueError("params must hold at least one tensor")
    _require_device(params[0], "params[0]")
    sizes = [t.numel() if isinstance(t, torch.Tensor) else -1 for t in params]
    _check_list(params, "params", _DTYPES.keys(), params[0].get_device(), sizes)
    return params[0].get_device(), sizes


def _check_masters(params, masters, device, sizes) -> None:
    low = [p.dtype == torch.bfloat16 for p in params]
    if masters is None:
        if any(low):
            raise ValueError("bfloat16 parameters need float32 masters")
        return
    if not isinstance(masters, (list, tuple)) or len(masters) != len(params):
        raise ValueError("masters must be a list of one entry for each parameter")
    if [m is not None for m in masters] != low:
        raise ValueError("masters must hold a tensor for every bfloat16 parameter and None for every float32 one")
    _check_list([m for m in masters if m is not None], "masters", {torch.float32}, device,
                [n for n, b in zip(sizes, low) if b])


def _check_apart(ts, name: str) -> None:
    """No two of the tensors share memory: a step reads and writes each at once."""
    spans = sorted((t.data_ptr(), t.numel() * t.element_size()) for t in ts if t is not None and t.numel())
    for (at, size), (next_at, _) in zip(spans, spans[1:]):
        if at + size > next_at:
            raise ValueError(f"{name} overlap in memory (or hold a tensor more than once)")


def _scalars(step: int, lr: float, betas, eps: float, weight_decay: float) -> AdamWScalars:
    step = int(step)
    b1, b2 = (float(b) for b in betas)
    if step < 1:
        raise ValueError(f"step must be >= 1, got {step}")
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
        raise ValueError(f"betas must be in [0, 1), got {betas}")
    if not (lr >= 0.0 and eps >= 0.0 and weight_decay >= 0.0 and max(lr, eps, weight_decay) < math.inf):
        raise ValueError("lr, eps and weight_decay must be finite and >= 0")
    return AdamWScalars(b1, 1.0 - b1, b2, 1.0 - b2, 1.0 / math.sqrt(1.0 - b2 ** step), eps, 1.0 - lr * weight_decay,
                        lr / (1.0 - b1 ** step))


def _check_scale(grad_scale, dev) -> None:
    if grad_scale is None:
        return
    _require_device(grad_scale, "grad_scale")
    if grad_scale.dtype != torch.float32 or grad_scale.numel() != 1 or grad_scale.device != dev:
        raise ValueError(f"grad_scale must be one float32 value on {dev}")


# --------------------------------------------------------------------------- #
# gradient norm
# --------------------------------------------------------------------------- #

def grad_norm(grads: Sequence[torch.Tensor], max_norm: Optional[float] = None, *,
              workspace: Optional[torch.Tensor] = None):
    """(norm, scale) of many gradients (f32 or bf16, contiguous): their global
    2-norm and min(1, max_norm / (norm + 1e-6)), one float32 value each on the
    device; scale is None without max_norm.  Squares and sums are binary64 in a
    fixed order.  Where the norm is not finite the scale is NaN, with which
    :func:`adamw_step_` and :func:`adamw8_step_` leave everything as it is.
    """
    if not isinstance(grads, (list, tuple)):
        raise TypeError("grads must be a list or a tuple of tensors")
    if not grads:
        raise ValueError("grads must hold at least one tensor")
    _require_device(grads[0], "grads[0]")
    if max_norm is not None and not max_norm > 0.0:
        raise ValueError(f"max_norm must be > 0, got {max_norm}")
    dev = grads[0].device
    sizes = [t.numel() if isinstance(t, torch.Tensor) else -1 for t in grads]
    _check_list(grads, "grads", _DTYPES.keys(), grads[0].get_device(), sizes)
    numel = _numel_array(sizes)
    wsb = int(lib().et_grad_norm_workspace_bytes(numel, len(sizes)))
    if workspace is None:
        workspace = torch.empty(max(wsb, 8), dtype=torch.uint8, device=dev)
    else:
        _require_workspace(workspace, wsb, dev, "workspace")
    out = torch.empty(2, dtype=torch.float32, device=dev)
    norm = out.data_ptr()
    dtypes = (ctypes.c_int32 * len(sizes))(*[_DTYPES[t.dtype] for t in grads])
    _call("et_grad_norm", dev, _pointers(grads), numel, dtypes, len(sizes),
          0.0 if max_norm is None else float(max_norm), norm, None if max_norm is None else norm + 4, _vp(workspace),
          workspace.numel() * workspace.element_size())
    return out[0], None if max_norm is None else out[1]


# --------------------------------------------------------------------------- #
# AdamW
# --------------------------------------------------------------------------- #

def _kinds(params, grads):
    """Index lists of the tensors that one library call can take: one parameter
    and one gradient type each (None where a single call takes all)."""
    pairs = [(p.dtype, g.dtype) for p, g in zip(params, grads)]
    if len(set(pairs)) == 1:
        return [None]
    return [[i for i, q in enumerate(pairs) if q == pair] for pair in dict.fromkeys(pairs)]


# The parameters have changed: a backward that kept one of them as it was before
# raises, as behind any in-place operation of torch (55 ns a tensor).
_changed = torch.autograd.graph.increment_version


def _step(fn: str, dev, params, grads, states, masters, sizes, scalars, grad_scale, *more) -> None:
    """The library calls of one step, its lists checked."""
    for at in _kinds(params, grads):
        def take(ts):
            return ts if at is None else [ts[i] for i in at]
        p, g = take(params), take(grads)
        low = p[0].dtype == torch.bfloat16
        _call(fn, dev, _pointers(p), _pointers(g),
              *(_pointers(take(s)) for s in states),
              _pointers(take(masters)) if low else None, _numel_array(take(sizes)), len(p),
              _DTYPES[p[0].dtype], _DTYPES[g[0].dtype], scalars, _vp(grad_scale), *more)


def adamw_step_(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avg: Sequence[torch.Tensor],
                exp_avg_sq: Sequence[torch.Tensor], *, step: int, lr: float, betas=(0.9, 0.999), eps: float = 1e-8,
                weight_decay: float = 0.01, masters: Optional[Sequence[Optional[torch.Tensor]]] = None,
                grad_scale: Optional[torch.Tensor] = None) -> None:
    """One AdamW step (decoupled weight decay), in place, over all tensors:
    with g = grad * grad_scale,

        m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
        w = (1 - lr wd) w - lr / (1 - b1^step) * m / (sqrt(v / (1 - b2^step)) + eps)

    in binary32.  A float32 parameter is w itself; a bfloat16 one is w rounded,
    w being its float32 master (``masters[i]``, None for float32 parameters).
    exp_avg (m) and exp_avg_sq (v) are float32; grads float32 or bfloat16.
    ``grad_scale`` is one float32 value on the device (:func:`grad_norm`'s); the
    step is skipped, every bit kept, where it is not finite.  No two tensors may
    share memory.
    """
    index, sizes = _check_params(params)
    dev = params[0].device
    _check_list(grads, "grads", _DTYPES.keys(), index, sizes)
    _check_list(exp_avg, "exp_avg", {torch.float32}, index, sizes)
    _check_list(exp_avg_sq, "exp_avg_sq", {torch.float32}, index, sizes)
    _check_masters(params, masters, index, sizes)
    _check_scale(grad_scale, dev)
    _step("et_adamw", dev, params, grads, (exp_avg, exp_avg_sq), masters, sizes,
          _scalars(step, lr, betas, eps, weight_decay), grad_scale)
    _changed(params)


def adamw8_scales(numel: int) -> int:
    """Entries of the scale tensor of an 8-bit state of `numel` elements."""
    return -(-int(numel) // ADAMW8_BLOCK)


def adamw8_step_(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avg: Sequence[torch.Tensor],
                 exp_avg_scale: Sequence[torch.Tensor], exp_avg_root: Sequence[torch.Tensor],
                 exp_avg_root_scale: Sequence[torch.Tensor], *, step: int, lr: float, betas=(0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 0.01,
                 masters: Optional[Sequence[Optional[torch.Tensor]]] = None,
                 grad_scale: Optional[torch.Tensor] = None, seed: Optional[int] = None) -> None:
    """:func:`adamw_step_` with 8-bit states: exp_avg (m) and exp_avg_root
    (sqrt(v)) are ``torch.float8_e4m3fn`` of the parameter's element count, and
    their scales float32 with one entry for every 256 elements; the value held
    is the e4m3 value times its block's scale.  All zero is the start.

    ``seed`` None rounds the states to nearest; a number (32 bits are used)
    rounds them stochastically, which a moving average needs to keep moving on
    so coarse a grid: give another one every step.
    """
    index, sizes = _check_params(params)
    dev = params[0].device
    blocks = list(map(adamw8_scales, sizes))
    _check_list(grads, "grads", _DTYPES.keys(), index, sizes)
    _check_list(exp_avg, "exp_avg", {torch.float8_e4m3fn}, index, sizes)
    _check_list(exp_avg_root, "exp_avg_root", {torch.float8_e4m3fn}, index, sizes)
    _check_list(exp_avg_scale, "exp_avg_scale", {torch.float32}, index, blocks)
    _check_list(exp_avg_root_scale, "exp_avg_root_scale", {torch.float32}, index, blocks)
    _check_masters(params, masters, index, sizes)
    _check_scale(grad_scale, dev)
    _step("et_adamw8", dev, params, grads, (exp_avg, exp_avg_scale, exp_avg_root, exp_avg_root_scale), masters, sizes,
          _scalars(step, lr, betas, eps, weight_decay), grad_scale, int(seed is not None), (seed or 0) & 0xFFFFFFFF)
    _changed(params)


class AdamW:
    """AdamW that holds its states, for a fixed list of parameters.

    ``state`` "f32" or "e4m3" (8 bits; ``stochastic`` rounding with the random
    words of ``seed + step number``, or to nearest).  The states (and the
    masters of bfloat16 parameters, unless given) are views of one allocation
    for each kind, ``flat[name]``, each tensor from a multiple of 256 elements
    on.  ``step(grads)`` takes one gradient for each parameter, or None for one
    that has none this time: it stays as it is, and the step number in its bias
    corrections counts its own steps.  ``steps`` counts the calls; setting it sets
    every parameter's number.  The parameters' own storage may move between
    steps (``p.data = ...``) as long as type, shape, layout and device stay.
    """

    def __init__(self, params: Sequence[torch.Tensor], *, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01, state: str = "f32",
                 masters: Optional[Sequence[Optional[torch.Tensor]]] = None, stochastic: bool = True, seed: int = 0):
        self.params = list(params)
        self._index, self._sizes = _check_params(self.params)
        self._dtypes = [p.dtype for p in self.params]
        dev = self.params[0].device
        _scalars(1, lr, betas, eps, weight_decay)
        if state not in ("f32", "e4m3"):
            raise ValueError(f"state must be 'f32' or 'e4m3', got {state!r}")
        self.lr, self.betas, self.eps, self.weight_decay = lr, betas, eps, weight_decay
        self.state, self.stochastic, self.seed, self.steps = state, bool(stochastic), int(seed), 0     # (and _counts)
        self._starts, n = [], 0
        for size in self._sizes:
            self._starts.append(n)
            n += adamw8_scales(size) * ADAMW8_BLOCK
        if masters is not None:
            _check_masters(self.params, masters, self._index, self._sizes)
        _check_apart(self.params + list(masters or ()), "parameters and masters")
        # (a list of None alone, for float32 parameters only, is no masters)
        self.masters = list(masters) if masters is not None and torch.bfloat16 in self._dtypes else None
        if state == "f32":
            kinds = dict(exp_avg=torch.float32, exp_avg_sq=torch.float32)
        else:
            e4m3 = torch.float8_e4m3fn
            kinds = dict(exp_avg=e4m3, exp_avg_scale=torch.float32, exp_avg_root=e4m3, exp_avg_root_scale=torch.float32)
        self._names = tuple(kinds)
        own = masters is None and torch.bfloat16 in self._dtypes
        if own:
            kinds["masters"] = torch.float32
        self.flat = {k: torch.zeros(n // self._per(k), dtype=t, device=dev) for k, t in kinds.items()}
        self._lay_out()
        if own:
            for v, p in zip(self.masters, self.params):
                if v is not None:
                    v.copy_(p.detach())

    @staticmethod
    def _per(name: str) -> int:
        """Elements of a parameter for each of a state's."""
        return ADAMW8_BLOCK if name.endswith("_scale") else 1

    def _views(self, name: str) -> list:
        flat, per = self.flat[name], self._per(name)
        if per > 1:
            return [flat[a // per:a // per + adamw8_scales(s)] for a, s in zip(self._starts, self._sizes)]
        return [flat[a:a + s].view(p.shape) for a, s, p in zip(self._starts, self._sizes, self.params)]

    def _lay_out(self) -> None:
        """The states as views of `flat`, and the tables of pointers that a step of
        all tensors hands over (the states' own buffers never move)."""
        self._states = tuple(map(self._views, self._names))
        for name, views in zip(self._names, self._states):
            setattr(self, name, views)
        if "masters" in self.flat:
            self.masters = [v if t == torch.bfloat16 else None for v, t in zip(self._views("masters"), self._dtypes)]
        self._one_type = len(set(self._dtypes)) == 1
        self._at = list(map(_data_ptr, self.params))
        self._param_table = _array(self._at)
        self._tables = [_pointers(s) for s in self._states]
        self._numel = _numel_array(self._sizes)

    def __getstate__(self) -> dict:
        """What a copy or a pickle holds: all but the views and the pointers."""
        state = dict(self.__dict__)
        for name in self._names + ("_states", "_at", "_param_table", "_tables", "_numel"):
            del state[name]
        if "masters" in self.flat:
            del state["masters"]
        return state

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state)
        self._index, _ = _check_params(self.params)     # (on another device, perhaps; never on the host)
        self._lay_out()

    @property
    def steps(self) -> int:
        return self._steps

    @steps.setter
    def steps(self, number: int) -> None:
        self._steps = number
        self._counts = None         # each parameter's steps, where they are not all this number

    def step(self, grads: Sequence[Optional[torch.Tensor]], *, grad_scale: Optional[torch.Tensor] = None,
             lr: Optional[float] = None) -> None:
        """One step; ``lr`` for this step only.  The step numbers count the steps
        that a grad_scale that is not finite made the device skip, too."""
        params, sizes, states, masters = self.params, self._sizes, self._states, self.masters
        dev = params[0].device
        if not isinstance(grads, (list, tuple)):
            raise TypeError("grads must be a list or a tuple of tensors")
        if len(grads) != len(params):
            raise ValueError(f"grads has {len(grads)} tensors, params has {len(params)}")
        at = list(map(_data_ptr, params))
        if at != self._at or list(map(_numel, params)) != sizes:      # storage that has moved is looked over again
            _check_list(params, "params", _DTYPES.keys(), self._index, sizes)
            if [p.dtype for p in params] != self._dtypes:
                raise TypeError("a parameter changed its type")
            self._at, self._param_table = at, _array(at)
        whole = True
        for g in grads:
            if g is None:
                whole = False
                break
        number, counts = self._steps, self._counts
        some = range(len(params))
        if not whole:
            some = [i for i, g in enumerate(grads) if g is not None]
            params, grads, sizes = ([ts[i] for i in some] for ts in (params, grads, sizes))
            states = [[s[i] for i in some] for s in states]
            masters = None if masters is None else [masters[i] for i in some]
        grad_types = _check_list(grads, "grads", _DTYPES.keys(), self._index, sizes)
        _check_scale(grad_scale, dev)
        hyper = self.lr if lr is None else lr, self.betas, self.eps, self.weight_decay
        scalars = _scalars(number + 1, *hyper)
        fn, more = "et_adamw", ()
        if self.state == "e4m3":
            fn, more = "et_adamw8", (int(self.stochastic), (self.seed + number + 1) & 0xFFFFFFFF)
        if counts is not None:          # one step number to a call
            ages = [counts[i] for i in some]
            for age in dict.fromkeys(ages):
                at = [j for j, n in enumerate(ages) if n == age]
                of = lambda ts: [ts[j] for j in at]  # noqa: E731
                _step(fn, dev, of(params), of(grads), [of(s) for s in states], None if masters is None else of(masters),
                      of(sizes), _scalars(age + 1, *hyper), grad_scale, *more)
        elif whole and self._one_type and len(grad_types) == 1:
            _call(fn, dev, self._param_table, _pointers(grads), *self._tables,
                  None if masters is None else _pointers(masters), self._numel, len(params),
                  _DTYPES[self._dtypes[0]], _DTYPES[grads[0].dtype], scalars, _vp(grad_scale), *more)
        elif params:
            _step(fn, dev, params, grads, states, masters, sizes, scalars, grad_scale, *more)
        _changed(params)
        if counts is not None or not whole:
            counts = self._counts = [number] * len(self.params) if counts is None else list(counts)
            for i in some:
                counts[i] += 1
        self._steps = number + 1

    def state_dict(self) -> dict:
        """Copies of the states and masters (flat), the step number and each parameter's."""
        held = {k: v.clone() for k, v in self.flat.items()}
        if self.masters is not None and "masters" not in held:
            held["masters"] = [None if m is None else m.clone() for m in self.masters]
        return dict(held, steps=self.steps, counts=[self.steps] * len(self.params) if self._counts is None else list(self._counts))

    def load_state_dict(self, held: dict) -> None:
        """Takes over :meth:`state_dict`'s values; the parameters are the caller's.
        Without ``counts`` every parameter has had ``steps`` steps."""
        names = set(self.flat) | ({"masters"} if self.masters is not None else set()) | {"steps"}
        if set(held) - {"counts"} != names:
            raise ValueError(f"state has {sorted(held)}, expected {sorted(names)}")
        # (everything is looked over before anything changes: copy_ would broadcast)
        def check(t, like, name):
            if not isinstance(t, torch.Tensor) or t.dtype != like.dtype or t.shape != like.shape:
                got = f"{t.dtype} of shape {tuple(t.shape)}" if isinstance(t, torch.Tensor) else type(t).__name__
                raise ValueError(f"{name} must be {like.dtype} of shape {tuple(like.shape)}, got {got}")

        for k, v in self.flat.items():
            check(held[k], v, k)
        pairs = [(v, held[k]) for k, v in self.flat.items()]
        if "masters" in held and "masters" not in self.flat:
            if not isinstance(held["masters"], (list, tuple)) or len(held["masters"]) != len(self.masters):
                raise ValueError("masters must be a list of one entry for each parameter")
            for i, (mine, other) in enumerate(zip(self.masters, held["masters"])):
                if mine is not None:
                    check(other, mine, f"masters[{i}]")
                    pairs.append((mine, other))
        steps = int(held["steps"])
        counts = list(map(int, held.get("counts", [steps] * len(self.params))))
        if steps < 0:
            raise ValueError(f"steps must be >= 0, got {steps}")
        if len(counts) != len(self.params) or not all(0 <= n <= steps for n in counts):
            raise ValueError("counts must hold a number of steps for each parameter, none above steps")
        for mine, other in pairs:
            mine.copy_(other)
        self.steps = steps
        if any(n != steps for n in counts):
            self._counts = counts
