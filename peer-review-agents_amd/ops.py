"""The path as PyTorch custom operators (namespace ``etmoe``).

Registered with ``torch.library.custom_op``, each with a fake (meta) kernel for
tracing and, where the operation has a gradient, ``register_autograd``.  So
``torch.compile(fullgraph=True)`` and ``torch.export`` see one opaque node per
operation instead of breaking the graph at a ctypes call.  The routing plan
travels as a tuple of tensors:

    (counts[E], expert_offsets[E+1], token_offsets[T+1],
     sorted_token[S], slot_gate[S], token_slot[S])

S, the routed slot count, is data-dependent: the fake kernel of ``route``
returns it as an unbacked symbolic size.  ``route_with_capacity`` fixes the
slot arrays at a caller-chosen capacity instead (no host synchronisation;
rows past expert_offsets[E] are then unused).

Every eager kernel calls the C ABI of libetmoe.so through the functions of
``expert_threshold`` (argument checks there); there is no CPU kernel.

    torch.ops.etmoe.route(logits, thr)                          -> plan tuple
    torch.ops.etmoe.route_with_capacity(logits, thr, capacity)  -> plan tuple
    torch.ops.etmoe.dispatch(x, token_offsets, token_slot)      -> Xp [rows, d]
    torch.ops.etmoe.combine(yp, logits, slot_gate, sorted_token, token_offsets,
                            token_slot, expert_offsets)         -> Y [T, d]
    torch.ops.etmoe.combine_backward(dy, yp, slot_gate, sorted_token,
                            token_offsets, token_slot, expert_offsets,
                            need_dlogits)                       -> (dYp, dgate, dlogits)
    torch.ops.etmoe.dispatch_backward(dxp, token_offsets, token_slot) -> dX [T, d]
    torch.ops.etmoe.threshold_update_(thr, logits, k_target, momentum) -> stat (thr updated in place)
    torch.ops.etmoe.layer_norm(x, weight, bias, eps)            -> (Y, mean, rstd)
    torch.ops.etmoe.add_layer_norm(x, residual, weight, bias, eps) -> (Y, sum, mean, rstd)
    torch.ops.etmoe.layer_norm_backward(dy, h, weight, mean, rstd, dsum) -> (dX, dweight, dbias)
    torch.ops.etmoe.gated_linear(x, w, activation)              -> H [T, F]
    torch.ops.etmoe.gated_linear_backward(dh, x, w, activation, need_dx, need_dw) -> (dX, dW)

Gradients: dispatch -> dispatch_backward; combine -> combine_backward, with
respect to yp, to the router logits (through the gates, which are the
sigmoid scores at the routed pairs: dlogits) and to slot_gate (dgate);
layer_norm and add_layer_norm -> layer_norm_backward, with respect to the rows,
the weight and the bias (mean and rstd are marked as not differentiable);
gated_linear -> gated_linear_backward, with respect to x and w.  The routing
itself is piecewise constant and has no gradient.
"""
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import expert_threshold as _et
from . import gated as _gated
from . import norm as _norm

Plan = Tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]


def plan_tensors(plan: _et.RoutingPlan) -> Plan:
    """A RoutingPlan as the tuple the operators take."""
    return (plan.counts, plan.expert_offsets, plan.token_offsets, plan.sorted_token, plan.slot_gate,
            plan.token_slot)


# --------------------------------------------------------------------------- #
# routing
# --------------------------------------------------------------------------- #

@torch.library.custom_op("etmoe::route", mutates_args=())
def route(logits: Tensor, thr: Tensor) -> Plan:
    """Threshold routing with exactly-sized slot arrays (one host
    synchronisation to read S)."""
    p = _et.route(logits, thr)
    return (p.counts, p.expert_offsets, p.token_offsets, p.sorted_token, p.slot_gate, p.token_slot)


@route.register_fake
def _route_fake(logits, thr):
    T, E = logits.shape
    S = torch.library.get_ctx().new_dynamic_size()
    i32 = dict(dtype=torch.int32, device=logits.device)
    return (logits.new_empty(E, **i32), logits.new_empty(E + 1, **i32), logits.new_empty(T + 1, **i32),
            logits.new_empty(S, **i32), logits.new_empty(S, dtype=torch.float32), logits.new_empty(S, **i32))


@torch.library.custom_op("etmoe::route_with_capacity", mutates_args=())
def route_with_capacity(logits: Tensor, thr: Tensor, slot_capacity: int) -> Plan:
    """Threshold routing into slot arrays of `slot_capacity` entries (no host
    synchronisation); the first expert_offsets[E] entries are the slots."""
    p = _et.route(logits, thr, slot_capacity=slot_capacity)
    return (p.counts, p.expert_offsets, p.token_offsets, p.sorted_token, p.slot_gate, p.token_slot)


@route_with_capacity.register_fake
def _route_cap_fake(logits, thr, slot_capacity):
    T, E = logits.shape
    i32 = dict(dtype=torch.int32, device=logits.device)
    cap = slot_capacity
    return (logits.new_empty(E, **i32), logits.new_empty(E + 1, **i32), logits.new_empty(T + 1, **i32),
            logits.new_empty(cap, **i32), logits.new_empty(cap, dtype=torch.float32), logits.new_empty(cap, **i32))


@torch.library.custom_op("etmoe::threshold_update_", mutates_args=("thr",))
def threshold_update_(thr: Tensor, logits: Tensor, k_target: int, momentum: float) -> Tensor:
    """EMA threshold update in place on thr; returns the per-expert statistic."""
    return _et.threshold_update_(thr, logits, k_target, momentum)


@threshold_update_.register_fake
def _threshold_update_fake(thr, logits, k_target, momentum):
    return thr.new_empty(thr.shape)


# --------------------------------------------------------------------------- #
# dispatch / combine and their backward
# --------------------------------------------------------------------------- #

def _rows_plan(token_offsets, token_slot, slot_gate=None, sorted_token=None, expert_offsets=None, counts=None):
    """A RoutingPlan over the given plan tensors (dispatch and its backward
    need only the token-major lists)."""
    T = token_offsets.shape[0] - 1
    E = expert_offsets.shape[0] - 1 if expert_offsets is not None else 0
    rows = token_slot.shape[0]
    return _et.RoutingPlan(counts, expert_offsets, token_offsets, sorted_token, slot_gate, token_slot, T, E, rows,
                           rows)


@torch.library.custom_op("etmoe::dispatch", mutates_args=())
def dispatch(x: Tensor, token_offsets: Tensor, token_slot: Tensor) -> Tensor:
    """Xp[slot] = X[token(slot)], one row per entry of token_slot."""
    return _et.dispatch(x, _rows_plan(token_offsets, token_slot))


@dispatch.register_fake
def _dispatch_fake(x, token_offsets, token_slot):
    return x.new_empty(token_slot.shape[0], x.shape[1])


@torch.library.custom_op("etmoe::dispatch_backward", mutates_args=())
def dispatch_backward(dxp: Tensor, token_offsets: Tensor, token_slot: Tensor) -> Tensor:
    """dX[t] = the sum of dXp over t's slots in ascending expert order."""
    return _et.dispatch_backward(dxp, _rows_plan(token_offsets, token_slot))


@dispatch_backward.register_fake
def _dispatch_backward_fake(dxp, token_offsets, token_slot):
    return dxp.new_empty(token_offsets.shape[0] - 1, dxp.shape[1])


@torch.library.custom_op("etmoe::combine", mutates_args=())
def combine(yp: Tensor, logits: Tensor, slot_gate: Tensor, sorted_token: Tensor, token_offsets: Tensor,
            token_slot: Tensor, expert_offsets: Tensor) -> Tensor:
    """Y[t] = sum over t's slots of slot_gate * Yp (fma chain, ascending
    expert).  `logits` is not read: it is the input the gradient through the
    gates flows to."""
    return _et.combine(yp, _rows_plan(token_offsets, token_slot, slot_gate, sorted_token, expert_offsets))


@combine.register_fake
def _combine_fake(yp, logits, slot_gate, sorted_token, token_offsets, token_slot, expert_offsets):
    return yp.new_empty(token_offsets.shape[0] - 1, yp.shape[1])


@torch.library.custom_op("etmoe::combine_backward", mutates_args=())
def combine_backward(dy: Tensor, yp: Tensor, slot_gate: Tensor, sorted_token: Tensor, token_offsets: Tensor,
                     token_slot: Tensor, expert_offsets: Tensor, need_dlogits: bool) -> Tuple[Tensor, Tensor, Tensor]:
    """(dYp, dgate, dlogits): dYp = gate * dY[token], dgate = <dY, Yp> in
    binary64 rounded once, dlogits [T, E] (or [0, E] when not requested)."""
    plan = _rows_plan(token_offsets, token_slot, slot_gate, sorted_token, expert_offsets)
    dyp, dgate, dl = _et.combine_backward(dy, yp, plan, need_dlogits=need_dlogits)
    if dl is None:
        dl = dy.new_empty(0, plan.num_experts, dtype=torch.float32)
    return dyp, dgate, dl


@combine_backward.register_fake
def _combine_backward_fake(dy, yp, slot_gate, sorted_token, token_offsets, token_slot, expert_offsets,
                           need_dlogits):
    T = token_offsets.shape[0] - 1
    E = expert_offsets.shape[0] - 1
    return (yp.new_empty(yp.shape), yp.new_empty(yp.shape[0], dtype=torch.float32),
            dy.new_empty(T if need_dlogits else 0, E, dtype=torch.float32))


# --------------------------------------------------------------------------- #
# autograd
# --------------------------------------------------------------------------- #

def _dispatch_setup(ctx, inputs, output):
    _x, token_offsets, token_slot = inputs
    ctx.save_for_backward(token_offsets, token_slot)


def _dispatch_grad(ctx, dxp):
    token_offsets, token_slot = ctx.saved_tensors
    return torch.ops.etmoe.dispatch_backward(dxp.contiguous(), token_offsets, token_slot), None, None


torch.library.register_autograd("etmoe::dispatch", _dispatch_grad, setup_context=_dispatch_setup)


def _combine_setup(ctx, inputs, output):
    yp, _logits, slot_gate, sorted_token, token_offsets, token_slot, expert_offsets = inputs
    ctx.save_for_backward(yp, slot_gate, sorted_token, token_offsets, token_slot, expert_offsets)


def _combine_grad(ctx, dy):
    yp, slot_gate, sorted_token, token_offsets, token_slot, expert_offsets = ctx.saved_tensors
    need_dl = bool(ctx.needs_input_grad[1])
    dyp, dgate, dl = torch.ops.etmoe.combine_backward(dy.contiguous(), yp, slot_gate, sorted_token, token_offsets,
                                                      token_slot, expert_offsets, need_dl)
    return dyp, (dl if need_dl else None), dgate, None, None, None, None


torch.library.register_autograd("etmoe::combine", _combine_grad, setup_context=_combine_setup)


# --------------------------------------------------------------------------- #
# layer norm
# --------------------------------------------------------------------------- #

@torch.library.custom_op("etmoe::layer_norm", mutates_args=())
def layer_norm(x: Tensor, weight: Tensor, bias: Optional[Tensor], eps: float) -> Tuple[Tensor, Tensor, Tensor]:
    """(Y, mean, rstd) of the rows of x."""
    return _norm.layer_norm(x, weight, bias, eps=eps, stats=True)


@layer_norm.register_fake
def _layer_norm_fake(x, weight, bias, eps):
    f32 = dict(dtype=torch.float32)
    return x.new_empty(x.shape), x.new_empty(x.shape[0], **f32), x.new_empty(x.shape[0], **f32)


@torch.library.custom_op("etmoe::add_layer_norm", mutates_args=())
def add_layer_norm(x: Tensor, residual: Tensor, weight: Tensor, bias: Optional[Tensor],
                   eps: float) -> Tuple[Tensor, Tensor, Tensor, Tensor]:
    """(Y, sum, mean, rstd) of the rows of sum = x + residual."""
    return _norm.layer_norm(x, weight, bias, eps=eps, residual=residual, stats=True)


@add_layer_norm.register_fake
def _add_layer_norm_fake(x, residual, weight, bias, eps):
    f32 = dict(dtype=torch.float32)
    return (x.new_empty(x.shape), x.new_empty(x.shape), x.new_empty(x.shape[0], **f32),
            x.new_empty(x.shape[0], **f32))


@torch.library.custom_op("etmoe::layer_norm_backward", mutates_args=())
def layer_norm_backward(dy: Tensor, h: Tensor, weight: Tensor, mean: Tensor, rstd: Tensor,
                        dsum: Optional[Tensor]) -> Tuple[Tensor, Tensor, Tensor]:
    """(dX, dweight, dbias), the last two float32; dsum is added to dX."""
    return _norm.layer_norm_backward(dy, h, weight, mean, rstd, dsum=dsum)


@layer_norm_backward.register_fake
def _layer_norm_backward_fake(dy, h, weight, mean, rstd, dsum):
    f32 = dict(dtype=torch.float32)
    return h.new_empty(h.shape), weight.new_empty(weight.shape, **f32), weight.new_empty(weight.shape, **f32)


def _norm_grads(ctx, dy, h, dsum):
    weight, mean, rstd = ctx.saved_tensors[:3]
    dy = torch.zeros_like(h) if dy is None else dy.contiguous()
    dx, dw, db = torch.ops.etmoe.layer_norm_backward(dy, h, weight, mean, rstd,
                                                     None if dsum is None else dsum.contiguous())
    return dx, dw.to(weight.dtype), db.to(weight.dtype) if ctx.has_bias else None


def _layer_norm_setup(ctx, inputs, output):
    x, weight, bias, _eps = inputs
    ctx.has_bias = bias is not None
    ctx.mark_non_differentiable(output[1], output[2])
    ctx.save_for_backward(weight, output[1], output[2], x)


def _layer_norm_grad(ctx, dy, _dmean, _drstd):
    return (*_norm_grads(ctx, dy, ctx.saved_tensors[3], None), None)


torch.library.register_autograd("etmoe::layer_norm", _layer_norm_grad, setup_context=_layer_norm_setup)


def _add_layer_norm_setup(ctx, inputs, output):
    _x, _residual, weight, bias, _eps = inputs
    ctx.has_bias = bias is not None
    ctx.mark_non_differentiable(output[2], output[3])
    ctx.save_for_backward(weight, output[2], output[3], output[1])


def _add_layer_norm_grad(ctx, dy, dsum, _dmean, _drstd):
    dx, dw, db = _norm_grads(ctx, dy, ctx.saved_tensors[3], dsum)
    return dx, dx.clone(), dw, db, None


torch.library.register_autograd("etmoe::add_layer_norm", _add_layer_norm_grad, setup_context=_add_layer_norm_setup)


# --------------------------------------------------------------------------- #
# gated projection
# --------------------------------------------------------------------------- #

@torch.library.custom_op("etmoe::gated_linear", mutates_args=())
def gated_linear(x: Tensor, w: Tensor, activation: str) -> Tensor:
    """H = act(x Wg^T) * (x Wu^T)."""
    return _gated.gated_linear(x, w, activation=activation)


@gated_linear.register_fake
def _gated_linear_fake(x, w, activation):
    return x.new_empty(x.shape[0], w.shape[0] // 2)


@torch.library.custom_op("etmoe::gated_linear_backward", mutates_args=())
def gated_linear_backward(dh: Tensor, x: Tensor, w: Tensor, activation: str, need_dx: bool,
                          need_dw: bool) -> Tuple[Tensor, Tensor]:
    """(dX, dW), one that is not needed without rows."""
    # (the gradient's place is known here only, not where a compiled backward is traced)
    dx, dw = _gated.gated_linear_backward(_gated._own_place(dh), x, w, activation=activation, need_dx=need_dx, need_dw=need_dw)
    return x.new_empty(0, x.shape[1]) if dx is None else dx, w.new_empty(0, w.shape[1]) if dw is None else dw


@gated_linear_backward.register_fake
def _gated_linear_backward_fake(dh, x, w, activation, need_dx, need_dw):
    return x.new_empty(x.shape[0] if need_dx else 0, x.shape[1]), w.new_empty(w.shape[0] if need_dw else 0, w.shape[1])


def _gated_setup(ctx, inputs, output):
    x, w, ctx.activation = inputs
    ctx.save_for_backward(x, w)


def _gated_grad(ctx, dh):
    x, w = ctx.saved_tensors
    need_dx, need_dw, _ = ctx.needs_input_grad
    dx, dw = torch.ops.etmoe.gated_linear_backward(dh.contiguous(), x, w, ctx.activation, need_dx, need_dw)
    return dx if need_dx else None, dw if need_dw else None, None


torch.library.register_autograd("etmoe::gated_linear", _gated_grad, setup_context=_gated_setup)
