"""The torch.library operators on the GPU: each eager operator gives the same
bits as the host API it wraps; torch.library.opcheck accepts the schema, fake
kernel and autograd registration of the row operators; and a small MoE layer
built from the operators (route -> dispatch -> an element-wise expert stand-in
-> combine, with the EMA update in training) runs under
torch.compile(fullgraph=True) -- so with no graph break -- and gives outputs,
gradients and thresholds bit-identical to eager, over several steps."""
import importlib

import pytest
import torch

et = importlib.import_module("peer-review-agents_amd")
ops = importlib.import_module("peer-review-agents_amd.ops")
W = importlib.import_module("peer-review-agents_amd.workloads")

pytestmark = pytest.mark.gpu


def _bits(t):
    return t.view(torch.int16) if t.element_size() == 2 else t.view(torch.int32)


def _case(dev, T=600, E=16, d=256, dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    logits = torch.randn(T, E, device=dev, generator=g) + torch.linspace(-1, 1, E, device=dev)
    thr = torch.quantile(torch.sigmoid(logits.double()), 0.8, dim=0).float().contiguous()
    x = torch.randn(T, d, device=dev, generator=g).to(dtype)
    return logits, thr, x, g


def test_eager_operators_equal_host_api(dev):
    logits, thr, x, g = _case(dev)
    plan = et.route(logits, thr)
    pt = torch.ops.etmoe.route(logits, thr)
    for a, b in zip(ops.plan_tensors(plan), pt):
        assert torch.equal(_bits(a), _bits(b))
    capped = torch.ops.etmoe.route_with_capacity(logits, thr, plan.num_slots + 7)
    assert capped[3].shape[0] == plan.num_slots + 7
    S = plan.num_slots
    for a, b in zip(pt[3:], capped[3:]):
        assert torch.equal(_bits(a), _bits(b[:S]))
    counts, eo, to, st, sg, ts = pt
    xp = torch.ops.etmoe.dispatch(x, to, ts)
    assert torch.equal(_bits(xp), _bits(et.dispatch(x, plan)))
    yp = torch.randn(S, x.shape[1], device=dev, generator=g).to(x.dtype)
    y = torch.ops.etmoe.combine(yp, logits, sg, st, to, ts, eo)
    assert torch.equal(_bits(y), _bits(et.combine(yp, plan)))
    dy = torch.randn_like(y)
    got = torch.ops.etmoe.combine_backward(dy, yp, sg, st, to, ts, eo, True)
    want = et.combine_backward(dy, yp, plan, need_dlogits=True)
    for a, b in zip(got, want):
        assert torch.equal(_bits(a), _bits(b))
    assert torch.ops.etmoe.combine_backward(dy, yp, sg, st, to, ts, eo, False)[2].numel() == 0
    assert torch.equal(_bits(torch.ops.etmoe.dispatch_backward(yp, to, ts)), _bits(et.dispatch_backward(yp, plan)))
    t1, t2 = thr.clone(), thr.clone()
    s1 = torch.ops.etmoe.threshold_update_(t1, logits, 4, 0.9)
    s2 = et.threshold_update_(t2, logits, 4, 0.9)
    assert torch.equal(_bits(t1), _bits(t2)) and torch.equal(_bits(s1), _bits(s2))


def test_opcheck_row_operators(dev):
    logits, thr, x, g = _case(dev, T=200, E=8, d=64, dtype=torch.float32)
    counts, eo, to, st, sg, ts = torch.ops.etmoe.route(logits, thr)
    S = st.shape[0]
    yp = torch.randn(S, 64, device=dev, generator=g, requires_grad=True)
    lg = logits.clone().requires_grad_(True)
    dy = torch.randn(200, 64, device=dev, generator=g)
    torch.library.opcheck(torch.ops.etmoe.dispatch.default, (x.requires_grad_(True), to, ts))
    torch.library.opcheck(torch.ops.etmoe.combine.default, (yp, lg, sg, st, to, ts, eo))
    torch.library.opcheck(torch.ops.etmoe.dispatch_backward.default, (yp.detach(), to, ts))
    torch.library.opcheck(torch.ops.etmoe.combine_backward.default, (dy, yp.detach(), sg, st, to, ts, eo, True))


class OpsMoE(torch.nn.Module):
    """route -> dispatch -> element-wise expert stand-in -> combine, with the
    EMA threshold update in training.  The stand-in is element-wise so that
    eager and compiled runs share every kernel, which makes bit-identity the
    bar."""

    def __init__(self, d, E, dev):
        super().__init__()
        g = torch.Generator().manual_seed(5)
        self.scale = torch.nn.Parameter((torch.randn(d, generator=g) * 0.5 + 1.0).to(dev))
        self.register_buffer("thr", torch.full((E,), 0.7, device=dev))

    def forward(self, x, logits):
        counts, eo, to, st, sg, ts = torch.ops.etmoe.route(logits.detach(), self.thr)
        if self.training:
            torch.ops.etmoe.threshold_update_(self.thr, logits.detach(), 4, 0.9)
        xp = torch.ops.etmoe.dispatch(x, to, ts)
        h = (torch.tanh(xp.float()) * self.scale).to(x.dtype)
        return torch.ops.etmoe.combine(h, logits, sg, st, to, ts, eo)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_compiled_layer_is_bit_identical_to_eager(dev, dtype):
    torch._dynamo.reset()
    T, E, d = 512, 16, 256
    eager, comp = OpsMoE(d, E, dev), OpsMoE(d, E, dev)
    compiled = torch.compile(comp, fullgraph=True, backend="aot_eager")
    for step in range(3):
        print(f"compile check {dtype} step {step}", flush=True)
        logits, _, x, g = _case(dev, T=T, E=E, d=d, dtype=dtype, seed=10 + step)
        outs = []
        for m in (eager, compiled):
            xi = x.clone().requires_grad_(True)
            li = logits.clone().requires_grad_(True)
            y = m(xi, li)
            dy = torch.ones_like(y) * 0.01 + torch.randn(y.shape, device=dev, generator=torch.Generator(
                device=dev).manual_seed(step)).to(y.dtype) * 0.02
            y.backward(dy)
            outs.append((y.detach(), xi.grad, li.grad))
        for a, b in zip(outs[0], outs[1]):
            assert torch.equal(_bits(a), _bits(b))
        assert torch.equal(_bits(eager.scale.grad), _bits(comp.scale.grad))
        assert torch.equal(_bits(eager.thr), _bits(comp.thr))
        eager.scale.grad = None
        comp.scale.grad = None
    # the EMA moved the thresholds, and the logits received gradient only at routed pairs
    assert not torch.equal(eager.thr, torch.full_like(eager.thr, 0.7))


def test_workspaces_that_only_look_large_are_refused(et, dev):
    """A workspace of enough elements on one element of memory."""
    T, E, d = 300, 8, 64
    logits, thr = torch.randn(T, E, device=dev), torch.zeros(E, device=dev)
    x, w = (torch.randn(n, d, device=dev).bfloat16() for n in (T, E))
    plan = et.route(logits, thr)
    yp = torch.randn(plan.rows, d, device=dev).bfloat16()
    dgate = torch.zeros(plan.rows, device=dev)
    bad = torch.zeros(4, device=dev)[:1].expand(1 << 24)
    for call in (lambda ws: et.route(logits, thr, workspace=ws),
                 lambda ws: et.route_update(logits, thr, 2, workspace=ws),
                 lambda ws: et.route_update(logits, thr, 2, thr_workspace=ws),
                 lambda ws: et.threshold_update_(thr, logits, 2, workspace=ws),
                 lambda ws: et.router_route(x, w, thr, workspace=ws),
                 lambda ws: et.router_weight_grad(logits, x, workspace=ws),
                 lambda ws: et.combine_backward(x, yp, plan, workspace=ws),
                 lambda ws: et.dispatch_backward(yp, plan, router_weight=w, dgate=dgate, workspace=ws)):
        with pytest.raises(ValueError, match="workspace"):
            call(bad)
