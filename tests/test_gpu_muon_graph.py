"""A captured Muon step: every way that a matrix can go, replayed between eager work."""
import pytest
import torch

from test_gpu_muon import _lists

pytestmark = pytest.mark.gpu

SHAPES = [(8, 64), (4, 32, 64), (64, 1024), (130, 77), (96, 264), (40, 384, 520), (24, 501, 154)]


@pytest.mark.parametrize("dtype,gdtype", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_a_captured_step(et, dev, dtype, gdtype):
    params, masters, momenta, grads = _lists(dev, SHAPES, dtype, gdtype)
    mine = [None if ts is None else [t.clone() for t in ts] for ts in (params, masters, momenta)]
    scale = torch.full((1,), 0.5, device=dev)
    kw = dict(lr=0.01, momentum=0.9, weight_decay=0.1, grad_scale=scale)
    spare = [None if ts is None else [t.clone() for t in ts] for ts in (params, masters, momenta)]
    et.muon_step_(spare[0], grads, spare[2], masters=spare[1], **kw)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        et.muon_step_(params, grads, momenta, masters=masters, **kw)
    for rep in range(4):
        for g, new in zip(grads, _lists(dev, SHAPES, dtype, gdtype, seed=rep + 1)[3]):
            g.copy_(new)
        scale.fill_((0.5, float("nan"), 0.25, 1.0)[rep])
        graph.replay()
        torch.cuda.synchronize()
        et.muon_step_(mine[0], grads, mine[2], masters=mine[1], **kw)
        for a, b in zip(params + momenta + (masters or []), mine[0] + mine[2] + (mine[1] or [])):
            assert torch.equal(a, b), rep
    del graph
