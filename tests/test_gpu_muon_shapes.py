"""A Muon step reads its lists under the parameters' matrices: tensors of as many elements that
are other matrices are refused, and nothing is changed."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _step(dev, shape=(3, 8, 16)):
    g = torch.Generator(device=dev).manual_seed(1)
    r = lambda: torch.randn(*shape, generator=g, device=dev)  # noqa: E731
    return dict(params=[r()], grads=[r()], momentum_buffers=[r()], lr=0.1)


def _other(t):
    """The same elements as other matrices: transposed, those of a batch side by side, without rows."""
    return [t.mT.contiguous(), t.transpose(0, 1).reshape(t.shape[1], -1).contiguous(), t.reshape(-1)]


@pytest.mark.parametrize("name", ["grads", "momentum_buffers", "masters"])
def test_other_matrices_are_refused(et, dev, name):
    step = _step(dev)
    if name == "masters":
        step["masters"] = [step["params"][0].clone()]
        step["params"] = [step["params"][0].bfloat16()]
    before = [t.clone() for t in (step["params"][0], step["momentum_buffers"][0])]
    for other in _other(step[name][0]):
        with pytest.raises(ValueError, match=name):
            et.muon_step_(**{**step, name: [other]})
    for a, b in zip(before, (step["params"][0], step["momentum_buffers"][0])):
        assert torch.equal(a, b)


def test_other_batch_dimensions_are_taken(et, dev):
    """The same matrices in the same order: [2, 3, m, n] is [6, m, n]."""
    step, again = _step(dev, (2, 3, 8, 16)), _step(dev, (2, 3, 8, 16))
    et.muon_step_(**step)
    again["grads"] = [again["grads"][0].view(6, 8, 16)]
    et.muon_step_(**again)
    assert torch.equal(step["params"][0], again["params"][0])
    assert torch.equal(step["momentum_buffers"][0], again["momentum_buffers"][0])


def test_the_held_optimizer(et, dev):
    step = _step(dev)
    p, g = step["params"][0], step["grads"][0]
    with pytest.raises(ValueError, match="masters"):
        et.Muon([p.bfloat16()], masters=[p.mT.contiguous()])
    opt = et.Muon([p, torch.randn(4, 6, device=dev)])
    before = p.clone()
    for other in _other(g):
        for second in (torch.randn(4, 6, device=dev), None):
            with pytest.raises(ValueError, match="grads"):
                opt.step([other, second])
    assert torch.equal(p, before) and not opt.momentum_buffers[0].any()
    # a parameter that has become another matrix since
    p.data = p.data.mT.contiguous()
    with pytest.raises(ValueError, match="params"):
        opt.step([g, None])
    with pytest.raises(ValueError, match="params"):
        opt.step([g.mT.contiguous(), None])
    p.data = before.clone()
    opt.step([g, None])
    assert not torch.equal(p, before)
