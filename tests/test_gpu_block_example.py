"""examples/moe_block.py: the norm, the experts, the optimizer and the 4-bit
serving path run together."""
import importlib.util
import os

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("moe_block", os.path.join(ROOT, "examples", "moe_block.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_block_trains_and_serves(et, dev, example):
    losses, errors = example.main(["--tokens", "512", "--width", "256", "--hidden", "128", "--steps", "40"])
    assert losses[-1] < 0.8 * losses[0]
    # 4-bit values of groups of 64 normal weights are off by scale / sqrt(12) =
    # max / 7.5 / 3.46, about 0.1 of their deviation; three projections of it
    assert all(e < 0.3 for e in errors)


@pytest.mark.parametrize("state", ["f32", "e4m3"])
def test_states_of_8_bits_train_like_those_of_32(et, dev, example, state):
    make = lambda seed: example.Block(256, 8, 128, 2, "cuda", seed)  # noqa: E731
    teacher, block = make(1), make(2)
    teacher.router.eval()
    losses = example.train(block, teacher, 512, 40, state=state)
    assert losses[-1] < 0.8 * losses[0]


def test_block_gradients_against_differences(et, dev, example):
    """The whole block's input gradient along a direction, against a central
    difference of the f64 sum of its bf16 outputs over many tokens: bf16 outputs
    of 512 tokens leave a noise of 2^-9 |y| sqrt(n) / step, 5% of the derivative here.
    Thresholds of 0 route every token to every expert: with others the
    output jumps where a step changes the routing, which no gradient has."""
    block = example.Block(256, 8, 128, 2, "cuda", 3)
    block.router.eval()
    block.router.thr.zero_()
    g = torch.Generator(device=dev).manual_seed(5)
    x = torch.randn(512, 256, generator=g, device=dev)
    v = torch.randn(512, 256, generator=g, device=dev)
    y, kept = block.forward(x.bfloat16())
    # the loss sum(c y) with c the direction's own image, so that the derivative is large
    step = 2.0 ** -4
    up, down = (block.forward((x + s * v).bfloat16())[0].double() for s in (step, -step))
    c = ((up - down) / (2 * step)).bfloat16()
    dx, _ = block.backward(c, kept)
    exact = (dx.double() * v.double()).sum().item()
    diff = (c.double() * (up - down)).sum().item() / (2 * step)
    assert abs(exact - diff) <= 0.1 * abs(diff)


def _float64_block(block, x, mask):
    """The block in float64 by torch's autograd, the routing that of `mask`."""
    gain, bias, w_router, w_gu, w_down = (p.detach().double().requires_grad_(True) for p in block.params)
    x = x.double().requires_grad_(True)
    c = x - x.mean(1, keepdim=True)
    h = c / (c.square().mean(1, keepdim=True) + 1e-5).sqrt() * gain + bias
    gate = torch.sigmoid(h @ w_router.t()) * mask
    y = x
    for e in range(len(w_gu)):
        gate_up = h @ w_gu[e].t()
        f = gate_up.shape[1] // 2
        g = gate_up[:, :f]
        y = y + gate[:, e:e + 1] * ((g * torch.sigmoid(g) * gate_up[:, f:]) @ w_down[e].t())
    return y, x, [gain, bias, w_router, w_gu, w_down]


@pytest.mark.parametrize("everyone", [True, False])
def test_every_gradient_against_64_bits(et, dev, example, everyone):
    """dx past the identity and the five parameters' gradients.  Ten roundings to
    bf16 on the way (h, gu, a, yp, dyp, da, dgu, dxp, dh, dx), each of
    2^-9 / sqrt(3) of a value at random, leave 0.4% of a gradient's size; dx, rounded
    with the identity's part in it, 2^-9 |dy| / sqrt(3) more.  Three times that is
    allowed.  The norm's own terms (the means over a row that it takes out of dh),
    which are 6% of it, are also looked at alone."""
    block = example.Block(256, 8, 128, 2, "cuda", 3)
    block.router.eval()
    g = torch.Generator(device=dev).manual_seed(5)
    block.gain.add_(torch.randn(256, generator=g, device=dev) * 0.2)
    block.bias.add_(torch.randn(256, generator=g, device=dev) * 0.2)
    block.router.thr.fill_(0.0 if everyone else 0.6)
    x = torch.randn(512, 256, generator=g, device=dev).bfloat16()
    dy = torch.randn(512, 256, generator=g, device=dev).bfloat16()
    y, kept = block.forward(x)
    dx, grads = block.backward(dy, kept)
    plan = kept[4]
    mask = torch.zeros(512, 8, dtype=torch.float64, device=dev)
    mask[plan.sorted_token.long(), torch.repeat_interleave(torch.arange(8, device=dev), plan.counts.long())] = 1.0
    want_y, x64, params = _float64_block(block, x, mask)
    want = torch.autograd.grad(want_y, [x64] + params, dy.double())
    allowed = 3 * 0.004
    assert (y.double() - want_y).norm() <= allowed * (want_y - x64).norm() + 2.0 ** -9 * want_y.norm()
    past, want_past = dx.double() - dy.double(), want[0] - dy.double()
    slack = 3 * 2.0 ** -9 / 3 ** 0.5 * dx.double().norm()
    assert (past - want_past).norm() <= allowed * want_past.norm() + slack
    for name, a, b in zip(("gain", "bias", "router", "gate_up", "down"), grads, want[1:]):
        assert (a.double() - b).norm() <= allowed * b.norm(), name
    # what the norm takes out of a row's gradient: its mean, and its share along xhat (both 0 of past)
    c = x.double() - x.double().mean(1, keepdim=True)
    xhat = c / c.square().mean(1, keepdim=True).sqrt()
    for along in (torch.ones_like(xhat), xhat):
        share = (past * along).sum(1) / 16.0        # (a row of 256: |along| = 16)
        # the roundings' part along one direction of 256
        assert share.norm() <= (allowed * want_past.norm() + slack) / 16.0
