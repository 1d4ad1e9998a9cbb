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
