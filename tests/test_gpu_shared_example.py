"""examples/shared_expert.py: the shared expert, the orthogonalised step and the
adapters run together, with the routed experts and their 4-bit serving."""
import importlib.util
import math
import os

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("shared_expert", os.path.join(ROOT, "examples", "shared_expert.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_it_runs(et, dev, example):
    losses = example.main(["--tokens", "256", "--width", "128", "--hidden", "64", "--steps", "6"])
    assert len(losses) == 6 and all(math.isfinite(v) for v in losses)


@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_block_gradients_against_differences(et, dev, example, activation):
    """The input gradient along a direction against a central difference of the
    block's outputs, thresholds at 0 (no step changes the routing): bf16 outputs of
    512 tokens leave a noise of 2^-9 |y| sqrt(n) / step, some 5% of the derivative."""
    block = example.SharedBlock(256, 8, 128, 2, "cuda", 3, activation)
    block.router.eval()
    block.router.thr.zero_()
    g = torch.Generator(device=dev).manual_seed(5)
    x, v = (torch.randn(512, 256, generator=g, device=dev) for _ in range(2))
    _, kept = block.forward(x.bfloat16())
    step = 2.0 ** -4
    up, down = (block.forward((x + s * v).bfloat16())[0].double() for s in (step, -step))
    c = ((up - down) / (2 * step)).bfloat16()
    dx, grads = block.backward(c, kept)
    diff = (c.double() * (up - down)).sum().item() / (2 * step)
    assert abs((dx.double() * v.double()).sum().item() - diff) <= 0.1 * abs(diff)
    assert [g.shape for g in grads] == [p.shape for p in block.params]


def test_shared_weights_gradients(et, dev, example):
    """Those of the shared expert's two weights and of the norm's gain, the routed experts' part
    taken out, against float64 autograd.  A value passes through six roundings to bf16 on the
    way (h, a, the products' outputs, dp and the gradient): 6 half steps of 2^-8 in norm."""
    block = example.SharedBlock(128, 4, 64, 2, "cuda", 7)
    block.router.eval()
    block.w_down.zero_()                # the routed experts give and take nothing
    g = torch.Generator(device=dev).manual_seed(1)
    x, dy = (torch.randn(96, 128, generator=g, device=dev).bfloat16() for _ in range(2))
    _, kept = block.forward(x)
    dx, grads = block.backward(dy, kept)
    leaves = [t.double().requires_grad_() for t in (x, block.gain, block.bias, block.w_shared, block.w_back)]
    xd, gain, bias, w, back = leaves
    z = (xd - xd.mean(1, keepdim=True)) / (xd.var(1, correction=0, keepdim=True) + 1e-5).sqrt()
    p = (z * gain + bias) @ w.t()
    y = xd + (torch.nn.functional.silu(p[:, :64]) * p[:, 64:]) @ back.t()
    want = torch.autograd.grad(y, leaves, dy.double())
    for got, exact, name in zip((dx, grads[0], grads[1], grads[5], grads[6]), want, ("x", "gain", "bias", "w", "back")):
        off = ((got.double() - exact).norm() / exact.norm()).item()
        assert off <= 6 * 2.0 ** -8, (name, off)


def test_every_matrix_is_stepped_and_served(et, dev, example):
    """One step changes every parameter; a batch served with adapters differs from one without
    in the rows that have one, and there by the adapter's formula."""
    block = example.SharedBlock(128, 4, 64, 2, "cuda", 9)
    before = [p.clone() for p in block.params]
    x = torch.randn(300, 128, device=dev).bfloat16()
    y, kept = block.forward(x)
    _, grads = block.backward(y, kept)
    example.Optimizers(block, 0.02).step(grads)
    for a, b in zip(before, block.params):
        assert not torch.equal(a, b) and torch.isfinite(b.float()).all()
    block.router.eval()
    bank = example.random_bank(block, 3, 8)
    server = example.SharedServer(block, bank)
    x = torch.randn(7, 128, device=dev).bfloat16()
    index = torch.tensor([0, -1, 2, 1, -1, 0, 2], dtype=torch.int32, device=dev)
    own, plain = server(x, index), server(x, torch.full_like(index, -1))
    assert torch.equal(own[index < 0], plain[index < 0])
    a = et.gated_linear(et.layer_norm(x, block.gain, block.bias), block.w_shared)
    at = index.clamp(min=0).long()
    delta = torch.einsum("tnr,tr->tn", bank.b[at].double(), torch.einsum("trk,tk->tr", bank.a[at].double(), a.double()))
    has = index >= 0
    # (the projection's output, the adapters' sum, and the block's sum, each rounded to bf16 on both sides)
    bound = 2.0 ** -8 * 3 * (own.double().abs() + plain.double().abs() + delta.abs() + 4)
    assert bool(((own.double() - plain.double() - delta).abs() <= bound)[has].all())
