"""The Muon step of matrices that one block does not take (a shorter side above 64), and of large ones that it
does, in every pair of types, against float64: bounds as test_gpu_muon derives them."""
import pytest
import torch

from test_gpu_muon import _check_step, _lists

pytestmark = pytest.mark.gpu

# products by 32 x 32 blocks; by the tile loop; wide and tall each, rows of whole 16 bytes and not; one
# block a matrix, of more than 32768 elements, whose momentum is read again
FEW = [(130, 77), (96, 264), (300, 72), (65, 65)]
MANY = [(40, 384, 520), (24, 501, 154), (2, 3, 128, 512), (70, 330)]
ONE = [(64, 1024), (2, 1100, 50), (33, 1501), (2, 40, 1200)]


@pytest.mark.parametrize("dtype,gdtype", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16),
                                          (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("nesterov,rms", [(True, 0.2), (False, None)])
@pytest.mark.parametrize("shapes", [FEW, MANY, ONE], ids=["few", "many", "one"])
def test_step(et, dev, shapes, dtype, gdtype, nesterov, rms):
    params, masters, momenta, grads = _lists(dev, shapes, dtype, gdtype)
    w = masters or params
    old = [(a.clone(), b.clone()) for a, b in zip(w, momenta)]
    scale = torch.full((), 0.37, device=dev)
    et.muon_step_(params, grads, momenta, lr=0.01, momentum=0.9, weight_decay=0.1, nesterov=nesterov, update_rms=rms,
                  masters=masters, grad_scale=scale)
    _check_step(old, list(zip(w, momenta)), grads, scale.double().item(), 0.9, nesterov, 0.01, 0.1, rms)
    if masters:
        assert all(torch.equal(p, m.bfloat16()) for p, m in zip(params, masters))


@pytest.mark.parametrize("dtype,gdtype", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_a_scale_that_is_not_finite_keeps_every_bit(et, dev, dtype, gdtype, bad):
    params, masters, momenta, grads = _lists(dev, FEW + MANY + ONE, dtype, gdtype)
    held = params + momenta + (masters or [])
    before = [t.clone() for t in held]
    kw = dict(lr=0.01, momentum=0.9, weight_decay=0.1, masters=masters)
    et.muon_step_(params, grads, momenta, grad_scale=torch.full((1,), bad, device=dev), **kw)
    assert all(torch.equal(a, b) for a, b in zip(held, before))
    et.muon_step_(params, grads, momenta, grad_scale=torch.ones(1, device=dev), **kw)
    assert not any(torch.equal(a, b) for a, b in zip(held, before))
    assert all(torch.isfinite(t.float()).all() for t in held)


def test_more_tensors_than_a_set(et, dev):
    """47 tensors of two kinds of types and every way: several launches of each, one behind the other."""
    shapes = [(66 + 5 * (i % 9), 100 + 9 * (i % 7)) if i % 2 else (140 - i, 70) if i % 3 else (2, 20, 30 + i) for i in range(47)]
    fp, _, momenta, grads = _lists(dev, shapes, torch.float32, torch.float32)
    params = [p.bfloat16() if i % 2 else p for i, p in enumerate(fp)]
    masters = [fp[i] if i % 2 else None for i in range(47)]
    old = [(a.clone(), b.clone()) for a, b in zip(fp, momenta)]
    et.muon_step_(params, grads, momenta, lr=0.01, momentum=0.9, weight_decay=0.1, masters=masters)
    _check_step(old, list(zip(fp, momenta)), grads, 1.0, 0.9, True, 0.01, 0.1, 0.2)
    assert all(torch.equal(p, m.bfloat16()) for p, m in zip(params, masters) if m is not None)


def test_a_callers_workspace_of_the_stated_size(et, dev):
    """Of all shapes at once, for a step of two kinds of types whose tensors alternate: the bits of the step with its own."""
    shapes = [(128, 200), (70, 66), (300, 90)] * 16
    a, b = (_lists(dev, shapes, torch.float32, torch.float32)[0::2] for _ in range(2))
    grads = [g.bfloat16() if i % 2 else g for i, g in enumerate(_lists(dev, shapes, torch.float32, torch.float32)[3])]
    et.muon_step_(a[0], grads, a[1], lr=0.01)
    n = et.orthogonalize_workspace_bytes(shapes)
    ws = torch.full((n + 4096,), 0x7f, device=dev, dtype=torch.uint8)        # (NaN as f16; as f32 and binary64 large)
    et.muon_step_(b[0], grads, b[1], lr=0.01, workspace=ws[:n])
    assert all(torch.equal(x, y) for x, y in zip(a[0] + a[1], b[0] + b[1]))
    assert bool((ws[n:] == 0x7f).all())
    with pytest.raises(ValueError, match="workspace"):
        et.muon_step_(b[0], grads, b[1], lr=0.01, workspace=ws[:1 << 20])
