"""Newton-Schulz orthogonalisation and the step that uses it, on the GPU, against
float64.

Bound.  Between the products X, A and S are held in f16 (half step 2^-11), which
the steps amplify by up to a per iteration while a singular value is small; how
much comes of it depends on the matrix.  So the reference does the same steps in
float64 twice, exactly and with X, A and S rounded to f16 where the kernels round
them: the kernel's binary32 sums move a few roundings to the neighbouring number,
so its distance from the exact result may be twice the rounded reference's (in
the Frobenius norm), and the bf16 result adds at most its half step, 2^-8."""
import copy
import math
import pickle

import pytest
import torch

pytestmark = pytest.mark.gpu

ABC = (3.4445, -4.7750, 2.0315)
EPS, HALF = 2.0 ** -24, 2.0 ** -8


def _f16(x, scale):
    return (x * scale).half().double() / scale


def _reference(u, steps=5, abc=ABC, eps=1e-7, rounded=False):
    """[E, m, n] float64"""
    a, b, c = abc
    rx = (lambda t: _f16(t, 2.0 ** 14)) if rounded else (lambda t: t)
    rs = (lambda t: _f16(t, 2.0 ** 14)) if rounded else (lambda t: t)
    u = u.double()
    tall = u.shape[1] > u.shape[2]
    x = u.mT.contiguous() if tall else u
    x = rx(x / (torch.sqrt((x * x).sum((1, 2), keepdim=True)) + eps))
    eye = torch.eye(x.shape[1], device=x.device, dtype=x.dtype)
    for _ in range(steps):
        g = rx(torch.bmm(x, x.mT.contiguous()))
        x = rx(torch.bmm(rs(a * eye + b * g + c * torch.bmm(g, g)), x))
    return x.mT if tall else x


def _off(got, u, **kw):
    """(distance, bound) in the Frobenius norm, of each matrix; X not rounded to bf16."""
    exact = _reference(u, **kw)
    near = (_reference(u, rounded=True, **kw) - exact).flatten(1).norm(dim=1)
    return (got.double() - exact).flatten(1).norm(dim=1), 2 * near + 2.0 ** -11 * exact.flatten(1).norm(dim=1), exact


def _check(got, u, what="", **kw):
    off, bound, exact = _off(got, u, **kw)
    bound = bound + HALF * exact.flatten(1).norm(dim=1) + 1e-30
    assert bool((off <= bound).all()), (what, (off / bound).max().item())


def _gradient(dev, E, m, n, seed=0, low_rank=True):
    g = torch.Generator(device=dev).manual_seed(seed * 977 + 31 * E + 7 * m + n)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    v = r(E, m, n)
    if low_rank:
        k = max(1, min(m, n) // 16)
        v = v + 3 * torch.bmm(r(E, m, k), r(E, k, n)) * k ** -0.5
    return v * 1e-3


SIZES = [(1, 1, 1), (1, 1, 7), (3, 9, 1), (2, 5, 3), (1, 16, 64), (1, 77, 130), (2, 130, 77), (3, 501, 154), (2, 154, 501),
         (4, 256, 256), (1, 520, 300), (1, 8, 2048), (2, 2048, 9), (3, 64, 1024), (2, 1100, 50), (2, 40, 4096), (40, 512, 384), (40, 384, 520)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E,m,n", SIZES)
def test_orthogonalize(et, dev, E, m, n, dtype):
    print(f"orthogonalize {E} x {m} x {n} {dtype}", flush=True)
    g = _gradient(dev, E, m, n).to(dtype)
    out = torch.full((E + 1, m, n), 5.0, device=dev, dtype=torch.bfloat16)
    got = et.orthogonalize(g, out=out[:E])
    _check(got, g, (E, m, n))
    assert bool((out[E:] == 5).all())
    assert torch.equal(got, et.orthogonalize(g))
    # one matrix of the batch alone: the same up to the order of the sums, which is the same
    assert torch.equal(et.orthogonalize(g[E - 1].contiguous()), got[E - 1]) or min(m, n) > 128


@pytest.mark.parametrize("E,m,n", [(1, 65, 65), (1, 66, 512), (3, 72, 520), (1, 300, 1300), (1, 1300, 200), (1, 90, 4104), (2, 1031, 97), (1, 512, 512)])
def test_products_of_few_tiles(et, dev, E, m, n):
    """Tiles of 32 x 32: sums of one chunk, of a chunk for each wave, of several turns, and lines that end inside a tile.
    The same bits again, beside other tensors."""
    u = _gradient(dev, E, m, n, seed=3)
    got = et.orthogonalize(u)
    _check(got, u, "few")
    assert torch.equal(got, et.orthogonalize(u))
    p = [torch.zeros_like(u), torch.zeros(70, 330, device=dev)]
    et.muon_step_(p, [u, torch.randn(70, 330, device=dev)], [torch.zeros_like(t) for t in p], lr=1.0, momentum=0.0, update_rms=None,
                  nesterov=False)
    size = max(1.0, m / n) ** 0.5
    assert bool((torch.isfinite(p[0])).all())
    _check(-p[0] / size, u, "beside others")


@pytest.mark.parametrize("m,n", [(1024, 2048), (64, 1024)])
def test_tensors_beyond_32_bits(et, dev, m, n):
    """The last matrices of a tensor of more than 4 GiB, through every way that takes many."""
    E = 2 ** 31 // (m * n) + 20
    g = torch.zeros(E, m, n, device=dev, dtype=torch.bfloat16)
    last = _gradient(dev, 3, m, n, seed=6).bfloat16()
    g[-3:] = last
    got = et.orthogonalize(g)
    _check(got[-3:], last.float(), "last")
    assert not got[:-3].any()


@pytest.mark.parametrize("m,n", [(2100, 2200), (1500, 5001)])
def test_norm_of_many_elements(et, dev, m, n):
    """More elements than the blocks of a norm take at once, whole rows of 16 bytes and not."""
    u = _gradient(dev, 1, m, n, seed=4)
    _check(et.orthogonalize(u), u, "large")
    p, mom = torch.zeros_like(u), torch.zeros_like(u)
    et.muon_step_([p], [u], [mom], lr=1.0, momentum=0.5, update_rms=None, nesterov=False)
    assert torch.equal(mom, 0.5 * u)
    _check(-p / max(1.0, m / n) ** 0.5, 0.5 * u, "large step")


@pytest.mark.parametrize("steps,abc", [(1, ABC), (3, ABC), (8, ABC), (10, (1.875, -1.25, 0.375)), (5, (1.5, -0.5, 0.0))])
def test_other_polynomials(et, dev, steps, abc):
    g = _gradient(dev, 2, 96, 200, low_rank=False)
    _check(et.orthogonalize(g, steps=steps, coefficients=abc), g, steps=steps, abc=abc)


def test_scale_zero_and_bad_matrices(et, dev):
    g = _gradient(dev, 4, 40, 72)
    want = et.orthogonalize(g, eps=0.0)
    # a power of two changes nothing, not where squares pass binary32's range either
    for k in (-90, -20, 30, 100):
        assert torch.equal(et.orthogonalize(g * 2.0 ** k, eps=0.0), want), k
    g[1] = 0
    g[2, 3, 4] = float("nan")
    got = et.orthogonalize(g)
    assert bool((got[1] == 0).all()) and bool(torch.isnan(got[2]).all())
    _check(got[[0, 3]], g[[0, 3]])
    for bad in (float("inf"), -float("inf")):
        g[2, 3, 4] = bad
        assert bool(torch.isnan(et.orthogonalize(g)[2]).all())
    assert et.orthogonalize(torch.empty(0, 4, 8, device=dev)).shape == (0, 4, 8)
    assert et.orthogonalize(torch.empty(3, 0, 8, device=dev)).shape == (3, 0, 8)
    # unaligned matrices: a view from an odd element on
    flat = torch.randn(1 + 2 * 24 * 40, device=dev)
    view = flat[1:].view(2, 24, 40)
    assert torch.equal(et.orthogonalize(view), et.orthogonalize(view.clone()))


def _lists(dev, shapes, dtype, gdtype, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + 5)
    masters = [torch.randn(s, generator=g, device=dev) * 0.02 for s in shapes]
    momenta = [_gradient(dev, math.prod(s[:-2]), *s[-2:], seed=seed + 1).view(s).contiguous() for s in shapes]
    grads = [_gradient(dev, math.prod(s[:-2]), *s[-2:], seed=seed + 2).view(s).to(gdtype).contiguous() for s in shapes]
    if dtype == torch.bfloat16:
        return [m.bfloat16() for m in masters], masters, momenta, grads
    return masters, None, momenta, grads


def _check_step(old, new, grads, scale, beta, nesterov, lr, decay, rms):
    """old, new: lists of (w, m) before and after."""
    for i, ((w0, m0), (w1, m1), g) in enumerate(zip(old, new, grads)):
        g = g.double() * scale
        m = beta * m0.double() + (1 - beta) * g
        # (four roundings, and beta and 1 - beta rounded to binary32)
        bound = 4 * EPS * (m0.double().abs() + g.abs())
        assert bool(((m1.double() - m).abs() <= bound + 1e-42).all()), i
        u = (1 - beta) * g + beta * m if nesterov else m
        shape = u.shape
        size = lr * (math.sqrt(max(1.0, shape[-2] / shape[-1])) if rms is None else rms * math.sqrt(max(shape[-2:])))
        x = _reference(u.reshape(-1, *shape[-2:])).reshape(shape)
        want = (1 - lr * decay) * w0.double() - size * x
        moved = ((1 - lr * decay) * w0.double() - w1.double()) / size
        off, near, _ = _off(moved.reshape(-1, *shape[-2:]), u.reshape(-1, *shape[-2:]))
        slack = 3 * EPS * (w0.double().flatten().norm() + want.flatten().norm()) / size
        assert bool((off <= near + slack).all()), (i, (off / (near + slack)).max().item())


SHAPES = [(8, 64), (4, 32, 64), (4, 64, 16), (1, 100), (100, 1), (2, 2, 33, 21)]


@pytest.mark.parametrize("dtype,gdtype", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16),
                                          (torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("nesterov,rms", [(True, 0.2), (False, None)])
def test_step(et, dev, dtype, gdtype, nesterov, rms):
    params, masters, momenta, grads = _lists(dev, SHAPES, dtype, gdtype)
    w = masters or params
    old = [(a.clone(), b.clone()) for a, b in zip(w, momenta)]
    scale = torch.full((), 0.37, device=dev)
    et.muon_step_(params, grads, momenta, lr=0.01, momentum=0.9, weight_decay=0.1, nesterov=nesterov, update_rms=rms,
                  masters=masters, grad_scale=scale)
    _check_step(old, list(zip(w, momenta)), grads, scale.double().item(), 0.9, nesterov, 0.01, 0.1, rms)
    if masters:
        assert all(torch.equal(p, m.bfloat16()) for p, m in zip(params, masters))


def test_many_tensors_and_the_held_optimizer(et, dev):
    """More tensors than one launch takes, wide and tall, two types; several steps of the optimizer
    against the function; a gradient that is missing; a scale that is not finite."""
    shapes = [(3 + i % 5, 8 + 3 * (i % 7)) if i % 2 else (2, 30 - i % 11, 9) for i in range(53)]
    low = [i % 3 == 0 for i in range(53)]
    fp, _, _, grads = _lists(dev, shapes, torch.float32, torch.float32)
    params = [p.bfloat16() if b else p for p, b in zip(fp, low)]
    mine = [p.clone() for p in params]
    masters = [p.float() if b else None for p, b in zip(mine, low)]
    momenta = [torch.zeros(s, device=dev) for s in shapes]
    opt = et.Muon(params, lr=0.02, weight_decay=0.05)
    versions = [p._version for p in params]
    for k in range(3):
        gs = [g * (k + 1) for g in grads]
        opt.step(gs)
        et.muon_step_(mine, gs, momenta, lr=0.02, weight_decay=0.05, masters=masters)
    for a, b in zip(params, mine):
        assert torch.equal(a, b)
    for a, b in zip(opt.momentum_buffers, momenta):
        assert torch.equal(a, b)
    assert all(p._version > v for p, v in zip(params, versions))
    held = opt.state_dict()
    before = [p.clone() for p in params]
    gs = list(grads)
    gs[7] = gs[20] = None
    opt.step(gs)
    for i, (a, b) in enumerate(zip(params, before)):
        assert torch.equal(a, b) == (i in (7, 20)), i
    assert torch.equal(opt.momentum_buffers[7], momenta[7])
    opt.step([None] * 53)
    # a copy, a pickle and a loaded state go on alike
    other = copy.deepcopy(opt)
    third = pickle.loads(pickle.dumps(opt))
    for o in (opt, other, third):
        o.step(grads, lr=0.001)
    for a, b, c in zip(opt.params, other.params, third.params):
        assert torch.equal(a, b) and torch.equal(a, c) and a.data_ptr() != b.data_ptr()
    opt.load_state_dict(held)
    assert all(torch.equal(a, b) for a, b in zip(opt.momentum_buffers, momenta))
    with pytest.raises(ValueError):
        opt.load_state_dict(dict(held, momentum_buffers=held["momentum_buffers"][:-1]))
    with pytest.raises(ValueError):
        opt.load_state_dict({})
    # skipped where the scale is not finite
    bits = [t.clone() for t in params + opt.momentum_buffers + [m for m in opt.masters if m is not None]]
    for bad in (float("nan"), float("inf")):
        opt.step(grads, grad_scale=torch.full((1,), bad, device=dev))
    for a, b in zip(params + opt.momentum_buffers + [m for m in opt.masters if m is not None], bits):
        assert torch.equal(a, b)


def test_graph_and_stream(et, dev):
    g = _gradient(dev, 3, 60, 130)
    want = et.orthogonalize(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = et.orthogonalize(g)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = et.orthogonalize(g)
    for rep in range(3):
        g.copy_(_gradient(dev, 3, 60, 130, seed=rep + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, et.orthogonalize(g)), rep
    del graph


@pytest.mark.parametrize("E,m,n", [(3, 16, 200), (2, 130, 264), (1, 300, 72)])
def test_in_place(et, dev, E, m, n):
    g = torch.randn(E, m, n, device=dev).bfloat16()
    want = et.orthogonalize(g)
    assert et.orthogonalize(g, out=g) is g and torch.equal(g, want)


def test_a_refused_workspace_leaves_every_kind_as_it_was(et, dev):
    """float32 and bfloat16 tensors are two calls: a workspace that is too small for the second one is
    refused before the first."""
    p = [torch.randn(16, 64, device=dev), torch.randn(200, 264, device=dev).bfloat16()]
    masters, momenta = [None, p[1].float()], [torch.zeros_like(t, dtype=torch.float32) for t in p]
    before = [t.clone() for t in p]
    with pytest.raises(ValueError, match="workspace"):
        et.muon_step_(p, [torch.ones_like(t) for t in p], momenta, lr=0.1, masters=masters,
                      workspace=torch.empty(256, dtype=torch.uint8, device=dev))
    assert all(torch.equal(a, b) for a, b in zip(p, before)) and not any(m.any() for m in momenta)


def test_refusals(et, dev):
    g = torch.randn(2, 8, 16, device=dev)
    for bad in (dict(g=g.double()), dict(out=torch.empty(2, 8, 16, device=dev))):
        with pytest.raises(TypeError):
            et.orthogonalize(**{**dict(g=g), **bad})
    for bad in (dict(g=g.mT), dict(g=g[0, 0]), dict(g=g.cpu()), dict(steps=0), dict(steps=65), dict(eps=-1.0),
                dict(coefficients=(3.0, 1.0)), dict(coefficients=(4.0, 0.0, 0.0)), dict(coefficients=(-1.0, 0.0, 0.0)),
                dict(coefficients=(20.0, -40.0, 20.5)), dict(out=torch.empty(2, 8, 8, device=dev, dtype=torch.bfloat16)),
                dict(g=torch.empty(2, 80, 96, device=dev), workspace=torch.empty(256, device=dev, dtype=torch.uint8)),
                dict(g=torch.empty(1, 65536, device=dev))):
        with pytest.raises(ValueError):
            et.orthogonalize(**{**dict(g=g), **bad})
    p, m = torch.zeros(2, 8, 16, device=dev), torch.zeros(2, 8, 16, device=dev)
    step = dict(params=[p], grads=[g], momentum_buffers=[m], lr=0.1)
    for bad in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=float("inf")), dict(update_rms=0.0), dict(grads=[g[:1]]),
                dict(params=[]), dict(params=[torch.zeros(8, device=dev)], grads=[g[0, 0, :8]], momentum_buffers=[m[0, 0, :8]]),
                dict(params=[p.bfloat16()]), dict(grad_scale=torch.zeros(2, device=dev))):
        with pytest.raises(ValueError):
            et.muon_step_(**{**step, **bad})
    with pytest.raises(ValueError, match="overlap"):
        et.Muon([p, p])
    opt = et.Muon([p])
    with pytest.raises(ValueError):
        opt.step([g, g])
    with pytest.raises(TypeError):
        opt.step(g)
