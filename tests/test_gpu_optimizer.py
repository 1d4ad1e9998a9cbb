"""AdamW over many tensors (f32 and 8-bit states) and the gradient norm against
a plain implementation in 64 bits, element by element with derived bounds; the
8-bit states also against the written definition in 32 bits, bit for bit."""
import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24          # unit roundoff of binary32
BF = 2.0 ** -8          # of bfloat16
BLOCK = 256

SIZES = [[1], [0, 1, 255, 256, 257, 3], [4095, 4096, 4097, 12289, 5], [1000] * 53 + [70001]]
HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


def _f32(v):
    return float(torch.tensor(v, dtype=torch.float32))


def _scalars(step, lr, betas, eps, weight_decay):
    """The constants as the call rounds them to binary32."""
    b1, b2 = betas
    return (_f32(b1), _f32(1 - b1), _f32(b2), _f32(1 - b2), _f32(1 / math.sqrt(1 - b2 ** step)), _f32(eps),
            _f32(1 - lr * weight_decay), _f32(lr / (1 - b1 ** step)))


def _make(sizes, pdtype, gdtype, seed, misalign=0, spread=2.0):
    """Host lists; with `misalign` each tensor starts that many elements into its buffer."""
    g = torch.Generator().manual_seed(seed)

    def buf(n, dtype, v):
        b = torch.zeros(n + misalign, dtype=dtype)
        b[misalign:] = v
        return b

    out = dict(p=[], g=[], m=[], v=[], w=[])
    for n in sizes:
        size = torch.exp(torch.randn(n, generator=g) * spread) * 1e-3
        w = torch.randn(n, generator=g) * 0.02
        out["w"].append(buf(n, torch.float32, w))
        out["p"].append(buf(n, pdtype, w.to(pdtype)))
        out["g"].append(buf(n, gdtype, (torch.randn(n, generator=g) * size).to(gdtype)))
        out["m"].append(buf(n, torch.float32, torch.randn(n, generator=g) * size * 0.3))
        out["v"].append(buf(n, torch.float32, (torch.randn(n, generator=g) * size).square() * 0.7))
    return out


def _dev(lists, dev, off):
    return [t.to(dev)[off:] for t in lists]


def _reference(w, g, m, v, c, scale):
    """(w, m, v) in 64 bits, and bounds of what the roundings of the 32-bit
    formula can add: each +, *, /, sqrt one unit of its result."""
    b1, o1, b2, o2, rb, eps, decay, size = c
    w, g, m, v = w.double(), g.double() * scale, m.double(), v.double()
    m2 = b1 * m + o1 * g
    em = 4 * U * (b1 * m.abs() + o1 * g.abs())          # g * scale, the two products, the sum
    v2 = b2 * v + o2 * g * g
    ev = 8 * U * v2                                     # (g * scale)^2: 3, the products, the sum; all >= 0
    d = v2.sqrt() * rb + eps
    ed = 8 * U * d                                      # half of v's, sqrt, *, +
    t = size * m2 / d
    et = size * em / d + t.abs() * (ed / d + 4 * U)
    w2 = w * decay - t
    ew = 2 * U * (w * decay).abs() + et + 2 * U * w2.abs()
    tiny = 2.0 ** -126                                  # (results below the normal range lose their last bits)
    return (w2, m2, v2), (ew + tiny, em + tiny, ev + tiny)


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("pdtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("gdtype", [torch.float32, torch.bfloat16], ids=["gf32", "gbf16"])
@pytest.mark.parametrize("misalign", [0, 1, 2])
@pytest.mark.parametrize("step,scale", [(1, None), (1000, 0.37)])
def test_adamw_against_64_bits(et, dev, sizes, pdtype, gdtype, misalign, step, scale):
    h = _make(sizes, pdtype, gdtype, 11 * step + len(sizes), misalign)
    p, g, m, v = (_dev(h[k], dev, misalign) for k in "pgmv")
    w = _dev(h["w"], dev, misalign) if pdtype == torch.bfloat16 else None
    gs = None if scale is None else torch.tensor([scale], device=dev)
    et.adamw_step_(p, g, m, v, step=step, masters=w, grad_scale=gs, **HYPER)
    c = _scalars(step, **HYPER)
    for i in range(len(sizes)):
        ref, bound = _reference(*(h[k][i][misalign:] for k in "wgmv"), c, 1.0 if scale is None else _f32(scale))
        got = ((w if w else p)[i], m[i], v[i])
        for name, r, b, x in zip("wmv", ref, bound, got):
            assert torch.all((x.cpu().double() - r).abs() <= b), (i, name)
        if w:
            assert torch.equal(p[i].cpu(), w[i].cpu().to(torch.bfloat16)), i


def test_adamw_in_front_of_and_behind_the_tensors_nothing_changes(et, dev):
    for n in (1, 5, 255, 1024, 4097):
        bufs = [torch.full((n + 64,), 7.0, device=dev) for _ in range(4)]
        p, g, m, v = ([b[32:32 + n]] for b in bufs)
        et.adamw_step_(p, g, m, v, step=3, **HYPER)
        for b in bufs:
            assert torch.all(b[:32] == 7.0) and torch.all(b[32 + n:] == 7.0)
        assert torch.all(bufs[1] == 7.0)


# --------------------------------------------------------------------------- #
# 8-bit states
# --------------------------------------------------------------------------- #

def _words(seed, start, n):
    low = 0xFFFFFFFF
    x = ((torch.arange(n, dtype=torch.int64) + start) * 0x9E3779B1 + seed) & low
    x = ((x ^ (x >> 15)) * 0x6A09E667) & low
    x = ((x ^ (x >> 13)) * 0xBB67AE85) & low
    return x ^ (x >> 16)


def _pad(x):
    return torch.nn.functional.pad(x, (0, -len(x) % BLOCK)).view(-1, BLOCK)


def _quantize(x, words, root):
    """The written definition, in binary32 on the host: (e4m3, scales)."""
    n = len(x)
    b = _pad(x)
    most = b.abs().amax(1, keepdim=True)
    zero = most < 1e-35
    scale = torch.where(zero, 0.0, most * _f32(1 / 448))
    inv = torch.where(zero, 0.0, torch.full_like(most, 448.0) / most)
    r = (b.abs() * inv).clamp(max=448.0)
    if words is not None:
        small = torch.where(r < 2.0 ** -6, _f32(2.0 ** -6), 0.0).float()
        bits = ((r + small).view(torch.int32) + (_pad(words) << 4).to(torch.int32)) & -(1 << 20)
        r = (bits.view(torch.float32) - small).clamp(max=448.0)
    if root:
        r = torch.where((b > 0) & ~zero, r.clamp(min=2.0 ** -9), r)
    q = torch.copysign(r, b).view(-1)[:n].to(torch.float8_e4m3fn)
    return q, scale.view(-1)


def _held(q, scale):
    return (_pad(q.float()) * scale[:, None]).view(-1)[:len(q)]


def _state8(h, misalign):
    st = []
    for m, v in zip(h["m"], h["v"]):
        st.append(_quantize(m[misalign:], None, False) + _quantize(v[misalign:].sqrt(), None, True))
    return st


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("pdtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("gdtype", [torch.float32, torch.bfloat16], ids=["gf32", "gbf16"])
@pytest.mark.parametrize("misalign", [0, 1])
@pytest.mark.parametrize("seed", [None, 12345])
def test_adamw8_against_64_bits_and_the_definition(et, dev, sizes, pdtype, gdtype, misalign, seed):
    step = 7
    h = _make(sizes, pdtype, gdtype, 5 + len(sizes), misalign)
    st = _state8(h, misalign)
    p, g = (_dev(h[k], dev, misalign) for k in "pg")
    w = _dev(h["w"], dev, misalign) if pdtype == torch.bfloat16 else None

    def buf(t):     # e4m3 at an odd address when misaligned
        b = torch.zeros(t.numel() + misalign, dtype=t.dtype, device=dev)[misalign:]
        b.copy_(t)
        return b
    m8, ms, u8, us = ([buf(s[k]) for s in st] for k in range(4))
    et.adamw8_step_(p, g, m8, ms, u8, us, step=step, masters=w, seed=seed, **HYPER)
    c = _scalars(step, **HYPER)
    b1, o1, b2, o2 = c[:4]
    start = 0
    for i, n in enumerate(sizes):
        q, qs, r, rs = st[i]
        m, u = _held(q, qs), _held(r, rs)
        gi, wi = h["g"][i][misalign:].float(), h["w"][i][misalign:]
        # the weight: as with f32 states (u * u adds one rounding, u's product another)
        ref, bound = _reference(wi, gi, m, u.double() ** 2, c, 1.0)
        x = (w if w else p)[i].cpu().double()
        assert torch.all((x - ref[0]).abs() <= bound[0] + 4 * U * (ref[0] - wi.double() * c[6]).abs()), i
        # the states: the definition's bits
        m2 = m * b1 + gi * o1
        # (a binary64 root rounded to binary32 is the correctly rounded one; the
        # host library's binary32 root is not always)
        u2 = torch.sqrt(((u * u) * b2 + (gi * gi) * o2).double()).float()
        words = None if seed is None else _words(seed, start, n)
        for x2, got, scale, half, root in ((m2, m8[i], ms[i], 16, False), (u2, u8[i], us[i], 0, True)):
            want, want_scale = _quantize(x2, None if words is None else (words >> half) & 0xFFFF, root)
            assert torch.equal(got.cpu().view(torch.uint8), want.view(torch.uint8)), (i, root)
            assert torch.equal(scale.cpu(), want_scale), (i, root)
            # and within a step of e4m3 (nearest: half a step) of the 64-bit value
            s = scale.cpu().double().repeat_interleave(BLOCK)[:n]
            exact = (ref[1] if not root else ref[2].sqrt())
            grid = torch.exp2((exact.abs() / s.clamp(min=1e-300)).clamp(min=2.0 ** -6).log2().floor() - 3) * s
            off = (got.cpu().double() * s - exact).abs()
            slack = 1e-5 * exact.abs() + 1e-5 * grid + (2.0 ** -9 * s if root else 0.0)
            assert torch.all(off <= grid * (1.0 if seed is not None else 0.5) + slack), (i, root)
        start += -(-n // BLOCK) * BLOCK


def test_adamw8_launches_share_one_count_of_elements(et, dev):
    """60 tensors take two launches; the random words go on counting."""
    n, k = 300, 60
    g = torch.Generator().manual_seed(3)
    grads = [torch.randn(n, generator=g) for _ in range(k)]
    z = lambda dt, c: [torch.zeros(c, dtype=dt, device=dev) for _ in range(k)]  # noqa: E731
    m8, u8, ms, us = z(torch.float8_e4m3fn, n), z(torch.float8_e4m3fn, n), z(torch.float32, 2), z(torch.float32, 2)
    et.adamw8_step_(z(torch.float32, n), [t.to(dev) for t in grads], m8, ms, u8, us, step=1, seed=99, **HYPER)
    o1 = _f32(1 - HYPER["betas"][0])
    for i in (0, 47, 48, 59):
        want, _ = _quantize(grads[i] * o1, _words(99, 512 * i, n) >> 16, False)
        assert torch.equal(m8[i].cpu().view(torch.uint8), want.view(torch.uint8)), i


def test_stochastic_rounding_is_unbiased_and_moves_the_average(et, dev):
    """With a gradient whose m is constant over a million elements, the mean of
    what is held is m within 6 standard errors (a value is one of two neighbours,
    s apart: deviation at most s / 2).  And an average that was 4 times too high
    comes down under stochastic rounding and not under rounding to nearest."""
    n = 1 << 20
    for value in (0.7, 0.0113, 0.3001):
        gval = torch.full((n,), value)
        gval[::BLOCK] = 1.0                            # every block's largest
        z = lambda dt, c: [torch.zeros(c, dtype=dt, device=dev)]  # noqa: E731
        m8, u8, ms, us = z(torch.float8_e4m3fn, n), z(torch.float8_e4m3fn, n), z(torch.float32, n // BLOCK), z(torch.float32, n // BLOCK)
        et.adamw8_step_(z(torch.float32, n), [gval.to(dev)], m8, ms, u8, us, step=1, lr=0.0, betas=(0.0, 0.0), seed=5)
        for q, s in ((m8, ms), (u8, us)):
            held = (q[0].double().view(-1, BLOCK) * s[0].double()[:, None])[:, 1:]
            r = value * 448
            grid = 2.0 ** (math.floor(math.log2(r)) - 3) / 448
            err = 6 * grid / 2 / math.sqrt(held.numel()) + 1e-6
            assert abs(held.mean().item() - value) <= err, value
            assert set(torch.unique((held * 448).round(decimals=3)).tolist()) <= {
                round(math.floor(r / (grid * 448)) * grid * 448, 3), round((math.floor(r / (grid * 448)) + 1) * grid * 448, 3)}
    n = 1 << 14
    finals = {}
    for stochastic in (False, True):
        opt = et.AdamW([torch.zeros(n, device=dev)], lr=0.0, betas=(0.9, 0.99), state="e4m3", stochastic=stochastic)
        spike = torch.full((n,), 0.25, device=dev)
        spike[::BLOCK] = 1.0
        for _ in range(800):
            opt.step([spike])
        small = spike.clone()
        small[small < 1] = 0.0625
        for _ in range(400):
            opt.step([small])
        root = (opt.exp_avg_root[0].float().view(-1, BLOCK) * opt.exp_avg_root_scale[0][:, None])[:, 1:]
        finals[stochastic] = root.mean().item()
    # 400 steps of 0.99: the excess of v is down to 2%
    assert abs(finals[True] - 0.0625) < 0.02, finals
    assert finals[False] > 0.2, finals


def test_scale_that_is_not_finite_skips_the_step(et, dev):
    for bad in (float("nan"), float("inf")):
        gs = torch.tensor(bad, device=dev)
        for state in ("f32", "e4m3"):
            p = [torch.randn(1000, device=dev).bfloat16(), torch.randn(77, device=dev).bfloat16()]
            opt = et.AdamW(p, state=state)
            opt.step([torch.randn(t.shape, device=dev) for t in p])
            before = {k: v.clone().view(torch.uint8) for k, v in opt.flat.items()}, [t.clone() for t in p]
            opt.step([torch.randn(t.shape, device=dev) for t in p], grad_scale=gs)
            assert all(torch.equal(v.view(torch.uint8), before[0][k]) for k, v in opt.flat.items())
            assert all(torch.equal(a, b) for a, b in zip(p, before[1]))


def test_infinite_and_nan_gradients_stay_in_their_element_or_block(et, dev):
    for bad in (float("nan"), float("inf"), -float("inf")):
        g = torch.randn(1024, device=dev)
        g[300] = bad
        p = [torch.zeros(1024, device=dev)]
        opt = et.AdamW(p)
        opt.step([g])
        ok = torch.ones(1024, dtype=torch.bool, device=dev)
        ok[300] = False
        assert torch.isfinite(p[0][ok]).all() and torch.isfinite(opt.exp_avg[0][ok]).all()
        assert not torch.isfinite(opt.exp_avg[0][300])
        p = [torch.zeros(1024, device=dev)]
        opt = et.AdamW(p, state="e4m3")
        opt.step([g])
        assert torch.isfinite(p[0][ok]).all()
        assert torch.isnan(opt.exp_avg_scale[0]).tolist() == [False, True, False, False]
        opt.step([torch.randn(1024, device=dev)])
        fine = torch.ones(1024, dtype=torch.bool, device=dev)
        fine[256:512] = False
        assert torch.isfinite(p[0][fine]).all() and torch.isnan(p[0][~fine]).all()


def test_zero_gradients_and_zero_states(et, dev):
    for state in ("f32", "e4m3"):
        p = [torch.ones(600, device=dev)]
        opt = et.AdamW(p, lr=0.1, weight_decay=0.5, state=state)
        opt.step([torch.zeros(600, device=dev)])
        assert torch.all(p[0] == _f32(1 - 0.1 * 0.5))
        assert all(torch.all(v.float() == 0) for v in opt.flat.values())
    # tiny gradients: squares that vanish, a block below the smallest scale
    p = [torch.zeros(600, device=dev)]
    opt = et.AdamW(p, state="e4m3")
    opt.step([torch.full((600,), 1e-38, device=dev)])
    assert torch.isfinite(p[0]).all() and torch.all(opt.exp_avg_scale[0] == 0)


# --------------------------------------------------------------------------- #
# the optimizer object, streams and graphs
# --------------------------------------------------------------------------- #

def _random_params(dev, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(s, generator=g).to(dev).to(dtype) for s in [(3, 5), (700,), (64, 129), (2, 40, 8)]]


@pytest.mark.parametrize("state", ["f32", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_optimizer_is_the_functions(et, dev, state, dtype):
    p = _random_params(dev, dtype)
    q = [t.clone() for t in p]
    opt = et.AdamW(p, state=state, seed=40, **HYPER)
    low = dtype == torch.bfloat16
    w = [t.float() for t in q] if low else None
    if state == "f32":
        st = [[torch.zeros(t.shape, device=dev) for t in q] for _ in range(2)]
    else:
        e4 = lambda: [torch.zeros(t.shape, dtype=torch.float8_e4m3fn, device=dev) for t in q]  # noqa: E731
        sc = lambda: [torch.zeros(et.adamw8_scales(t.numel()), device=dev) for t in q]  # noqa: E731
        st = [e4(), sc(), e4(), sc()]
    for step in range(1, 4):
        g = [torch.randn(t.shape, device=dev) * 0.1 for t in p]
        norm, scale = et.grad_norm(g, max_norm=0.5)
        opt.step(g, grad_scale=scale)
        if state == "f32":
            et.adamw_step_(q, g, *st, step=step, masters=w, grad_scale=scale, **HYPER)
        else:
            et.adamw8_step_(q, g, *st, step=step, masters=w, grad_scale=scale, seed=40 + step, **HYPER)
    for a, b in zip(p, q):
        assert torch.equal(a, b)
    for mine, other in zip(opt._states, st):
        for a, b in zip(mine, other):
            assert torch.equal(a.reshape(-1).view(torch.uint8), b.reshape(-1).view(torch.uint8))


def test_optimizer_mixed_types_missing_gradients_and_moved_storage(et, dev):
    p = _random_params(dev, torch.float32)
    p[1] = p[1].bfloat16()
    p[3] = p[3].bfloat16()
    q = [t.clone() for t in p]
    a, b = et.AdamW(p), et.AdamW(q)
    g = [torch.randn(t.shape, device=dev) for t in p]
    g[0] = g[0].bfloat16()
    a.step(g)
    for i in range(4):            # one by one: the same, tensor by tensor
        b.steps = 0
        b.step([t if j == i else None for j, t in enumerate(g)])
    assert all(torch.equal(x, y) for x, y in zip(p, q))
    a.step([None] * 4)
    assert a.steps == 2 and all(torch.equal(x, y) for x, y in zip(p, q))
    old = p[2].clone()
    p[2].data = p[2].data.clone()
    keep = q[2].clone()
    a.steps, b.steps = 1, 1
    a.step(g), b.step(g)
    assert torch.equal(p[2], q[2]) and not torch.equal(p[2], old) and torch.equal(keep, old)


@pytest.mark.parametrize("state", ["f32", "e4m3"])
def test_optimizer_state_dict_resumes_bit_for_bit(et, dev, state):
    p = _random_params(dev, torch.bfloat16)
    opt = et.AdamW(p, state=state, **HYPER)
    g = [[torch.randn(t.shape, device=dev) for t in p] for _ in range(4)]
    opt.step(g[0]), opt.step(g[1])
    held, q = opt.state_dict(), [t.clone() for t in p]
    opt.step(g[2]), opt.step(g[3])
    other = et.AdamW(q, state=state, **HYPER)
    other.load_state_dict(held)
    other.step(g[2]), other.step(g[3])
    assert all(torch.equal(a, b) for a, b in zip(p, q)) and other.steps == 4


def test_side_stream_and_graph_replays(et, dev):
    p = _random_params(dev, torch.bfloat16)
    q = [t.clone() for t in p]
    g = [torch.randn(t.shape, device=dev) for t in p]
    a, b = et.AdamW(p, state="e4m3", lr=1e-2), et.AdamW(q, state="e4m3", lr=1e-2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _, scale = et.grad_norm(g, max_norm=1.0)
        a.step(g, grad_scale=scale)
    torch.cuda.current_stream().wait_stream(s)
    _, scale_b = et.grad_norm(g, max_norm=1.0)
    b.step(g, grad_scale=scale_b)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(p, q))
    # the captured step (its scalars fixed) replayed four times against eager steps of the same number
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, scale = et.grad_norm(g, max_norm=1.0)
        a.step(g, grad_scale=scale)
    for _ in range(4):
        for t in g:
            t.mul_(0.9)
        graph.replay()
        torch.cuda.synchronize()
        b.steps = 1
        _, scale_b = et.grad_norm(g, max_norm=1.0)
        b.step(g, grad_scale=scale_b)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(p, q))
        assert all(torch.equal(a.flat[k].view(torch.uint8), b.flat[k].view(torch.uint8)) for k in a.flat)


# --------------------------------------------------------------------------- #
# gradient norm
# --------------------------------------------------------------------------- #

@pytest.mark.parametrize("sizes", [[1], [0, 3], [16383, 16384, 16385, 7], [33] * 130 + [100003]], ids=lambda s: str(len(s)))
@pytest.mark.parametrize("misalign", [0, 1])
def test_grad_norm_against_64_bits(et, dev, sizes, misalign):
    gen = torch.Generator().manual_seed(len(sizes))
    host = []
    for i, n in enumerate(sizes):
        t = torch.exp(torch.randn(n + misalign, generator=gen) * 4)
        host.append(t.bfloat16() if i % 3 == 1 else t)
    g = [t.to(dev)[misalign:] for t in host]
    want = math.sqrt(sum(float(t[misalign:].double().square().sum()) for t in host))
    norm, scale = et.grad_norm(g, max_norm=0.75)
    # 64-bit sums of exact squares: one rounding to 32 bits (and 2^-40 of the sums' order)
    assert abs(norm.item() - want) <= (U + 2.0 ** -40) * want
    ref = min(1.0, 0.75 / (want + 1e-6))
    assert abs(scale.item() - ref) <= 4 * U * ref
    again, none = et.grad_norm(g)
    assert again.item() == norm.item() and none is None


def test_grad_norm_of_extreme_values(et, dev):
    big = torch.full((1000,), 1e30, device=dev)
    norm, scale = et.grad_norm([big], max_norm=1.0)      # squares pass binary32's range
    assert abs(norm.item() - math.sqrt(1000) * _f32(1e30)) <= 2 * U * norm.item()
    assert 0 < scale.item() < 1e-31
    norm, scale = et.grad_norm([torch.zeros(10, device=dev)], max_norm=2.0)
    assert norm.item() == 0 and scale.item() == 1
    norm, scale = et.grad_norm([torch.empty(0, device=dev)], max_norm=2.0)
    assert norm.item() == 0 and scale.item() == 1
    for bad in (float("inf"), float("nan")):
        big[17] = bad
        norm, scale = et.grad_norm([big, torch.ones(5, device=dev)], max_norm=1.0)
        assert not math.isfinite(norm.item()) and math.isnan(scale.item())


# --------------------------------------------------------------------------- #
# refusals
# --------------------------------------------------------------------------- #

def test_refusals(et, dev):
    t = lambda n=8, dt=torch.float32: torch.zeros(n, dtype=dt, device=dev)  # noqa: E731
    ok = dict(step=1, lr=0.1)
    with pytest.raises(TypeError):
        et.adamw_step_(t(), [t()], [t()], [t()], **ok)
    with pytest.raises(ValueError, match="at least one"):
        et.adamw_step_([], [], [], [], **ok)
    with pytest.raises(ValueError, match="HIP device"):
        et.adamw_step_([torch.zeros(8)], [t()], [t()], [t()], **ok)
    with pytest.raises(TypeError, match="float32 or"):
        et.adamw_step_([t(8, torch.float16)], [t()], [t()], [t()], **ok)
    with pytest.raises(ValueError, match="elements"):
        et.adamw_step_([t()], [t(9)], [t()], [t()], **ok)
    with pytest.raises(ValueError, match="tensors"):
        et.adamw_step_([t(), t()], [t()], [t(), t()], [t(), t()], **ok)
    with pytest.raises(ValueError, match="contiguous"):
        et.adamw_step_([t(16)[::2]], [t()], [t()], [t()], **ok)
    with pytest.raises(TypeError, match="exp_avg"):
        et.adamw_step_([t()], [t()], [t(8, torch.bfloat16)], [t()], **ok)
    with pytest.raises(ValueError, match="masters"):
        et.adamw_step_([t(8, torch.bfloat16)], [t()], [t()], [t()], **ok)
    with pytest.raises(ValueError, match="masters"):
        et.adamw_step_([t()], [t()], [t()], [t()], masters=[t()], **ok)
    for bad in (dict(step=0, lr=0.1), dict(step=1, lr=-1.0), dict(step=1, lr=float("nan")),
                dict(step=1, lr=0.1, betas=(1.0, 0.9)), dict(step=1, lr=0.1, eps=-1e-8)):
        with pytest.raises(ValueError):
            et.adamw_step_([t()], [t()], [t()], [t()], **bad)
    with pytest.raises(ValueError, match="grad_scale"):
        et.adamw_step_([t()], [t()], [t()], [t()], grad_scale=t(2), **ok)
    e4 = torch.float8_e4m3fn
    with pytest.raises(ValueError, match="exp_avg_scale"):
        et.adamw8_step_([t(257)], [t(257)], [t(257, e4)], [t(1)], [t(257, e4)], [t(2)], **ok)
    with pytest.raises(TypeError, match="exp_avg_root"):
        et.adamw8_step_([t()], [t()], [t(8, e4)], [t(1)], [t(8, torch.uint8)], [t(1)], **ok)
    with pytest.raises(ValueError, match="max_norm"):
        et.grad_norm([t()], max_norm=0.0)
    with pytest.raises(ValueError, match="workspace"):
        et.grad_norm([t(100000)], workspace=t(1, torch.uint8))
    opt = et.AdamW([t(), t(4)])
    with pytest.raises(ValueError, match="tensors"):
        opt.step([t()])
    with pytest.raises(ValueError, match="elements"):
        opt.step([t(), t(5)])
    assert opt.steps == 0
    with pytest.raises(ValueError, match="state"):
        et.AdamW([t()], state="int8")
    with pytest.raises(ValueError, match="expected"):
        opt.load_state_dict({"steps": 3})
    assert ctypes.sizeof(ctypes.c_void_p) == 8


def test_masters_that_are_all_none(et, dev):
    g = [torch.randn(33, device=dev), torch.randn(5, device=dev)]
    p, q = ([torch.ones(33, device=dev), torch.ones(5, device=dev)] for _ in range(2))
    a, b = et.AdamW(p, masters=[None, None]), et.AdamW(q)
    for _ in range(2):
        a.step(g), b.step(g)
        a.step([g[0], None]), b.step([g[0], None])
    assert all(torch.equal(x, y) for x, y in zip(p, q))
    b.load_state_dict(a.state_dict())
    a.load_state_dict(b.state_dict())


# --------------------------------------------------------------------------- #
# parameters of different ages, copies, what a state may hold
# --------------------------------------------------------------------------- #

@pytest.mark.parametrize("state", ["f32", "e4m3"])
@pytest.mark.parametrize("dtypes", [(torch.float32,) * 3, (torch.bfloat16, torch.float32, torch.bfloat16)], ids=["one", "two"])
def test_a_parameter_without_gradients_keeps_its_step_number(et, dev, state, dtypes):
    """A parameter whose first gradient arrives late takes its first step: the
    bits of an optimizer of its own that began then."""
    late = 1000
    shapes = [(700,), (3, 5), (300,)]
    g = torch.Generator().manual_seed(2)
    p = [torch.randn(s, generator=g).to(dev).to(t) for s, t in zip(shapes, dtypes)]
    q = [t.clone() for t in p]
    kw = dict(state=state, stochastic=False, **HYPER)
    opt, alone = et.AdamW(p, **kw), [et.AdamW([t], **kw) for t in q]
    opt.steps = late                # (as after so many steps with every gradient)
    alone[0].steps = alone[2].steps = late
    opt._counts = [late, 0, late]   # but for the second parameter, which had none
    for turn in range(4):
        grads = [torch.randn(s, generator=g).to(dev) for s in shapes]
        if turn == 2:
            grads[2] = None
        opt.step(grads)
        for a, t in zip(alone, grads):
            if t is not None:
                a.step([t])
        assert opt.steps == late + turn + 1
        assert all(torch.equal(x, y) for x, y in zip(p, q)), turn
        if turn == 2:               # a state that is loaded goes on the same way
            held = opt.state_dict()
            opt = et.AdamW(p, **kw)
            opt.load_state_dict(held)


def test_step_numbers_against_64_bits(et, dev):
    """Four parameters, gradients in some of twelve steps: every weight is that
    of the formula with its own number of steps."""
    g = torch.Generator().manual_seed(7)
    w = [torch.randn(50, generator=g) for _ in range(4)]
    p = [t.to(dev) for t in w]
    opt = et.AdamW(p, **HYPER)
    (b1, b2), lr, eps, wd = HYPER["betas"], HYPER["lr"], HYPER["eps"], HYPER["weight_decay"]
    w, m, v, n = [t.double() for t in w], [0.0] * 4, [0.0] * 4, [0] * 4
    for turn in range(12):
        # gradients of one sign: the denominator stays away from 0
        grads = [torch.rand(50, generator=g) + 0.5 for _ in range(4)]
        has = [True, turn >= 9, turn % 3 == 1, turn < 2]
        opt.step([t.to(dev) if h else None for t, h in zip(grads, has)])
        for i in range(4):
            if has[i]:
                x = grads[i].double()
                n[i] += 1
                m[i], v[i] = b1 * m[i] + (1 - b1) * x, b2 * v[i] + (1 - b2) * x * x
                w[i] = w[i] * (1 - lr * wd) - lr / (1 - b1 ** n[i]) * m[i] / ((v[i] / (1 - b2 ** n[i])).sqrt() + eps)
    for i in range(4):
        # a step moves a weight by 1.3 lr at most (m and sqrt(v) are averages of [0.5, 1.5]) with some 40
        # roundings (of the constants and of both averages' histories), and rounds it three times
        bound = n[i] * (1.3 * lr * 40 * U + 3 * U * (w[i].abs() + 1.3 * lr * n[i]))
        assert torch.all((p[i].cpu().double() - w[i]).abs() <= bound), i


@pytest.mark.parametrize("state", ["f32", "e4m3"])
@pytest.mark.parametrize("given", [False, True])
def test_copies_and_pickles_go_on_alike(et, dev, state, given):
    import copy
    import io
    p = _random_params(dev, torch.bfloat16)
    opt = et.AdamW(p, state=state, masters=[t.float() for t in p] if given else None, **HYPER)
    g = [[torch.randn(t.shape, device=dev) for t in p] for _ in range(3)]
    opt.step(g[0])
    opt.step([None] + g[0][1:])
    buf = io.BytesIO()
    torch.save(opt, buf)
    buf.seek(0)
    others = [copy.deepcopy(opt), torch.load(buf, weights_only=False)]
    buf.seek(0)
    with pytest.raises(ValueError, match="HIP device"):
        torch.load(buf, weights_only=False, map_location="cpu")
    for other in others:
        assert all(a.data_ptr() != b.data_ptr() for a, b in zip(opt.params, other.params))
        assert all(v.untyped_storage().data_ptr() == other.flat["exp_avg"].untyped_storage().data_ptr()
                   for v in other.exp_avg)
        other.step(g[1]), other.step(g[2])
    mid = [t.clone() for t in p]
    opt.step(g[1]), opt.step(g[2])
    assert not all(torch.equal(a, b) for a, b in zip(mid, p))
    for other in others:
        assert all(torch.equal(a, b) for a, b in zip(p, other.params))
        assert all(torch.equal(a, b) for a, b in zip(opt.masters, other.masters))
        assert other.steps == 4


def test_a_state_that_does_not_fit_changes_nothing(et, dev):
    p = _random_params(dev, torch.bfloat16)
    opt = et.AdamW(p, masters=[t.float() for t in p])
    opt.step([torch.randn(t.shape, device=dev) for t in p])
    before, flat = [t.clone() for t in opt.masters], {k: v.clone() for k, v in opt.flat.items()}

    def wrong(change):
        held = opt.state_dict()
        held["masters"] = [torch.zeros_like(t) for t in held["masters"]]
        held.update({k: torch.ones_like(v) for k, v in held.items() if k.startswith("exp_avg")})
        change(held)
        with pytest.raises((ValueError, TypeError)):
            opt.load_state_dict(held)
        assert all(torch.equal(a, b) for a, b in zip(before, opt.masters))
        assert all(torch.equal(flat[k], opt.flat[k]) for k in flat) and opt.steps == 1

    wrong(lambda h: h["masters"].__setitem__(2, None))
    wrong(lambda h: h["masters"].__setitem__(2, torch.zeros(1, device=dev)))     # (would broadcast)
    wrong(lambda h: h["masters"].__setitem__(3, h["masters"][3].bfloat16()))
    wrong(lambda h: h["masters"].pop())
    wrong(lambda h: h.update(exp_avg_sq=h["exp_avg_sq"][1:]))
    wrong(lambda h: h.update(exp_avg=None))
    wrong(lambda h: h.update(steps=-1))
    wrong(lambda h: h.update(steps="many"))
    wrong(lambda h: h.update(counts=[1, 1]))
    wrong(lambda h: h.update(counts=[1, 1, 1, 2]))


def test_a_parameter_given_twice_is_refused(et, dev):
    t = torch.zeros(64, device=dev)
    with pytest.raises(ValueError, match="more than once|overlap"):
        et.AdamW([t, torch.zeros(3, device=dev), t])
    with pytest.raises(ValueError, match="overlap"):
        et.AdamW([t[:40], t[32:]])
    with pytest.raises(ValueError, match="overlap"):
        et.AdamW([t.bfloat16(), torch.zeros(64, device=dev).bfloat16()], masters=[t, t])
    et.AdamW([t[:32], t[32:], t[:0], t[:0]])


def test_steps_count_as_changes_of_the_parameters(et, dev):
    """A weight that the forward kept and a step has changed since is an error in
    the backward, not a gradient of another weight."""
    for state, dtype in (("f32", torch.float32), ("e4m3", torch.bfloat16)):
        x = torch.randn(4, 8, device=dev, dtype=dtype, requires_grad=True)
        w = torch.randn(8, 8, device=dev, dtype=dtype, requires_grad=True)
        opt = et.AdamW([w], state=state)
        y = (x.float() @ w.float().mul(w.float())).sum() + (x * w[0]).sum()
        opt.step([torch.randn(8, 8, device=dev)])
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
        z = lambda dt=torch.float32, n=64: [torch.zeros(n, dtype=dt, device=dev)]  # noqa: E731
        e4 = torch.float8_e4m3fn
        p, s = z(), w._version
        et.adamw_step_(p, z(), z(), z(), step=1, lr=0.1)
        assert p[0]._version == 1
        et.adamw8_step_(p, z(), z(e4), z(n=1), z(e4), z(n=1), step=1, lr=0.1)
        assert p[0]._version == 2
        opt.step([None])
        assert w._version == s
    with torch.inference_mode():
        w = torch.ones(8, device=dev)
        et.AdamW([w]).step([torch.ones(8, device=dev)])
        assert torch.all(w < 1)


def test_workspaces_that_only_look_large_are_refused(et, dev):
    """A workspace of enough elements on one element of memory."""
    small = torch.zeros(2, dtype=torch.float64, device=dev)
    for bad in (small[:1].expand(4096), small[:1].expand(64, 64), torch.zeros(9000, device=dev)[::2]):
        with pytest.raises(ValueError, match="workspace"):
            et.grad_norm([torch.ones(1 << 20, device=dev)], workspace=bad)


def test_a_shallow_copy_counts_for_itself(et, dev):
    import copy
    p = [torch.zeros(8, device=dev), torch.zeros(8, device=dev)]
    g = torch.ones(8, device=dev)
    opt = et.AdamW(p)
    opt.step([g, None])
    other = copy.copy(opt)
    other.step([g, g])
    assert opt.state_dict()["counts"] == [1, 0] and other.state_dict()["counts"] == [2, 1]
