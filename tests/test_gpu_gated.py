"""The gated projection and its backward on the GPU, against the formulas in
float64 on the same bf16 inputs.

Bounds, element by element, with eps(binary32) = 2^-24 and bf16's half step
2^-8: a product's sum of n terms is off by at most n 2^-24 sum|terms| (any
order); act' is at most 1.13 in size and act(g) at most |g|; the activation's
own arithmetic is good to 2^-20 of its value (some ten roundings, erfc's few
units).  What a later step makes of an error is the same formula on absolute
values.  Sizes cover one token, one chunk of K, rows and hidden units that end
inside a tile, both tile sizes of every product, and rows that are a slice."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

EPS, HALF = 2.0 ** -24, 2.0 ** -8


def _inputs(dev, T, K, F, pad=0, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed * 131 + T + K + F)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    x = torch.full((T, K + pad), float("nan"), device=dev, dtype=torch.bfloat16)
    x[:, :K] = r(T, K)
    return x[:, :K], (r(2 * F, K) * K ** -0.5).bfloat16(), (r(T, F) * 0.1).bfloat16()


def _act(g, activation):
    """(act(g), act'(g)) in float64."""
    if activation == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    p = 0.5 * torch.special.erfc(-g / math.sqrt(2))
    return g * p, p + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def _want(x, w, activation, dh=None):
    """{name: (value, bound)}"""
    x, w = x.double(), w.double()
    T, K = x.shape
    F = w.shape[0] // 2
    p = x @ w.t()
    dp_sum = K * EPS * (x.abs() @ w.abs().t())          # error of g and u
    g, u = p[:, :F], p[:, F:]
    eg, eu = dp_sum[:, :F], dp_sum[:, F:]
    a, s = _act(g, activation)
    e_a = 1.13 * eg + 2.0 ** -20 * a.abs()
    h = a * u
    out = dict(h=(h, HALF * h.abs() + 1.01 * (e_a * (u.abs() + eu) + a.abs() * eu) + 1e-38))
    if dh is None:
        return out
    dh = dh.double()
    # (act'' is at most 1 in size for both; 2^-20 of the slope's terms, which are at most 1.2)
    e_s = eg + 2.0 ** -20 * 1.2
    dp = torch.cat([dh * u * s, dh * a], 1)
    e = torch.cat([dh.abs() * (e_s * (u.abs() + eu) + s.abs() * eu), dh.abs() * e_a], 1)
    e = 1.01 * e + HALF * (dp.abs() + e)
    big = dp.abs() + e
    dx, dw = dp @ w, dp.t() @ x
    out["dx"] = dx, HALF * dx.abs() + 1.01 * (e @ w.abs() + 2 * F * EPS * (big @ w.abs()))
    # (splits of the tokens are added in binary32 as well: T terms in all)
    out["dw"] = dw, HALF * dw.abs() + 1.01 * (e.t() @ x.abs() + T * EPS * (big.t() @ x.abs()))
    out["dw32"] = dw, out["dw"][1] - HALF * dw.abs() + EPS * dw.abs()
    return out


def _close(got, want, name):
    value, bound = want
    off = (got.double() - value).abs()
    assert torch.isfinite(got.double()).all(), name
    worst = (off / bound.clamp(min=1e-300)).max().item() if off.numel() else 0.0
    assert worst <= 1.0, (name, worst)


SIZES = [(1, 8, 8), (1, 64, 8), (2, 72, 24), (17, 136, 40), (33, 1032, 16), (64, 512, 104), (65, 200, 72), (200, 72, 48), (128, 64, 64), (130, 64, 136),
         (257, 1000, 712), (1025, 136, 264)]


@pytest.mark.parametrize("activation", ["silu", "gelu"])
@pytest.mark.parametrize("T,K,F", SIZES)
def test_forward_and_backward(et, dev, T, K, F, activation):
    print(f"gated T={T} K={K} F={F} {activation}", flush=True)
    x, w, dh = _inputs(dev, T, K, F, pad=8 * (T % 3))
    want = _want(x, w, activation, dh)
    wide = torch.full((T + 3, F), 7.0, device=dev, dtype=torch.bfloat16)
    h = et.gated_linear(x, w, activation=activation, out=wide[:T])
    _close(h, want["h"], "h")
    assert bool((wide[T:] == 7).all())
    dx, dw = et.gated_linear_backward(dh, x, w, activation=activation)
    _close(dx, want["dx"], "dx")
    _close(dw, want["dw"], "dw")
    dw32 = torch.empty(2 * F, K, device=dev)
    none, again = et.gated_linear_backward(dh, x, w, activation=activation, need_dx=False, out_dw=dw32)
    assert none is None and again is dw32
    _close(dw32, want["dw32"], "dw32")
    # the same bits again
    assert torch.equal(h, et.gated_linear(x, w, activation=activation))
    dx2, dw2 = et.gated_linear_backward(dh, x, w, activation=activation)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)


@pytest.mark.parametrize("side", [2, 4, 6, 8])
@pytest.mark.parametrize("T,K,F", [(1, 8, 8), (5, 64, 24), (300, 72, 136), (513, 256, 520), (1100, 136, 40), (700, 328, 4104), (700, 136, 4104), (300, 64, 8200)])
def test_all_tiles_of_the_forward(et, dev, T, K, F, side):
    print(f"gated tile {side} T={T} K={K} F={F}", flush=True)
    x, w, _ = _inputs(dev, T, K, F)
    x = x.contiguous()
    h = torch.empty(T, F, device=dev, dtype=torch.bfloat16)
    rc = et.lib().et_gated_linear_impl(x.data_ptr(), K, w.data_ptr(), T, K, F, 0, h.data_ptr(), side,
                                       torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    _close(h, _want(x, w, "silu")["h"], "h")


@pytest.mark.parametrize("T,K,F", [(8200, 1088, 600), (150, 3584, 1800), (5000, 520, 2200), (3001, 72, 712), (3001, 1400, 72), (3003, 2824, 1408)])
def test_large_tiles_of_the_backward(et, dev, T, K, F):
    """Enough tiles for 192 x 128 or 256 x 256 ones in the recomputation, dx (alone too) or dw, and a block that
    walks several."""
    print(f"gated large T={T} K={K} F={F}", flush=True)
    x, w, dh = _inputs(dev, T, K, F)
    want = _want(x, w, "silu", dh)
    _close(et.gated_linear(x, w), want["h"], "h")
    dx, dw = et.gated_linear_backward(dh, x, w)
    _close(dx, want["dx"], "dx")
    _close(dw, want["dw"], "dw")
    _close(et.gated_linear_backward(dh, x, w, need_dw=False)[0], want["dx"], "dx")


@pytest.mark.parametrize("T,K,F", [(20001, 264, 72), (40000, 64, 16), (9000, 72, 200)])
def test_long_sums_of_the_weight_gradient(et, dev, T, K, F):
    """Many tokens for few weights: dW's sum split beside dx, which alone fills the GPU; and alone, whose
    splits differ."""
    print(f"gated long T={T} K={K} F={F}", flush=True)
    x, w, dh = _inputs(dev, T, K, F)
    want = _want(x, w, "silu", dh)
    for need_dx in (True, False):
        dx, dw = et.gated_linear_backward(dh, x, w, need_dx=need_dx)
        _close(dw, want["dw"], "dw")
        if need_dx:
            _close(dx, want["dx"], "dx")


def test_no_rows_and_wide_strides(et, dev):
    w = torch.randn(48, 64, device=dev).bfloat16()
    x = torch.empty(0, 64, device=dev, dtype=torch.bfloat16)
    assert et.gated_linear(x, w).shape == (0, 24)
    dx, dw = et.gated_linear_backward(torch.empty(0, 24, device=dev, dtype=torch.bfloat16), x, w)
    assert dx.shape == (0, 64) and bool((dw == 0).all())
    # rows far apart: the last row's offset in x passes 32 bits
    big = torch.empty(530, 1 << 22, device=dev, dtype=torch.bfloat16)[:, :64 + 64]
    x = big[:, 64:][:, :64]
    assert (x.shape[0] - 1) * x.stride(0) * 2 > 2 ** 32 - 2 ** 23
    with pytest.raises(ValueError, match="2\\^22"):
        et.gated_linear(x, w)
    big = torch.empty(1100, (1 << 21) + 8, device=dev, dtype=torch.bfloat16)
    x = big[:, 64:128]
    x.copy_(torch.randn(1100, 64, device=dev))
    dh = torch.randn(1100, 24, device=dev).bfloat16()
    want = _want(x, w, "silu", dh)
    _close(et.gated_linear(x, w), want["h"], "h")
    dx, dw = et.gated_linear_backward(dh, x, w)
    _close(dx, want["dx"], "dx")
    _close(dw, want["dw"], "dw")


def test_rows_beyond_32_bits(et, dev):
    """h, dh and the projections' gradient of more than 4 GiB: the last rows' results."""
    T, K, F, n = (1 << 20) + 77, 64, 2056, 70
    last, w, dlast = _inputs(dev, n, K, F)
    x = torch.zeros(T, K, device=dev, dtype=torch.bfloat16)
    dh = torch.zeros(T, F, device=dev, dtype=torch.bfloat16)
    x[-n:], dh[-n:] = last, dlast
    want = _want(last, w, "silu", dlast)
    h = et.gated_linear(x, w)
    _close(h[-n:], want["h"], "h")
    assert not h[:-n].any()
    del h
    dx, dw = et.gated_linear_backward(dh, x, w)
    _close(dx[-n:], want["dx"], "dx")
    _close(dw, want["dw"], "dw")
    assert not dx[:-n].any()


def test_a_bad_row_stays_a_row(et, dev):
    x, w, dh = _inputs(dev, 70, 72, 40)
    x = x.contiguous()
    clean = et.gated_linear(x, w)
    clean_dx, _ = et.gated_linear_backward(dh, x, w)
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[33, 5] = bad
        h = et.gated_linear(y, w)
        dx, dw = et.gated_linear_backward(dh, y, w)
        others = torch.arange(70, device=dev) != 33
        assert torch.equal(h[others], clean[others]) and not torch.isfinite(h[33]).all()
        assert torch.equal(dx[others], clean_dx[others])
        assert torch.isnan(dw).any()


def test_large_values_saturate_as_the_formula(et, dev):
    """Gates far out on both sides: act(g) -> g or 0, act' -> 1 or 0; no NaN from exp."""
    K = 64
    x = torch.zeros(4, K, device=dev, dtype=torch.bfloat16)
    x[:, 0] = torch.tensor([200.0, -200.0, 1e4, -1e4], device=dev)
    w = torch.zeros(32, K, device=dev, dtype=torch.bfloat16)
    w[:, 0] = 1
    dh = torch.ones(4, 16, device=dev, dtype=torch.bfloat16)
    for activation in ("silu", "gelu"):
        h = et.gated_linear(x, w, activation=activation)
        dx, dw = et.gated_linear_backward(dh, x, w, activation=activation)
        g = x[:, :1].double()
        assert torch.equal(h.double(), torch.where(g > 0, g * g, 0.0).expand(4, 16).bfloat16().double())
        assert torch.isfinite(dx.double()).all() and torch.isfinite(dw.double()).all()
        assert bool((dx[1] == 0).all()) and bool((dx[3] == 0).all())


def test_gelu_over_its_range(et, dev):
    """g Phi(g) of every bf16 g in [-13, 40], against erfc in float64: 2^-20 of the value and the
    rounding to bf16 (below -13 the value is under 2^-120)."""
    bits = torch.arange(1 << 16, device=dev, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    g = bits[torch.isfinite(bits.float()) & (bits.float() >= -13) & (bits.float() <= 40)]
    x = torch.zeros(len(g), 8, device=dev, dtype=torch.bfloat16)
    x[:, 0], x[:, 1] = g, 1
    w = torch.zeros(16, 8, device=dev, dtype=torch.bfloat16)
    w[:8, 0] = 1                    # the gates: g
    w[8:, 1] = 1                    # up: 1
    h = et.gated_linear(x, w, activation="gelu").double()
    want = _act(g.double(), "gelu")[0][:, None]
    off = (h - want).abs()
    assert bool((off <= (HALF + 2.0 ** -20) * want.abs() + 2.0 ** -133).all()), (off / want.abs()).max().item()
    # the slope: dx[:, 0] is the sum of 8 units' slopes, each rounded to bf16 (they are equal)
    dx, _ = et.gated_linear_backward(torch.ones(len(g), 8, device=dev, dtype=torch.bfloat16), x, w, activation="gelu")
    slope = _act(g.double(), "gelu")[1] * 8
    assert bool(((dx[:, 0].double() - slope).abs() <= 2 * (HALF + 2.0 ** -20) * slope.abs() + 8 * 2.0 ** -22).all())


@pytest.mark.parametrize("activation", ["silu", "gelu"])
def test_gradients_against_differences(et, dev, activation):
    """The loss sum(h c) along a direction: the float64 formula's central difference against <dx, v> + <dw, z>."""
    x, w, dh = _inputs(dev, 40, 64, 32, seed=3)
    dx, dw = et.gated_linear_backward(dh, x, w, activation=activation)
    g = torch.Generator(device=dev).manual_seed(9)
    v, z = (torch.randn(t.shape, generator=g, device=dev, dtype=torch.float64) for t in (x, w))

    def loss(s):
        p = (x.double() + s * v) @ (w.double() + s * z).t()
        return (_act(p[:, :32], activation)[0] * p[:, 32:] * dh.double()).sum()

    step = 1e-4
    by_difference = ((loss(step) - loss(-step)) / (2 * step)).item()
    want = _want(x, w, activation, dh)
    bound = ((want["dx"][1] * v.abs()).sum() + (want["dw"][1] * z.abs()).sum()).item()
    got = ((dx.double() * v).sum() + (dw.double() * z).sum()).item()
    # (the difference's own error: step^2 / 6 of the third derivative, far below)
    assert abs(got - by_difference) <= bound + 1e-5 * abs(by_difference)


def test_autograd_and_needs(et, dev):
    x, w, dh = _inputs(dev, 33, 72, 24)
    x = x.contiguous()
    want = et.gated_linear_backward(dh, x, w)
    for need_x, need_w in ((True, True), (True, False), (False, True)):
        a, b = x.clone().requires_grad_(need_x), w.clone().requires_grad_(need_w)
        h = et.gated_linear_autograd(a, b)
        h.backward(dh)
        assert (a.grad is not None) == need_x and (b.grad is not None) == need_w
        if need_x:
            assert torch.equal(a.grad, want[0])
        if need_w:
            assert torch.equal(b.grad, want[1])
    # a gradient that is broadcast (of a sum), and a second derivative
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    et.gated_linear_autograd(a, b).sum().backward()
    ones = et.gated_linear_backward(torch.ones_like(dh), x, w)
    assert torch.equal(a.grad, ones[0]) and torch.equal(b.grad, ones[1])
    a = x.clone().requires_grad_()
    grad, = torch.autograd.grad(et.gated_linear_autograd(a, w).float().square().sum(), a, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_streams_and_graph(et, dev):
    """On another stream than the current one of other work, and captured: replays with new inputs
    between eager calls, each against the eager result."""
    T, K, F = 300, 136, 72
    x, w, dh = (t.contiguous() for t in _inputs(dev, T, K, F))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        h = et.gated_linear(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(h, et.gated_linear(x, w))
    et.gated_linear_backward(dh, x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gh = et.gated_linear(x, w)
        gdx, gdw = et.gated_linear_backward(dh, x, w)
    for rep in range(3):
        x2, w2, dh2 = _inputs(dev, T, K, F, seed=rep + 5)
        x.copy_(x2), w.copy_(w2), dh.copy_(dh2)
        graph.replay()
        torch.cuda.synchronize()
        want = et.gated_linear(x, w), *et.gated_linear_backward(dh, x, w)
        for a, b in zip((gh, gdx, gdw), want):
            assert torch.equal(a, b), rep
    del graph


def test_operators(et, dev):
    x, w, dh = (t.contiguous() for t in _inputs(dev, 20, 72, 40))
    ops = torch.ops.etmoe
    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    torch.library.opcheck(ops.gated_linear.default, (x.clone().requires_grad_(), w.clone().requires_grad_(), "gelu"),
                          test_utils=tests)
    for need in ((True, True), (False, True), (True, False)):
        torch.library.opcheck(ops.gated_linear_backward.default, (dh, x, w, "silu", *need),
                              test_utils=("test_schema", "test_faketensor"))
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()

    def f(a, b):
        return ops.gated_linear(a, b, "silu").float().square().sum()

    f(a, b).backward()
    c, d = x.clone().requires_grad_(), w.clone().requires_grad_()
    torch.compile(f, fullgraph=True, backend="aot_eager")(c, d).backward()
    assert torch.equal(a.grad, c.grad) and torch.equal(b.grad, d.grad)


def test_refusals(et, dev):
    x, w, dh = _inputs(dev, 4, 64, 16)
    for bad in (dict(x=x.float()), dict(w=w.float())):
        with pytest.raises(TypeError):
            et.gated_linear(**{**dict(x=x, w=w), **bad})
    for bad in (dict(w=w[:, :56].contiguous()), dict(w=w[:24].contiguous()), dict(w=w[:, ::2]), dict(activation="relu"),
                dict(x=x.t()), dict(x=x[:, 4:60], w=w[:, :56].contiguous()), dict(w=w.cpu()),
                dict(x=x[0]), dict(out=torch.empty(4, 8, device=dev, dtype=torch.bfloat16)),
                dict(x=torch.empty(4, 68, device=dev, dtype=torch.bfloat16)[:, :64])):
        with pytest.raises(ValueError):
            et.gated_linear(**{**dict(x=x, w=w), **bad})
    with pytest.raises(ValueError):
        et.gated_linear_backward(dh[:, :8].contiguous(), x, w)
    with pytest.raises(ValueError):
        et.gated_linear_backward(dh, x, w, workspace=torch.empty(16, dtype=torch.uint8, device=dev))
