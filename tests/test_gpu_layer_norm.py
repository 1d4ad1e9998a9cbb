"""Layer norm and its backward against a plain implementation in 64 bits, with
bounds derived from the number of roundings."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24                    # unit roundoff of binary32
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}   # unit roundoff of the output type (24 and 8 bits)
# longest chain of additions of a row's sum: 64 elements of a thread, 6 steps of a wave, 16 waves
CHAIN = 96
# of a column's: rows of a block, then the blocks of one of four waves, then 2
COLS = 300

F32, BF16 = torch.float32, torch.bfloat16
TYPES = [(F32, F32), (BF16, F32), (BF16, BF16)]
IDS = ["f32", "bf16_w32", "bf16"]
# one element; below a vector; odd; the edges of the variants (1, 2, 4 vectors a lane, 4 and 16 waves a row)
WIDTHS = [1, 3, 7, 64, 255, 512, 513, 1000, 1024, 1025, 2048, 2049, 2889, 4096, 4100, 7168, 8192, 8193, 16383, 16384]


def _rows(g, T, d, dtype, pad=0, scale=1.0, offset=0.0):
    wide = torch.full((T, d + pad), 9.0, dtype=dtype)
    wide[:, :d] = (torch.randn(T, d, generator=g) * scale + offset).to(dtype)
    return wide


def _case(T, d, types, seed, pad=0, residual=False):
    g = torch.Generator().manual_seed(seed)
    dtype, wdtype = types
    return dict(x=_rows(g, T, d, dtype, pad, 1.5, 0.7), r=_rows(g, T, d, dtype, pad, 0.5) if residual else None,
                w=(1 + torch.randn(d, generator=g) * 0.3).to(wdtype), b=(torch.randn(d, generator=g) * 0.2).to(wdtype),
                dy=_rows(g, T, d, dtype, pad, 0.02), ds=_rows(g, T, d, dtype, pad, 0.03))


def _forward64(h, w, b, eps):
    h, w = h.double(), w.double()
    d = h.shape[1]
    mean = h.sum(1, keepdim=True) / d
    c = h - mean
    var = (c * c).sum(1, keepdim=True) / d
    rstd = (var + eps).rsqrt()
    y = c * rstd * w + (0.0 if b is None else b.double())
    # what the roundings add
    em = CHAIN * U * h.abs().mean(1, keepdim=True) + U * mean.abs()
    ec = em + U * h.abs()
    ev = (CHAIN + 4) * U * var + 2 * (c.abs() * ec).mean(1, keepdim=True) + (ec * ec).mean(1, keepdim=True)
    er = rstd * (0.5 * ev / (var + eps) + 4 * U)
    ey = w.abs() * (rstd * ec + c.abs() * er + 3 * U * (c * rstd).abs()) + 2 * U * y.abs()
    return mean[:, 0], rstd[:, 0], y, em[:, 0], er[:, 0], ey


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("T,pad,residual,bias", [(1, 0, False, True), (5, 0, True, True), (67, 5, True, False),
                                                 (6, 8, False, True)])
def test_forward_against_64_bits(et, dev, types, d, T, pad, residual, bias):
    c = _case(T, d, types, d + T, pad, residual)
    x = c["x"].to(dev)[:, :d]
    r = c["r"].to(dev)[:, :d] if residual else None
    b = c["b"].to(dev) if bias else None
    eps = 1e-5
    got = et.layer_norm(x, c["w"].to(dev), b, eps=eps, residual=r, stats=True)
    h = c["x"][:, :d]
    if residual:
        h = (h.float() + c["r"][:, :d].float()).to(types[0])
        assert torch.equal(got[1].cpu(), h)
    mean, rstd, y, em, er, ey = _forward64(h, c["w"], c["b"] if bias else None, eps)
    assert torch.all((got[-2].cpu().double() - mean).abs() <= em)
    assert torch.all((got[-1].cpu().double() - rstd).abs() <= er)
    assert torch.all((got[0].cpu().double() - y).abs() <= ey + HALF[types[0]] * (y.abs() + ey))
    # the form without statistics, and the same bits again
    again = et.layer_norm(x, c["w"].to(dev), b, eps=eps, residual=r)
    again = again if residual else (again,)
    assert all(torch.equal(p, q) for p, q in zip(again, got))
    assert torch.all(c["x"].to(dev)[:, d:] == 9.0) and torch.equal(x.cpu(), c["x"][:, :d])


def _backward64(dy, h, w, mean, rstd, ds):
    dy, h, w = dy.double(), h.double(), w.double()
    mean, rstd = mean.double()[:, None], rstd.double()[:, None]
    d = h.shape[1]
    xh = (h - mean) * rstd
    g = dy * w
    c1, c2 = g.sum(1, keepdim=True) / d, (g * xh).sum(1, keepdim=True) / d
    dx = rstd * (g - c1 - xh * c2)
    a1, a2 = g.abs().mean(1, keepdim=True), (g * xh).abs().mean(1, keepdim=True)
    ex = rstd * (CHAIN + 16) * U * (g.abs() + a1 + xh.abs() * a2) + 4 * U * dx.abs()
    if ds is not None:
        dx = dx + ds.double()
        ex = ex + U * (dx.abs() + ds.double().abs())
    ew = (COLS + 6) * U * (dy * xh).abs().sum(0)
    eb = COLS * U * dy.abs().sum(0)
    return dx, (dy * xh).sum(0), dy.sum(0), ex, ew, eb


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("T,pad,dsum,bias", [(1, 0, False, True), (4, 3, True, True), (71, 0, True, False),
                                             (1030, 8, False, True)])
def test_backward_against_64_bits(et, dev, types, d, T, pad, dsum, bias):
    if T * d > 1 << 22:
        T = 260
    c = _case(T, d, types, 3 * d + T, pad)
    cut = lambda k: c[k].to(dev)[:, :d]  # noqa: E731
    w = c["w"].to(dev)
    _, mean, rstd = et.layer_norm(cut("x"), w, stats=True)
    got = et.layer_norm_backward(cut("dy"), cut("x"), w, mean, rstd, dsum=cut("ds") if dsum else None, need_dbias=bias)
    dx, dw, db, ex, ew, eb = _backward64(c["dy"][:, :d], c["x"][:, :d], c["w"], mean.cpu(), rstd.cpu(),
                                         c["ds"][:, :d] if dsum else None)
    assert torch.all((got[0].cpu().double() - dx).abs() <= ex + HALF[types[0]] * (dx.abs() + ex))
    assert torch.all((got[1].cpu().double() - dw).abs() <= ew)
    if bias:
        assert torch.all((got[2].cpu().double() - db).abs() <= eb)
    else:
        assert got[2] is None
    again = et.layer_norm_backward(cut("dy"), cut("x"), w, mean, rstd, dsum=cut("ds") if dsum else None)
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])


def test_many_rows(et, dev):
    """More rows than a launch has blocks: 70001 rows of 40, and 9000 of 4096."""
    for T, d, dtype in ((70001, 40, F32), (9000, 4096, BF16)):
        g = torch.Generator().manual_seed(T)
        x = _rows(g, T, d, dtype).to(dev)
        dy = _rows(g, T, d, dtype, scale=0.02).to(dev)
        w = torch.ones(d, device=dev)
        y, mean, rstd = et.layer_norm(x, w, stats=True)
        m, r, want, em, er, ey = _forward64(x, w, None, 1e-5)
        assert torch.all((y.double() - want).abs() <= ey + HALF[dtype] * (want.abs() + ey))
        dx, dw, db = et.layer_norm_backward(dy, x, w, mean, rstd)
        rx, rw, rb, ex, ew, eb = _backward64(dy, x, w, mean, rstd, None)
        # (a block's chain is T / blocks rows here)
        assert torch.all((dx.double() - rx).abs() <= ex + HALF[dtype] * (rx.abs() + ex))
        assert torch.all((dw.double() - rw).abs() <= 2 * ew) and torch.all((db.double() - rb).abs() <= 2 * eb)


def test_more_rows_than_one_launch_takes(et, dev):
    """67108865 rows of 8: the forward's launches hold 2^24 - 1 blocks of 4 rows."""
    T = 4 * (2 ** 24 - 1) + 5
    x = torch.empty(T, 8, dtype=BF16, device=dev)
    for i in range(0, T, 1 << 24):
        x[i:i + (1 << 24)].normal_()
    w = torch.arange(1.0, 9.0, device=dev)
    y, s, mean, rstd = et.layer_norm(x, w, residual=x, stats=True)
    for a, b in ((0, 1000), (T - 1000, T), (4 * (2 ** 24 - 1) - 500, 4 * (2 ** 24 - 1) + 3)):
        part = et.layer_norm(x[a:b].clone(), w, residual=x[a:b].clone(), stats=True)
        assert all(torch.equal(p, q[a:b]) for p, q in zip(part, (y, s, mean, rstd)))


def test_gradients_against_differences(et, dev):
    """<dL, v> against central differences of L = sum(c1 y) + sum(c2 sum) in f32
    rows of 33: a step of 2^-7 leaves a truncation of about step^2 and U * |L| /
    step of rounding, 1e-3 of the gradient's size each at the most."""
    g = torch.Generator().manual_seed(0)
    T, d, step = 9, 33, 2.0 ** -7
    x, r, w, b, c1, c2 = (torch.randn(s, generator=g).to(dev) for s in ((T, d), (T, d), (d,), (d,), (T, d), (T, d)))

    def loss(x, r, w, b):
        y, s = et.layer_norm(x, w, b, residual=r)
        return ((y.double() * c1.double()).sum() + (s.double() * c2.double()).sum()).item()

    leaves = [t.clone().requires_grad_(True) for t in (x, r, w, b)]
    y, s = et.layer_norm_autograd(leaves[0], leaves[2], leaves[3], residual=leaves[1])
    ((y * c1).sum() + (s * c2).sum()).backward()
    args = [x, r, w, b]
    for i, leaf in enumerate(leaves):
        v = torch.randn(leaf.shape, generator=g).to(dev)
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + step * v, args[i] - step * v
        diff = (loss(*up) - loss(*down)) / (2 * step)
        size = leaf.grad.double().norm().item() * v.double().norm().item()
        assert abs((leaf.grad.double() * v.double()).sum().item() - diff) <= 2e-3 * size, i


def test_autograd_parts(et, dev):
    x = torch.randn(10, 64, device=dev, dtype=BF16, requires_grad=True)
    r = torch.randn(10, 64, device=dev, dtype=BF16, requires_grad=True)
    w = torch.ones(64, device=dev, requires_grad=True)
    y = et.layer_norm_autograd(x, w)
    y.sum().backward()
    assert x.grad.shape == x.shape and w.grad.dtype == F32
    x.grad = w.grad = None
    _, s = et.layer_norm_autograd(x, w, residual=r)       # the norm's output unused
    s.sum().backward()
    assert torch.all(x.grad == 1) and torch.all(r.grad == 1) and w.grad is None
    x.grad = r.grad = None
    y, _ = et.layer_norm_autograd(x, w, residual=r)       # the sum unused
    y.sum().backward()
    assert torch.equal(x.grad, r.grad)


def test_operators(et, dev):
    """torch.ops.etmoe.layer_norm under torch.compile, with its gradient."""
    x = torch.randn(33, 96, device=dev, requires_grad=True)
    w = torch.randn(96, device=dev, requires_grad=True)
    b = torch.randn(96, device=dev, requires_grad=True)

    def f(x, w, b):
        return (torch.ops.etmoe.layer_norm(x, w, b, 1e-5)[0] ** 2).sum()

    torch.compile(f, fullgraph=True, backend="aot_eager")(x, w, b).backward()
    got = x.grad, w.grad, b.grad
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b)]
    (et.layer_norm_autograd(*leaves) ** 2).sum().backward()
    assert all(torch.equal(p, q.grad) for p, q in zip(got, leaves))


def test_no_rows_and_constant_rows(et, dev):
    w = torch.randn(100, device=dev)
    x = torch.empty(0, 100, device=dev)
    y, mean, rstd = et.layer_norm(x, w, stats=True)
    assert y.shape == (0, 100) and mean.shape == (0,)
    dx, dw, db = et.layer_norm_backward(x, x, w, mean, rstd)
    assert dx.shape == (0, 100) and torch.all(dw == 0) and torch.all(db == 0)
    # a constant row has no variance: its output is the bias
    b = torch.randn(100, device=dev)
    y = et.layer_norm(torch.full((3, 100), 2.0, device=dev), w, b)
    assert torch.equal(y, b.expand(3, 100))


def test_non_finite_rows_stay_alone(et, dev):
    x = torch.randn(9, 300, device=dev)
    w = torch.ones(300, device=dev)
    clean, mean, rstd = et.layer_norm(x, w, stats=True)
    for bad in (float("nan"), float("inf")):
        z = x.clone()
        z[4, 299] = bad
        y = et.layer_norm(z, w)
        assert torch.isnan(y[4]).all()
        keep = torch.arange(9, device=dev) != 4
        assert torch.equal(y[keep], clean[keep])
        dy = torch.randn(9, 300, device=dev)
        good = et.layer_norm_backward(dy, x, w, mean, rstd)[0]
        dy[4, 0] = bad
        dx = et.layer_norm_backward(dy, x, w, mean, rstd)[0]
        assert torch.equal(dx[keep], good[keep]) and not torch.isfinite(dx[4]).any()


def test_large_offsets_keep_the_variance(et, dev):
    """Rows around 1000 with a deviation of 1: the variance is that of the
    centred values, not a difference of large sums."""
    x = torch.randn(50, 4096, device=dev) + 1000.0
    y = et.layer_norm(x, torch.ones(4096, device=dev), eps=0.0)
    m, r, want, em, er, ey = _forward64(x, torch.ones(4096, device=dev), None, 0.0)
    assert torch.all((y.double() - want).abs() <= ey + U * want.abs())


def test_in_place_outputs_streams_and_graphs(et, dev):
    x, r = (torch.randn(130, 1000, device=dev, dtype=BF16) for _ in range(2))
    w = torch.randn(1000, device=dev)
    y, s = et.layer_norm(x, w, residual=r)
    z = x.clone()
    q = r.clone()
    got = et.layer_norm(z, w, residual=q, out=z, out_sum=q)
    assert torch.equal(z, y) and torch.equal(q, s) and got[0] is z
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2, s2 = et.layer_norm(x, w, residual=r)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y2, y) and torch.equal(s2, s)
    dy = torch.randn_like(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        yg, sg, mean, rstd = et.layer_norm(x, w, residual=r, stats=True)
        dg = et.layer_norm_backward(dy, sg, w, mean, rstd, dsum=dy)
    for i in range(4):
        x.mul_(1.1)
        graph.replay()
        torch.cuda.synchronize()
        ye, se, me, re = et.layer_norm(x, w, residual=r, stats=True)
        de = et.layer_norm_backward(dy, se, w, me, re, dsum=dy)
        torch.cuda.synchronize()
        assert torch.equal(yg, ye) and torch.equal(sg, se) and all(torch.equal(a, b) for a, b in zip(dg, de))


def test_neighbours_of_the_outputs_stay(et, dev):
    for d in (1, 7, 100, 513):
        buf = torch.full((6, d), 5.0, device=dev, dtype=BF16)
        et.layer_norm(torch.randn(4, d, device=dev, dtype=BF16), torch.ones(d, device=dev), out=buf[1:5])
        assert torch.all(buf[0] == 5.0) and torch.all(buf[5] == 5.0)
        wide = torch.full((3 * d,), 5.0, device=dev)
        x = torch.randn(40, d, device=dev)
        _, mean, rstd = et.layer_norm(x, torch.ones(d, device=dev), stats=True)
        et.layer_norm_backward(x, x, torch.ones(d, device=dev), mean, rstd, out_dweight=wide[d:2 * d])
        assert torch.all(wide[:d] == 5.0) and torch.all(wide[2 * d:] == 5.0)


def test_refusals(et, dev):
    x = torch.zeros(4, 16, device=dev)
    w = torch.ones(16, device=dev)
    with pytest.raises(ValueError, match="HIP device"):
        et.layer_norm(x.cpu(), w)
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        et.layer_norm(x.half(), w)
    with pytest.raises(ValueError, match="2-D"):
        et.layer_norm(x[0], w)
    with pytest.raises(ValueError, match="contiguous"):
        et.layer_norm(x.t().contiguous().t(), w)
    with pytest.raises(ValueError, match="overlap"):
        et.layer_norm(x[:1].expand(4, 16), w)
    with pytest.raises(TypeError, match="weight"):
        et.layer_norm(x, w.bfloat16())
    with pytest.raises(TypeError, match="same dtype"):
        et.layer_norm(x.bfloat16(), w, w.bfloat16())
    with pytest.raises(ValueError, match="entries"):
        et.layer_norm(x, w[:8])
    with pytest.raises(ValueError, match="eps"):
        et.layer_norm(x, w, eps=-1.0)
    with pytest.raises(TypeError, match="residual"):
        et.layer_norm(x, w, residual=x.bfloat16())
    with pytest.raises(ValueError, match="residual"):
        et.layer_norm(x, w, residual=x[:2])
    with pytest.raises(ValueError, match="residual"):
        et.layer_norm(x, w, out_sum=x)
    with pytest.raises(ValueError, match="16384"):
        et.layer_norm(torch.zeros(1, 16385, device=dev), torch.ones(16385, device=dev))
    m = torch.zeros(4, device=dev)
    with pytest.raises(ValueError, match="mean"):
        et.layer_norm_backward(x, x, w, m[:3], m)
    with pytest.raises(ValueError, match="dy"):
        et.layer_norm_backward(x[:, :8], x, w, m, m)
    with pytest.raises(ValueError, match="workspace"):
        et.layer_norm_backward(x, x, w, m, m, workspace=torch.zeros(8, dtype=torch.uint8, device=dev))


def test_a_second_derivative_is_an_error(et, dev):
    """Not a gradient that lacks the terms through this one."""
    def refuses(f, x):
        grad, = torch.autograd.grad(f(x).float().square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            (grad.square().sum() + x.float().square().sum()).backward()

    w = torch.ones(40, device=dev, requires_grad=True)
    rows = lambda: torch.randn(5, 40, device=dev, requires_grad=True)  # noqa: E731
    r = rows()
    refuses(lambda x: et.layer_norm_autograd(x, w), rows())
    refuses(lambda x: et.layer_norm_autograd(x, w, residual=r)[0], rows())
    refuses(lambda x: torch.ops.etmoe.layer_norm(x, w, None, 1e-5)[0], rows())
    refuses(lambda x: torch.ops.etmoe.add_layer_norm(x, r, w, None, 1e-5)[0], rows())
    plan = et.route(torch.randn(5, 4, device=dev), torch.full((4,), 0.5, device=dev))
    refuses(lambda x: et.dispatch_autograd(x, plan), rows())
    yp = torch.randn(plan.rows, 40, device=dev, requires_grad=True)
    refuses(lambda x: et.combine_autograd(x, torch.zeros(5, 4, device=dev), plan), yp)


def test_statistics_carry_no_gradient(et, dev):
    x, r = (torch.randn(5, 40, device=dev, requires_grad=True) for _ in range(2))
    w = torch.ones(40, device=dev, requires_grad=True)
    y, mean, rstd = torch.ops.etmoe.layer_norm(x, w, None, 1e-5)
    assert y.requires_grad and not mean.requires_grad and not rstd.requires_grad
    y, s, mean, rstd = torch.ops.etmoe.add_layer_norm(x, r, w, None, 1e-5)
    assert y.requires_grad and s.requires_grad and not mean.requires_grad and not rstd.requires_grad


def test_add_layer_norm_operator(et, dev):
    """torch.ops.etmoe.add_layer_norm under torch.compile, both outputs used."""
    x, r = (torch.randn(33, 96, device=dev, requires_grad=True) for _ in range(2))
    w, b = (torch.randn(96, device=dev, requires_grad=True) for _ in range(2))

    def f(x, r, w, b):
        y, s, _, _ = torch.ops.etmoe.add_layer_norm(x, r, w, b, 1e-5)
        return (y ** 2).sum() + (s ** 3).sum()

    torch.compile(f, fullgraph=True, backend="aot_eager")(x, r, w, b).backward()
    got = x.grad, r.grad, w.grad, b.grad
    leaves = [t.detach().clone().requires_grad_(True) for t in (x, r, w, b)]
    y, s = et.layer_norm_autograd(leaves[0], leaves[2], leaves[3], residual=leaves[1])
    ((y ** 2).sum() + (s ** 3).sum()).backward()
    assert all(torch.equal(p, q.grad) for p, q in zip(got, leaves))
    # one output alone
    for pick in (0, 1):
        for t in (x, r):
            t.grad = None
        torch.ops.etmoe.add_layer_norm(x, r, w, None, 1e-5)[pick].sum().backward()
        assert torch.equal(x.grad, r.grad) and (pick == 0 or torch.all(x.grad == 1))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_opcheck(et, dev, dtype):
    x, r = (torch.randn(9, 40, device=dev).to(dtype).requires_grad_(True) for _ in range(2))
    w, b = (torch.randn(40, device=dev, requires_grad=True) for _ in range(2))
    tests = ("test_schema", "test_faketensor", "test_autograd_registration")
    ops = torch.ops.etmoe
    for bias in (b, None):
        torch.library.opcheck(ops.layer_norm.default, (x, w, bias, 1e-5), test_utils=tests)
        torch.library.opcheck(ops.add_layer_norm.default, (x, r, w, bias, 1e-5), test_utils=tests)
    _, mean, rstd = ops.layer_norm(x.detach(), w.detach(), None, 1e-5)
    for ds in (None, r.detach()):
        torch.library.opcheck(ops.layer_norm_backward.default, (r.detach(), x.detach(), w.detach(), mean, rstd, ds),
                              test_utils=("test_schema", "test_faketensor"))


def test_workspaces_that_only_look_large_are_refused(et, dev):
    """A workspace of enough elements on one element of memory."""
    x, w, m = torch.ones(400, 64, device=dev), torch.ones(64, device=dev), torch.ones(400, device=dev)
    small = torch.zeros(4, device=dev)
    for bad in (small[:1].expand(1 << 20), small[:1].expand(1 << 10, 1 << 10), torch.zeros(1 << 17, device=dev)[::2]):
        with pytest.raises(ValueError, match="workspace"):
            et.layer_norm_backward(x, x, w, m, m, workspace=bad)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("d", [3, 9, 100, 1000, 1500, 2889, 6000, 9000])
def test_backward_of_rows_far_from_zero(et, dev, dtype, d):
    """Constant rows of 2^112: mean * rstd passes binary32's range, but x - mean is
    0 in every column, so dx = rstd (g - mean(g)) + dsum is not large."""
    g = torch.Generator().manual_seed(d)
    x = torch.full((6, d), 2.0 ** 112, device=dev, dtype=dtype)
    w = (1 + torch.randn(d, generator=g) * 0.3).to(dev)
    mean, rstd = torch.full((6,), 2.0 ** 112, device=dev), torch.full((6,), 2.0 ** 20, device=dev)
    dy, ds = (torch.randn(6, d, generator=g).to(dev).to(dtype) for _ in range(2))
    got = et.layer_norm_backward(dy, x, w, mean, rstd, dsum=ds)
    dx, dw, db, ex, ew, eb = _backward64(dy, x, w, mean, rstd, ds)
    assert torch.all((got[0].double() - dx).abs() <= ex + HALF[dtype] * (dx.abs() + ex))
    assert torch.all(got[1] == 0) and torch.all((got[2].double() - db).abs() <= eb)


@pytest.mark.parametrize("dtype,d", [(F32, 3), (BF16, 64), (F32, 520), (BF16, 520), (F32, 8200), (BF16, 8200)])
def test_column_sums_over_many_rows(et, dev, dtype, d):
    """The error of dweight and dbias does not grow with the rows.  A sum of n
    terms of deviation 1 and random signs in chains of lengths l_1, l_2, ... (a chain's
    results are the next one's terms) is off by about 0.3 U sqrt(l_1 + l_2 + ...) times
    its size, sqrt(n): an addition errs by 0.4 U (deviation) of a partial sum that
    grows as the root.  Chains of 32 and T / 256 / 32 rows, 20 for the blocks, and one U of the
    terms' own roundings: below 4 U up to 2^18 rows, where a single
    chain of T / 256 gives 9 U."""
    T = (1 << 18) if d < 4096 else (1 << 16)
    g = torch.Generator(device=dev).manual_seed(d)
    x, dy = torch.empty(T, d, dtype=dtype, device=dev), torch.empty(T, d, dtype=dtype, device=dev)
    step = 1 << 13
    for i in range(0, T, step):
        x[i:i + step] = torch.randn(step, d, generator=g, device=dev)
        dy[i:i + step] = torch.randn(step, d, generator=g, device=dev)
    w = torch.ones(d, device=dev)
    mean, rstd = torch.zeros(T, device=dev), torch.ones(T, device=dev)     # (xhat = x, exactly)
    _, dw, db = et.layer_norm_backward(dy, x, w, mean, rstd)
    rw, rb = (torch.zeros(d, dtype=torch.float64, device=dev) for _ in range(2))
    for i in range(0, T, step):
        a = dy[i:i + step].double()
        rw += (a * x[i:i + step].double()).sum(0)
        rb += a.sum(0)
    for got, want in ((dw, rw), (db, rb)):
        assert (got.double() - want).norm() <= 4 * U * (T * d) ** 0.5
