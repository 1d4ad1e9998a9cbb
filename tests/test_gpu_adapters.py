"""Low-rank adapters on the GPU against the formula in float64.

Bound, element by element: the inner sum of K terms is off by at most
K 2^-24 sum|a x|, times the scale one rounding more; it enters the second
product as two bf16 numbers, off by at most 2^-16 of its value (a half step of
2^-8 twice; 2^-15 with the second's own half step); that product has 2 rank
terms in binary32, and the sum with y is rounded to bf16 once (half a step, 2^-8)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

EPS, HALF = 2.0 ** -24, 2.0 ** -8


def _bank(et, dev, n, rank, K, N, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed * 71 + n + rank + K + N)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    return et.AdapterBank((r(n, rank, K) * K ** -0.5).bfloat16(), r(n, N, rank).bfloat16(), torch.exp(r(n)))


def _batch(dev, T, K, N, n, seed=0, none=0.25):
    g = torch.Generator(device=dev).manual_seed(seed * 113 + T + K + N)
    x = torch.randn(T, K, generator=g, device=dev).bfloat16()
    y = torch.randn(T, N, generator=g, device=dev).bfloat16()
    index = torch.randint(0, n, (T,), generator=g, device=dev, dtype=torch.int32)
    index[torch.rand(T, generator=g, device=dev) < none] = -1
    return x, y, index


def _want(y, x, bank, index):
    value, bound = y.double(), torch.zeros(y.shape, device=y.device, dtype=torch.float64)
    x, K, rank = x.double(), x.shape[1], bank.a.shape[1]
    for i in range(bank.num_adapters):
        at = (index == i).nonzero()[:, 0]
        if not len(at):
            continue
        a, b, s = bank.a[i].double(), bank.b[i].double(), bank.scale[i].double()
        v = s * (x[at] @ a.t())
        e = s * (K * EPS * (x[at].abs() @ a.abs().t())) + (2 * EPS + 2.0 ** -15) * v.abs()
        value[at] += v @ b.t()
        bound[at] = 1.01 * (e @ b.abs().t() + 2 * rank * EPS * (v.abs() @ b.abs().t()) + EPS * value[at].abs())
    return value, bound + HALF * (value.abs() + bound)


def _check(got, y, x, bank, index):
    value, bound = _want(y, x, bank, index)
    off = (got.double() - value).abs()
    assert bool((off <= bound + 1e-30).all()), (off / (bound + 1e-30)).max().item()
    none = (index < 0) | (index >= bank.num_adapters)
    assert torch.equal(got[none], y[none])


@pytest.mark.parametrize("T,K,N,rank,n", [
    (1, 8, 8, 8, 1), (1, 512, 72, 16, 3), (2, 64, 64, 8, 5), (15, 264, 200, 16, 4), (16, 1032, 256, 16, 1), (17, 2056, 264, 24, 2),
    (48, 512, 520, 16, 64), (61, 136, 1000, 32, 7), (300, 200, 136, 40, 9), (1000, 256, 312, 64, 33), (2048, 72, 64, 16, 5),
    (2049, 136, 72, 8, 2), (5000, 264, 328, 32, 24), (3001, 72, 200, 128, 3), (4100, 64, 136, 72, 600), (40, 520, 264, 128, 4096)])
def test_adapter_add(et, dev, T, K, N, rank, n):
    print(f"adapters T={T} K={K} N={N} rank={rank} n={n}", flush=True)
    bank = _bank(et, dev, n, rank, K, N)
    x, y, index = _batch(dev, T, K, N, n)
    plan = et.adapter_plan(index, n)
    # the plan: every token once, items of one adapter
    count = int(plan.num_items)
    assert count <= plan.items.shape[0]
    order, items = plan.order.long(), plan.items[:count].tolist()
    assert torch.equal(order.sort().values, torch.arange(T, device=dev))
    assert sum(rows for _, _, rows, _ in items) == T and sorted(first for _, first, _, _ in items)[0] == 0
    sorted_index = index[order].tolist()
    for adapter, first, rows, _ in items:
        assert 1 <= rows <= 64 and set(sorted_index[first:first + rows]) == {adapter}
    before = y.clone()
    got = et.adapter_add(y, x, bank, plan)
    assert torch.equal(y, before)
    _check(got, y, x, bank, index)
    # in place, and again: the same bits
    again = y.clone()
    assert et.adapter_add(again, x, bank, plan, out=again) is again
    assert torch.equal(again, got)
    assert torch.equal(et.adapter_add(y, x, bank, et.adapter_plan(index, n)), got)


def test_runs_one_adapter_and_none(et, dev):
    T, K, N, n = 700, 136, 200, 12
    bank = _bank(et, dev, n, 16, K, N)
    x, y, index = _batch(dev, T, K, N, n)
    for index in (index.sort().values.contiguous(), torch.full_like(index, 11), torch.full_like(index, -1),
                  torch.full_like(index, n), torch.full_like(index, -2 ** 31), torch.full_like(index, 2 ** 31 - 1)):
        _check(et.adapter_add(y, x, bank, et.adapter_plan(index, n)), y, x, bank, index)
    empty = et.adapter_plan(index[:0], n)
    assert int(empty.num_items) == 0
    assert et.adapter_add(y[:0], x[:0], bank, empty).shape == (0, N)


def test_slices_of_wider_rows(et, dev):
    """x, y and out as columns of wider buffers (a fused projection's output), rows and columns
    beside them left as they were; rows whose offsets pass 32 bits."""
    T, K, N, n = 100, 72, 136, 6
    bank = _bank(et, dev, n, 24, K, N)
    x, y, index = _batch(dev, T, K, N, n)
    plan = et.adapter_plan(index, n)
    want = et.adapter_add(y, x, bank, plan)
    xs = torch.full((T, K + 16), float("nan"), device=dev, dtype=torch.bfloat16)
    ys = torch.full((T + 2, 3 * N), 3.0, device=dev, dtype=torch.bfloat16)
    xs[:, 8:8 + K], ys[:T, N:2 * N] = x, y
    part = ys[:T, N:2 * N]
    et.adapter_add(part, xs[:, 8:8 + K], bank, plan, out=part)
    assert torch.equal(part, want)
    assert bool((ys[:T, :N] == 3).all()) and bool((ys[:, 2 * N:] == 3).all()) and bool((ys[T:] == 3).all())
    far = torch.zeros(T, (1 << 25) + 8, device=dev, dtype=torch.bfloat16)
    assert (T - 1) * far.stride(0) * 2 > 2 ** 32
    far[:, :K] = x
    far[:, K:K + N] = y
    assert torch.equal(et.adapter_add(far[:, K:K + N], far[:, :K], bank, plan), want)
    et.adapter_add(far[:, K:K + N], far[:, :K], bank, plan, out=far[:, K:K + N])
    assert torch.equal(far[:, K:K + N], want)


@pytest.mark.parametrize("T", [40, 2100])
def test_a_bank_beyond_32_bits(et, dev, T):
    """The last of 4096 adapters lies more than 4 GiB into a and b."""
    n, rank, K, N = 4096, 128, 4120, 4128
    few = _bank(et, dev, 2, rank, K, N)
    a = torch.zeros(n, rank, K, device=dev, dtype=torch.bfloat16)
    b = torch.zeros(n, N, rank, device=dev, dtype=torch.bfloat16)
    assert (n - 1) * rank * K * 2 > 2 ** 32
    scale = torch.zeros(n, device=dev)
    for at, i in ((0, 0), (n - 1, 1)):
        a[at], b[at], scale[at] = few.a[i], few.b[i], few.scale[i]
    bank = et.AdapterBank(a, b, scale)
    x, y, index = _batch(dev, T, K, N, 2)
    got = et.adapter_add(y, x, bank, et.adapter_plan(torch.where(index == 1, n - 1, index), n))
    _check(got, y, x, few, index)


def test_a_bad_token_stays_a_token(et, dev):
    T, K, N, n = 60, 72, 64, 3
    bank = _bank(et, dev, n, 16, K, N)
    x, y, index = _batch(dev, T, K, N, n, none=0.1)
    index[10] = 1
    plan = et.adapter_plan(index, n)
    want = et.adapter_add(y, x, bank, plan)
    others = torch.arange(T, device=dev) != 10
    for bad in (float("nan"), float("inf")):
        x2 = x.clone()
        x2[10, 3] = bad
        got = et.adapter_add(y, x2, bank, plan)
        assert torch.equal(got[others], want[others]) and bool(torch.isnan(got[10]).all())
    # an adapter that holds NaN, of another token
    bank.a[2] = float("nan")
    got = et.adapter_add(y, x, bank, plan)
    fine = index != 2
    assert torch.equal(got[fine], want[fine])


def test_beside_a_shared_4_bit_projection(et, dev):
    """As a server runs it: the shared projection from 4-bit weights, one plan for two projections,
    captured, replayed for other batches."""
    T, K, N, n = 40, 256, 192, 9
    g = torch.Generator(device=dev).manual_seed(2)
    w = [et.pack_w4(*et.quantize_w4(torch.randn(N, k, generator=g, device=dev) * 0.05, group=64), group=64) for k in (K, N)]
    banks = [_bank(et, dev, n, 16, K, N), _bank(et, dev, n, 8, N, N, seed=1)]
    x, _, index = _batch(dev, T, K, N, n)

    def run(plan=None):
        plan = et.adapter_plan(index, n)
        h = et.linear_w4(x, w[0])
        h = et.adapter_add(h, x, banks[0], plan, out=h)
        z = et.linear_w4(h, w[1])
        return h, et.adapter_add(z, h, banks[1], plan), z

    h, out, z = run()
    _check(h, et.linear_w4(x, w[0]), x, banks[0], index)
    _check(out, z, h, banks[1], index)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gh, gout, _ = run()
    for rep in range(3):
        x2, _, i2 = _batch(dev, T, K, N, n, seed=rep + 3)
        x.copy_(x2), index.copy_(i2)
        graph.replay()
        torch.cuda.synchronize()
        h, out, _ = run()
        assert torch.equal(gh, h) and torch.equal(gout, out), rep
    del graph
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other[1], out)


def test_a_plan_of_other_tensors(et, dev):
    """What a plan is made of is checked where it is made, and neither it nor a bank can be changed after that."""
    index = torch.zeros(5, dtype=torch.int32, device=dev)
    plan = et.adapter_plan(index, 3)
    good = dict(order=plan.order, items=plan.items, num_items=plan.num_items, num_tokens=5, num_adapters=3)
    et.AdapterPlan(**good)
    for bad in (dict(order=plan.order[:4]), dict(items=plan.items[:1]), dict(items=plan.items.view(-1, 2)), dict(num_tokens=500),
                dict(items=torch.zeros(9, 5, dtype=torch.int32, device=dev)), dict(num_adapters=4000, num_tokens=6),
                dict(num_items=plan.order), dict(num_items=plan.num_items.cpu())):
        with pytest.raises(ValueError):
            et.AdapterPlan(**{**good, **bad})
    with pytest.raises(TypeError):
        et.AdapterPlan(**{**good, "order": plan.order.long()})
    bank = _bank(et, dev, 3, 16, 64, 72)
    for thing, name in ((plan, "order"), (bank, "a")):
        with pytest.raises(AttributeError):
            setattr(thing, name, getattr(thing, name)[:1])


def test_refusals(et, dev):
    bank = _bank(et, dev, 3, 16, 64, 72)
    x, y, index = _batch(dev, 5, 64, 72, 3)
    plan = et.adapter_plan(index, 3)
    a, b, s = bank.a, bank.b, bank.scale
    for bad in (dict(a=a.float()), dict(b=b.half()), dict(scale=s.double())):
        with pytest.raises(TypeError):
            et.AdapterBank(**{**dict(a=a, b=b, scale=s), **bad})
    for bad in (dict(a=a[:2].contiguous()), dict(b=b[:, :, :8].contiguous()), dict(scale=s[:2]), dict(a=a[:, :, :60].contiguous()),
                dict(a=a[:, :12].contiguous(), b=b[:, :, :12].contiguous()), dict(b=b[:, :70].contiguous()), dict(a=a.cpu()),
                dict(a=a[:0], b=b[:0], scale=s[:0]), dict(a=a.transpose(1, 2))):
        with pytest.raises(ValueError):
            et.AdapterBank(**{**dict(a=a, b=b, scale=s), **bad})
    with pytest.raises(TypeError):
        et.adapter_plan(index.long(), 3)
    for i, n in ((index, 0), (index, 4097), (index.cpu(), 3), (index[::2], 3)):
        with pytest.raises(ValueError):
            et.adapter_plan(i, n)
    call = dict(y=y, x=x, bank=bank, plan=plan)
    for bad in (dict(bank=(a, b, s)), dict(plan=index), dict(x=x.float())):
        with pytest.raises(TypeError):
            et.adapter_add(**{**call, **bad})
    wide = torch.empty(5, 76, device=dev, dtype=torch.bfloat16)
    for bad in (dict(y=y[:4]), dict(x=x[:, :56].contiguous()), dict(plan=et.adapter_plan(index, 4)), dict(y=wide[:, :72]),
                dict(out=y[:4]), dict(workspace=torch.empty(8, device=dev, dtype=torch.uint8)), dict(x=x.cpu())):
        with pytest.raises(ValueError):
            et.adapter_add(**{**call, **bad})
