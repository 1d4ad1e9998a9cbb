"""The dense operators on two streams at once, and as two captured graphs replayed in
turn: every result has the bits of the call alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _work(et, dev, seed):
    """A list of calls, each of fixed inputs, that return tensors."""
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=dev).bfloat16()  # noqa: E731
    x, w, dh, few = r(700, 136), r(2 * 72, 136), r(700, 72), r(5, 136)
    small, wide, tall = r(3, 40, 200), r(2, 200, 264), r(1, 600, 130)
    bank = et.AdapterBank(r(4, 16, 136), r(4, 72, 16), torch.rand(4, generator=g, device=dev))
    index = torch.randint(-1, 4, (700,), generator=g, device=dev, dtype=torch.int32)

    def adapters():
        return [et.adapter_add(dh, x, bank, et.adapter_plan(index, 4))]

    return [lambda: [et.gated_linear(x, w)], lambda: [et.gated_linear(few, w)], lambda: list(et.gated_linear_backward(dh, x, w)),
            lambda: [et.orthogonalize(small)], lambda: [et.orthogonalize(wide)], lambda: [et.orthogonalize(tall)], adapters]


def test_two_streams(et, dev):
    works = [_work(et, dev, s) for s in (1, 2)]
    want = [[t.clone() for f in w for t in f()] for w in works]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for fs in zip(*works):
            for k in (0, 1):
                with torch.cuda.stream(streams[k]):
                    got[k].append(fs[k]())
    torch.cuda.synchronize()
    for k in (0, 1):
        flat = [t for call in got[k] for t in call]
        assert len(flat) == 4 * len(want[k])
        for i, t in enumerate(flat):
            assert torch.equal(t, want[k][i % len(want[k])]), (k, i)


def test_two_graphs(et, dev):
    works = [_work(et, dev, s) for s in (3, 4)]
    want = [[t.clone() for f in w for t in f()] for w in works]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for w in works:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([t for f in w for t in f()])
        graphs.append(graph)
    for rep in range(3):
        for k in (rep & 1, 1 - (rep & 1)):
            for t in outs[k]:
                t.zero_()
            graphs[k].replay()
            eager = [t for f in works[1 - k] for t in f()]
            torch.cuda.synchronize()
            for a, b in zip(outs[k] + eager, want[k] + want[1 - k]):
                assert torch.equal(a, b), (rep, k)
