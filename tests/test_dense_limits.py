"""What the dense operators refuse at the far ends of their ranges, and the sizes they
report, through the C ABI and the Python checks; no GPU."""
import ctypes
import importlib

import pytest

ET_ERR_INVALID_ARGUMENT = -1


def _err(et):
    return et.lib().et_last_error().decode()


def _shapes(*s):
    return (ctypes.c_int64 * (3 * len(s)))(*[v for t in s for v in t])


def _polynomial(et, abc, iterations):
    """Status of a call that has nothing to do: what it says of its coefficients."""
    return et.lib().et_orthogonalize((ctypes.c_void_p * 1)(), (ctypes.c_void_p * 1)(), _shapes((0, 8, 8)), 1, 0, iterations,
                                     (ctypes.c_float * 3)(*abc), 1e-7, None, 0, None)


@pytest.mark.parametrize("abc,steps", [((1.07, 0.0, 0.0), 20), ((1.05, -0.01, 0.0), 64), ((1.02, 0.0, 0.0), 40)])
def test_polynomials_that_leave_the_range_late_are_refused(et, abc, steps):
    """A singular value of 1 grows by a few percent a step and passes 1.9 behind the eighth."""
    muon = importlib.import_module("peer-review-agents_amd.muon")
    s, a = 1.0, abc
    for _ in range(steps):
        s *= a[0] + a[1] * s * s + a[2] * s ** 4
    assert s > 1.9
    with pytest.raises(ValueError, match="singular"):
        muon._coefficients(abc, steps, 1e-7)
    assert _polynomial(et, abc, steps) == ET_ERR_INVALID_ARGUMENT and "singular" in _err(et)


@pytest.mark.parametrize("abc,steps", [((1.5, -0.5, 0.0), 64), ((3.4445, -4.7750, 2.0315), 64), ((1.875, -1.25, 0.375), 64),
                                       ((1.07, 0.0, 0.0), 6), ((1.0, 0.0, 0.0), 1)])
def test_polynomials_that_stay_are_taken(et, abc, steps):
    muon = importlib.import_module("peer-review-agents_amd.muon")
    assert muon._coefficients(abc, steps, 1e-7) == abc
    assert _polynomial(et, abc, steps) == 0


def test_launches_stay_below_2_32_threads(et):
    """A matrix that goes one block has 512 threads; an item of the adapters' first kernel two blocks of up to 512."""
    lib, P = et.lib(), ctypes.c_void_p(0x1000)
    one, abc, step = (ctypes.c_void_p * 1)(0x1000), (ctypes.c_float * 3)(3.4445, -4.775, 2.0315), (ctypes.c_float * 1)(0.1)
    scalars = importlib.import_module("peer-review-agents_amd._lib").MuonScalars(0.95, 0.05, 1.0, 1e-7, 3.4445, -4.775, 2.0315, 5, 1)
    for E, m, n in ((1 << 23, 2, 2), (1 << 23, 1, 1), ((1 << 24) - 1, 8, 8)):
        shape = _shapes((E, m, n))
        assert lib.et_orthogonalize(one, one, shape, 1, 0, 5, abc, 1e-7, P, 1 << 40, None) == ET_ERR_INVALID_ARGUMENT
        assert "2^23" in _err(et)
        assert lib.et_muon(one, one, one, None, step, shape, 1, 0, 0, scalars, None, P, 1 << 40, None) == ET_ERR_INVALID_ARGUMENT
        assert lib.et_orthogonalize_workspace_bytes(shape, 1) == 0
    for T, rank in ((1 << 28, 8), ((1 << 28) + 64, 32), ((1 << 29) - 64, 8)):
        rc = lib.et_adapter_add(P, 8, P, 8, P, P, P, P, P, P, T, 4, 8, 8, rank, P, 8, P, 1 << 62, None)
        assert rc == ET_ERR_INVALID_ARGUMENT and "too large" in _err(et), T


def test_workspace_sizes_of_sizes_that_are_refused(et):
    """0, as the header says, for whatever the call itself refuses."""
    lib = et.lib()
    gated, adapters = lib.et_gated_linear_bwd_workspace_bytes, lib.et_adapter_add_workspace_bytes
    assert gated(100, 64, 16) > 0 and adapters(100, 4, 64, 16) > 0
    for T, K, F in ((-1, 64, 16), (1 << 31, 64, 16), (1 << 62, 64, 16), (100, 60, 16), (100, 0, 16), (100, 1 << 21, 8), (100, 64, 12),
                    (100, 64, 0), (100, 8, 1 << 20), (100, 1 << 20, 1 << 10), (100, 1 << 62, 16), (100, 64, 1 << 62)):
        assert gated(T, K, F) == 0, (T, K, F)
    for T, n, K, r in ((-1, 4, 64, 16), (1 << 30, 4, 64, 16), (8, 0, 64, 16), (8, 4097, 64, 16), (8, 4, 60, 16), (8, 4, 0, 16),
                       (8, 4, 1 << 22, 16), (8, 4, 64, 12), (8, 4, 64, 0), (8, 4, 64, 136), (1 << 28, 4, 64, 16)):
        assert adapters(T, n, K, r) == 0, (T, n, K, r)


def test_the_backwards_workspace_goes_by_the_tensors_device(et, monkeypatch):
    """Its splits go by a device's CUs: those of the device that the call runs on, not of the current one."""
    gated = importlib.import_module("peer-review-agents_amd.gated")
    current = [0]

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            current.append(self.index)

        def __exit__(self, *_):
            current.pop()

    class Library:
        @staticmethod
        def et_gated_linear_bwd_workspace_bytes(rows, K, F):
            return 1000 * rows + current[-1]

    monkeypatch.setattr(gated.torch.cuda, "device", Device)
    monkeypatch.setattr(gated, "lib", lambda: Library)
    try:
        assert gated.gated_linear_backward_workspace_bytes(5, 64, 16) == 5000
        assert gated.gated_linear_backward_workspace_bytes(5, 64, 16, device=3) == 5003
        assert gated.gated_linear_backward_workspace_bytes(5, 64, 16, device=gated.torch.device("cuda:2")) == 5002
    finally:
        gated._workspace_bytes.cache_clear()


def test_sets_of_tensors_share_the_workspace(et):
    """At most 20 tensors run at a time, wide ones and tall ones apart: a step needs what the largest of these needs."""
    size = lambda *s: et.lib().et_orthogonalize_workspace_bytes(_shapes(*s), len(s))  # noqa: E731
    one, tall = size((4, 200, 520)), size((2, 900, 136))
    assert 4 * 4 * 200 * 520 < one < 4 * 4 * (200 * 520 + 200 * 200) * 1.1 and tall > 0
    assert size(*[(4, 200, 520)] * 20) == 20 * one
    assert size(*[(4, 200, 520)] * 100) == 20 * one
    assert size(*[(4, 200, 520), (2, 900, 136)] * 5) == max(5 * one, 5 * tall)
    assert size((4, 200, 520), *[(8, 64, 512)] * 50) == one and size(*[(8, 64, 512)] * 50) == 0
    assert size((0, 200, 520), (3, 0, 200)) == 0
    # whatever the order, and enough for a part of the list (the tensors of one pair of types)
    mixed = [(4, 200, 520), (1, 100, 100)] * 20
    assert size(*mixed) == size(*mixed[::2]) == 20 * one == size(*mixed[::-1])
    assert size(*mixed[:10]) < size(*mixed[:30]) < size(*mixed)
