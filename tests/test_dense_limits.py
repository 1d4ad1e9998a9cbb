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
