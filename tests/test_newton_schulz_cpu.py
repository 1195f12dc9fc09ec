"""Which coefficients of Newton-Schulz steps are accepted: those that keep singular values at 8 or below, wherever they were on the way."""
import ctypes

import numpy as np
import pytest

import difflogic_b200 as D
from difflogic_b200 import _native as N


def largest(coefficients, points=200001):
    """Over a grid that is laid anew over what the step before has reached."""
    reach = 1.0
    for a, b, c in coefficients:
        s = np.linspace(0, reach, points)
        reach = np.abs(s * (a + s * s * (b + s * s * c))).max()
    return reach


@pytest.mark.parametrize("seed", range(40))
def test_the_largest_value_is_found(seed):
    rng = np.random.default_rng(seed)
    sets = [tuple(rng.uniform(-1, 1, 3) * 10.0 ** rng.uniform(-1, 1.5)) for _ in range(3)]
    if seed % 4 == 0:
        sets = [(a, b, 0.0) for a, b, c in sets]
    reach = 1.0
    for s in sets:
        reach = min(D.ops._largest_value(*s, reach), 50.0)
    got, grid = 1.0, 1.0
    for s in sets:
        got = D.ops._largest_value(*s, got)
        grid = largest([s], 20001) if grid == 1.0 else np.abs(np.polyval([s[2], 0, s[1], 0, s[0], 0], np.linspace(0, grid, 20001))).max()
        assert abs(got - grid) <= 1e-5 * grid + 1e-12
        got = grid = min(got, 50.0)


@pytest.mark.parametrize("coefficients, fits", [(((20.0, -60.0, 48.0),), True), (((8.0, 0.0, 0.0),), True), (((8.1, 0.0, 0.0),), False),
                                                (((8.0, 0.0, 0.0), (1.0, 0.0, 0.0)), True), (((8.0, 0.0, 0.0), (1.01, 0.0, 0.0)), False),
                                                (((64.0, -64.0, 0.0),), False), (((24.0, -60.0, 44.0),), True), (((-8.0, 0.0, 0.0),), True),
                                                # between the images of a grid over [0, 1] the second step's peak would be missed
                                                (((8.0, 0.0, 0.0), (0.0, 0.0, -0.001)), False)])
def test_coefficients_at_the_edge(coefficients, fits):
    assert (largest(coefficients) <= 8.0 + 1e-6) == fits
    steps, lib = len(coefficients), N.lib()
    table = (ctypes.c_float * (3 * steps))(*[v for s in coefficients for v in s])
    status = lib.dl_orthogonalize(None, None, 0, 4, 4, 0, steps, table, 1e-7, None, None)
    assert lib.dl_muon_step_f32(None, 0, 0.1, 0.9, 1, 0.0, steps, table, 1e-7, None, None) == status
    if fits:
        assert status == N.DL_OK and list(D.ops._newton_schulz(coefficients, steps)) == list(table)
    else:
        assert status == N.DL_ERR_INVALID_ARG and "singular values" in N.last_error()
        with pytest.raises(ValueError, match="near 1"):
            D.ops._newton_schulz(coefficients, steps)


def test_the_library_refuses_what_is_not_a_number():
    for bad in ((float("nan"), 0.0, 0.0), (1.0, float("inf"), 0.0), (1.0, 0.0, -65.0)):
        table = (ctypes.c_float * 3)(*bad)
        assert N.lib().dl_orthogonalize(None, None, 0, 4, 4, 0, 1, table, 1e-7, None, None) == N.DL_ERR_INVALID_ARG
        with pytest.raises(ValueError, match="near 1"):
            D.ops._newton_schulz(bad, 1)


def test_what_was_refused_once_is_refused_after_a_call_that_equals_it():
    """1, 1.0 and True are one key of a table that does not look at types."""
    for steps in (1, 2):
        table = D.ops._newton_schulz((1.5, -0.5, 0.0), steps)
        assert D.ops._newton_schulz((1.5, -0.5, 0.0), steps) is table
        for wrong in (float(steps), True) if steps == 1 else (float(steps),):
            with pytest.raises(ValueError, match="whole number"):
                D.ops._newton_schulz((1.5, -0.5, 0.0), wrong)


@pytest.mark.parametrize("c", [0.0, 1e-8, -1e-8, 1e-15, -1e-15, 1e-20, -1e-20, 1e-36, 1e-45])
@pytest.mark.parametrize("b", [-60.0, -20.0])
def test_small_coefficients_hide_no_peak(b, c):
    """The peak of a s + b s^3 beside a last coefficient that is next to nothing."""
    a = -b
    peak = a * 2 / 3 / 3 ** 0.5
    assert D.ops._largest_value(a, b, c, 1.0) == pytest.approx(peak, rel=1e-6)
    table = (ctypes.c_float * 3)(a, b, c)
    status = N.lib().dl_orthogonalize(None, None, 0, 4, 4, 0, 1, table, 1e-7, None, None)
    assert (status == N.DL_OK) == (peak <= 8)
    assert D.ops._largest_value(0.0, 0.0, c, 1.0) == abs(c) and D.ops._largest_value(a, 0.0, 0.0, 1.0) == a
    assert D.ops._largest_value(0.0, b, 0.0, 1.0) == -b and D.ops._largest_value(0.0, b, c, 1.0) == pytest.approx(-b, rel=1e-6)
