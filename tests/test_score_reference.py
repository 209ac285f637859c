"""The arithmetic of the softmax reference (csrc/score_reference.cuh), built for the host: scores of every finite size."""
import ctypes
import math
import os
import subprocess
from fractions import Fraction

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
MOST = 3.4028234663852886e38


@pytest.fixture(scope="module")
def probe(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("probe") / "probe.so")
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-ffp-contract=off", "-fPIC", "-shared", os.path.join(HERE, "score_reference_probe.cpp"), "-o", out])
    lib = ctypes.CDLL(out)
    f = ctypes.c_float
    for name, args in (("probe_exponent", [ctypes.POINTER(f), f, f, f]), ("probe_move", [ctypes.POINTER(f), f, f, f]),
                       ("probe_negative_reference", [f, f])):
        getattr(lib, name).argtypes, getattr(lib, name).restype = args, f
    return lib


def _state():
    return (ctypes.c_float * 3)()


def _exact(y, q):
    return Fraction(float(y)) * Fraction(float(q))


@pytest.mark.parametrize("e", list(range(0, 48)) + [60, 90, 120, 125])
def test_exponents_of_a_row_are_right_at_any_size(probe, e):
    """The score the reference was made from comes out at `lift` and the others below it by their exact distance: within
    1/4 for a near reference (half a step of a number below 2^22), the same for the whole row, and otherwise within 2^-22
    of the distance (three roundings of half a step)."""
    rng = np.random.default_rng(e)
    for lift in (-3.0, 0.0, 41.0, -100.0, 100.0):
        for _ in range(20):
            y, q = np.float32(rng.uniform(0.5, 2.0) * rng.choice([-1, 1])), np.float32(2.0 ** e * rng.uniform(0.5, 0.99))
            st = _state()
            probe.probe_move(st, y, q, lift)
            assert st[2] == (abs(float(np.float32(y * q))) >= 2.0 ** 22)
            own = probe.probe_exponent(st, y, q, lift)
            assert abs(own - lift) <= (2.0 ** -16 if st[2] else 0.25 + 2.0 ** -16)
            for steps in (1, 2, 7, 1000, 10 ** 6):
                y2 = np.float32(y - steps * float(np.spacing(abs(y))))
                far = float(_exact(y, q) - _exact(y2, q))
                got = own - probe.probe_exponent(st, y2, q, lift)
                assert abs(got - far) <= 2.0 ** -22 * far + 2.0 ** -14, (got, far)


def test_moving_the_reference_changes_all_exponents_alike(probe):
    rng = np.random.default_rng(1)
    for _ in range(2000):
        e0, e1 = rng.integers(0, 60, 2)
        lift = float(rng.integers(-100, 100))
        q = np.float32(rng.uniform(0.5, 1.0))
        a, b = np.float32(rng.uniform(-1, 1) * 2.0 ** e0), np.float32(rng.uniform(0.5, 1) * 2.0 ** e1)
        if not b * q > a * q + 8:
            continue
        st = _state()
        probe.probe_move(st, a, q, lift)
        before = probe.probe_exponent(st, a, q, lift)
        change = probe.probe_move(st, b, q, lift)
        after = probe.probe_exponent(st, a, q, lift)
        assert change < 0
        if change > -200:                                                  # further away the factor is zero either way
            assert abs((after - before) - change) <= 2.0 ** -13             # a few fp32 steps of exponents up to 300 are 2^-13
        else:
            assert after < before - 150


def test_a_row_walked_in_tiles_ends_and_keeps_its_maximum(probe):
    """The order of the kernel: a first reference, then tile after tile, moved where a tile's largest score is more than
    8 ahead, at most once.  Whatever the sizes, no exponent is above lift + 8 by more than rounding, and the largest
    score of the row ends at most 8 above and 1/2 below the reference."""
    rng = np.random.default_rng(2)
    lift = 5.0
    for e in list(range(16, 44)) + [70, 120]:
        for _ in range(10):
            q = np.float32(rng.uniform(0.5, 1.0) * 2.0 ** (e / 2))
            y = np.float32(rng.standard_normal((4, 128)) * 2.0 ** (e / 2) * (2.0 ** rng.integers(-30, 1, (4, 1)) if e % 2 else 1.0))
            st, best = _state(), -math.inf
            for j, tile in enumerate(y):
                top = tile.max()
                if j == 0 or probe.probe_exponent(st, top, q, lift) > lift + 8:
                    probe.probe_move(st, top, q, lift)
                best = max(best, top)
                assert probe.probe_exponent(st, top, q, lift) <= lift + 8.5
            assert lift - 0.5 <= probe.probe_exponent(st, best, q, lift) <= lift + 8.5


def test_scores_beyond_the_range_make_the_row_nan(probe):
    for y, q in ((math.inf, 1.0), (-math.inf, 1.0), (math.nan, 1.0), (1.0, math.inf), (1.0, math.nan), (3e38, 3e38), (1e38, 1.0)):
        st = _state()
        assert math.isnan(probe.probe_move(st, y, q, 3.0))
        assert math.isnan(probe.probe_exponent(st, 1.0, 1.0, 3.0)) and not st[2]
    st = _state()
    st[0] = math.inf                                                       # no reference yet: any score is ahead of it
    assert probe.probe_exponent(st, -3e30, 1.0, 3.0) == math.inf and probe.probe_move(st, -3e30, 1.0, 3.0) == -math.inf
    assert abs(probe.probe_exponent(st, -3e30, 1.0, 3.0) - 3.0) < 2.0 ** -16
    st = _state()
    probe.probe_move(st, 1.5, 2.0 ** 80, 3.0)
    assert probe.probe_exponent(st, -math.inf, 2.0 ** 80, 3.0) == -math.inf        # a removed position stays removed


@pytest.mark.parametrize("e", list(range(0, 40)) + [80, 127])
def test_reference_for_rounded_scores(probe, e):
    rng = np.random.default_rng(e)
    for at in (15.0, 0.5, -3.0, 33.0):
        for sign in (-1, 1):
            mx = np.float32(sign * min(rng.uniform(1, 2) * 2.0 ** e, MOST))
            neg = np.float32(probe.probe_negative_reference(mx, at))
            x = float(np.float32(mx + neg))
            assert abs(x - (at if abs(mx) < 2.0 ** 22 else 0.0)) <= 0.25
