"""Which logits of a row have a weight (sample_shape.h): those at most 45 temperatures below the largest, exactly, whatever f32's steps are there."""
import os
import subprocess
from fractions import Fraction

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LOWEST = np.float32(-3.4028234663852886e38)


@pytest.fixture(scope="module")
def floors(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("sample") / "sample_floor_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-I", os.path.join(ROOT, "moe4all_b200", "csrc"), os.path.join(ROOT, "tests", "cpp", "sample_floor_check.cpp"), "-o", exe],
                   check=True)

    def ask(top, t):
        pairs = "".join(f"{a:08x} {b:08x}\n" for a, b in zip(np.float32(top).view(np.uint32), np.float32(t).view(np.uint32)))
        out = subprocess.run([exe], input=pairs, capture_output=True, text=True, check=True).stdout.split()
        return np.array([int(x, 16) for x in out], np.uint32).view(np.float32)

    return ask


def test_the_floor_is_the_least_number_within_reach(floors):
    r = np.random.default_rng(1)
    top = np.concatenate([r.normal(size=3000) * 10.0 ** r.uniform(-30, 30, 3000), [100, 12, 20, 1e10, 1e5, 100, 100, 1e17, -3e38, 3e38, 0.0, 0.0, -2.99e38, 3.4028234663852886e38, 1e-39]])
    t = np.concatenate([10.0 ** r.uniform(-40, 38, 3000), [1e-8, 1e-9, 2e-9, 1, 1e-6, 1.69e-7, 1.72e-7, 1, 1e30, 1e-3, 1e-45, 1e-41, 3e37, 1e-45, 1e-41]])
    t[:2000] = np.abs(top[:2000]) * 10.0 ** r.uniform(-12, 1, 2000)  # (around a step of the largest)
    top, t = top.astype(np.float32), np.maximum(t.astype(np.float32), np.float32(1.4e-45))
    for a, b, f in zip(top, t, floors(top, t)):
        assert LOWEST <= f <= a
        reach = float(a) - 45.0 * float(b)  # in 64 bits, as it is meant
        if f > LOWEST or reach > float(LOWEST):
            assert float(f) >= reach, (a, b, f)
            # so a weight's exponent is in range: 45 temperatures, and what 64 bits round of the reach
            assert Fraction(float(a)) - Fraction(float(f)) <= Fraction(45) * Fraction(float(b)) + abs(Fraction(float(a))) * Fraction(2) ** -52 + Fraction(45) * Fraction(float(b)) * Fraction(2) ** -50
            below = np.nextafter(f, np.float32(-np.inf), dtype=np.float32)
            assert float(below) < reach, (a, b, f)


def test_nothing_finite_is_near_an_infinite_one(floors):
    inf = np.float32(np.inf)
    assert floors([np.inf, np.inf], [1.0, np.inf]).tolist() == [inf, inf]
    assert floors([5.0, 5.0, -3e38], [np.inf, 3e38, 1e38]).tolist() == [LOWEST] * 3
