"""CPU check of a softmax row's exponents (a host build of fast-mac-gsplat_amd/csrc/exponent.h, the source the
kernels compile) for largest logits from 0 to the float's limits and temperatures from 1e-20 to 1e3.

The row's exponents are t + shift, t taken to the power of two before shift is added.  So the shift has to be
small beside the range of the powers (1 of 126), and t + shift off by few roundings of the exponent itself:
  fast  t = fma(x, c, -k) is rounded once, shift holds the rest of k up to 2^-24 of itself: E |t| + E
  slow  a difference, a product and a difference, each rounded:                            3 E (|t| + |l|)
with E = 2^-24, t the exponent."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
E = 2.0 ** -24
F = np.float32


@pytest.fixture(scope="module")
def exponents(tmp_path_factory):
    out = tmp_path_factory.mktemp("exponent") / "libexponentcheck.so"
    subprocess.run(["g++", "-O2", "-std=c++17", "-fPIC", "-shared", "-mfma", "-ffp-contract=off",
                    os.path.join(HERE, "exponent_check.cpp"), "-o", str(out)], check=True)
    lib = ctypes.CDLL(str(out))
    lib.exponent_check.restype = ctypes.c_int
    lib.exponent_check.argtypes = [ctypes.c_float] * 3 + [ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p]

    def f(m, l, c, x):
        x = np.ascontiguousarray(x, F)
        t, shift = np.empty_like(x), np.empty(1, F)
        plain = lib.exponent_check(m, l, c, x.ctypes.data, x.size, t.ctypes.data, shift.ctypes.data)
        return t, float(shift[0]), bool(plain)
    return f


SIZES = [0.0, 1e-3, 0.7, 3.0, 5.5, 88.0, 1e3, 1e5, 3e6, 1e7, 2e7, 1e8, 1e9, 1e10, 1e15, 1e20, 1e29, 1e30, 1e31, 3e38]


@pytest.mark.parametrize("T", [1e3, 1.0, 0.3, 1e-3, 1e-6, 1e-9, 1e-10, 1e-20])
@pytest.mark.parametrize("l", [0.0, 5.25, -32.0, -17.5])
def test_exponents_of_far_rows(exponents, T, l):
    rng = np.random.default_rng(3)
    c = F(F(1.0) / F(T)) * F(1.4426950408889634)
    for size in SIZES:
        for m in (F(size), F(-size)):
            with np.errstate(over="ignore"):
                x = (m - np.abs(rng.normal(size=64)).astype(F) * F(T) * F(8)).astype(F)
                x[:4] = m
                x[4:8] = np.nextafter(m, F(-np.inf))
                x[8] = m - abs(m) * F(2.0 ** -7)
            t, shift, plain = exponents(float(m), l, float(c), x)
            assert abs(shift) <= 1.0, f"m={m} T={T}: shift {shift}"
            true = (x.astype(np.float64) - float(m)) * float(c) - l
            near = true > -1000.0  # (below: no probability)
            got = t.astype(np.float64) + shift
            bound = 3 * E * (np.abs(true) + abs(l)) + E
            assert np.all(np.abs(got - true)[near] <= bound[near]), f"m={m} T={T} plain={plain}"
            assert np.all(got[~near] <= -999.0), f"m={m} T={T} plain={plain}"


def test_rows_without_probabilities(exponents):
    """log2 s = inf: every exponent is -inf, the shift 0; a NaN row's shift is NaN."""
    t, shift, plain = exponents(3.0, float("inf"), 1.44, np.array([3.0, -1.0, -np.inf], F))
    assert not plain and shift == 0.0 and np.all(t == -np.inf)
    _, shift, plain = exponents(3.0, float("nan"), 1.44, np.array([3.0], F))
    assert not plain and np.isnan(shift)
