# SPDX-License-Identifier: Apache-2.0
"""The fp32 SwiGLU of the int8 quantizer (csrc/dsv4_swiglu_math.h), built for
the host, against fp64, over every exponent of gate and up value.

The bound. A code and a scale follow from values within 2^-21 of the row's
largest. A value may so be off by 2^-21 of itself (8 x 2^-24, the header's sum of
steps) plus 2^-21 of the least largest value with which its row would still be
served by fp32. A value that is NaN sends its row to fp64, one beyond 2^120 too."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from conftest import PKG_DIR

SHIM = """
#include "dsv4_swiglu_math.h"
using namespace dsv4_swiglu;
extern "C" void values(const float *g, const float *u, float limit, float *v, long n)
{
    for (long i = 0; i < n; i++) v[i] = value32(g[i], u[i], limit);
}
/* the least power of two that a row's largest value may be with up values of size u */
extern "C" void least(const float *u, float limit, float *a, long n)
{
    for (long i = 0; i < n; i++) {
        const float um = !unbounded(limit) ? 0.0f : limit > 0 ? fminf(fabsf(u[i]), limit) : fabsf(u[i]);
        for (a[i] = 0x1p-149f; !fp32_serves(a[i], um); a[i] *= 2) ;
    }
}
extern "C" int serves(float amax, float umax) { return fp32_serves(amax, umax); }
"""


@pytest.fixture(scope="module")
def values(tmp_path_factory):
    d = tmp_path_factory.mktemp("swiglu")
    src, so = d / "shim.cpp", d / "shim.so"
    src.write_text(SHIM)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-ffp-contract=off", "-shared", "-fPIC", "-I",
                    os.path.join(PKG_DIR, "csrc"), str(src), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    P = np.ctypeslib.ndpointer(np.float32, flags="C_CONTIGUOUS")
    lib.values.argtypes, lib.values.restype = [P, P, C.c_float, P, C.c_long], None
    lib.least.argtypes, lib.least.restype = [P, C.c_float, P, C.c_long], None
    lib.serves.argtypes, lib.serves.restype = [C.c_float, C.c_float], C.c_int

    def run(g, u, limit):
        """values, and the least largest value of a row that fp32 serves"""
        v, a = np.empty_like(g), np.empty_like(g)
        lib.values(g, u, limit, v, g.size)
        lib.least(u, limit, a, u.size)
        return v, a.astype(np.float64)
    run.serves = lib.serves
    return run


def grid():
    """gates and up values of every exponent and sign, and gates around exp's ends"""
    r = np.random.default_rng(1)
    with np.errstate(over="ignore"):
        mag = np.concatenate([np.ldexp(1 + r.random(2), e) for e in range(-149, 128)])
    gates = np.concatenate([mag, -mag, -np.linspace(60, 130, 1401), np.linspace(-12, 12, 481), [0.0, -0.0]])
    ups = np.concatenate([mag, -mag[::5], [0.0, 1e37, 3.4e38, 1.0]])
    g, u = np.meshgrid(gates.astype(np.float32), ups.astype(np.float32), indexing="ij")
    return g.ravel().copy(), u.ravel().copy()


def exact(g, u, limit):
    g, u = g.astype(np.float64), u.astype(np.float64)
    if limit > 0:
        g, u = np.minimum(g, limit), np.clip(u, -limit, limit)
    with np.errstate(over="ignore"):
        return g / (1 + np.exp(-g)) * u


def in_bound(v, want, least):
    with np.errstate(over="ignore", invalid="ignore"):
        ok = np.abs(v.astype(np.float64) - want) <= 2.0 ** -21 * (np.abs(want) + least)
    return ok | ((np.abs(want) > 2.0 ** 120) & (np.abs(v) > 2.0 ** 120))


@pytest.mark.parametrize("limit", [0.0, -1.0, 10.0, 2.0 ** 32, 2.0 ** 33, 1e20, 3e38])
def test_values_hold_their_bound_or_are_nan(values, limit):
    g, u = grid()
    v, least = values(g, u, limit)
    assert (np.isnan(v) | in_bound(v, exact(g, u, limit), least)).all()


@pytest.mark.parametrize("g,u", [(-89.0, 1e37), (-87.5, 1e37), (-90.0, 1e37), (-100.0, 2.0 ** 110), (4.2e-45, 1e38),
                                 (3 * 2.0 ** -149, 2.0 ** 100)])
def test_a_value_that_is_lost_has_its_row_decided_in_fp64(values, g, u):
    """Be it the row's largest value or one that is 64 times smaller."""
    size = abs(exact(np.float32([g]), np.float32([u]), 0.0)[0])
    for largest in (size, 64 * size):
        assert not values.serves(largest, u)


def test_large_up_values_under_ordinary_gates_are_served(values):
    for u in (1.0, 1e12, 1e30):
        assert values.serves(0.5 * u, u) and values.serves(1e-25 * u + 1e-15, u)


@pytest.mark.parametrize("amax", [0.0, 1e-19, 2e36, float("inf"), float("nan")])
def test_rows_beyond_fp32s_reach_are_not(values, amax):
    assert not values.serves(amax, 0.0)


@pytest.mark.parametrize("limit", [0.0, 10.0, 2.0 ** 32])
def test_no_finite_gate_sends_its_row_to_fp64(values, limit):
    """With up values of a model a value is finite however negative its gate: one
    that is not costs all of its row two fp64 values an element."""
    r = np.random.default_rng(2).random(2000)
    g = np.concatenate([-np.linspace(60, 130, 7001), -np.ldexp(1 + r, 7 + np.arange(2000) % 120)]).astype(np.float32)
    for u in (1.0, -0.03, 700.0):
        u = np.full_like(g, u)
        v, least = values(g, u, limit)
        assert np.isfinite(v).all() and in_bound(v, exact(g, u, limit), least).all()


@pytest.mark.parametrize("limit", [0.0, 10.0])
def test_infinite_and_nan_gates_do(values, limit):
    g = np.float32([-np.inf, np.nan] + ([np.inf] if limit == 0 else []))
    assert np.isnan(values(g, np.ones_like(g), limit)[0]).all()
