# SPDX-License-Identifier: Apache-2.0
"""The fp32 SwiGLU of the int8 quantizer (csrc/dsv4_swiglu_math.h), built for
the host, against fp64: a value is within its bound or NaN, over every exponent
of gate and up value.

The bound. A row is served by fp32 values only where its largest is 2^-60 or
more, and a code or scale follows from values within 2^-21 of the largest: so a
value may be off by 2^-21 of itself (8 x 2^-24, the header's sum of steps) plus
2^-81. Beyond fp32's range a value is infinite and its row goes to fp64."""
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
    const bool un = unbounded(limit);
    for (long i = 0; i < n; i++) {
        v[i] = value32(g[i], u[i], limit);
        if (un && lost(g[i], u[i], v[i])) v[i] = NAN;
    }
}
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

    def run(g, u, limit):
        v = np.empty_like(g)
        lib.values(g, u, limit, v, g.size)
        return v
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


def in_bound(v, want):
    big = np.abs(want) >= np.finfo(np.float32).max * (1 - 2.0 ** -20)
    with np.errstate(over="ignore", invalid="ignore"):
        ok = np.abs(v.astype(np.float64) - want) <= 2.0 ** -21 * np.abs(want) + 2.0 ** -81
    return ok | (big & (np.abs(v) >= 3.4e38))


@pytest.mark.parametrize("limit", [0.0, -1.0, 10.0, 2.0 ** 32, 2.0 ** 33, 1e20, 3e38])
def test_values_hold_their_bound_or_are_nan(values, limit):
    g, u = grid()
    v, want = values(g, u, limit), exact(g, u, limit)
    assert (np.isnan(v) | in_bound(v, want)).all()


@pytest.mark.parametrize("g,u", [(-89.0, 1e37), (-87.5, 1e37), (-90.0, 1e37), (-95.0, 1e37), (-100.0, 2.0 ** 110),
                                 (4.2e-45, 1e38), (3 * 2.0 ** -149, 2.0 ** 100)])
def test_a_lost_value_is_nan(values, g, u):
    """Gates whose silu leaves fp32's normal range under up values that make it count."""
    assert np.isnan(values(np.float32([g]), np.float32([u]), 0.0)).all()


def test_ordinary_gates_keep_large_up_values(values):
    """Only a lost value becomes NaN, not every product with a large up value."""
    g = np.float32([-80, -20, -1, -1e-30, 0, 1e-30, 1, 50] * 2)
    u = np.float32([1e12] * 8 + [-1e30] * 8)
    v = values(g, u, 0.0)
    assert in_bound(v, exact(g, u, 0.0)).all()
