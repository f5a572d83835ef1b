# SPDX-License-Identifier: Apache-2.0
"""What the int8 product and expert-order calls refuse, before any device is
touched: every bad argument gives -1 with its reason, and the same call with
good arguments gets as far as the device."""
import ctypes as C

import pytest
import torch

from conftest import load_pkg

P = 1 << 20                       # an aligned address that no refused call reads


@pytest.fixture(scope="module")
def calls():
    if torch.cuda.is_available():
        pytest.skip("the last of these calls would reach the device")
    pkg = load_pkg()
    lib = pkg.Lib()
    L = lib.lib

    def w(**kw):
        f = dict(w=P, s=P, wdt=pkg.DSV4_WI8, rows=32, cols=64, blk_r=1, blk_c=64) | kw
        return C.byref(pkg.QMat(*(f[k] for k in ("w", "s", "wdt", "rows", "cols", "blk_r", "blk_c"))))

    good = {
        "quant": (L.dsv4_hip_quant_i8_dev, dict(Q=P, S=P, a=P, type=0, ld=64, n=3, k=64, st=None)),
        "swiglu": (L.dsv4_hip_swiglu_quant_i8_dev,
                   dict(Q=P, S=P, g=P, u=P, type=1, ld=64, n=3, k=64, limit=10.0, st=None)),
        "gemm": (L.dsv4_hip_gemm_i8_dev, dict(C=P, out=0, Aq=P, Sa=P, M=3, W=w(), st=None)),
        "grouped": (L.dsv4_hip_gemm_i8_grouped_dev,
                    dict(C=P, out=0, Aq=P, Sa=P, n_a=4, row_tok=P, n_rows=8, ex_off=P, table=P, E=5, N=32, K=64,
                         st=None)),
        "permute": (L.dsv4_hip_moe_permute_dev,
                    dict(rows=P, ex_off=P, row_tok=P, pos=P, x=P, type=0, idx=P, n=3, topk=2, E=5, h=8, st=None)),
        "permute_bwd": (L.dsv4_hip_moe_permute_bwd_dev,
                        dict(dx=P, drows=P, type=0, pos=P, n=3, topk=2, h=8, st=None)),
        "unpermute": (L.dsv4_hip_moe_unpermute_dev,
                      dict(out=P, rows=P, type=0, pos=P, w=P, shared=None, n=3, topk=2, h=8, st=None)),
        "unpermute_bwd": (L.dsv4_hip_moe_unpermute_bwd_dev,
                          dict(drows=P, dw=P, dout=P, rows=P, type=0, pos=P, w=P, n=3, topk=2, h=8, st=None)),
    }

    def run(name, **bad):
        fn, args = good[name]
        assert set(bad) <= set(args)
        return fn(*(args | bad).values()), lib.error()
    return run, w


GOOD = ["quant", "swiglu", "gemm", "grouped", "permute", "permute_bwd", "unpermute", "unpermute_bwd"]


@pytest.mark.parametrize("name", GOOD)
def test_good_arguments_get_to_the_device(calls, name):
    rc, why = calls[0](name)
    assert rc == -1 and "init" in why


@pytest.mark.parametrize("name,zero", [("quant", "n"), ("swiglu", "n"), ("gemm", "M"), ("grouped", "n_rows"),
                                       ("permute", "n"), ("permute_bwd", "n"), ("unpermute", "n"),
                                       ("unpermute_bwd", "n")])
def test_no_rows_is_no_fault_of_the_call(calls, name, zero):
    """Without a device they are refused for that, and not for the size."""
    rc, why = calls[0](name, **{zero: 0})
    assert rc == -1 and "init" in why
    rc, why = calls[0](name, **{zero: -1})
    assert rc == -1 and "init" not in why


BAD = [("quant", k, v) for k, v in [("Q", None), ("S", None), ("a", None), ("type", 3), ("type", -1), ("ld", 63),
                                    ("ld", 66), ("k", 0), ("k", 24), ("a", P + 4), ("Q", P + 4), ("S", P + 2),
                                    ("ld", (1 << 40) + 16)]]
BAD += [("swiglu", k, v) for k, v in [("g", None), ("u", None), ("u", P + 8), ("ld", 48), ("k", 40)]]
BAD += [("gemm", k, v) for k, v in [("C", None), ("Aq", None), ("Sa", None), ("W", None), ("out", 7), ("Aq", P + 8),
                                    ("C", P + 2), ("Sa", P + 1)]]
BAD += [("grouped", k, v) for k, v in [("C", None), ("ex_off", None), ("table", None), ("E", 0), ("E", 1025),
                                       ("N", 0), ("K", 8), ("K", 72), ("K", 131072), ("n_a", 0), ("out", -2),
                                       ("Aq", P + 1), ("table", P + 4), ("row_tok", P + 2), ("n_a", 1 << 25)]]
BAD += [("permute", k, v) for k, v in [("rows", None), ("ex_off", None), ("row_tok", None), ("pos", None), ("x", None),
                                       ("idx", None), ("type", 5), ("topk", 0), ("topk", 17), ("E", 0), ("E", 1025),
                                       ("h", 0), ("n", 1 << 26), ("x", P + 2), ("pos", P + 1)]]
BAD += [("permute_bwd", k, v) for k, v in [("dx", None), ("drows", None), ("pos", None), ("topk", 17), ("type", 9)]]
BAD += [("unpermute", k, v) for k, v in [("out", None), ("rows", None), ("pos", None), ("w", None), ("shared", P + 1),
                                         ("topk", 0), ("h", -4)]]
BAD += [("unpermute_bwd", k, v) for k, v in [("drows", None), ("dw", None), ("dout", None), ("rows", None),
                                             ("pos", None), ("w", None), ("type", 3)]]


@pytest.mark.parametrize("name,arg,value", BAD)
def test_bad_argument_is_refused(calls, name, arg, value):
    rc, why = calls[0](name, **{arg: value})
    assert rc == -1 and why and "init" not in why


@pytest.mark.parametrize("m,n", [((1 << 31) - 1, 1 << 20), (1 << 28, 1 << 20), ((1 << 31) - 1, 64), (1, (1 << 31) - 1),
                                 (1 << 24, 1 << 16), ((1 << 31) - 100, 3)])
def test_more_than_a_launch_takes_is_refused(calls, m, n):
    run, w = calls
    rc, why = run("gemm", M=m, W=w(rows=n))
    assert rc == -1 and "too many" in why
    rc, why = run("grouped", n_rows=m, N=n)
    assert rc == -1 and "too many" in why


@pytest.mark.parametrize("n", [1 << 22, (1 << 31) - 1])
def test_more_rows_than_a_launch_takes_are_refused(calls, n):
    for name in ("quant", "swiglu"):
        rc, why = calls[0](name, n=n)
        assert rc == -1 and "too many" in why


@pytest.mark.parametrize("k", [(1 << 24) + 16, (1 << 31) - 16])
def test_rows_whose_elements_an_index_does_not_hold_are_refused(calls, k):
    for name in ("quant", "swiglu"):
        rc, why = calls[0](name, k=k, ld=k)
        assert rc == -1 and "2^24" in why
        rc, why = calls[0](name, k=1 << 24, ld=k)
        assert rc == -1 and "init" in why


@pytest.mark.parametrize("field,value", [("wdt", 2), ("rows", 0), ("cols", 0), ("cols", 40), ("cols", 131072),
                                         ("w", None), ("s", None), ("w", P + 8), ("s", P + 2)])
def test_bad_matrix_is_refused(calls, field, value):
    run, w = calls
    rc, why = run("gemm", W=w(**{field: value}))
    assert rc == -1 and why and "init" not in why
