# SPDX-License-Identifier: Apache-2.0
"""What the 4-bit rows and products and the router with groups refuse, before any
device is touched: every bad argument gives -1 with its reason, and the same call
with good arguments gets as far as the device."""
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
        f = dict(w=P, s=P, wdt=pkg.DSV4_WFP4, rows=32, cols=64, blk_r=1, blk_c=32) | kw
        return C.byref(pkg.QMat(*(f[k] for k in ("w", "s", "wdt", "rows", "cols", "blk_r", "blk_c"))))

    def r(**kw):
        f = dict(score=1, n_experts=24, topk=4, n_group=6, topk_group=2, group_top=2, renorm=1, scale=1.0) | kw
        return C.byref(pkg.Router(*f.values()))

    good = {
        "rows": (L.dsv4_hip_quant_mxfp4_dev, dict(Q=P, S=P, a=P, type=0, ld=64, n=3, k=64, st=None)),
        "swiglu": (L.dsv4_hip_swiglu_quant_mxfp4_dev,
                   dict(Q=P, S=P, g=P, u=P, type=1, ld=64, n=3, k=64, limit=10.0, st=None)),
        "columns": (L.dsv4_hip_quant_mxfp4_t_dev, dict(Q=P, S=P, a=P, type=1, ld=63, n=3, k=61, st=None)),
        "gemm": (L.dsv4_hip_gemm_mxfp4q_dev, dict(C=P, out=0, Aq=P, As=P, M=3, W=w(), st=None)),
        "grouped": (L.dsv4_hip_gemm_mxfp4q_grouped_dev,
                    dict(C=P, out=0, Aq=P, As=P, n_a=4, row_tok=P, n_rows=8, ex_off=P, table=P, E=5, N=32, K=64,
                         st=None)),
        "route": (L.dsv4_hip_route_groups_dev,
                  dict(idx=P, w=P, scores=None, logits=P, type=0, n=3, bias=None, r=r(), st=None)),
        "route_bwd": (L.dsv4_hip_route_groups_bwd_dev,
                      dict(dlogits=P, dw=P, dscores=None, logits=P, type=0, idx=P, n=3, r=r(), st=None)),
    }

    def run(name, **bad):
        fn, args = good[name]
        assert set(bad) <= set(args)
        return fn(*(args | bad).values()), lib.error()
    return run, w, r


GOOD = ["rows", "swiglu", "columns", "gemm", "grouped", "route", "route_bwd"]
COUNT = {"gemm": "M", "grouped": "n_rows"}


@pytest.mark.parametrize("name", GOOD)
def test_good_arguments_get_to_the_device(calls, name):
    rc, why = calls[0](name)
    assert rc == -1 and "init" in why


@pytest.mark.parametrize("name", GOOD)
def test_no_rows_is_no_fault_of_the_call(calls, name):
    """Without a device they are refused for that, and not for the size."""
    n = COUNT.get(name, "n")
    rc, why = calls[0](name, **{n: 0})
    assert rc == -1 and "init" in why
    rc, why = calls[0](name, **{n: -1})
    assert rc == -1 and "init" not in why


def test_scales_and_codes_of_any_alignment_get_to_the_device(calls):
    for name, args in (("rows", dict(Q=P + 4, S=P + 1)), ("columns", dict(S=P + 3, a=P + 2)), ("columns", dict(k=1, n=1)),
                       ("gemm", dict(As=P + 1, C=P + 4)), ("grouped", dict(As=P + 3, row_tok=None)),
                       ("route", dict(scores=P + 4, bias=P + 8))):
        rc, why = calls[0](name, **args)
        assert rc == -1 and "init" in why
    rc, why = calls[0]("gemm", W=calls[1](s=P + 3))
    assert rc == -1 and "init" in why


BAD = [("rows", k, v) for k, v in [("Q", None), ("S", None), ("a", None), ("type", 3), ("type", -1), ("ld", 63),
                                   ("ld", 66), ("k", 0), ("k", 48), ("a", P + 4), ("Q", P + 2), ("ld", (1 << 40) + 16)]]
BAD += [("swiglu", k, v) for k, v in [("g", None), ("u", None), ("u", P + 8), ("ld", 48), ("k", 40)]]
BAD += [("columns", k, v) for k, v in [("Q", None), ("a", None), ("a", P + 1), ("Q", P + 8), ("ld", 60), ("k", -1),
                                       ("n", 1 << 24), ("type", 4)]]
BAD += [("gemm", k, v) for k, v in [("C", None), ("Aq", None), ("As", None), ("W", None), ("out", 7), ("Aq", P + 8),
                                    ("C", P + 2)]]
BAD += [("grouped", k, v) for k, v in [("C", None), ("ex_off", None), ("table", None), ("E", 0), ("E", 1025),
                                       ("N", 0), ("K", 16), ("K", 80), ("K", (1 << 20) + 32), ("n_a", 0), ("out", -2),
                                       ("Aq", P + 1), ("table", P + 4), ("row_tok", P + 2), ("n_a", 1 << 26)]]
BAD += [("route", k, v) for k, v in [("idx", None), ("w", None), ("logits", None), ("r", None), ("type", 5), ("idx", P + 2),
                                     ("scores", P + 1), ("bias", P + 2), ("logits", P + 2), ("n", (1 << 26) - 3)]]
BAD += [("route_bwd", k, v) for k, v in [("dlogits", None), ("dw", None), ("logits", None), ("idx", None), ("r", None),
                                         ("type", 9), ("dscores", P + 1), ("dlogits", P + 1), ("n", (1 << 26) - 3)]]


@pytest.mark.parametrize("name,arg,value", BAD)
def test_bad_argument_is_refused(calls, name, arg, value):
    rc, why = calls[0](name, **{arg: value})
    assert rc == -1 and why and "init" not in why


@pytest.mark.parametrize("field,value", [("wdt", 2), ("wdt", 5), ("rows", 0), ("cols", 0), ("cols", 40),
                                         ("cols", (1 << 20) + 32), ("w", None), ("s", None), ("w", P + 8), ("blk_r", 2),
                                         ("blk_c", 64)])
def test_bad_matrix_is_refused(calls, field, value):
    run, w, _ = calls
    rc, why = run("gemm", W=w(**{field: value}))
    assert rc == -1 and why and "init" not in why


@pytest.mark.parametrize("bad", [dict(score=3), dict(score=-1), dict(n_experts=0), dict(n_experts=1025, n_group=1, topk_group=1),
                                 dict(topk=0), dict(topk=17), dict(topk=9), dict(n_group=0), dict(n_group=5),
                                 dict(n_group=7), dict(topk_group=0), dict(topk_group=7), dict(group_top=0),
                                 dict(group_top=3), dict(n_experts=130, n_group=65)])
def test_bad_router_is_refused(calls, bad):
    run, _, r = calls
    rc, why = run("route", r=r(**bad))
    assert rc == -1 and why and "init" not in why


def test_the_backward_call_reads_no_groups(calls):
    run, _, r = calls
    rc, why = run("route_bwd", r=r(n_group=0, topk_group=0, group_top=0))
    assert rc == -1 and "init" in why
    for bad in (dict(topk=17), dict(score=9), dict(n_experts=3)):
        rc, why = run("route_bwd", r=r(**bad))
        assert rc == -1 and "init" not in why


@pytest.mark.parametrize("m,n", [((1 << 31) - 1, 1 << 20), (1 << 28, 1 << 20), ((1 << 31) - 1, 64), (1, (1 << 31) - 1),
                                 (1 << 24, 1 << 16), ((1 << 31) - 100, 3)])
def test_more_than_a_launch_takes_is_refused(calls, m, n):
    run, w, _ = calls
    if m > 8 or n > 1 << 26:
        rc, why = run("gemm", M=m, W=w(rows=n))
        assert rc == -1 and "too many" in why
    rc, why = run("grouped", n_rows=m, N=n)
    assert rc == -1 and "too many" in why


@pytest.mark.parametrize("name,n,k", [("rows", (1 << 31) - 1, 64), ("rows", 1 << 11, 1 << 24), ("swiglu", 1 << 29, 64),
                                      ("swiglu", (1 << 30) - 127, 32),
                                      ("columns", 1 << 20, 1 << 15), ("columns", (1 << 24) - 1, 1 << 12)])
def test_more_elements_than_a_launch_takes_are_refused(calls, name, n, k):
    rc, why = calls[0](name, n=n, k=k, ld=k)
    assert rc == -1 and "too many" in why
