# SPDX-License-Identifier: Apache-2.0
"""The rules that pick an int8 product's form by its sizes (csrc/dsv4_choose.h),
compiled for the host: the forms that were measured to be the faster ones, and
that the GPU tests of the products reach every form."""
import ctypes as C
import os
import subprocess

import pytest

import test_gpu_i8
import test_gpu_i8_forms
from conftest import PKG_DIR

SHIM = """
#include "dsv4_choose.h"
using namespace dsv4;
extern "C" {
int c_form(int M, int N, int K) { return i8_form(M, N, K); }
int c_grouped(int M, int N, int K, int ne) { return i8_grouped_form(M, N, K, ne); }
long c_waves(int form, long M, long N, long ne) { return i8_waves((I8Form)form, M, N, ne); }
}
"""
PAIR, T64x2, T64x2_DEEP, T64x4, T128x4, T128x8, T256x8 = range(1, 8)


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("i8")
    src, so = d / "shim.cpp", d / "shim.so"
    src.write_text(SHIM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(PKG_DIR, "csrc"), str(src), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    lib.c_waves.argtypes, lib.c_waves.restype = [C.c_int, C.c_long, C.c_long, C.c_long], C.c_long
    return lib


@pytest.mark.parametrize("M,N,K,form", [
    (1, 4096, 4096, PAIR), (8, 4096, 4096, PAIR), (12, 1024, 4096, PAIR), (16, 4096, 4096, T64x2_DEEP),
    (128, 4096, 4096, T64x2_DEEP), (333, 1024, 4096, T64x2_DEEP), (5, 32768, 1024, T64x2), (333, 4096, 4096, T128x4),
    (1000, 2048, 2048, T128x4), (1024, 4096, 4096, T128x8), (2048, 4096, 4096, T256x8), (1000, 32768, 1024, T256x8)])
def test_product_form(rules, M, N, K, form):
    assert rules.c_form(M, N, K) == form


@pytest.mark.parametrize("M,N,K,ne,form", [
    (6, 2048, 4096, 256, T64x2), (42, 2048, 4096, 256, PAIR), (1536, 2048, 4096, 256, PAIR),
    (160, 512, 1024, 64, T64x2), (7680, 2048, 4096, 256, T128x4), (12288, 2048, 4096, 256, T256x8),
    (24576, 2048, 4096, 256, T256x8), (800, 512, 512, 1000, T64x2), (384, 2048, 2048, 256, PAIR),
    (6144, 2048, 4096, 64, T256x8)])
def test_experts_form(rules, M, N, K, ne, form):
    assert rules.c_grouped(M, N, K, ne) == form


def test_gpu_tests_reach_every_form(rules):
    assert {rules.c_form(*s) for s in test_gpu_i8.SHAPES} == set(range(1, 8))
    groups = {rules.c_grouped(sum(c) + 5, N, K, len(c)) for c, N, K in test_gpu_i8.GROUPS}
    assert groups == {PAIR, T64x2, T128x4, T256x8}
    for c in ([2500, 3, 0, 300], 2100, 8208), ([1, 0, 1200, 0, 60, 200, 1100] * 3, 781, 4112):
        assert c in test_gpu_i8.GROUPS and rules.c_grouped(sum(c[0]) + 5, c[1], c[2], len(c[0])) == T256x8
    assert rules.c_grouped(2900, 1701, 8208, 5) == T256x8        # the large product with bad offsets


@pytest.mark.parametrize("form,F,TR,waves", [(PAIR, 8, 8, 8), (T64x2, 64, 32, 4), (T64x2_DEEP, 64, 32, 4),
                                             (T64x4, 64, 64, 8), (T128x4, 128, 64, 8), (T128x8, 128, 128, 8),
                                             (T256x8, 256, 128, 8)])
def test_waves_of_a_launch(rules, form, F, TR, waves):
    """A tile for every F features and TR rows; rows and features of 2^31 - 1 do
    not wrap."""
    for M, N in ((1, 1), (TR, F), (TR + 1, F + 1), (1000, 777), ((1 << 31) - 1, (1 << 31) - 1)):
        assert rules.c_waves(form, M, N, 0) == -(-M // TR) * -(-N // F) * waves


@pytest.mark.parametrize("form,F,TR,waves", [(PAIR, 32, 16, 4), (T64x2, 64, 32, 4), (T128x4, 128, 64, 8),
                                             (T256x8, 256, 128, 8)])
@pytest.mark.parametrize("counts", [[0, 0, 5], [1] * 300, [127, 129, 0, 31, 33], [2000]])
def test_waves_hold_every_bucket(rules, form, F, TR, waves, counts):
    tiles = sum(-(-c // TR) for c in counts)
    assert rules.c_waves(form, sum(counts), 100, len(counts)) >= tiles * -(-100 // F) * waves


FORMS = {"pair": PAIR, "64x2": T64x2, "64x2 deep": T64x2_DEEP, "64x4": T64x4, "128x4": T128x4, "128x8": T128x8,
         "256x8": T256x8}
TILES = {"pair": (8, 8), "64x2": (64, 32), "64x2 deep": (64, 32), "64x4": (64, 64), "128x4": (128, 64),
         "128x8": (128, 128), "256x8": (256, 128)}                 # features, rows


def test_gpu_tests_reach_the_forms_that_they_name(rules):
    """and each with rows, features and K that end inside a tile"""
    for cases in (test_gpu_i8_forms.ONE, test_gpu_i8_forms.WIDE, test_gpu_i8_forms.SLICES, test_gpu_i8_forms.EVEN):
        assert set(cases) == set(FORMS)
    for form, (F, TR) in TILES.items():
        for M, N, K in test_gpu_i8_forms.ONE[form]:
            assert rules.c_form(M, N, K) == FORMS[form] and M % TR and N % F and K % 128
        assert rules.c_form(*test_gpu_i8_forms.WIDE[form], test_gpu_i8_forms.KMAX) == FORMS[form]
        assert rules.c_form(test_gpu_i8_forms.SLICES[form], test_gpu_i8_forms.SLICES_N,
                            test_gpu_i8_forms.SLICES_K) == FORMS[form]
        M, N, K = test_gpu_i8_forms.EVEN[form]
        assert rules.c_form(M, N, K) == FORMS[form] and N % 8 == 0


def test_gpu_tests_reach_the_forms_of_the_experts_product(rules):
    for cases in (test_gpu_i8_forms.GROUPED, test_gpu_i8_forms.GROUPED_WIDE):
        for form in ("pair", "64x2", "128x4", "256x8"):
            counts, N, K = cases[form]
            assert rules.c_grouped(sum(counts), N, K, len(counts)) == FORMS[form]


@pytest.mark.parametrize("M,N,K", [(1 << 30, 256, 16), ((1 << 30) - 128, 256, 4096), (1 << 30, 1, 16),
                                   ((1 << 30) - 127, 1, 131056), (1 << 26, 4096, 64), ((1 << 26) - 128, 4096, 64),
                                   (1 << 18, 1 << 20, 16), ((1 << 18) - 128, 1 << 20, 16), ((1 << 31) - 1, 1, 16),
                                   ((1 << 27) - 5, 256, 16), ((1 << 27) + 5, 200, 16), ((1 << 22) - 300, 8000, 16)])
def test_the_limit_of_a_launch(rules, M, N, K):
    """less than 2^23 tiles of 128 x 256 results, whatever form a size takes"""
    fits = -(-M // 128) * -(-N // 256) < 1 << 23
    assert (rules.c_waves(rules.c_form(M, N, K), M, N, 0) < 1 << 26) == fits
