# SPDX-License-Identifier: Apache-2.0
"""The rules that pick a 4-bit product's form by its sizes (csrc/dsv4_choose.h),
compiled for the host: the launches cover what they have to, and the GPU tests of
the products reach every form."""
import ctypes as C
import os
import subprocess

import pytest

import test_gpu_mxfp4
from conftest import PKG_DIR

SHIM = """
#include "dsv4_choose.h"
using namespace dsv4;
extern "C" {
int c_form(int M, int N, int K) { return fp4_form(M, N, K); }
int c_grouped(int M, int N, int K, int ne) { return fp4_grouped_form(M, N, K, ne); }
long c_waves(int form, long M, long N, long ne) { return fp4_waves((Fp4Form)form, M, N, ne); }
int c_stream(int M, int N, int K, int ne) { return fp4_stream(M, N, K, ne); }
int c_shape(int form, int what)
{
    const Fp4Shape s = fp4_shape((Fp4Form)form);
    return what == 0 ? s.F : what == 1 ? s.TR : s.waves;
}
int c_last() { return FP4_256x256; }
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("fp4")
    src, so = d / "shim.cpp", d / "shim.so"
    src.write_text(SHIM)
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-I",
                    os.path.join(PKG_DIR, "csrc"), str(src), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    lib.c_waves.argtypes, lib.c_waves.restype = [C.c_int, C.c_long, C.c_long, C.c_long], C.c_long
    return lib


def test_gpu_tests_reach_every_form(rules):
    """each with rows, features and K that end inside a tile"""
    every = {rules.c_form(M, N, K) for N in (100, 1024, 4096, 32768) for K in (256, 1024, 4096)
             for M in (1, 8, 30, 100, 333, 700, 1500, 2803, 4096, 8192)}
    ragged = set()
    for M, N, K in test_gpu_mxfp4.SHAPES:
        f = rules.c_form(M, N, K)
        if M % rules.c_shape(f, 1) and N % rules.c_shape(f, 0) and K % 256:
            ragged.add(f)
    assert {rules.c_form(*s) for s in test_gpu_mxfp4.SHAPES} == ragged == every and len(every) == 10


def test_gpu_tests_reach_every_form_of_the_experts_product(rules):
    """and each with weights that go past the caches"""
    def of(M, N, K, E):
        return rules.c_grouped(M, N, K, E), rules.c_stream(M, N, K, E)
    forms = {of(sum(c) + 5, N, K, len(c)) for c, N, K in test_gpu_mxfp4.GROUPS + test_gpu_mxfp4.STREAMS}
    assert forms == {of(M, N, K, E) for E in (1, 8, 64, 256) for N in (64, 512, 2048, 4096) for K in (512, 1024, 4096)
                     for M in range(1, 300 * E, 1 + E // 2)}


@pytest.mark.parametrize("ne", [0, 7])
def test_waves_of_a_launch(rules, ne):
    """A tile for every F features and TR rows, one more row tile for each expert;
    rows and features of 2^31 - 1 do not wrap."""
    for form in range(1, rules.c_last() + 1):
        F, TR, waves = (rules.c_shape(form, i) for i in range(3))
        for M, N in ((1, 1), (TR, F), (TR + 1, F + 1), (1000, 777), ((1 << 31) - 1, (1 << 31) - 1)):
            rows = M // TR + min(M, ne) if ne else -(-M // TR)
            assert rules.c_waves(form, M, N, ne) == rows * -(-N // F) * waves


@pytest.mark.parametrize("counts", [[0, 0, 5], [1] * 300, [127, 129, 0, 31, 33], [2000], [257, 255, 1, 1]])
def test_waves_hold_every_bucket(rules, counts):
    for form in range(1, rules.c_last() + 1):
        F, TR, waves = (rules.c_shape(form, i) for i in range(3))
        tiles = sum(-(-c // TR) for c in counts)
        assert rules.c_waves(form, sum(counts), 100, len(counts)) >= tiles * -(-100 // F) * waves


@pytest.mark.parametrize("M,N,K", [(1 << 30, 128, 32), (1 << 27, 128, 4096), ((1 << 30) - 128, 64, 32), (1 << 26, 2048, 64),
                                   ((1 << 26) - 128, 2048, 64), ((1 << 31) - 1, 1, 32), (9, (1 << 31) - 1, 32),
                                   ((1 << 22) - 300, 8000, 32), (1, 1 << 26, 32), (8, 1 << 25, 64)])
def test_the_limit_of_a_launch(rules, M, N, K):
    """what covers less than 2^23 tiles of 128 x 128 results is taken, whatever form its size takes"""
    if -(-M // 128) * -(-N // 128) < 1 << 23:
        assert rules.c_waves(rules.c_form(M, N, K), M, N, 0) < 1 << 26
