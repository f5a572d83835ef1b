# SPDX-License-Identifier: Apache-2.0
"""Where the router's score is 0 (csrc/dsv4_route_math.h, route_orig_zero), which
the gradient of renormalised weights asks: exactly where route_orig is. Every fp32
input from -100 to -110, elsewhere every 997th, and the specials."""
import os
import subprocess

from conftest import PKG_DIR

SRC = r"""
#include "dsv4_route_math.h"
#include <cstdio>
#include <initializer_list>
using namespace dsv4_route;
static long bad = 0, zeros = 0;
static void one(float x)
{
    bad += route_orig_zero(x) != (route_orig(x) == 0.0f);
    zeros += route_orig_zero(x);
}
int main()
{
    for (uint32_t u = fbits(-100.0f); u <= fbits(-110.0f); u++) one(fof(u));
    for (uint64_t u = 0; u <= 0xFFFFFFFFull; u += 997) one(fof((uint32_t)u));
    for (float x : {0.0f, -0.0f, 20.0f, 3.4028235e38f, -3.4028235e38f, INFINITY, -INFINITY, (float)NAN}) one(x);
    printf("%ld %d\n", bad, zeros > 1000000);
}
"""


def test_zero_scores(tmp_path):
    src, exe = tmp_path / "zero.cpp", tmp_path / "zero"
    src.write_text(SRC)
    flags = ["-mfma"] if " fma " in open("/proc/cpuinfo").read() else []
    subprocess.run(["g++", "-O2", "-std=c++17", "-ffp-contract=off", *flags, "-I", os.path.join(PKG_DIR, "csrc"),
                    str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=600).stdout.split() == ["0", "1"]
