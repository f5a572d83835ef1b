# SPDX-License-Identifier: Apache-2.0
"""The router's score without branches (csrc/dsv4_route_math.h, route_orig_most)
against the branching one, which is pinned to the host's libm: the same bits
wherever it does not call its input rare, and rare inputs lie between expf's
underflow and -20 alone. Every fp32 input near the borders and near 0, elsewhere
every 13th, and the specials."""
import os
import subprocess

from conftest import PKG_DIR

SRC = r"""
#include "dsv4_route_math.h"
#include <cstdio>
#include <initializer_list>
using namespace dsv4_route;
static long bad = 0, rare = 0, wrong = 0, seen = 0;
static void one(uint32_t u)
{
    const float x = fof(u);
    bool r = false;
    const float a = route_orig_most(x, r);
    seen++;
    rare += r;
    if (r) wrong += !(x < -20.0f && x >= -0x1.9fe368p6f);
    else bad += fbits(a) != fbits(route_orig(x));
}
static void range(float lo, float hi, uint32_t step)       /* of one sign, by magnitude */
{
    for (uint32_t u = fbits(lo); u <= fbits(hi); u += step) one(u);
}
int main()
{
    range(0.0f, 20.5f, 13);
    range(-0.0f, -110.0f, 13);
    const float at[] = {-0.8813736f, 20.0f, -20.0f, -0x1.9fe368p6f, -87.5f, 1.0986123f, 1.9459101f, 9.7e-7f, 1e-6f, -1e-6f};
    for (float x : at) {
        const uint32_t u = fbits(x);
        for (uint32_t v = u - 300000; v < u + 300000; v++) one(v);
    }
    for (float x : {0.0f, -0.0f, 1e30f, -1e30f, 3.4028235e38f, -3.4028235e38f, -INFINITY, INFINITY}) one(fbits(x));
    printf("%ld %ld %d %d\n", bad, wrong, seen > 100000000, rare > 1000000);
}
"""


def test_the_same_bits(tmp_path):
    src, exe = tmp_path / "flat.cpp", tmp_path / "flat"
    src.write_text(SRC)
    flags = ["-mfma"] if " fma " in open("/proc/cpuinfo").read() else []
    subprocess.run(["g++", "-O2", "-std=c++17", "-ffp-contract=off", *flags, "-I", os.path.join(PKG_DIR, "csrc"),
                    str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=600).stdout.split()
    assert out == ["0", "0", "1", "1"]
