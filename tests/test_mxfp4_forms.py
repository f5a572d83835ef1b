# SPDX-License-Identifier: Apache-2.0
"""The GPU tests of far tokens and of bad tables, tokens and offsets
(test_gpu_mxfp4_forms.py) run every form of the 4-bit experts' product, through
the caches and past them."""
import pytest

import test_gpu_mxfp4_forms
from test_mxfp4_choice import rules  # noqa: F401


def of(rules, M, N, K, E):
    return rules.c_grouped(M, N, K, E), rules.c_stream(M, N, K, E)


@pytest.mark.parametrize("cases", [test_gpu_mxfp4_forms.FAR, test_gpu_mxfp4_forms.BAD])
def test_every_form(rules, cases):  # noqa: F811
    every = {of(rules, M, N, K, E) for E in (1, 8, 64, 256) for N in (64, 512, 2048, 4096) for K in (512, 1024, 4096, 8192)
             for M in range(1, 300 * E, 1 + E // 2)}
    assert {of(rules, sum(c), N, K, len(c)) for c, N, K in cases} == every


def test_far_tokens(rules):  # noqa: F811
    """the last token's codes end within a row of the last byte that an offset reaches"""
    for _, _, K in test_gpu_mxfp4_forms.FAR:
        n_a = (2 ** 32 - 1) // K
        assert 2 ** 31 - K < n_a * (K // 2) < 2 ** 31
