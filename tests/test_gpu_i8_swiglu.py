# SPDX-License-Identifier: Apache-2.0
"""SwiGLU rows to int8 on the GPU where fp32 alone would go wrong, against the
64-bit form: codes equal, scales one rounding off at most."""
import pytest
import torch

from test_gpu_i8 import DEV, TYPES, check_rows, gen, swiglu64, swiglu_quant

pytestmark = pytest.mark.gpu

# gates whose silu leaves fp32's normal range, with up values that make it count
LOST = [(-89.0, 1e37), (-87.5, 1e37), (-90.0, 1e37), (-95.0, 1e37), (-100.0, 2.0 ** 110), (1e-40, 1e38),
        (4.2e-45, 1e38), (3 * 2.0 ** -149, 2.0 ** 100), (-3e-39, -2e30)]


def rows_around(dtype, n, k, odd, ratio, seed):
    """n ordinary rows whose largest value is `ratio` times that of the odd
    element (g, u), which each row holds somewhere"""
    g, u = (torch.randn(n, k, device=DEV, generator=gen(seed + i)).to(dtype) for i in range(2))
    go, uo = (torch.tensor([[v]], dtype=torch.float64, device=DEV).to(dtype) for v in odd)
    size = float(swiglu64(go, uo, 0.0).abs())
    u = (u.double() * (ratio * size / swiglu64(g, u, 0.0).abs().amax(1, keepdim=True))).to(dtype)
    at = torch.arange(n, device=DEV) * 37 % k
    g[torch.arange(n), at], u[torch.arange(n), at] = go[0, 0], uo[0, 0]
    return g, u


@pytest.mark.parametrize("odd", LOST)
@pytest.mark.parametrize("ratio", [0.2, 5.0])
@pytest.mark.parametrize("limit", [0.0, 3e38])
def test_values_that_fp32_loses(lib, odd, ratio, limit):
    """One in each row, the row's largest value or an ordinary one."""
    for dtype in (torch.float32, torch.bfloat16):
        if dtype == torch.bfloat16 and 0 < odd[0] < 2.0 ** -133:
            continue                               # bf16 has no such gate
        for n, k in ((5, 64), (3, 528), (2, 4096), (1, 8208)):
            g, u = rows_around(dtype, n, k, odd, ratio, n + k)
            check_rows(*swiglu_quant(lib, g, u, limit), swiglu64(g, u, limit))


@pytest.mark.parametrize("limit", [10.0, 2.0 ** 32, 2.0 ** 33])
def test_a_clamp_bounds_what_fp32_loses(lib, limit):
    for dtype in (torch.float32, torch.bfloat16):
        for odd in LOST:
            g, u = rows_around(dtype, 4, 528, (odd[0], 1.0), 1.0, 9)
            g[:, 5:9], u[:, 5:9] = odd[0], odd[1]
            u[:, 20] = 1.0 / 128                   # beside the clamped values, ordinary ones
            check_rows(*swiglu_quant(lib, g, u, limit), swiglu64(g, u, limit))


@pytest.mark.parametrize("limit", [0.0, 10.0])
@pytest.mark.parametrize("gate", [-88.5, -90.5, -92.5, -95.0, -1000.0, -65504.0])
def test_a_very_negative_gate_among_ordinary_ones(lib, gate, limit):
    """Its value is 0 beside the others', which keep their codes."""
    for dtype in TYPES:
        for n, k in ((5, 64), (300, 2048), (2, 8208)):
            g, u = (torch.randn(n, k, device=DEV, generator=gen(n + i)).to(dtype) for i in range(2))
            g[torch.arange(n), torch.arange(n, device=DEV) * 37 % k] = gate
            check_rows(*swiglu_quant(lib, g, u, limit), swiglu64(g, u, limit))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("limit", [0.0, 10.0])
@pytest.mark.parametrize("k", [16400, 20000, 33024])
def test_rows_that_are_read_again(lib, dtype, limit, k):
    """Rows that no workgroup holds at once: the largest value in any pass, rows
    in fp64, rows of zeros and with a value that is not finite."""
    g, u = (torch.randn(9, k, device=DEV, generator=gen(k + i)).to(dtype) for i in range(2))
    for r, at in ((1, 3), (2, 16390), (3, k - 1)):
        g[r, at], u[r, at] = 9.0, -9.5             # the row's largest
    u[4] = u[4].double().mul(1e-30).to(dtype)      # below what fp32 serves
    g[5], u[6] = 0.0, 0.0
    g[7, k - 5] = float("nan")
    g[8, 16384::7] = -95.0
    q, s = swiglu_quant(lib, g, u, limit)
    check_rows(q, s, swiglu64(g, u, limit))
    assert torch.isnan(s[7]) and (q[7] == 0).all()
