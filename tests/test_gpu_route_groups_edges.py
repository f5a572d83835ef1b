# SPDX-License-Identifier: Apache-2.0
"""The router with groups at its edges on the GPU: weights that are constant, tokens
that are refused, experts that are not there.

Bounds as in test_gpu_route_groups.py: what is exactly 0 is compared with 0, a
gradient is an fp64 value with one rounding to the logits' type, and an absolute
part of 2e-11 for what cancels."""
import pytest
import torch

from test_gpu_route_groups import DEV, HALF, SIGMOID, SOFTMAX, SQRT, TINY, TYPES, backward, gen, route, want_grad

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.mark.parametrize("kind", [SQRT, SOFTMAX, SIGMOID])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,E", [(6, 4), (40, 700), (4103, 200)])
def test_constant_weights_have_no_gradient(lib, pkg, kind, dtype, n, E):
    """Where every chosen score is 0 the weights are 0 whatever the logits: exactly no gradient.
    sqrt(softplus) of fp32 is 0 from -104 down, its exact value e^(x / 2) only from -207 down."""
    x = -104.0 - 100.0 * torch.rand(n, E, device=DEV, generator=gen(n + E))
    x[0] = torch.arange(E, device=DEV) - (119.0 + E)
    x[2, 1:] = -INF
    x[3] = -INF
    x[4] = torch.linspace(-300.0, -1000.0, E, device=DEV)
    x[5::2] += 110.0                               # scores that are not 0
    x = x.to(dtype)
    dw = torch.randn(n, 3, device=DEV, generator=gen(2))
    r = pkg.Router(kind, E, 3, 1, 1, 1, 1, 2.5)
    lib.status()
    idx, w, _ = route(lib, r, x)
    got = backward(lib, r, x, idx, dw)
    assert lib.status() == 0
    none = (w == 0).all(1)
    # softmax: a token's largest score is 1 / (experts near it) or more, so only one without experts has none
    zeros = torch.ones(n, dtype=torch.bool, device=DEV)
    zeros[5::2] = False
    if kind == SOFTMAX:
        zeros[:] = False
        zeros[3] = True
    assert torch.equal(none, zeros)
    assert (got[none] == 0).all()
    want = want_grad(r, x[~none], idx[~none], dw[~none], None)
    # an id of -1 in a row of -inf differentiates to NaN beside it
    want = torch.where(x[~none] > -INF, want, 0.0)
    assert ((got[~none].double() - want).abs() <= 1.001 * HALF[dtype] * want.abs() + 1e-12 * 20 + TINY[dtype]).all()
    assert (got[~none] != 0).any()


@pytest.mark.parametrize("kind", [SQRT, SOFTMAX, SIGMOID])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("renorm", [0, 1])
@pytest.mark.parametrize("n,E", [(9, 70), (8205, 200), (21, 600)])
def test_refused_tokens_have_no_gradient(lib, pkg, kind, dtype, renorm, n, E):
    """A logit of NaN or +inf: ids of -1, gradient 0 whatever comes back for the weights and scores,
    the other tokens' bits those of a batch without it."""
    good = torch.randn(n, E, device=DEV, generator=gen(n + E)).to(dtype)
    bad = torch.tensor([2, 5, n - 1, n - 2], device=DEV)
    x = good.clone()
    x[2, E - 1], x[5, 0], x[n - 1], x[n - 2, 7] = float("nan"), INF, float("nan"), INF
    x[2, 3], x[5, 1:4] = INF, -INF
    others = torch.ones(n, dtype=torch.bool, device=DEV)
    others[bad] = False
    r = pkg.Router(kind, E, 4, 5, 3, 2, renorm, 2.5)
    idx, _, _ = route(lib, r, x)
    i2, _, _ = route(lib, r, good)
    dw, ds = (torch.randn(n, k, device=DEV, generator=gen(k)) for k in (4, E))
    dw[5], ds[2], ds[n - 1] = float("nan"), float("nan"), INF
    dw2, ds2 = dw.clone(), ds.clone()
    dw2[bad], ds2[bad] = 0.0, 0.0
    assert lib.status() == 1
    for d, d2 in ((None, None), (ds, ds2)):
        want = backward(lib, r, good, i2, dw2, d2)
        assert lib.status() == 0
        got = backward(lib, r, x, idx, dw, d)
        # without scores' gradients only softmax reads a token whose ids are -1
        assert lib.status() == (1 if d is not None or kind == SOFTMAX else 0)
        assert (got[bad] == 0).all() and torch.equal(got[others], want[others])
        assert (got[others] != 0).any()


@pytest.mark.parametrize("kind", [SQRT, SOFTMAX, SIGMOID])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,E", [(9, 70), (8205, 200), (21, 600)])
def test_experts_that_are_not_there_take_no_gradient(lib, pkg, kind, dtype, n, E):
    """What a loss sends to the score of an expert whose logit is -inf (1 / 0 of a logarithm, NaN)
    goes nowhere: gradient 0 for it, for the others the bits of a call with 0 there."""
    x = torch.randn(n, E, device=DEV, generator=gen(n + E)).to(dtype)
    x[torch.rand(n, E, device=DEV, generator=gen(7)) < 0.3] = -INF
    x[4] = -INF
    gone = x == -INF
    r = pkg.Router(kind, E, 4, 1, 1, 1, 1, 2.5)
    idx, _, _ = route(lib, r, x)
    dw, ds = (torch.randn(n, k, device=DEV, generator=gen(k)) for k in (4, E))
    ds[gone] = 0.0
    want = backward(lib, r, x, idx, dw, ds)
    for v in (INF, -INF, float("nan")):
        got = backward(lib, r, x, idx, dw, torch.where(gone, v, ds))
        assert (got[gone] == 0).all() and torch.equal(got, want)
    assert lib.status() == 0 and (want != 0).any()
