# SPDX-License-Identifier: Apache-2.0
"""The router with groups at its edges on the GPU: weights that are constant, tokens
that are refused, experts that are not there, the token counts from which four
tokens share a wave.

Bounds as in test_gpu_route_groups.py: what is exactly 0 is compared with 0, a
gradient is an fp64 value with one rounding to the logits' type, and an absolute
part of 2e-11 for what cancels."""
import pytest
import torch

from test_gpu_route_groups import (DEV, HALF, SIGMOID, SOFTMAX, SQRT, TINY, TYPES, U, backward, check, gen, route, want_grad,
                                   with_masks)

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


# Tokens share a wave, with up to 256 experts, from 3,500 forward, 6,144 with sqrt(softplus); backward from
# 4,096, 8,192 with scores' gradients. Experts: each number of quads a lane.
@pytest.mark.parametrize("kind,n", [(SOFTMAX, 3500), (SIGMOID, 3500), (SQRT, 6144)])
@pytest.mark.parametrize("E,topk,G,kept", [(60, 4, 5, 2), (128, 6, 8, 3), (250, 8, 10, 4)])
def test_one_token_less_than_share_a_wave(lib, pkg, kind, n, E, topk, G, kept):
    """Both sides by the definition, and alike. Softmax adds up in another order: fp64 sums of 250
    terms, 2^-44 of them, so a score may round to the other side, a step of 2^-23, and a weight,
    a quotient of two sums of scores, to three of them."""
    x = with_masks(1.5 * torch.randn(n, E, device=DEV, generator=gen(n + E)))
    bias = 0.1 * torch.randn(E, device=DEV, generator=gen(3))
    r = pkg.Router(kind, E, topk, G, kept, 2, 1, 2.5)
    lib.status()
    check(lib, r, x, bias)
    check(lib, r, x[:-1], bias)
    more, less = route(lib, r, x, bias), route(lib, r, x[:-1], bias)
    assert lib.status() == 0 and torch.equal(more[0][:-1], less[0])
    for a, b, steps in ((more[1][:-1], less[1], 3), (more[2][:-1], less[2], 1)):
        if kind == SOFTMAX:
            assert ((a - b).abs() <= steps * 2 * U * b + 2.0 ** -149).all()
        else:
            assert torch.equal(a, b)


@pytest.mark.parametrize("kind", [SQRT, SOFTMAX, SIGMOID])
@pytest.mark.parametrize("scores,n", [(False, 4096), (True, 8192)])
@pytest.mark.parametrize("E,topk", [(60, 4), (128, 6), (250, 8)])
def test_gradients_of_one_token_less_than_share_a_wave(lib, pkg, kind, scores, n, E, topk):
    """As above; softmax: 1e-12 of what adds up, and the rounding to fp32 may fall to the other side."""
    x = 1.5 * torch.randn(n, E, device=DEV, generator=gen(n + E))
    dw = torch.randn(n, topk, device=DEV, generator=gen(2))
    ds = torch.randn(n, E, device=DEV, generator=gen(5)) if scores else None
    for renorm in (0, 1):
        r = pkg.Router(kind, E, topk, 1, 1, 1, renorm, 2.5)
        idx, _, _ = route(lib, r, x)
        more = backward(lib, r, x, idx, dw, ds)
        less = backward(lib, r, x[:-1], idx[:-1], dw[:-1], ds[:-1] if scores else None)
        want = want_grad(r, x, idx, dw, ds)
        assert ((more.double() - want).abs() <= 1.001 * HALF[torch.float32] * want.abs() + 1e-12 * 20 + 2.0 ** -149).all()
        if kind == SOFTMAX:
            assert ((more[:-1].double() - less.double()).abs() <= 1e-12 * 20 + 2 * U * less.abs()).all()
        else:
            assert torch.equal(more[:-1], less)
