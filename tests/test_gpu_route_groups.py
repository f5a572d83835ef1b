# SPDX-License-Identifier: Apache-2.0
"""The router with groups on the GPU against its definition in 64 bits.

Bounds. u = 2^-24 is fp32's half step. A score is an fp64 value rounded once (u,
and fp64's own error, far below). The choice is made from fp32 scores and one fp32
addition: equal, ties included. A weight is scale s / sum of fp32 scores in fp64,
rounded once: against unrounded scores (1 + u)^3 - 1 < 3.01 u. Gradients are fp64
with one rounding to the logits' type: its half step, and an absolute part for
what cancels (1e-12 of the largest term)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}
SQRT, SOFTMAX, SIGMOID = 0, 1, 2
INF = float("inf")


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def scores64(x, kind):
    x = x.double()
    if kind == SIGMOID:
        return 1 / (1 + torch.exp(-x))
    if kind == SQRT:
        return torch.where(x > 20, x.clamp(min=1e-300), torch.log1p(torch.exp(x.clamp(max=20)))).sqrt()
    m = x.amax(-1, keepdim=True)
    p = torch.where(x > -INF, torch.exp(x - torch.where(m > -INF, m, 0.0)), 0.0)
    t = p.sum(-1, keepdim=True)
    return torch.where(t > 0, p / torch.where(t > 0, t, 1.0), 0.0)


def choose(score, x, bias, r):
    """ids by the definition, from fp32 scores, one token at a time on the host"""
    score, x = score.cpu().numpy().astype(np.float32), x.float().cpu().numpy()
    n, E = score.shape
    b = np.zeros(E, np.float32) if bias is None else bias.cpu().numpy()
    with np.errstate(invalid="ignore"):
        c = (score + b[None]).astype(np.float32)
    there = (x > -np.inf) & (c > -np.inf)
    G, per = r.n_group, E // r.n_group
    ids = np.full((n, r.topk), -1, np.int64)
    for t in range(n):
        if not (x[t] < np.inf).all():
            continue
        live = there[t].copy()
        if r.topk_group < G:
            worth = np.full(G, -np.inf, np.float32)
            for g in range(G):
                v = np.sort(c[t, g * per:(g + 1) * per][live[g * per:(g + 1) * per]])[::-1][:r.group_top]
                if v.size:
                    worth[g] = v[0] if v.size == 1 else np.float32(v[0] + v[1])
            for g in np.argsort(-worth.astype(np.float64), kind="stable")[r.topk_group:]:
                live[g * per:(g + 1) * per] = False
        at = np.nonzero(live)[0]
        at = at[np.argsort(-c[t, at].astype(np.float64), kind="stable")][:r.topk]
        ids[t, :at.size] = at
    return torch.from_numpy(ids).to(DEV)


def weights64(s, ids, r):
    got = torch.where(ids >= 0, s.gather(1, ids.clamp(min=0)), 0.0)
    if not r.renorm:
        return r.scale * got
    t = got.sum(-1, keepdim=True)
    return torch.where(t > 0, r.scale * got / torch.where(t > 0, t, 1.0), 0.0)


def route(lib, r, x, bias=None, scores=True, stream=None):
    n, E = x.shape
    idx = torch.full((n + 1, r.topk), 55, dtype=torch.int32, device=DEV)
    w = torch.full((n + 1, r.topk), 55.0, device=DEV)
    s = torch.full((n + 1, E), 55.0, device=DEV) if scores else None
    lib.route_groups_dev(idx.data_ptr(), w.data_ptr(), s.data_ptr() if scores else None, x.data_ptr(), CODE[x.dtype], n,
                         bias.data_ptr() if bias is not None else None, r, stream)
    torch.cuda.synchronize()
    assert (idx[n] == 55).all() and (w[n] == 55).all() and (not scores or (s[n] == 55).all())
    return idx[:n], w[:n], s[:n] if scores else None


def check(lib, r, x, bias=None):
    s64 = scores64(x, r.score)
    idx, w, s = route(lib, r, x, bias)
    if r.score == SQRT:
        # the router's own bits, one step from the rounded value. Its softplus is an fp32 value: below
        # fp32's normal range it is off by up to two of the smallest steps, 2^-148, and so a square root
        # by up to 2^-74 (|sqrt p - sqrt q| <= sqrt |p - q|)
        assert ((s.double() - s64).abs() <= 2 * U * s64 + 2.0 ** -74).all()
        ids = choose(s, x, bias, r)
    else:
        assert ((s.double() - s64).abs() <= 1.001 * U * s64 + 2.0 ** -150).all()
        ids = choose(s64.float(), x, bias, r)
    assert torch.equal(idx.long(), ids)
    want = weights64(s64, ids, r)
    wide = s64.gather(1, ids.clamp(min=0)).clamp(max=1.0)
    fine = (wide > 1e-30) | (ids < 0)              # scores that fp32 holds to 24 bits
    far = (w.double() - want).abs() <= (7 if r.score == SQRT else 3.01) * U * want + 2.0 ** -149
    assert (far | ~fine.all(1, keepdim=True)).all()
    i2, w2, _ = route(lib, r, x, bias, scores=False)
    assert torch.equal(i2, idx) and torch.equal(w2, w)


CASES = [  # n, experts, topk, groups, kept, top
    (1, 1, 1, 1, 1, 1), (5, 7, 3, 1, 1, 1), (3, 64, 6, 8, 3, 2), (1, 256, 6, 8, 4, 2), (67, 256, 8, 8, 4, 2),
    (33, 160, 6, 8, 3, 1), (9, 100, 16, 5, 2, 2), (4, 1024, 16, 64, 7, 2), (130, 257, 4, 1, 1, 1), (3, 90, 5, 45, 44, 1),
    (20, 512, 8, 2, 1, 2), (7, 1000, 10, 8, 8, 2), (12, 13, 13, 13, 13, 1), (2, 63, 9, 7, 1, 2)]


@pytest.mark.parametrize("kind", [SQRT, SOFTMAX, SIGMOID])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,E,topk,G,kept,top", CASES)
def test_routing(lib, pkg, kind, dtype, n, E, topk, G, kept, top):
    x = (1.5 * torch.randn(n, E, device=DEV, generator=gen(n + E))).to(dtype)
    bias = 0.1 * torch.randn(E, device=DEV, generator=gen(3))
    for renorm, b in ((1, bias), (0, bias), (1, None)):
        check(lib, pkg.Router(kind, E, topk, G, kept, top, renorm, 2.5), x, b)


# tokens that share a wave: 6,144 do, 16,384 with sqrt(softplus) and 8,244 backward, of up to 256 experts
MANY = [(6147, 60, 4, 5, 2, 2), (6145, 128, 6, 8, 3, 1), (6149, 256, 8, 8, 4, 2), (6146, 160, 16, 32, 9, 2),
        (6144, 250, 5, 1, 1, 1), (6150, 64, 8, 64, 20, 1), (6151, 3, 2, 1, 1, 1), (6148, 200, 12, 10, 6, 2),
        (6153, 256, 16, 1, 1, 1)]


def with_masks(x):
    """in every fourth token some experts, in some all but one, in some all are not there"""
    x[1::4][torch.rand(x[1::4].shape, device=DEV, generator=gen(7)) < 0.7] = -INF
    x[5::64, 1:] = -INF
    x[7::64] = -INF
    x[9::64] = torch.finfo(x.dtype).min
    return x


@pytest.mark.parametrize("kind", [SQRT, SOFTMAX, SIGMOID])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,E,topk,G,kept,top", MANY)
def test_routing_many(lib, pkg, kind, dtype, n, E, topk, G, kept, top):
    n += (16384 - 6144) * (kind == SQRT)
    x = with_masks((1.5 * torch.randn(n, E, device=DEV, generator=gen(n + E))).to(dtype))
    bias = 0.1 * torch.randn(E, device=DEV, generator=gen(3))
    lib.status()
    check(lib, pkg.Router(kind, E, topk, G, kept, top, 1, 2.5), x, bias)
    assert lib.status() == 0


@pytest.mark.parametrize("kind", [SOFTMAX, SIGMOID])
def test_ties_of_many(lib, pkg, kind):
    x = torch.randint(-1, 2, (6200, 256), device=DEV, generator=gen(1)).float()
    check(lib, pkg.Router(kind, 256, 8, 8, 3, 2, 1, 1.0), x)
    x = torch.randint(17, 40, (6200, 96), device=DEV, generator=gen(2)).float()
    check(lib, pkg.Router(kind, 96, 8, 6, 2, 1, 0, 1.0), x)


@pytest.mark.parametrize("kind", [SQRT, SOFTMAX, SIGMOID])
def test_refused_among_many(lib, pkg, kind):
    """The same bits for a token in a small call and among many; refusals stay with their tokens."""
    n = 16390 if kind == SQRT else 6150
    x = torch.randn(n, 200, device=DEV, generator=gen(1))
    x[3, 199], x[n - 1, 0], x[n - 2, 77] = float("nan"), INF, float("nan")
    r = pkg.Router(kind, 200, 5, 10, 3, 2, 1, 1.0)
    lib.status()
    many = route(lib, r, x)
    assert lib.status() == 1
    few = route(lib, r, x[-50:].contiguous())
    lib.status()
    for a, b in zip(many, few):
        assert torch.equal(a[-50:].contiguous().view(torch.int32), b.contiguous().view(torch.int32))
    for t in (3, n - 1, n - 2):
        assert (many[0][t] == -1).all() and torch.isnan(many[1][t]).all() and torch.isnan(many[2][t]).all()
    assert (many[0][[0, 1, 2, 4, 5, n - 3]] >= 0).all()


@pytest.mark.parametrize("kind", [SOFTMAX, SIGMOID])
def test_ties_go_to_the_lower_id(lib, pkg, kind):
    """Few distinct logits: experts and groups of equal worth; sigmoids that round to 1."""
    for E, G, kept, top in ((256, 8, 3, 2), (96, 6, 2, 1), (512, 1, 1, 1)):
        for lo, hi in ((-1, 2), (17, 40)):
            x = torch.randint(lo, hi, (50, E), device=DEV, generator=gen(E)).float()
            check(lib, pkg.Router(kind, E, 8, G, kept, top, 1, 1.0), x)
            check(lib, pkg.Router(kind, E, 8, G, kept, top, 1, 1.0), x, torch.zeros(E, device=DEV))


@pytest.mark.parametrize("kind", [SQRT, SOFTMAX, SIGMOID])
def test_experts_that_are_not_there(lib, pkg, kind):
    """Logits of -inf, biases of -inf and NaN, rows that leave fewer than topk, one or none."""
    E = 128
    x = torch.randn(40, E, device=DEV, generator=gen(1))
    x[torch.rand(40, E, device=DEV, generator=gen(2)) < 0.5] = -INF
    x[3] = -INF
    x[4] = -INF
    x[4, 77] = 0.5
    x[5, 5:] = -INF
    x[6] = -INF
    x[6, ::40] = -3.0e38
    x[7] = torch.finfo(torch.float32).min
    x[8] = -200.0
    bias = 0.1 * torch.randn(E, device=DEV, generator=gen(3))
    bias[9], bias[10] = -INF, float("nan")
    lib.status()
    for G, kept, top in ((1, 1, 1), (8, 2, 2), (16, 15, 1)):
        for b in (None, bias):
            for renorm in (0, 1):
                r = pkg.Router(kind, E, 6, G, kept, top, renorm, 1.5)
                check(lib, r, x, b)
                idx, w, s = route(lib, r, x, b)
                assert (idx[3] == -1).all() and (w[3] == 0).all() and (s[3] == 0).all()
                assert idx[4, 0] == 77 and (idx[4, 1:] == -1).all()
                assert torch.isfinite(w).all()
    assert lib.status() == 0


@pytest.mark.parametrize("kind", [SQRT, SOFTMAX, SIGMOID])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_are_refused(lib, pkg, kind, dtype):
    x = torch.randn(9, 70, device=DEV, generator=gen(1)).to(dtype)
    x[2, 69] = float("nan")
    x[5, 0] = INF
    good = [0, 1, 3, 4, 6, 7, 8]
    r = pkg.Router(kind, 70, 5, 7, 3, 2, 1, 1.0)
    lib.status()
    idx, w, s = route(lib, r, x)
    assert lib.status() == 1
    i2, w2, s2 = route(lib, r, x[good].contiguous())
    assert lib.status() == 0
    assert torch.equal(idx[good], i2) and torch.equal(w[good], w2) and torch.equal(s[good], s2)
    for t in (2, 5):
        assert (idx[t] == -1).all() and torch.isnan(w[t]).all() and torch.isnan(s[t]).all()


def test_the_same_bits_as_the_router_without_groups(lib, pkg):
    n, E, k = 300, 256, 6
    x = 3 * torch.randn(n, E, device=DEV, generator=gen(8))
    bias = 0.3 * torch.randn(E, device=DEV, generator=gen(9))
    idx, w, s = route(lib, pkg.Router(SQRT, E, k, 1, 1, 1, 1, 1.5), x, bias)
    i2, w2, s2 = torch.zeros_like(idx), torch.zeros_like(w), torch.zeros_like(s)
    lib.route_dev(i2.data_ptr(), w2.data_ptr(), s2.data_ptr(), x.data_ptr(), n, E, k, 1.5, bias.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(idx, i2) and torch.equal(s, s2)
    assert ((w - w2).abs() <= 4 * U * w).all()


# --------------------------------------------------------------- gradients ----

def backward(lib, r, x, idx, dw, ds=None):
    n, E = x.shape
    dx = torch.full((n + 1, E), 55.0, dtype=x.dtype, device=DEV)
    lib.route_groups_bwd_dev(dx.data_ptr(), dw.data_ptr(), ds.data_ptr() if ds is not None else None, x.data_ptr(),
                             CODE[x.dtype], idx.data_ptr(), n, r)
    torch.cuda.synchronize()
    assert (dx[n] == 55).all()
    return dx[:n]


def want_grad(r, x, idx, dw, ds):
    """by differentiation of the definition in fp64"""
    v = x.double().clone().requires_grad_(True)
    if r.score == SOFTMAX:
        s = torch.softmax(v, -1)
    elif r.score == SIGMOID:
        s = torch.sigmoid(v)
    else:
        s = torch.where(v > 20, v, torch.log1p(torch.exp(v.clamp(max=20)))).clamp(min=0).sqrt()
    ids = idx.long()
    got = torch.where(ids >= 0, s.gather(1, ids.clamp(min=0)), 0.0)
    w = r.scale * (got / got.sum(-1, keepdim=True) if r.renorm else got)
    loss = (torch.where(ids >= 0, w, 0.0) * dw.double()).sum()
    if ds is not None:
        loss = loss + (s * ds.double()).sum()
    return torch.autograd.grad(loss, v)[0]


@pytest.mark.parametrize("kind", [SQRT, SOFTMAX, SIGMOID])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,E,topk,G,kept,top", CASES)
def test_gradients(lib, pkg, kind, dtype, n, E, topk, G, kept, top):
    x = (1.5 * torch.randn(n, E, device=DEV, generator=gen(n + E))).to(dtype)
    dw = torch.randn(n, topk, device=DEV, generator=gen(2))
    for renorm in (0, 1):
        r = pkg.Router(kind, E, topk, G, kept, top, renorm, 2.5)
        idx, _, _ = route(lib, r, x)
        for ds in (None, torch.randn(n, E, device=DEV, generator=gen(5))):
            want = want_grad(r, x, idx, dw, ds)
            got = backward(lib, r, x, idx, dw, ds).double()
            assert ((got - want).abs() <= 1.001 * HALF[dtype] * want.abs() + 1e-12 * 20 + TINY[dtype]).all()


@pytest.mark.parametrize("kind", [SQRT, SOFTMAX, SIGMOID])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,E,topk,G,kept,top", MANY)
def test_gradients_of_many(lib, pkg, kind, dtype, n, E, topk, G, kept, top):
    n += 16384 - 6144 if kind == SQRT else 2100
    x = (1.5 * torch.randn(n, E, device=DEV, generator=gen(n + E))).to(dtype)
    dw = torch.randn(n, topk, device=DEV, generator=gen(2))
    ds = torch.randn(n, E, device=DEV, generator=gen(5))
    for renorm, d in ((0, ds), (1, None), (1, ds), (0, None)):
        r = pkg.Router(kind, E, topk, G, kept, top, renorm, 2.5)
        idx, _, _ = route(lib, r, x)
        want = want_grad(r, x, idx, dw, d)
        got = backward(lib, r, x, idx, dw, d).double()
        assert ((got - want).abs() <= 1.001 * HALF[dtype] * want.abs() + 1e-12 * 20 + TINY[dtype]).all()


def test_gradients_of_masked_tokens(lib, pkg):
    """Tokens without experts have gradient 0, masked experts too; a token's gradient is the
    same among few and many. Softmax adds up its 96 terms, of at most 30, in fp64 in
    another order there: 2 x 96 x 2^-53 x 30 < 1e-12, and the rounding to fp32 may then
    fall to the other side, 2^-23 of the value."""
    for kind in (SQRT, SOFTMAX, SIGMOID):
        x = with_masks(torch.randn(16390, 96, device=DEV, generator=gen(3)))
        dw, ds = (torch.randn(16390, k, device=DEV, generator=gen(4)) for k in (6, 96))
        r = pkg.Router(kind, 96, 6, 8, 3, 2, 1, 2.5)
        idx, _, _ = route(lib, r, x)
        for d in (None, ds):
            got = backward(lib, r, x, idx, dw, d)
            assert torch.isfinite(got).all() and (got[x == -INF] == 0).all()
            t = slice(16390 - 77, 16390)
            few = backward(lib, r, x[t].contiguous(), idx[t].contiguous(), dw[t].contiguous(), d[t].contiguous() if d is not None else None)
            if kind == SOFTMAX:
                assert ((got[t].double() - few.double()).abs() <= 1e-12 + 2 * U * few.abs()).all()
            else:
                assert torch.equal(got[t], few)


def test_tokens_past_4_gib(lib, pkg):
    """The last tokens of 4.4 GB of logits as by themselves, both ways."""
    n, E = (1 << 22) + 3, 260
    x = torch.empty(n, E, device=DEV)
    x.normal_(generator=gen(1))
    r = pkg.Router(SIGMOID, E, 4, 4, 2, 2, 1, 1.0)
    big, few = route(lib, r, x), route(lib, r, x[-9:].contiguous())
    for a, b in zip(big, few):
        assert torch.equal(a[-9:], b)
    dw = torch.randn(n, 4, device=DEV, generator=gen(2))
    a = backward(lib, r, x, big[0].contiguous(), dw, big[2].contiguous())
    b = backward(lib, r, x[-9:].contiguous(), few[0].contiguous(), dw[-9:].contiguous(), few[2].contiguous())
    assert torch.equal(a[-9:], b)


@pytest.mark.parametrize("kind", [SQRT, SOFTMAX, SIGMOID])
@pytest.mark.parametrize("renorm", [0, 1])
def test_gradients_against_differences(lib, pkg, kind, renorm):
    """Central differences of the fp64 definition at fixed ids, h = 1e-4: off by h^2 / 6
    of a third derivative of at most a few, 1e-7 with what cancels."""
    n, E, topk, h = 3, 12, 4, 1e-4
    x = torch.randn(n, E, device=DEV, generator=gen(4))
    dw = torch.randn(n, topk, device=DEV, generator=gen(5))
    ds = torch.randn(n, E, device=DEV, generator=gen(6))
    r = pkg.Router(kind, E, topk, 3, 2, 2, renorm, 1.5)
    idx, _, _ = route(lib, r, x)

    def loss(v):
        s = scores64(v, kind)
        return (weights64(s, idx.long(), r) * dw.double()).sum(-1) + (s * ds.double()).sum(-1)

    want = torch.zeros(n, E, dtype=torch.float64, device=DEV)
    for e in range(E):
        d = torch.zeros(E, dtype=torch.float64, device=DEV)
        d[e] = h
        want[:, e] = (loss(x.double() + d) - loss(x.double() - d)) / (2 * h)
    assert ((backward(lib, r, x, idx, dw, ds).double() - want).abs() <= 1e-6).all()


def test_gradients_of_ids_that_are_not_there(lib, pkg):
    """-1 adds nothing and is no fault, others out of range raise bit 0; an id twice adds twice."""
    n, E = 4, 100
    x = torch.randn(n, E, device=DEV, generator=gen(4))
    x[3] = -INF
    dw = torch.randn(n, 3, device=DEV, generator=gen(5))
    idx = torch.tensor([[5, -1, 99], [-1, -1, -1], [7, 7, 2], [-1, -1, -1]], dtype=torch.int32, device=DEV)
    lib.status()
    for kind in (SQRT, SOFTMAX, SIGMOID):
        for renorm in (0, 1):
            r = pkg.Router(kind, E, 3, 1, 1, 1, renorm, 1.0)
            got = backward(lib, r, x, idx, dw).double()
            want = want_grad(r, x[:3], idx[:3], dw[:3], None).nan_to_num(0.0)
            assert ((got[:3] - want).abs() <= 1.001 * U * want.abs() + 1e-12).all()
            assert (got[1] == 0).all() and (got[3] == 0).all()
    assert lib.status() == 0
    bad = idx.clone()
    bad[0, 1], bad[1, 0] = 100, -7
    a, b = backward(lib, r, x, bad, dw), backward(lib, r, x, idx, dw)
    assert lib.status() == 1 and torch.equal(a, b)


def test_gradients_far_from_zero(lib, pkg):
    """Logits where scores saturate or vanish: finite, and constant weights have none."""
    x = torch.tensor([[-200.0, -150.0, -120.0, -300.0], [200.0, 150.0, 30.0, 21.0], [-1e30, 1e30, 0.0, -5.0],
                      [-800.0, -900.0, -1e38, -2000.0]], device=DEV)
    for kind in (SQRT, SOFTMAX, SIGMOID):
        for renorm in (0, 1):
            r = pkg.Router(kind, 4, 2, 1, 1, 1, renorm, 1.0)
            idx, w, _ = route(lib, r, x)
            got = backward(lib, r, x, idx, torch.ones(4, 2, device=DEV), torch.ones(4, 4, device=DEV))
            assert torch.isfinite(got).all() and torch.isfinite(w).all()


def test_no_tokens(lib, pkg):
    r = pkg.Router(SIGMOID, 8, 2, 1, 1, 1, 1, 1.0)
    lib.route_groups_dev(None, None, None, None, 0, 0, None, r)
    lib.route_groups_bwd_dev(None, None, None, None, 0, None, 0, r)


@pytest.mark.parametrize("kind", [SQRT, SOFTMAX, SIGMOID])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [5, 8203, 16391])
def test_gradients_in_place(lib, pkg, kind, dtype, n):
    """Over the logits, and over the scores' gradients, the bits of a call of its own."""
    x = with_masks((1.5 * torch.randn(n, 70, device=DEV, generator=gen(n))).to(dtype))
    dw, ds = (torch.randn(n, k, device=DEV, generator=gen(k)) for k in (6, 70))
    r = pkg.Router(kind, 70, 6, 7, 4, 2, 1, 2.5)
    idx, _, _ = route(lib, r, x)
    want = backward(lib, r, x, idx, dw, ds)
    y = x.clone()
    lib.route_groups_bwd_dev(y.data_ptr(), dw.data_ptr(), ds.data_ptr(), y.data_ptr(), CODE[dtype], idx.data_ptr(), n, r)
    assert torch.equal(y, want)
    if dtype == torch.float32:
        lib.route_groups_bwd_dev(ds.data_ptr(), dw.data_ptr(), ds.data_ptr(), x.data_ptr(), 0, idx.data_ptr(), n, r)
        assert torch.equal(ds, want)


@pytest.mark.parametrize("E", [3, 300])
def test_most_tokens(lib, pkg, E):
    """2^26 - 4 tokens, a wave's worth for three experts, past four waves a workgroup for 300."""
    n = (1 << 26) - 4
    x = torch.empty(n, E, dtype=torch.bfloat16, device=DEV).normal_(generator=gen(E))
    r = pkg.Router(SIGMOID, E, 1, 1, 1, 1, 0, 1.0)
    idx, w, _ = route(lib, r, x, scores=False)
    few, w2, _ = route(lib, r, x[-9:].contiguous(), scores=False)
    assert torch.equal(idx[-9:], few) and torch.equal(w[-9:], w2)
    assert (idx[:: 1 << 20] >= 0).all()
    dw = torch.ones(n, 1, device=DEV)
    dx = backward(lib, r, x, idx.contiguous(), dw)
    assert torch.equal(dx[-9:], backward(lib, r, x[-9:].contiguous(), few.contiguous(), dw[-9:].contiguous()))
    assert lib.status() == 0
