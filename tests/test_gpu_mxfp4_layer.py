# SPDX-License-Identifier: Apache-2.0
"""A routed expert layer in 4 bits as a program runs it: router with groups, tokens
in expert order, 4-bit rows, the experts' products, the weighted way back, and the
gradients of the way back, the router and the order. One by one against plain forms
of each call's own inputs; on several streams at once and captured, the bits of the
calls made one by one."""
import numpy as np
import pytest
import torch

from test_gpu_mxfp4 import DEV, U, gen, operand, table_of, values, want_codes
from test_gpu_route_groups import choose, scores64, want_grad, weights64

pytestmark = pytest.mark.gpu

E, TOPK, H, INTER, LIMIT = 24, 4, 512, 256, 10.0


class Layer:
    """One caller's buffers; the weights are shared between callers."""

    def __init__(self, lib, pkg, n, weights, kind=2):
        R, i32 = n * TOPK, dict(dtype=torch.int32, device=DEV)
        bf = dict(dtype=torch.bfloat16, device=DEV)
        u8 = dict(dtype=torch.uint8, device=DEV)
        self.lib, self.n, self.R, self.tables = lib, n, R, [table_of(pkg, w, s) for w, s in weights]
        self.r = pkg.Router(kind, E, TOPK, 6, 3, 2, 1, 2.5)
        self.x, self.dout, self.logits = torch.zeros(n, H, **bf), torch.zeros(n, H, **bf), torch.zeros(n, E, **bf)
        self.bias = 0.05 * torch.randn(E, device=DEV, generator=gen(99))
        self.idx, self.w, self.scores = torch.zeros(n, TOPK, **i32), torch.zeros(n, TOPK, device=DEV), torch.zeros(n, E, device=DEV)
        self.off, self.tok, self.pos = torch.zeros(E + 1, **i32), torch.zeros(R, **i32), torch.zeros(n, TOPK, **i32)
        self.rows, self.y, self.drows = (torch.zeros(R, H, **bf) for _ in range(3))
        self.gate, self.up = torch.zeros(R, INTER, **bf), torch.zeros(R, INTER, **bf)
        self.xq, self.xs = torch.zeros(n, H // 2, **u8), torch.zeros(n, H // 32, **u8)
        self.mq, self.ms = torch.zeros(R, INTER // 2, **u8), torch.zeros(R, INTER // 32, **u8)
        self.out, self.dx, self.dw = torch.zeros(n, H, **bf), torch.zeros(n, H, **bf), torch.zeros(n, TOPK, device=DEV)
        self.ds, self.dlogits = 0.01 * torch.randn(n, E, device=DEV, generator=gen(98)), torch.zeros(n, E, **bf)

    def fill(self, seed):
        for i, t in enumerate((self.x, self.dout, self.logits)):
            t.copy_(torch.randn(t.shape, device=DEV, generator=gen(seed + i)))
        if self.n > 2:                                 # a token without experts, one with a single one left
            self.logits[1] = -float("inf")
            self.logits[2, 1:] = -float("inf")

    def run(self, st):
        lib, n, R, p = self.lib, self.n, self.R, lambda t: t.data_ptr()
        w1, w3, w2 = self.tables
        lib.route_groups_dev(p(self.idx), p(self.w), p(self.scores), p(self.logits), 1, n, p(self.bias), self.r, st)
        lib.moe_permute_dev(p(self.rows), p(self.off), p(self.tok), p(self.pos), p(self.x), 1, p(self.idx), n, TOPK, E,
                            H, st)
        lib.quant_mxfp4_dev(p(self.xq), p(self.xs), p(self.x), 1, H, n, H, st)
        for c, t in ((self.gate, w1), (self.up, w3)):
            lib.gemm_mxfp4q_grouped_dev(p(c), 1, p(self.xq), p(self.xs), n, p(self.tok), R, p(self.off), p(t), E, INTER,
                                        H, st)
        lib.swiglu_quant_mxfp4_dev(p(self.mq), p(self.ms), p(self.gate), p(self.up), 1, INTER, R, INTER, LIMIT, st)
        lib.gemm_mxfp4q_grouped_dev(p(self.y), 1, p(self.mq), p(self.ms), R, None, R, p(self.off), p(w2), E, H, INTER,
                                    st)
        lib.moe_unpermute_dev(p(self.out), p(self.y), 1, p(self.pos), p(self.w), p(self.x), n, TOPK, H, st)
        lib.moe_unpermute_bwd_dev(p(self.drows), p(self.dw), p(self.dout), p(self.y), 1, p(self.pos), p(self.w), n,
                                  TOPK, H, st)
        lib.route_groups_bwd_dev(p(self.dlogits), p(self.dw), p(self.ds), p(self.logits), 1, p(self.idx), n, self.r, st)
        lib.moe_permute_bwd_dev(p(self.dx), p(self.drows), 1, p(self.pos), n, TOPK, H, st)

    def results(self):
        live = int(self.off[-1])
        return [self.idx, self.w, self.scores, self.off, self.pos, self.out, self.dx, self.dw, self.dlogits, self.xq,
                self.xs] + [t[:live] for t in (self.tok, self.rows, self.gate, self.up, self.mq, self.ms, self.y,
                                               self.drows)]


@pytest.fixture(scope="module")
def weights():
    out = []
    for i, (r, c) in enumerate(((INTER, H), (INTER, H), (H, INTER))):
        q, s = operand(E * r, c, 50 + i)
        out.append((q.view(E, r, -1), s.view(E, r, -1).sub_(9)))     # values around 2^-8
    return out


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("n", [1, 5, 300])
def test_a_layer_step_by_step(lib, pkg, weights, n, kind):
    """Every call's outputs against the plain form of the inputs that it had."""
    y = Layer(lib, pkg, n, weights, kind)
    y.fill(n)
    lib.status()
    torch.cuda.synchronize()
    y.run(None)
    torch.cuda.synchronize()
    assert lib.status() == 0
    live = int(y.off[-1])
    ids = choose(y.scores, y.logits, y.bias, y.r)
    assert torch.equal(y.idx.long(), ids)
    s64 = scores64(y.logits, kind)
    assert ((y.w.double() - weights64(s64, ids, y.r)).abs() <= 7 * U * y.w).all()
    assert n < 3 or ((y.idx[1] == -1).all() and int((y.idx[2] >= 0).sum()) == 1)
    q, s = want_codes(y.x.double())
    np.testing.assert_array_equal(y.xq.cpu().numpy(), q)
    np.testing.assert_array_equal(y.xs.cpu().numpy(), s)
    xv = values(y.xq, y.xs)
    e_of = torch.searchsorted(y.off.long()[1:], torch.arange(live, device=DEV), right=True)

    def product(a, w, got):
        """each row by its expert: a bf16 rounding of the fp64 sum, and what fp32 sums may be off by"""
        for e in range(E):
            rows = e_of == e
            if rows.any():
                v = values(w[0][e], w[1][e]).t().contiguous()
                want, most = a[rows] @ v, a[rows].abs() @ v.abs()
                assert ((got[rows].double() - want).abs() <= 2.0 ** -8 * want.abs() + 40 * U * most).all()

    tok = y.tok[:live].long()
    product(xv[tok], weights[0], y.gate[:live])
    product(xv[tok], weights[1], y.up[:live])
    g, u = y.gate[:live].double().clamp(max=LIMIT), y.up[:live].double().clamp(-LIMIT, LIMIT)
    q, s = want_codes(g / (1 + torch.exp(-g)) * u) if live else (np.zeros((0, INTER // 2)), np.zeros((0, INTER // 32)))
    np.testing.assert_array_equal(y.mq[:live].cpu().numpy(), q)
    np.testing.assert_array_equal(y.ms[:live].cpu().numpy(), s)
    product(values(y.mq[:live], y.ms[:live]), weights[2], y.y[:live])
    pos = y.pos.long()
    rows = torch.where((pos >= 0)[..., None], y.y[pos.clamp(min=0)].double(), 0.0)
    out = (y.w.double()[..., None] * rows).sum(1) + y.x.double()
    most = (y.w.double()[..., None] * rows).abs().sum(1) + y.x.double().abs()
    assert ((y.out.double() - out).abs() <= 2.0 ** -8 * out.abs() + 10 * U * most).all()
    dw = (rows * y.dout.double()[:, None]).sum(-1)
    most = (rows * y.dout.double()[:, None]).abs().sum(-1)
    assert ((y.dw.double() - dw).abs() <= 80 * U * most).all()
    want = want_grad(y.r, y.logits, y.idx, y.dw, y.ds).nan_to_num(0.0)
    there = y.logits.float() > -float("inf")           # differentiation leaves NaN where nothing is
    got = y.dlogits.double()
    assert (got[~there] == 0).all()
    ok = there & (there.sum(-1, keepdim=True) > 1) if kind == 1 else there
    assert ((got - want).abs() <= 1.001 * 2.0 ** -8 * want.abs() + 1e-10)[ok].all()


def one_by_one(layer, lib, pkg, weights):
    """the same inputs through calls that are waited for one after the other"""
    ref = Layer(lib, pkg, layer.n, weights)
    for a in ("x", "dout", "logits"):
        getattr(ref, a).copy_(getattr(layer, a))
    torch.cuda.synchronize()
    ref.run(None)
    torch.cuda.synchronize()
    return ref.results()


def same(got, want):
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_layers_on_streams(lib, pkg, weights):
    layers = [Layer(lib, pkg, n, weights) for n in (5, 5, 300, 300)]
    streams = [torch.cuda.Stream() for _ in layers]
    for i, y in enumerate(layers):
        y.fill(10 * i)
    lib.status()
    torch.cuda.synchronize()
    for _ in range(4):
        for y, s in zip(layers, streams):
            y.run(s.cuda_stream)
    torch.cuda.synchronize()
    for y in layers:
        same(y.results(), one_by_one(y, lib, pkg, weights))
    assert lib.status() == 0


@pytest.mark.parametrize("n", [1, 64, 700])
def test_a_captured_layer(lib, pkg, weights, n):
    """Two graphs of one layer each, replayed with other routings and with eager
    work between."""
    layers, graphs = [Layer(lib, pkg, n, weights) for _ in range(2)], []
    for y in layers:
        y.fill(n)
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=torch.cuda.Stream()):
            y.run(torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    lib.status()
    for i in range(4):
        for j, (y, g) in enumerate(zip(layers, graphs)):
            y.fill(100 * i + 10 * j + n)
            torch.cuda.synchronize()
            g.replay()
        torch.cuda.synchronize()
        for y in layers:
            same(y.results(), one_by_one(y, lib, pkg, weights))
    assert lib.status() == 0
    assert np.isfinite(float(layers[0].out.float().abs().max()))


def test_a_captured_projection(lib, pkg):
    """Forward and both gradients of a projection in one graph, its inputs replaced
    between replays; a second graph of the same calls beside it."""
    M, N, K = 77, 160, 288
    mp = 96
    bufs = []
    for _ in range(2):
        b = {n: torch.zeros(r, c, dtype=torch.bfloat16, device=DEV) for n, r, c in (("x", M, K), ("w", N, K), ("dy", M, N))}
        for n, r, c in (("xq", M, K), ("wq", N, K), ("dyq", M, N), ("xt", K, mp), ("wt", K, N), ("dyt", N, mp)):
            b[n] = torch.zeros(r, c // 2, dtype=torch.uint8, device=DEV), torch.zeros(r, c // 32, dtype=torch.uint8, device=DEV)
        b["y"], b["dx"], b["dw"] = (torch.zeros(r, c, device=DEV) for r, c in ((M, N), (M, K), (N, K)))
        bufs.append(b)

    def run(b, st):
        for q, s, x in (("xq", "x", (M, K)), ("wq", "w", (N, K)), ("dyq", "dy", (M, N))):
            lib.quant_mxfp4_dev(b[q][0].data_ptr(), b[q][1].data_ptr(), b[s].data_ptr(), 1, x[1], *x, st)
        for q, s, x in (("xt", "x", (M, K)), ("wt", "w", (N, K)), ("dyt", "dy", (M, N))):
            lib.quant_mxfp4_t_dev(b[q][0].data_ptr(), b[q][1].data_ptr(), b[s].data_ptr(), 1, x[1], *x, st)
        for c, a, w in (("y", "xq", "wq"), ("dx", "dyq", "wt"), ("dw", "dyt", "xt")):
            m = pkg.qmat(pkg.DSV4_WFP4, b[w][0].data_ptr(), b[w][1].data_ptr(), b[w][0].shape[0], 2 * b[w][0].shape[1], 1, 32)
            lib.gemm_mxfp4q_dev(b[c].data_ptr(), 0, b[a][0].data_ptr(), b[a][1].data_ptr(), b[a][0].shape[0], m, st)

    graphs = []
    for b in bufs:
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=torch.cuda.Stream()):
            run(b, torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for i in range(4):
        for j, (b, g) in enumerate(zip(bufs, graphs)):
            for k, n in enumerate(("x", "w", "dy")):
                b[n].copy_(torch.randn(b[n].shape, device=DEV, generator=gen(10 * i + 3 * j + k)))
            torch.cuda.synchronize()
            g.replay()
        torch.cuda.synchronize()
        for b in bufs:
            got = [b[n].clone() for n in ("y", "dx", "dw")]
            run(b, None)
            torch.cuda.synchronize()
            for a, n in zip(got, ("y", "dx", "dw")):
                assert torch.equal(a, b[n]) and float(a.abs().max()) > 0
