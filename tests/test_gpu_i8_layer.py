# SPDX-License-Identifier: Apache-2.0
"""The whole int8 expert layer, its gradients of the way back and of the sort
behind it, on two streams at once and captured: each run gives the bits of the
calls made one by one."""
import numpy as np
import pytest
import torch

from test_gpu_i8 import DEV, gen, operands, table_of
from test_gpu_permute import routing

pytestmark = pytest.mark.gpu

E, TOPK, H, INTER, LIMIT = 12, 4, 512, 256, 10.0


class Layer:
    """One caller's buffers; the weights are shared between callers."""

    def __init__(self, lib, pkg, n, weights):
        R, i32 = n * TOPK, dict(dtype=torch.int32, device=DEV)
        bf = dict(dtype=torch.bfloat16, device=DEV)
        self.lib, self.n, self.R, self.tables = lib, n, R, [table_of(pkg, w, s) for w, s in weights]
        self.x, self.dout = torch.zeros(n, H, **bf), torch.zeros(n, H, **bf)
        self.idx, self.w = torch.full((n, TOPK), -1, **i32), torch.zeros(n, TOPK, device=DEV)
        self.off, self.tok, self.pos = torch.zeros(E + 1, **i32), torch.zeros(R, **i32), torch.zeros(R, **i32)
        self.rows, self.y, self.drows = (torch.zeros(R, H, **bf) for _ in range(3))
        self.gate, self.up = torch.zeros(R, INTER, **bf), torch.zeros(R, INTER, **bf)
        self.xq, self.xs = torch.zeros(n, H, dtype=torch.int8, device=DEV), torch.zeros(n, device=DEV)
        self.mq, self.ms = torch.zeros(R, INTER, dtype=torch.int8, device=DEV), torch.zeros(R, device=DEV)
        self.out, self.dx, self.dw = torch.zeros(n, H, **bf), torch.zeros(n, H, **bf), torch.zeros(n, TOPK, device=DEV)

    def fill(self, seed):
        self.x.copy_(torch.randn(self.n, H, device=DEV, generator=gen(seed)))
        self.dout.copy_(torch.randn(self.n, H, device=DEV, generator=gen(seed + 1)))
        self.w.copy_(torch.rand(self.n, TOPK, device=DEV, generator=gen(seed + 2)))
        self.idx.copy_(torch.from_numpy(routing(self.n, TOPK, E, seed, 0.2)))

    def run(self, st):
        lib, n, R, p = self.lib, self.n, self.R, lambda t: t.data_ptr()
        w1, w3, w2 = self.tables
        lib.moe_permute_dev(p(self.rows), p(self.off), p(self.tok), p(self.pos), p(self.x), 1, p(self.idx), n, TOPK, E,
                            H, st)
        lib.quant_i8_dev(p(self.xq), p(self.xs), p(self.x), 1, H, n, H, st)
        for c, t in ((self.gate, w1), (self.up, w3)):
            lib.gemm_i8_grouped_dev(p(c), 1, p(self.xq), p(self.xs), n, p(self.tok), R, p(self.off), p(t), E, INTER, H,
                                    st)
        lib.swiglu_quant_i8_dev(p(self.mq), p(self.ms), p(self.gate), p(self.up), 1, INTER, R, INTER, LIMIT, st)
        lib.gemm_i8_grouped_dev(p(self.y), 1, p(self.mq), p(self.ms), R, None, R, p(self.off), p(w2), E, H, INTER, st)
        lib.moe_unpermute_dev(p(self.out), p(self.y), 1, p(self.pos), p(self.w), p(self.x), n, TOPK, H, st)
        lib.moe_unpermute_bwd_dev(p(self.drows), p(self.dw), p(self.dout), p(self.y), 1, p(self.pos), p(self.w), n,
                                  TOPK, H, st)
        lib.moe_permute_bwd_dev(p(self.dx), p(self.drows), 1, p(self.pos), n, TOPK, H, st)

    def results(self):
        live = int(self.off[-1])
        return [self.off, self.pos, self.out, self.dx, self.dw, self.xq, self.xs] + \
            [t[:live] for t in (self.tok, self.rows, self.gate, self.up, self.mq, self.ms, self.y, self.drows)]


@pytest.fixture(scope="module")
def weights():
    out = []
    for i, (r, c) in enumerate(((INTER, H), (INTER, H), (H, INTER))):
        _, _, w, s = operands(1, E * r, c, 50 + i)
        out.append((w.view(E, r, c), s.view(E, r) * 0.02))
    return out


def one_by_one(layer, lib, pkg, weights):
    """the same inputs through calls that are waited for one after the other"""
    ref = Layer(lib, pkg, layer.n, weights)
    for a in ("x", "dout", "w", "idx"):
        getattr(ref, a).copy_(getattr(layer, a))
    torch.cuda.synchronize()
    ref.run(None)
    torch.cuda.synchronize()
    return ref.results()


def same(got, want):
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_layers_on_two_streams(lib, pkg, weights):
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
