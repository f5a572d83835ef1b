# SPDX-License-Identifier: Apache-2.0
"""Tokens to expert order and back on the GPU against plain 64-bit forms, the
gradients against their formulas and against differences, and the whole int8
expert layer that these calls make together.

Bounds, u = 2^-24 (fp32's half step, relative): a sum of topk products in fp32
is off by at most (topk + 1) u times the sum of the products' magnitudes, a dot
product of h elements by h u times theirs, whatever the order; a 16-bit result
adds its half step (bf16 2^-8, fp16 2^-11, or half fp16's least subnormal)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def routing(n, topk, E, seed, dropped=0.0, skew=False):
    """ids, one expert possibly several times in a token; -1 for dropped pairs"""
    r = np.random.default_rng(seed)
    ids = r.integers(0, E, (n, topk)) if not skew else np.minimum(r.geometric(0.3, (n, topk)) - 1, E - 1)
    ids = np.where(r.random((n, topk)) < dropped, -1, ids)
    return ids.astype(np.int32)


def want_order(ids, E):
    """first rows, token of each row, row of each pair, pair by pair"""
    flat = ids.reshape(-1)
    good = (flat >= 0) & (flat < E)
    cnt = np.bincount(flat[good], minlength=E)
    off = np.concatenate([[0], np.cumsum(cnt)])
    cur, pos, tok = off[:-1].copy(), np.full(flat.size, -1), np.full(flat.size, -1)
    for p in np.nonzero(good)[0]:
        pos[p] = cur[flat[p]]
        cur[flat[p]] += 1
        tok[pos[p]] = p // ids.shape[1]
    return off, tok, pos


def room(x, ids, E):
    """the sort's outputs with guard entries around them"""
    R = ids.numel()
    return dict(rows=torch.full((R + 2, x.shape[1]), 7.0, dtype=x.dtype, device=DEV),
                off=torch.full((E + 3,), -7, dtype=torch.int32, device=DEV),
                tok=torch.full((R + 2,), -7, dtype=torch.int32, device=DEV),
                pos=torch.full((R + 2,), -7, dtype=torch.int32, device=DEV))


def permute_into(lib, out, x, ids, E, stream=None):
    n, topk = ids.shape
    lib.moe_permute_dev(out["rows"][1:].data_ptr(), out["off"][1:].data_ptr(), out["tok"][1:].data_ptr(),
                        out["pos"][1:].data_ptr(), x.data_ptr(), CODE[x.dtype], ids.data_ptr(), n, topk, E, x.shape[1],
                        stream)
    return out


def permute(lib, x, ids, E):
    return permute_into(lib, room(x, ids, E), x, ids, E)


def check_order(out, ids, E, x):
    n, topk = ids.shape
    R = n * topk
    off, tok, pos = want_order(ids, E)
    live = off[-1]
    got = {k: v.cpu() for k, v in out.items()}
    for k in got:                                  # nothing outside the arrays
        assert (got[k][0] == (7 if k == "rows" else -7)).all() and (got[k][-1] == (7 if k == "rows" else -7)).all()
    np.testing.assert_array_equal(got["off"][1:-1].numpy(), off)
    np.testing.assert_array_equal(got["pos"][1:-1].numpy(), pos)
    np.testing.assert_array_equal(got["tok"][1:-1].numpy()[:live], tok[:live])
    assert (got["tok"][1:-1][live:] == -7).all() and (got["rows"][1:-1][live:] == 7).all()
    assert torch.equal(got["rows"][1:-1][:live], x.cpu()[tok[:live]])
    return pos.reshape(n, topk)


@pytest.mark.parametrize("n,topk,E,h", [(1, 1, 1, 8), (1, 6, 256, 4096), (7, 6, 256, 1024), (8, 16, 5, 64),
                                        (9, 16, 1024, 7), (64, 6, 256, 4096), (65, 2, 3, 100), (300, 8, 64, 520),
                                        (1000, 6, 384, 33), (4096, 8, 1000, 16), (129, 1, 64, 1)])
@pytest.mark.parametrize("kind", ["all", "dropped", "skew"])
def test_order(lib, n, topk, E, h, kind):
    dtype = TYPES[(n + h) % 3]
    ids = routing(n, topk, E, n + topk, 0.4 if kind == "dropped" else 0.0, kind == "skew")
    x = torch.randn(n, h, device=DEV, generator=gen(n)).to(dtype)
    lib.status()
    check_order(permute(lib, x, torch.from_numpy(ids).to(DEV), E), ids, E, x)
    assert lib.status() == 0


@pytest.mark.parametrize("n,topk,E,h", [(32769, 1, 256, 16), (5500, 6, 256, 64), (4100, 8, 1024, 24), (2200, 16, 1, 9),
                                        (20000, 6, 100, 8), (33000, 2, 1024, 4), (32768, 1, 64, 24), (16383, 2, 1000, 40),
                                        (8000, 4, 7, 72), (5461, 6, 128, 100), (4100, 7, 40, 33), (4097, 2, 16, 8208)])
@pytest.mark.parametrize("kind", ["all", "dropped", "skew"])
def test_order_of_many_pairs(lib, n, topk, E, h, kind):
    dtype = TYPES[n % 3]
    ids = routing(n, topk, E, n, 0.7 if kind == "dropped" else 0.0, kind == "skew")
    x = torch.randn(n, h, device=DEV, generator=gen(n)).to(dtype)
    check_order(permute(lib, x, torch.from_numpy(ids).to(DEV), E), ids, E, x)


@pytest.mark.parametrize("n", [40, 12000])
def test_order_with_nothing_to_do(lib, n):
    """every pair dropped, one expert for all, and ids that are no expert"""
    E, topk, h = 12, 4, 32
    x = torch.randn(n, h, device=DEV, generator=gen(1))
    for ids, bits in ((np.full((n, topk), -1), 0), (np.full((n, topk), 11), 0), (np.full((n, topk), 12), 1),
                      (np.where(np.arange(n * topk).reshape(n, topk) % 7 == 3, -5, 2), 1)):
        ids = ids.astype(np.int32)
        lib.status()
        check_order(permute(lib, x, torch.from_numpy(ids).to(DEV), E), ids, E, x)
        assert lib.status() == bits


def test_special_stream_handles(lib):
    """the calling thread's own stream works, the default stream is NULL only"""
    n, topk, E, h = 40, 3, 8, 64
    ids = routing(n, topk, E, 3, 0.2, False)
    idx, x = torch.from_numpy(ids).to(DEV), torch.randn(n, h, device=DEV, generator=gen(3))
    off, tok, pos = (torch.zeros(k, dtype=torch.int32, device=DEV) for k in (E + 1, n * topk, n * topk))
    rows = torch.zeros(n * topk, h, device=DEV)
    torch.cuda.synchronize()
    args = (rows.data_ptr(), off.data_ptr(), tok.data_ptr(), pos.data_ptr(), x.data_ptr(), 0, idx.data_ptr(), n, topk, E, h)
    with pytest.raises(Exception, match="NULL for the default stream"):
        lib.moe_permute_dev(*args, 1)
    torch.cuda.synchronize()
    assert (off == 0).all()
    lib.moe_permute_dev(*args, 2)
    torch.cuda.synchronize()
    assert off[-1] == (ids >= 0).sum()
    used = pos >= 0
    assert torch.equal(rows[pos[used].long()], x.repeat_interleave(topk, 0)[used])


def test_order_of_no_tokens(lib):
    off = torch.full((9,), 5, dtype=torch.int32, device=DEV)
    lib.moe_permute_dev(None, off.data_ptr(), None, None, None, 0, None, 0, 6, 8, 64)
    assert (off == 0).all()
    lib.moe_permute_bwd_dev(None, None, 0, None, 0, 6, 64)
    lib.moe_unpermute_dev(None, None, 0, None, None, None, 0, 6, 64)
    lib.moe_unpermute_bwd_dev(None, None, None, None, 0, None, None, 0, 6, 64)


def rows_of_elements(n, h, dtype, off, seed):
    """n x h values that begin `off` elements after a 16-byte boundary"""
    buf = torch.randn(n * h + 16, device=DEV, generator=gen(seed)).to(dtype)
    return buf[off:off + n * h].view(n, h)


def close(got, want, mag, factor):
    bound = HALF[got.dtype] * (want.abs() + factor * mag) + factor * mag + TINY[got.dtype]
    assert ((got.double() - want).abs() <= bound).all()


BACK = [(1, 1, 8, 0), (1, 6, 4096, 0), (7, 6, 1024, 0), (64, 6, 4096, 0), (33, 16, 520, 0), (10, 3, 7, 0), (65, 8, 64, 1),
        (300, 2, 33, 0), (500, 6, 2048, 0), (12, 9, 4096, 3)]


@pytest.mark.parametrize("n,topk,h,shift", BACK)
@pytest.mark.parametrize("dtype", TYPES)
def test_way_back(lib, n, topk, h, shift, dtype):
    E = 16
    ids = routing(n, topk, E, n, 0.3)
    _, _, pos = want_order(ids, E)
    p = torch.from_numpy(pos.reshape(n, topk)).to(DEV)
    p32 = p.to(torch.int32)
    rows = rows_of_elements(n * topk, h, dtype, shift, 1)
    used = torch.zeros(n * topk, dtype=torch.bool, device=DEV)
    used[p[p >= 0]] = True
    rows[~used] = float("nan")                     # nothing of a row that no pair has
    shared = rows_of_elements(n, h, dtype, shift, 2)
    w = torch.rand(n, topk, device=DEV, generator=gen(3)) - 0.3
    there = (p >= 0)[..., None]
    y = torch.where(there, rows[p.clamp(min=0)].double(), 0.0)
    prod = w.double()[..., None] * y
    for sh in (shared, None):
        out = torch.full((n + 2, h), 7.0, dtype=dtype, device=DEV)
        lib.moe_unpermute_dev(out[1:].data_ptr(), rows.data_ptr(), CODE[dtype], p32.data_ptr(), w.data_ptr(),
                              None if sh is None else sh.data_ptr(), n, topk, h)
        s = 0 if sh is None else sh.double()
        close(out[1:-1], prod.sum(1) + s, prod.abs().sum(1) + (0 if sh is None else sh.double().abs()), (topk + 1) * U)
        assert (out[0] == 7).all() and (out[-1] == 7).all()
    # the sort's gradient: the same without weights
    dx = torch.empty(n, h, dtype=dtype, device=DEV)
    lib.moe_permute_bwd_dev(dx.data_ptr(), rows.data_ptr(), CODE[dtype], p32.data_ptr(), n, topk, h)
    close(dx, y.sum(1), y.abs().sum(1), topk * U)
    # gradients of the way back
    dout = rows_of_elements(n, h, dtype, shift, 4)
    drows = torch.full((n * topk, h), 7.0, dtype=dtype, device=DEV)
    dw = torch.full((n, topk), 7.0, device=DEV)
    lib.moe_unpermute_bwd_dev(drows.data_ptr(), dw.data_ptr(), dout.data_ptr(), rows.data_ptr(), CODE[dtype],
                              p32.data_ptr(), w.data_ptr(), n, topk, h)
    assert (drows[~used] == 7).all()
    want = w.double()[..., None] * dout.double()[:, None]
    close(drows[p.clamp(min=0)] * there, want * there, want.abs() * there, U)
    dots = dout.double()[:, None] * y
    assert ((dw.double() - dots.sum(-1)).abs() <= h * U * dots.abs().sum(-1) + 2.0 ** -149).all()
    assert (dw[p < 0] == 0).all()
    # drows over rows itself
    rows2, dw2 = rows.clone(), torch.empty_like(dw)
    lib.moe_unpermute_bwd_dev(rows2.data_ptr(), dw2.data_ptr(), dout.data_ptr(), rows2.data_ptr(), CODE[dtype],
                              p32.data_ptr(), w.data_ptr(), n, topk, h)
    assert torch.equal(dw2, dw) and torch.equal(rows2[used], drows[used])


def test_way_back_of_millions_of_tokens(lib):
    """a workgroup a token: as many as one launch takes threads for"""
    n, h = 4_300_001, 8
    rows = torch.randn(n, h, device=DEV, generator=gen(5)).to(torch.bfloat16)
    dout = torch.randn(n, h, device=DEV, generator=gen(6)).to(torch.bfloat16)
    w = torch.rand(n, 1, device=DEV, generator=gen(7))
    pos = torch.arange(n - 1, -1, -1, dtype=torch.int32, device=DEV)[:, None].contiguous()
    drows, dw = torch.empty_like(rows), torch.empty_like(w)
    lib.moe_unpermute_bwd_dev(drows.data_ptr(), dw.data_ptr(), dout.data_ptr(), rows.data_ptr(), 1, pos.data_ptr(),
                              w.data_ptr(), n, 1, h)
    want = w.double() * dout.double()
    close(drows.flip(0), want, want.abs(), U)
    dots = dout.double() * rows.flip(0).double()
    assert ((dw.double() - dots.sum(-1, keepdim=True)).abs() <= h * U * dots.abs().sum(-1, keepdim=True)).all()


def test_way_back_ignores_rows_out_of_range(lib):
    n, topk, h = 6, 4, 64
    rows = torch.randn(n * topk, h, device=DEV, generator=gen(1))
    w = torch.rand(n, topk, device=DEV, generator=gen(2))
    pos = torch.randperm(n * topk, device=DEV, generator=gen(3)).to(torch.int32).view(n, topk)
    bad = pos.clone()
    bad[0, 0], bad[3, 2], bad[5] = n * topk, 1 << 30, -3
    out = torch.empty(n, h, device=DEV)
    lib.moe_unpermute_dev(out.data_ptr(), rows.data_ptr(), 0, bad.data_ptr(), w.data_ptr(), None, n, topk, h)
    ok = (bad >= 0) & (bad < n * topk)
    prod = torch.where(ok, w, 0.0).double()[..., None] * rows[pos.long()].double()
    close(out, prod.sum(1), prod.abs().sum(1), (topk + 1) * U)
    assert (out[5] == 0).all()
    drows, dw = torch.full_like(rows, 7.0), torch.empty_like(w)
    lib.moe_unpermute_bwd_dev(drows.data_ptr(), dw.data_ptr(), out.data_ptr(), rows.data_ptr(), 0, bad.data_ptr(),
                              w.data_ptr(), n, topk, h)
    assert (drows[pos[~ok].long()] == 7).all() and (dw[~ok] == 0).all()


def test_out_may_be_the_shared_output(lib):
    n, topk, h = 20, 6, 512
    rows = torch.randn(n * topk, h, device=DEV, generator=gen(1)).to(torch.bfloat16)
    w = torch.rand(n, topk, device=DEV, generator=gen(2))
    pos = torch.randperm(n * topk, device=DEV, generator=gen(3)).to(torch.int32)
    sh = torch.randn(n, h, device=DEV, generator=gen(4)).to(torch.bfloat16)
    out = torch.empty_like(sh)
    for o, s in ((out, sh), (sh, sh)):
        lib.moe_unpermute_dev(o.data_ptr(), rows.data_ptr(), 1, pos.data_ptr(), w.data_ptr(), s.data_ptr(), n, topk, h)
    assert torch.equal(out, sh)


def test_gradients_against_differences(lib):
    """loss = sum(c * unpermute(permute(x), w)) in fp32: linear in x and in w,
    so a difference over a step of one is the gradient up to the rounding of
    the two losses' terms."""
    n, topk, E, h = 6, 3, 4, 8
    ids = routing(n, topk, E, 5, 0.25)
    idx = torch.from_numpy(ids).to(DEV)
    x = torch.randn(n, h, device=DEV, generator=gen(1))
    w = torch.rand(n, topk, device=DEV, generator=gen(2))
    c = torch.randn(n, h, device=DEV, generator=gen(3))

    def forward(x, w):
        o = permute(lib, x, idx, E)
        rows, pos = o["rows"][1:-1].contiguous(), o["pos"][1:-1].contiguous()
        out = torch.empty_like(x)
        lib.moe_unpermute_dev(out.data_ptr(), rows.data_ptr(), 0, pos.data_ptr(), w.data_ptr(), None, n, topk, h)
        return out, rows, pos

    out, rows, pos = forward(x, w)
    drows, dw, dx = torch.zeros_like(rows), torch.empty_like(w), torch.empty_like(x)
    lib.moe_unpermute_bwd_dev(drows.data_ptr(), dw.data_ptr(), c.data_ptr(), rows.data_ptr(), 0, pos.data_ptr(),
                              w.data_ptr(), n, topk, h)
    lib.moe_permute_bwd_dev(dx.data_ptr(), drows.data_ptr(), 0, pos.data_ptr(), n, topk, h)
    # a loss has at most n h terms of topk products, each within (topk + 2) u of
    # its magnitude; two losses and the gradient's own rounding, bounded by the
    # magnitudes with every factor one larger
    mag = float((c.abs() * ((x.abs() + 1) * (w.abs() + 1).sum(1, keepdim=True))).sum().double())
    bound = 3 * (topk + 2) * U * mag
    for grad, var, of in ((dx, x, 0), (dw, w, 1)):
        for i in np.ndindex(*var.shape):
            moved = var.clone()
            moved[i] += 1
            o = forward(*((moved, w) if of == 0 else (x, moved)))[0]
            diff = float(((o.double() - out.double()) * c.double()).sum())
            step = float(moved[i].double() - var[i].double())
            assert abs(diff - step * float(grad[i])) <= bound


def test_on_streams_and_in_a_graph(lib):
    """Calls on two streams at once, both sorting forms, and a captured chain
    replayed with other work between: none shares anything with another."""
    E, topk, h = 64, 6, 64
    sets = []
    for n in (50, 6000):
        ids = routing(n, topk, E, n)
        x = torch.randn(n, h, device=DEV, generator=gen(n)).to(torch.bfloat16)
        idx = torch.from_numpy(ids).to(DEV)
        sets += [(x, ids, idx, room(x, idx, E), torch.cuda.Stream()) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(4):
        for x, _, idx, o, s in sets:
            permute_into(lib, o, x, idx, E, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for x, ids, _, o, _ in sets:
        check_order(o, ids, E, x)
    for n in (50, 6000):
        x = torch.randn(n, h, device=DEV, generator=gen(n))
        idx = torch.from_numpy(routing(n, topk, E, 1)).to(DEV)
        w = torch.rand(n, topk, device=DEV, generator=gen(4))
        o = permute(lib, x, idx, E)
        out = torch.empty_like(x)
        g = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=side):
            st = torch.cuda.current_stream().cuda_stream
            permute_into(lib, o, x, idx, E, stream=st)
            lib.moe_unpermute_dev(out.data_ptr(), o["rows"][1:].data_ptr(), 0, o["pos"][1:].data_ptr(), w.data_ptr(),
                                  x.data_ptr(), n, topk, h, st)
        for i in range(4):
            ids = routing(n, topk, E, 20 + i)
            idx.copy_(torch.from_numpy(ids))
            x.normal_(generator=gen(i))
            g.replay()
            torch.cuda.synchronize()
            check_order(o, ids, E, x)
            want = x.double() * (1 + w.double().sum(1, keepdim=True))
            close(out, want, x.double().abs() * (1 + w.double().sum(1, keepdim=True)), (topk + 1) * U)


def test_rows_beyond_4_gib(lib):
    n, topk, E, h = 70001, 8, 256, 4096
    ids = routing(n, topk, E, 1)
    idx = torch.from_numpy(ids).to(DEV)
    x = torch.empty(n, h, dtype=torch.bfloat16, device=DEV).normal_(generator=gen(1))
    o = room(x, idx, E)
    permute_into(lib, o, x, idx, E)
    off, tok, pos = want_order(ids, E)
    assert torch.equal(o["pos"][1:-1].cpu(), torch.from_numpy(pos).int())
    assert torch.equal(o["off"][1:-1].cpu(), torch.from_numpy(off).int())
    rows, p32 = o["rows"][1:-1], o["pos"][1:-1].contiguous()
    for r in (slice(0, 50), slice(524280, 524300), slice(n * topk - 50, n * topk)):
        assert torch.equal(rows[r], x[torch.from_numpy(tok[r]).to(DEV)])
    w = torch.rand(n, topk, device=DEV, generator=gen(2))
    out = torch.empty_like(x)
    lib.moe_unpermute_dev(out.data_ptr(), rows.data_ptr(), 1, p32.data_ptr(), w.data_ptr(), None, n, topk, h)
    drows, dw = torch.empty_like(o["rows"]), torch.empty_like(w)
    lib.moe_unpermute_bwd_dev(drows[1:].data_ptr(), dw.data_ptr(), x.data_ptr(), rows.data_ptr(), 1, p32.data_ptr(),
                              w.data_ptr(), n, topk, h)
    for t in (0, 65530, n - 1):
        want = x[t].double() * w[t].double().sum()
        close(out[t], want, want.abs(), (topk + 1) * U)
        sq = (x[t].double() ** 2).sum()
        assert ((dw[t].double() - sq).abs() <= h * U * sq).all()
        for k in range(topk):
            d = w[t, k].double() * x[t].double()
            close(drows[1 + int(pos[t * topk + k])], d, d.abs(), U)


def test_route_dev_orders_the_rows_of_these_calls(lib):
    """The framework's own permutation gives the same order, so its arrays serve
    the way back and the experts' products as well."""
    n, topk, E, h = 321, 6, 40, 64
    ids = routing(n, topk, E, 3)
    idx = torch.from_numpy(ids).to(DEV)
    x = torch.randn(n, h, device=DEV, generator=gen(1))
    o = permute(lib, x, idx, E)
    off, tok, k, pos = (torch.empty(s, dtype=torch.int32, device=DEV) for s in (E + 1, n * topk, n * topk, n * topk))
    lib.moe_route_dev(off.data_ptr(), tok.data_ptr(), k.data_ptr(), pos.data_ptr(), idx.data_ptr(), n, topk, E)
    assert torch.equal(off, o["off"][1:-1]) and torch.equal(tok, o["tok"][1:-1]) and torch.equal(pos, o["pos"][1:-1])


# ------------------------------------------------------- an expert layer ----

@pytest.mark.parametrize("n,dropped", [(1, 0.0), (7, 0.0), (77, 0.3), (300, 0.0)])
def test_int8_expert_layer(lib, pkg, n, dropped):
    """The calls together: tokens to int8, sorted by expert, gate and up
    products with the tokens taken through row_tok, SwiGLU to int8 rows, the
    down products, and the weighted way back. Each step is held to its own
    64-bit form on the inputs that the step before gave it, so no bound has to
    follow a code through the next quantization."""
    E, topk, H, I, limit = 12, 4, 512, 256, 10.0
    ids = routing(n, topk, E, n, dropped)
    off, tok, pos = want_order(ids, E)
    R, live = n * topk, int(off[-1])
    x = torch.randn(n, H, device=DEV, generator=gen(n)).to(torch.bfloat16)
    idx = torch.from_numpy(ids).to(DEV)
    mats, tables = {}, {}
    for name, (r, c) in (("w1", (I, H)), ("w3", (I, H)), ("w2", (H, I))):
        wf = 0.05 * torch.randn(E * r, c, device=DEV, generator=gen(len(mats)))
        q, s = torch.empty(E * r, c, dtype=torch.int8, device=DEV), torch.empty(E * r, device=DEV)
        lib.quant_i8_dev(q.data_ptr(), s.data_ptr(), wf.data_ptr(), 0, c, E * r, c)
        mats[name] = (q.view(E, r, c), s.view(E, r))
        ms = [pkg.qmat(pkg.DSV4_WI8, mats[name][0][e].data_ptr(), mats[name][1][e].data_ptr(), r, c, 1, c)
              for e in range(E)]
        tables[name] = torch.frombuffer(bytearray(bytes((pkg.QMat * E)(*ms))), dtype=torch.uint8).to(DEV)
    lib.status()
    o = permute(lib, x, idx, E)
    check_order(o, ids, E, x)
    dev = {k: o[k][1:-1].contiguous() for k in o}
    xq, xs = torch.empty(n, H, dtype=torch.int8, device=DEV), torch.empty(n, device=DEV)
    lib.quant_i8_dev(xq.data_ptr(), xs.data_ptr(), x.data_ptr(), 1, H, n, H)
    gu = [torch.zeros(R, I, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    for c, name in zip(gu, ("w1", "w3")):
        lib.gemm_i8_grouped_dev(c.data_ptr(), 1, xq.data_ptr(), xs.data_ptr(), n, dev["tok"].data_ptr(), R,
                                dev["off"].data_ptr(), tables[name].data_ptr(), E, I, H)
    mq, ms = torch.empty(R, I, dtype=torch.int8, device=DEV), torch.empty(R, device=DEV)
    lib.swiglu_quant_i8_dev(mq.data_ptr(), ms.data_ptr(), gu[0].data_ptr(), gu[1].data_ptr(), 1, I, R, I, limit)
    y = torch.zeros(R, H, dtype=torch.bfloat16, device=DEV)
    lib.gemm_i8_grouped_dev(y.data_ptr(), 1, mq.data_ptr(), ms.data_ptr(), R, None, R, dev["off"].data_ptr(),
                            tables["w2"].data_ptr(), E, H, I)
    w = torch.rand(n, topk, device=DEV, generator=gen(9))
    out = torch.empty(n, H, dtype=torch.bfloat16, device=DEV)
    lib.moe_unpermute_dev(out.data_ptr(), y.data_ptr(), 1, dev["pos"].data_ptr(), w.data_ptr(), x.data_ptr(), n, topk, H)
    assert lib.status() == 0

    ex = np.searchsorted(off, np.arange(live), side="right") - 1
    step = HALF[torch.bfloat16] * (1 + 4 * U) + 3.01 * U

    def products(a, sa, name, src):
        q, s = mats[name]
        return torch.stack([(a[t].double() @ q[e].double().t().contiguous()) * sa[t].double() * s[e].double()
                            for e, t in zip(ex, src)]) if live else torch.zeros(0, q.shape[1], device=DEV)
    for c, name in zip(gu, ("w1", "w3")):
        want = products(xq, xs, name, tok[:live])
        assert ((c[:live].double() - want).abs() <= step * want.abs() + 2.0 ** -134).all()
    g, u = (c[:live].double() for c in gu)
    g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    v = g / (1 + torch.exp(-g)) * u
    amax = v.abs().amax(1, keepdim=True)
    assert torch.equal(mq[:live], torch.round(v * 127 / amax).to(torch.int8))
    want = products(mq, ms, "w2", range(live))
    assert ((y[:live].double() - want).abs() <= step * want.abs() + 2.0 ** -134).all()
    p = torch.from_numpy(pos.reshape(n, topk)).to(DEV)
    prod = torch.where((p >= 0)[..., None], w.double()[..., None] * y[p.clamp(min=0)].double(), 0.0)
    close(out, prod.sum(1) + x.double(), prod.abs().sum(1) + x.double().abs(), (topk + 1) * U)
