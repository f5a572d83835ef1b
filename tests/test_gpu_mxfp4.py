# SPDX-License-Identifier: Apache-2.0
"""Microscaled 4-bit rows and their products on the GPU against plain 64-bit
forms.

Bounds. Codes and scale bytes are defined by exact arithmetic (SwiGLU: by fp64
values): equal. Products of codes are multiples of 1/4 up to 36; with scales of
2^-1, 1 and 2 on both sides every partial sum is a multiple of 2^-4 below 2^20 up
to K = 5,000, so fp32 holds it exactly in any order and the results are equal, or
the exact sum rounded once to 16 bits. With scales over a wide range: u = 2^-24 is
fp32's half step, an addition to a sum of at most A = sum |a w| errs by at most 2 u
A (a matrix instruction may cut where fp32 rounds), there are K / 32 blocks and up
to 16 sums of waves: (K / 32 + 16) 2 u A, and the output's own half step."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
CODE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def ceil32(n):
    return (n + 31) // 32 * 32


def want_codes(v):
    """packed codes and scale bytes of fp64 rows"""
    v = v.cpu().numpy().astype(np.float64)
    b = v.reshape(v.shape[0], -1, 32)
    ok = np.isfinite(b).all(-1)
    amax = np.abs(np.where(ok[..., None], b, 0)).max(-1)
    f, e = np.frexp(amax)
    byte = np.clip(127 + e - 3 + (f > 0.75), 0, 254)
    byte = np.where(ok, np.where(amax > 0, byte, 127), 255)
    x = np.where(ok[..., None], b, 0.0) * np.exp2(127.0 - np.minimum(byte, 254))[..., None]
    a = np.abs(x)
    c = sum((a > t).astype(np.uint8) for t in (0.25, 1.25, 2.5, 5.0)) + sum((a >= t).astype(np.uint8) for t in (0.75, 1.75, 3.5))
    c = (c | (np.signbit(x) * 8).astype(np.uint8)) * ok[..., None]
    c = c.reshape(v.shape).astype(np.uint8)
    return c[:, 0::2] | (c[:, 1::2] << 4), byte.astype(np.uint8)


def quant(lib, a, k=None, ld=None, form="rows", u=None, limit=10.0, stream=None):
    n, k = a.shape[0], k or a.shape[1]
    rows, cols = (k, ceil32(n)) if form == "columns" else (n, k)
    q = torch.full((rows + 1, cols // 2), 0x99, dtype=torch.uint8, device=DEV)
    s = torch.full((rows + 1, cols // 32), 0x77, dtype=torch.uint8, device=DEV)
    args = (CODE[a.dtype], ld or a.stride(0), n, k)
    if form == "swiglu":
        lib.swiglu_quant_mxfp4_dev(q.data_ptr(), s.data_ptr(), a.data_ptr(), u.data_ptr(), *args, limit, stream)
    else:
        f = lib.quant_mxfp4_t_dev if form == "columns" else lib.quant_mxfp4_dev
        f(q.data_ptr(), s.data_ptr(), a.data_ptr(), *args, stream)
    torch.cuda.synchronize()
    assert (q[rows] == 0x99).all() and (s[rows] == 0x77).all()
    return q[:rows], s[:rows]


def check_rows(got, v):
    qw, sw = want_codes(v)
    np.testing.assert_array_equal(got[1].cpu().numpy(), sw)
    np.testing.assert_array_equal(got[0].cpu().numpy(), qw)


def columns(v):
    out = torch.zeros(v.shape[1], ceil32(v.shape[0]), dtype=torch.float64, device=v.device)
    out[:, :v.shape[0]] = v.double().t()
    return out


# ------------------------------------------------------------------- rows ----

SIZES = [(1, 32), (1, 4096), (3, 96), (33, 1024), (7, 2080), (2, 20000 // 32 * 32), (1030, 512), (1303, 4128)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k", SIZES)
def test_rows(lib, dtype, n, k):
    x = torch.randn(n, k, device=DEV, generator=gen(n + k)).to(dtype)
    check_rows(quant(lib, x), x.double())


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_are_those_of_the_weight_quantizer(lib, dtype):
    x = torch.randn(65, 352, device=DEV, generator=gen(1)).to(dtype)
    q, s = quant(lib, x)
    w, f = torch.zeros_like(q), x.float()
    sw = torch.zeros_like(s)
    lib.quant_fp4_mx_dev(w.data_ptr(), sw.data_ptr(), f.data_ptr(), 65, 352)
    torch.cuda.synchronize()
    assert torch.equal(q, w) and torch.equal(s, sw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k", [(1, 1), (1, 37), (31, 2), (32, 128), (33, 129), (255, 3), (256, 256), (257, 100),
                                 (2803, 77), (5, 5000)])
def test_columns(lib, dtype, n, k):
    x = torch.randn(n, k, device=DEV, generator=gen(n + k)).to(dtype)
    check_rows(quant(lib, x, form="columns"), columns(x))


def borders(n, k, dtype, seed):
    """values at, just below and just above every border of their block, blocks of many scales"""
    b = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 0.0], device=DEV)
    x = b[torch.randint(0, 9, (n, k), device=DEV, generator=gen(seed))]
    x = x * (1 - 2 * torch.randint(0, 2, (n, k), device=DEV, generator=gen(seed + 1)))
    x[:, ::32] = 6.0
    lo, hi = (-10, 9) if dtype == torch.float16 else (-60, 60)
    e = torch.randint(lo, hi, (n, k // 32), device=DEV, generator=gen(seed + 2)).repeat_interleave(32, 1)
    x = torch.ldexp(x, e).to(dtype)
    bits = x.view(torch.int32 if dtype == torch.float32 else torch.int16)
    d = torch.randint(-1, 2, (n, k), device=DEV, generator=gen(seed + 3)).to(bits.dtype)
    d[:, ::32] = torch.randint(-1, 2, (n, k // 32), device=DEV, generator=gen(seed + 4)).to(bits.dtype)
    return torch.where(x == 0, x, (bits + d).view(dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_borders(lib, dtype):
    x = borders(64, 1024, dtype, 7)
    check_rows(quant(lib, x), x.double())
    y = x.t().contiguous()
    check_rows(quant(lib, y, form="columns"), columns(y))


def extremes(k=96):
    x = torch.randn(12, k, device=DEV, generator=gen(5))
    x[0] = 0
    x[1] = 0
    x[1, 5] = 2.0 ** -149
    x[2] *= 2.0 ** -140
    x[3] = x[3] / x[3].abs().max() * 3.4e38
    x[4, 17] = float("nan")
    x[5, 95] = float("inf")
    x[6, 0] = -float("inf")
    x[7] = -0.0
    x[8] = 1.0
    x[9, 3] = 1e30
    x[10] *= 2.0 ** -110
    x[11] *= 2.0 ** -126
    return x


def test_rows_of_extremes(lib):
    x = extremes()
    q, s = quant(lib, x)
    check_rows((q, s), x.double())
    assert s[4, 0] == 255 and (q[4, :16] == 0).all() and s[4, 1] != 255 and s[5, 2] == 255 and s[6, 0] == 255
    assert (s[0] == 127).all()
    y = torch.zeros(96, 12, device=DEV)
    y.copy_(x.t())
    check_rows(quant(lib, y, form="columns"), columns(y))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_with_a_pitch(lib, dtype):
    """Rows that lie apart; what lies between them is not read into them. Columns at
    odd pitches and addresses."""
    big = torch.full((9, 160), 1e4, device=DEV, dtype=dtype)
    big[:, :96] = torch.randn(9, 96, device=DEV, generator=gen(3)).to(dtype)
    check_rows(quant(lib, big[:, :96], ld=160, k=96), big[:, :96].double())
    for c, k, ld in ((0, 96, 160), (1, 95, 160), (3, 2, 160), (1, 61, 97)):
        flat = big.view(-1)[c:]
        x = torch.as_strided(flat, (7, k), (ld, 1))
        check_rows(quant(lib, x, ld=ld, k=k, form="columns"), columns(x))


def test_rows_past_4_gib(lib):
    """The last rows, and columns, of more than 4 GiB as by themselves."""
    x = torch.empty((1 << 21) + 3, 1056, dtype=torch.bfloat16, device=DEV).normal_(generator=gen(1))
    q, s = quant(lib, x)
    check_rows((q[-5:], s[-5:]), x[-5:].double())
    u = x.flip(0)
    q, s = quant(lib, x, form="swiglu", u=u)
    check_rows((q[-5:], s[-5:]), swiglu64(x[-5:], u[-5:], 10.0))
    del u
    x = x.view(-1)[:40037 * 55000].view(40037, 55000)
    q, s = quant(lib, x, form="columns")
    check_rows((q[-3:], s[-3:]), columns(x[:, -3:]))


def swiglu64(g, u, limit):
    g, u = g.double(), u.double()
    lim = float(np.float32(limit))
    if lim > 0:
        g, u = torch.where(g > lim, lim, g), torch.where(u > lim, lim, torch.where(u < -lim, -lim, u))
    return g / (1 + torch.exp(-g)) * u


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("limit", [0.0, 10.0, 0.5])
@pytest.mark.parametrize("n,k", [(1, 32), (3, 2048), (70, 544), (1100, 2048)])
def test_swiglu_rows(lib, dtype, limit, n, k):
    g, u = (4 * torch.randn(n, k, device=DEV, generator=gen(n + k + i)).to(dtype) for i in range(2))
    check_rows(quant(lib, g, form="swiglu", u=u, limit=limit), swiglu64(g, u, limit))


def test_swiglu_rows_next_to_borders(lib):
    """Up values that put the product within a few steps of fp32 of a border: the
    fp64 value decides, for codes and for the largest value's power of two."""
    n, k = 256, 512
    g = 3 * torch.randn(n, k, device=DEV, generator=gen(11))
    silu = g.double() / (1 + torch.exp(-g.double()))
    b = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV, dtype=torch.float64)
    t = b[torch.randint(0, 7, (n, k), device=DEV, generator=gen(12))]
    t[:, ::32] = 6.0
    u = (t / silu).float()
    d = torch.randint(-3, 4, (n, k), device=DEV, generator=gen(13), dtype=torch.int32)
    u = (u.view(torch.int32) + d).view(torch.float32)
    check_rows(quant(lib, g, form="swiglu", u=u, limit=0.0), swiglu64(g, u, 0.0))


def test_swiglu_rows_of_extremes(lib):
    k = 64
    g, u = (torch.randn(12, k, device=DEV, generator=gen(i)) for i in range(2))
    g[0], u[0] = 0, 0
    g[1] = -95.0
    g[2], u[2] = 1e15, u[2] * 1e20
    u[3] = u[3] * 1e-30
    g[4, 9] = float("nan")
    u[5, 2] = float("inf")
    g[6, 1] = -float("inf")
    g[7] = -60.0
    u[8] = 3e38
    g[9, 5] = 88.0
    g[10], u[10] = -80.0, 1e38
    g[11, ::2] = -100.0
    u[11] = 1e30
    check_rows(quant(lib, g, form="swiglu", u=u, limit=0.0), swiglu64(g, u, 0.0))


@pytest.mark.parametrize("dtype", TYPES)
def test_swiglu_of_the_halves_of_one_array(lib, dtype):
    gu = torch.randn(9, 2 * 96, device=DEV, generator=gen(21)).to(dtype)
    g, u = gu[:, :96], gu[:, 96:]
    check_rows(quant(lib, g, form="swiglu", u=u, limit=10.0, ld=192, k=96), swiglu64(g, u, 10.0))


def test_no_rows(lib):
    q = torch.full((4,), 9, dtype=torch.uint8, device=DEV)
    for f in (lib.quant_mxfp4_dev, lib.quant_mxfp4_t_dev):
        f(q.data_ptr(), q.data_ptr(), None, 0, 32, 0, 32)
    lib.quant_mxfp4_t_dev(q.data_ptr(), q.data_ptr(), q.data_ptr(), 0, 0, 5, 0)
    torch.cuda.synchronize()
    assert (q == 9).all()


# --------------------------------------------------------------- products ----

def values(q, s):
    """fp64 values of packed rows"""
    g = torch.cat([GRID, -GRID]).to(q.device)
    v = torch.empty(*q.shape[:-1], 2 * q.shape[-1], dtype=torch.float64, device=q.device)
    v[..., 0::2], v[..., 1::2] = g[(q & 15).long()], g[(q >> 4).long()]
    scale = torch.tensor([2.0 ** (i - 127) for i in range(255)] + [float("nan")], dtype=torch.float64, device=q.device)
    return v * scale[s.long()].repeat_interleave(32, -1)


def operand(rows, k, seed, wide=False, at=0):
    """packed rows and scales; `at`: how far from alignment the scales lie"""
    q = torch.randint(0, 256, (rows, k // 2), device=DEV, generator=gen(seed), dtype=torch.uint8)
    lo, hi = (110, 140) if wide else (126, 129)
    s = torch.empty(rows * (k // 32) + at, dtype=torch.uint8, device=DEV)[at:].view(rows, k // 32)
    s.copy_(torch.randint(lo, hi, s.shape, device=DEV, generator=gen(seed + 1), dtype=torch.uint8))
    return q, s


def qmat(pkg, q, s):
    return pkg.qmat(pkg.DSV4_WFP4, q.data_ptr(), s.data_ptr(), q.shape[0], 2 * q.shape[1], 1, 32)


def product(lib, pkg, a, w, out=torch.float32, off=0):
    """C with `off` elements before it and guards behind"""
    M, N = a[0].shape[0], w[0].shape[0]
    buf = torch.full((M * N + off + 64,), 77.0, dtype=out, device=DEV)
    c = buf[off:off + M * N]
    lib.gemm_mxfp4q_dev(c.data_ptr(), CODE[out], a[0].data_ptr(), a[1].data_ptr(), M, qmat(pkg, *w))
    torch.cuda.synchronize()
    assert (buf[:off] == 77).all() and (buf[off + M * N:] == 77).all()
    return c.view(M, N)


# every form with rows, features and K that end inside a tile, whole ones too
SHAPES = [(1, 1, 32), (1, 77, 4128), (3, 130, 96), (8, 4096, 544), (5, 1000, 256), (9, 33, 32), (17, 100, 4096),
          (32, 64, 512), (45, 257, 672), (100, 300, 1056), (200, 1500, 288), (333, 1024, 4096), (700, 1001, 160),
          (130, 8200, 224), (300, 8192, 512), (900, 3333, 320), (1100, 4104, 96), (700, 6000, 1184), (2048, 2048, 768),
          (1300, 6001, 160), (2100, 8200, 288), (4100, 4097, 64), (2048, 8192, 1280), (4097, 4352, 32), (70, 15000, 544),
          (40, 20001, 1120), (333, 2111, 2080), (500, 4111, 2080), (1001, 4099, 1056), (2803, 4100, 2080), (1999, 4097, 4128),
          (1, 20000, 4128), (1990, 3416, 3040), (2044, 3357, 1632), (333, 2111, 160), (70, 999, 2720), (64, 4100, 4128),
          (3658, 3624, 800), (312, 2659, 1216), (1609, 1153, 160), (431, 6829, 160)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_exact(lib, pkg, M, N, K):
    a, w = operand(M, K, M + K), operand(N, K, N + K + 1)
    want = values(*a) @ values(*w).t().contiguous()
    assert torch.equal(product(lib, pkg, a, w).double(), want)


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_exact_16_bits(lib, pkg, M, N, K, out):
    """one rounding of the exact sum; unaligned rows and scales"""
    a, w = operand(M, K, M, at=1), operand(N, K, N, at=3)
    if out == torch.float16:
        a[1].sub_(8)                                # within its range
    want = (values(*a) @ values(*w).t().contiguous()).to(out)
    assert torch.equal(product(lib, pkg, a, w, out, off=1), want)


@pytest.mark.parametrize("M,N,K", [(1, 4096, 4096), (4, 100, 8224), (40, 512, 4096), (333, 1024, 4096), (520, 2048, 2048),
                                   (1100, 4096, 2080), (1100, 6144, 2048), (2100, 8192, 4096)])
def test_product_of_many_scales(lib, pkg, M, N, K):
    a, w = operand(M, K, M, wide=True), operand(N, K, N, wide=True)
    va, vw = values(*a), values(*w)
    want = va @ vw.t().contiguous()
    most = va.abs() @ vw.abs().t().contiguous()
    assert ((product(lib, pkg, a, w).double() - want).abs() <= (K / 32 + 16) * 2 * U * most).all()


@pytest.mark.parametrize("M,N,K", [(2, 40, 288), (40, 70, 4128), (200, 1500, 288), (300, 8192, 512), (700, 6000, 1184),
                                   (2100, 8200, 288)])
def test_scales_of_nan(lib, pkg, M, N, K):
    """A byte of 255 reaches the results of its row and no others, in K's last block too."""
    a, w = operand(M, K, M), operand(N, K, N)
    want = values(*a) @ values(*w).t().contiguous()
    a[1][M - 1, -1] = 255
    w[1][1, 0] = 255
    w[1][N - 1, -1] = 255
    got = product(lib, pkg, a, w)
    nan = torch.zeros(M, N, dtype=torch.bool, device=DEV)
    nan[M - 1], nan[:, 1], nan[:, N - 1] = True, True, True
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan].double(), want[~nan])


def test_scales_of_the_ends(lib, pkg):
    """Scales at both ends of their range: 2^-127 times 2^127, and results at fp32's ends."""
    a, w = operand(3, 64, 1), operand(5, 64, 2)
    a[1].fill_(0)
    w[1].fill_(254)
    assert torch.equal(product(lib, pkg, a, w).double(), values(*a) @ values(*w).t().contiguous())
    a[1].fill_(254)
    got = product(lib, pkg, a, w)
    assert (torch.isinf(got) | torch.isnan(got) | (got == 0)).all()


@pytest.mark.parametrize("M,N,K", [(70001, 16390, 32), (3, 70003, 1 << 17), (40, 70003, 1 << 17), (70003, 9, 1 << 17)])
def test_matrices_past_4_gib(lib, pkg, M, N, K):
    """Results, weights and tokens beyond 4 GiB: the last of them, and a call's guards."""
    a, w = operand(M, K, 1, wide=True), operand(N, K, 2, wide=True)
    got = product(lib, pkg, a, w)
    m, n = min(M, 40), min(N, 40)
    va, vw = values(a[0][-m:], a[1][-m:]), values(w[0][-n:], w[1][-n:])
    want, most = va @ vw.t().contiguous(), va.abs() @ vw.abs().t().contiguous()
    assert ((got[-m:, -n:].double() - want).abs() <= (K / 32 + 16) * 2 * U * most).all()


def test_wide_rows(lib, pkg):
    """K at its limit, one token and a few."""
    K = 1 << 20
    for M, N in ((1, 9), (20, 33)):
        a, w = operand(M, K, M, wide=True), operand(N, K, N, wide=True)
        va, vw = values(*a), values(*w)
        want, most = va @ vw.t().contiguous(), va.abs() @ vw.abs().t().contiguous()
        assert ((product(lib, pkg, a, w).double() - want).abs() <= (K / 32 + 16) * 2 * U * most).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_projection_and_its_gradients(lib, pkg, dtype):
    """Y = X W^T, dX = dY W, dW = dY^T X from rows and columns quantized by the calls,
    against the products of the quantized values; and those against the unquantized
    ones: a value is off by at most a sixth of its block's largest... of the norm, well
    within a quarter."""
    M, N, K = 77, 160, 288
    x, w, dy = (torch.randn(r, c, device=DEV, generator=gen(i)).to(dtype) for i, (r, c) in enumerate(((M, K), (N, K), (M, N))))
    rows = {n: quant(lib, t) for n, t in (("x", x), ("w", w), ("dy", dy))}
    cols = {n: quant(lib, t, form="columns") for n, t in (("x", x), ("w", w), ("dy", dy))}
    for a, b, plain in ((rows["x"], rows["w"], x.double() @ w.double().t().contiguous()),
                        (rows["dy"], cols["w"], dy.double() @ w.double()),
                        (cols["dy"], cols["x"], dy.double().t().contiguous() @ x.double())):
        va, vb = values(*a), values(*b)
        want, most = va @ vb.t().contiguous(), va.abs() @ vb.abs().t().contiguous()
        got = product(lib, pkg, a, b).double()
        assert ((got - want).abs() <= (va.shape[1] / 32 + 16) * 2 * U * most).all()
        assert float((got - plain).norm() / plain.norm()) < 0.25


# ---------------------------------------------------------------- experts ----

def table_of(pkg, w, s, wdt=3, k=None):
    E, N, kb = w.shape
    i = torch.arange(E, device=DEV)
    k = k or 2 * kb
    return torch.stack([w.data_ptr() + i * (N * kb), s.data_ptr() + i * (N * s.shape[2]), 0 * i + (wdt + (N << 32)),
                        0 * i + (k + (1 << 32)), 0 * i + 32], 1).contiguous()


def grouped(lib, pkg, counts, N, K, n_a, seed, out=torch.float32, row_tok=True, table=None, w=None):
    E, R = len(counts), sum(counts)
    if w is None:
        wq, ws = operand(E * N, K, seed)
        w = wq.view(E, N, -1), ws.view(E, N, -1)
    a = operand(n_a, K, seed + 7)
    off = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device=DEV)
    tok = torch.randint(0, n_a, (R + 5,), device=DEV, generator=gen(seed + 9), dtype=torch.int32) if row_tok else \
        torch.arange(R + 5, device=DEV, dtype=torch.int32)
    c = torch.full((R + 5, N), 77.0, dtype=out, device=DEV)
    t = table_of(pkg, *w) if table is None else table
    lib.gemm_mxfp4q_grouped_dev(c.data_ptr(), CODE[out], a[0].data_ptr(), a[1].data_ptr(), n_a,
                                tok.data_ptr() if row_tok else None, R + 5, off.data_ptr(), t.data_ptr(), E, N, K)
    torch.cuda.synchronize()
    want = torch.full((R + 5, N), 77.0, dtype=torch.float64, device=DEV)
    va = values(*a)
    r = 0
    for e, n in enumerate(counts):
        if n:
            vw = values(w[0][e], w[1][e]).t().contiguous()
            want[r:r + n] = va[tok[r:r + n].long()] @ vw
            assert K <= 5000 or float((va[tok[r:r + n].long()].abs() @ vw.abs()).max()) < 2 ** 20
        r += n
    return c, want


GROUPS = [([1], 1, 32), ([0, 0, 3, 0], 40, 96), ([1] * 40, 64, 544), ([5, 0, 9, 1, 12, 0, 3] * 3, 100, 288),
          ([20, 0, 31, 18, 2, 40], 77, 1056), ([64, 10, 0, 30, 33, 48], 130, 352), ([100, 0, 60, 130, 1, 90], 333, 608),
          ([300, 0, 3, 129, 128, 127, 500], 300, 416), ([0, 700, 0, 0, 20], 520, 96), ([2500, 3, 0, 300], 1000, 160),
          ([1, 0, 1200, 0, 60, 200, 1100] * 2, 300, 288), ([1] * 300 + [0] * 700 + [4] * 24, 33, 64),
          ([33, 64, 65, 0, 1, 31, 32, 96] * 4, 1000, 1056), ([257, 128, 129, 1, 0, 127, 31, 65] * 4, 1030, 544),
          ([700, 0, 128, 129, 256, 257, 1, 1500, 900], 4111, 288), ([2000, 31, 255, 0, 1900, 65], 2100, 1120)]
# weights that go past the caches: 128 MB and more of them, few rows an expert
STREAMS = [([1, 0, 2, 1, 0, 0, 3] * 9, 2051, 4128), ([5, 0, 9, 1, 12, 0, 3] * 9, 2051, 4128),
           ([60, 33, 64, 0, 1, 20, 50, 31], 8200, 8224)]


@pytest.mark.parametrize("counts,N,K", GROUPS)
def test_experts(lib, pkg, counts, N, K):
    lib.status()
    c, want = grouped(lib, pkg, counts, N, K, 211, len(counts) + N)
    assert torch.equal(c.double(), want) and lib.status() == 0


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("counts,N,K", STREAMS)
def test_experts_past_the_caches(lib, pkg, counts, N, K, out):
    """K beyond 5,000: the sums of magnitudes, which bound every partial sum, are below 2^20"""
    c, want = grouped(lib, pkg, counts, N, K, 211, len(counts) + N, out)
    assert torch.equal(c, want.to(out))


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts,N,K", GROUPS)
def test_experts_16_bits_in_row_order(lib, pkg, counts, N, K, out):
    c, want = grouped(lib, pkg, counts, N, K, sum(counts) + 5, N + K, out, row_tok=False)
    if out == torch.float16:
        want = want.clamp(-1e30, 1e30)
    assert torch.equal(c, want.to(out))


def test_experts_of_bad_descriptors_tokens_and_offsets(lib, pkg):
    for counts, N, K in (([3, 4, 2], 40, 96), ([20, 30, 25], 100, 288), ([40, 60, 50], 130, 352), ([200, 300, 250], 300, 96)):
        E, R = len(counts), sum(counts)
        wq, ws = operand(E * N, K, 3)
        w = wq.view(E, N, -1), ws.view(E, N, -1)
        t = table_of(pkg, *w)
        t[1, 2] = 5 + (N << 32)                    # int8 weights
        lib.status()
        c, want = grouped(lib, pkg, counts, N, K, 50, 3, table=t, w=w)
        assert lib.status() == 2
        lo, hi = counts[0], counts[0] + counts[1]
        assert torch.isnan(c[lo:hi]).all()
        assert torch.equal(c[:lo].double(), want[:lo]) and torch.equal(c[hi:].double(), want[hi:])
        # tokens out of range, offsets that fall and pass the rows
        a = operand(50, K, 10)
        tok = torch.randint(0, 50, (R,), device=DEV, generator=gen(1), dtype=torch.int32)
        tok[2], tok[R - 1] = -1, 50
        good = table_of(pkg, *w)
        off = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device=DEV)
        c = torch.zeros(R, N, device=DEV)
        args = (a[0].data_ptr(), a[1].data_ptr(), 50, tok.data_ptr(), R)
        lib.gemm_mxfp4q_grouped_dev(c.data_ptr(), 0, *args, off.data_ptr(), good.data_ptr(), E, N, K)
        assert lib.status() == 1
        nan = torch.zeros(R, dtype=torch.bool, device=DEV)
        nan[2], nan[R - 1] = True, True
        assert torch.equal(torch.isnan(c).all(1), nan) and torch.equal(torch.isnan(c).any(1), nan)
        for bad in ([-5, counts[0], 2, R + 900], [R, 0, R, 0], [7, 5, 3, 1]):
            off = torch.tensor(bad, dtype=torch.int32, device=DEV)
            buf = torch.full((R + 8, N), 5.0, device=DEV)
            lib.gemm_mxfp4q_grouped_dev(buf.data_ptr(), 0, *args, off.data_ptr(), good.data_ptr(), E, N, K)
            torch.cuda.synchronize()
            assert (buf[R:] == 5).all()
        lib.status()


def test_no_results(lib, pkg):
    a, w = operand(3, 64, 1), operand(5, 64, 2)
    c = torch.full((3, 5), 9.0, device=DEV)
    lib.gemm_mxfp4q_dev(c.data_ptr(), 0, None, None, 0, qmat(pkg, *w))
    lib.gemm_mxfp4q_grouped_dev(c.data_ptr(), 0, None, None, 0, None, 0, None, None, 4, 5, 64)
    off = torch.zeros(3, dtype=torch.int32, device=DEV)
    t = table_of(pkg, w[0].view(1, 5, -1), w[1].view(1, 5, -1)).repeat(2, 1)
    lib.gemm_mxfp4q_grouped_dev(c.data_ptr(), 0, a[0].data_ptr(), a[1].data_ptr(), 3, None, 3, off.data_ptr(), t.data_ptr(),
                                2, 5, 64)
    torch.cuda.synchronize()
    assert (c == 9).all()


def test_tokens_past_4_gib(lib, pkg):
    """A token in the last bytes of 2 GiB of codes: offsets use all of 32 bits."""
    K, n_a, N = 8192, (1 << 19) - 1, 40
    q = torch.zeros(n_a, K // 2, dtype=torch.uint8, device=DEV)
    s = torch.full((n_a, K // 32), 127, dtype=torch.uint8, device=DEV)
    a = operand(3, K, 5)
    at = torch.tensor([0, n_a // 2, n_a - 1], device=DEV)
    q[at], s[at] = a[0], a[1]
    for R in (3, 60, 200, 700):                    # each form
        wq, ws = operand(N, K, 6)
        tok = at.repeat(R // 3 + 1)[:R].to(torch.int32)
        off = torch.tensor([0, R], dtype=torch.int32, device=DEV)
        c = torch.zeros(R, N, device=DEV)
        t = table_of(pkg, wq.view(1, N, -1), ws.view(1, N, -1))
        lib.gemm_mxfp4q_grouped_dev(c.data_ptr(), 0, q.data_ptr(), s.data_ptr(), n_a, tok.data_ptr(), R, off.data_ptr(),
                                    t.data_ptr(), 1, N, K)
        torch.cuda.synchronize()
        want = (values(*a) @ values(wq, ws).t().contiguous()).repeat(R // 3 + 1, 1)[:R]
        most = (values(*a).abs() @ values(wq, ws).abs().t().contiguous()).repeat(R // 3 + 1, 1)[:R]
        assert ((c.double() - want).abs() <= (K / 32 + 16) * 2 * U * most).all()
