# SPDX-License-Identifier: Apache-2.0
"""Int8 rows and int8 products on the GPU against plain 64-bit forms.

Bounds. u = 2^-24 is fp32's half step, relative. Codes are defined by exact
arithmetic: equal. A scale is one rounding of amax / 127 (one u, or half the
smallest subnormal). A product is (float)sum * Sa * s: three roundings of u
each, (1 + u)^3 - 1 < 3.01 u, and an integer sum; a 16-bit output adds its own
half step (bf16 2^-8, fp16 2^-11, or half fp16's smallest subnormal)."""
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


def quant(lib, a, ld=None, k=None, stream=None):
    n, k = a.shape[0], k or a.shape[1]
    q = torch.full((n, k), 99, dtype=torch.int8, device=DEV)
    s = torch.full((n,), 7.0, device=DEV)
    lib.quant_i8_dev(q.data_ptr(), s.data_ptr(), a.data_ptr(), CODE[a.dtype], ld or a.stride(0), n, k, stream)
    return q, s


def swiglu_quant(lib, g, u, limit):
    n, k = g.shape
    q = torch.full((n, k), 99, dtype=torch.int8, device=DEV)
    s = torch.full((n,), 7.0, device=DEV)
    lib.swiglu_quant_i8_dev(q.data_ptr(), s.data_ptr(), g.data_ptr(), u.data_ptr(), CODE[g.dtype], g.stride(0), n, k,
                            limit, None)
    return q, s


def want_codes(v):
    """codes and scales of fp64 rows; a row that is not all finite: NaN and zeros"""
    v = v.cpu().numpy().astype(np.float64)
    ok = np.isfinite(v).all(1)
    amax = np.abs(np.where(ok[:, None], v, 0)).max(1)
    live = ok & (amax > 0)
    x = np.where(live[:, None], v, 0) / np.where(live, amax, 1)[:, None] * 127.0 if (amax > 1e300).any() else \
        np.where(live[:, None], v, 0) * 127.0 / np.where(live, amax, 1)[:, None]
    return np.rint(x).astype(np.int8), np.where(ok, np.where(amax > 0, amax / 127, 1.0), np.nan)


def check_rows(q, s, v):
    qw, sw = want_codes(v)
    np.testing.assert_array_equal(q.cpu().numpy(), qw)
    got = s.cpu().numpy().astype(np.float64)
    fine = np.isfinite(sw)
    assert (np.isnan(got) == ~fine).all()
    assert (np.abs(got - sw)[fine] <= 1.01 * U * sw[fine] + 2.0 ** -150).all()


# ------------------------------------------------------------------- rows ----

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k", [(1, 16), (1, 4096), (3, 48), (33, 1024), (7, 2064), (5, 8192), (2, 8208), (2, 20000),
                                 (1030, 512), (2100, 4112)])
def test_rows(lib, dtype, n, k):
    x = torch.randn(n, k, device=DEV, generator=gen(n + k)).to(dtype)
    check_rows(*quant(lib, x), x.double())


def test_widest_row(lib):
    x = torch.randn(1, 1 << 24, device=DEV, generator=gen(24)).to(torch.bfloat16)
    check_rows(*quant(lib, x), x.double())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k", [64, 4096, 8208])
def test_rows_of_borders(lib, dtype, k):
    """Values at, just below and just above every half step of their row, and ties."""
    n = 40
    amax = torch.linspace(0.3, 9.7, n, dtype=torch.float64, device=DEV).to(dtype).double()
    half = torch.randint(-127, 127, (n, k), device=DEV, generator=gen(k)) + 0.5
    x = (half * amax[:, None] / 127).to(dtype)
    x[:, 0] = amax.to(dtype)
    x[:, 1] = (amax / 2).to(dtype)                 # exactly 63.5 steps: an even 64
    x[:, 2] = (-amax / 2).to(dtype)
    x = torch.where(x.abs() > x[:, :1], x[:, :1], x)
    if dtype == torch.float32:                     # one step of fp32 to either side
        d = torch.randint(-1, 2, (n, k), device=DEV, generator=gen(k + 1), dtype=torch.int32)
        d[:, :3] = 0
        x = (x.view(torch.int32) + d).view(torch.float32)
        x = torch.where(x.abs() > x[:, :1], x[:, :1], x)
    q, s = quant(lib, x)
    assert (q[:, 1] == 64).all() and (q[:, 2] == -64).all()
    check_rows(q, s, x.double())


def test_rows_of_extremes(lib):
    k = 96
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
    q, s = quant(lib, x)
    check_rows(q, s, x.double())
    for r in (4, 5, 6):
        assert torch.isnan(s[r]) and (q[r] == 0).all()
    assert s[0] == 1 and s[7] == 1 and (q[0] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_with_a_pitch(lib, dtype):
    """Rows that lie apart; what lies between them is not read into them."""
    big = torch.full((9, 160), 1e4, device=DEV, dtype=dtype)
    big[:, :112] = torch.randn(9, 112, device=DEV, generator=gen(3)).to(dtype)
    check_rows(*quant(lib, big[:, :112], ld=160, k=112), big[:, :112].double())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("limit", [0.0, 10.0, 0.5])
@pytest.mark.parametrize("n,k", [(1, 16), (3, 2048), (70, 528), (2, 8208), (1100, 2048)])
def test_swiglu_rows(lib, dtype, limit, n, k):
    g, u = (4 * torch.randn(n, k, device=DEV, generator=gen(n + k + i)).to(dtype) for i in range(2))
    check_rows(*swiglu_quant(lib, g, u, limit), swiglu64(g, u, limit))


def swiglu64(g, u, limit):
    g, u = g.double(), u.double()
    lim = float(np.float32(limit))
    if lim > 0:
        g, u = torch.where(g > lim, lim, g), torch.where(u > lim, lim, torch.where(u < -lim, -lim, u))
    return g / (1 + torch.exp(-g)) * u


def test_swiglu_rows_of_extremes(lib):
    k = 64
    g, u = (torch.randn(12, k, device=DEV, generator=gen(i)) for i in range(2))
    g[0], u[0] = 0, 0
    g[1] = -95.0                                   # silu below fp32's normal range
    g[2], u[2] = 1e25, u[2] * 1e25                 # the product beyond fp32
    u[3] = u[3] * 1e-30                            # a row of tiny values
    g[4, 9] = float("nan")
    u[5, 2] = float("inf")
    g[6, 1] = -float("inf")                        # silu(-inf) is -inf / inf
    g[7] = -60.0
    u[8] = 3e38
    g[9, 5] = 88.0
    q, s = swiglu_quant(lib, g, u, 0.0)
    v = swiglu64(g, u, 0.0)
    qw, sw = want_codes(v)
    np.testing.assert_array_equal(q.cpu().numpy(), qw)
    got = s.cpu().numpy().astype(np.float64)
    for r in range(12):
        if np.isnan(sw[r]) or sw[r] > 3.5e38:
            assert not np.isfinite(got[r])
        else:
            assert abs(got[r] - sw[r]) <= 1.01 * U * sw[r] + 2.0 ** -150
    assert np.isnan(got[4]) and np.isnan(got[5]) and np.isnan(got[6])
    # the clamp makes infinities finite
    q, s = swiglu_quant(lib, g, u, 10.0)
    check_rows(q, s, swiglu64(g, u, 10.0))
    assert torch.isfinite(s[5])


def test_swiglu_halves_of_one_array(lib):
    gu = torch.randn(6, 2 * 80, device=DEV, generator=gen(8)).to(torch.bfloat16)
    g, u = gu[:, :80], gu[:, 80:]
    check_rows(*swiglu_quant(lib, g, u, 10.0), swiglu64(g, u, 10.0))


# ---------------------------------------------------------------- product ----

def operands(n_a, N, K, seed, full=False):
    g = gen(seed)
    lo, hi = (-128, 128) if full else (-127, 128)
    a = torch.randint(lo, hi, (n_a, K), dtype=torch.int8, device=DEV, generator=g)
    w = torch.randint(lo, hi, (N, K), dtype=torch.int8, device=DEV, generator=g)
    sa = 0.01 + torch.rand(n_a, device=DEV, generator=g)
    sw = (0.01 + torch.rand(N, device=DEV, generator=g)) / K
    return a, sa, w, sw


def close(got, a, sa, w, sw):
    """got against sums of codes that fp64 holds exactly"""
    acc = a.double() @ w.double().t().contiguous()
    want = acc * sa.double()[:, None] * sw.double()[None]
    bound = want.abs() * (HALF[got.dtype] * (1 + 4 * U) + 3.01 * U) + TINY[got.dtype]
    assert ((got.double() - want).abs() <= bound).all()


def run_gemm(lib, pkg, a, sa, w, sw, dtype, stream=None, C=None):
    M, N = a.shape[0], w.shape[0]
    pad = 64
    if C is None:
        buf = torch.full((M * N + 2 * pad,), 7.0, dtype=dtype, device=DEV)
        C = buf[pad:pad + M * N].view(M, N)
    d = pkg.qmat(pkg.DSV4_WI8, w.data_ptr(), sw.data_ptr(), N, w.shape[1], 1, w.shape[1])
    lib.gemm_i8_dev(C.data_ptr(), CODE[dtype], a.data_ptr(), sa.data_ptr(), M, d, stream)
    if stream is None and C.storage_offset() == pad:
        assert (buf[:pad] == 7).all() and (buf[-pad:] == 7).all()      # nothing beyond C
    return C


SHAPES = [(1, 4096, 4096), (1, 1, 16), (1, 17, 48), (2, 255, 1040), (5, 300, 512), (7, 4096, 1024), (8, 130, 2064),
          (9, 64, 128), (15, 33, 4096), (16, 16, 64), (17, 257, 80), (31, 1024, 144), (33, 515, 1024), (63, 48, 272),
          (64, 64, 4096), (65, 129, 96), (100, 1000, 512), (129, 128, 128), (130, 384, 1136), (257, 260, 2048),
          (300, 1024, 4096), (333, 777, 4112), (512, 513, 640), (1000, 1023, 208), (2048, 256, 1024),
          (701, 2048, 4096), (1300, 1536, 16), (3, 5, 16384), (2, 40000, 256), (4097, 100, 192), (2051, 4099, 528),
          (1000, 4096, 528), (1025, 4080, 272), (2048, 4096, 4096), (2050, 4100, 1040), (40, 32768, 1024), (14, 700, 8208),
          (1000, 4095, 4096)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product(lib, pkg, M, N, K):
    dtype = TYPES[(M + N) % 3]
    a, sa, w, sw = operands(M, N, K, M + N + K)
    close(run_gemm(lib, pkg, a, sa, w, sw, dtype), a, sa, w, sw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,N,K", [(1, 512, 4096), (13, 513, 272), (70, 254, 512), (300, 515, 1024), (520, 1030, 144)])
def test_product_of_every_type(lib, pkg, dtype, M, N, K):
    a, sa, w, sw = operands(M, N, K, 3 * M)
    close(run_gemm(lib, pkg, a, sa, w, sw, dtype), a, sa, w, sw)


@pytest.mark.parametrize("M", [1, 20, 200])
@pytest.mark.parametrize("K", [4096, 131056])
def test_product_of_extreme_codes(lib, pkg, M, K):
    """-128 times -128 everywhere: the largest sum that the widest rows reach."""
    a = torch.full((M, K), -128, dtype=torch.int8, device=DEV)
    w = torch.full((140, K), -128, dtype=torch.int8, device=DEV)
    w[1::2] = 127
    sa, sw = torch.ones(M, device=DEV), torch.ones(140, device=DEV)
    close(run_gemm(lib, pkg, a, sa, w, sw, torch.float32), a, sa, w, sw)


def test_product_nan_scale_makes_its_row_nan(lib, pkg):
    a, sa, w, sw = operands(40, 200, 256, 1)
    sa[7] = float("nan")
    c = run_gemm(lib, pkg, a, sa, w, sw, torch.bfloat16)
    assert torch.isnan(c[7]).all() and torch.isfinite(c[:7]).all() and torch.isfinite(c[8:]).all()


def test_product_beyond_fp16_is_infinite(lib, pkg):
    a = torch.full((3, 64), 127, dtype=torch.int8, device=DEV)
    w = torch.full((20, 64), 127, dtype=torch.int8, device=DEV)
    w[1] = -127
    one = torch.ones(20, device=DEV)
    c = run_gemm(lib, pkg, a, one[:3], w, one, torch.float16)
    assert (c[:, 0] == float("inf")).all() and (c[:, 1] == -float("inf")).all()


@pytest.mark.parametrize("M", [1, 5, 16, 17, 64, 200, 333])
def test_rows_of_a_product_do_not_depend_on_their_number(lib, pkg, M):
    """Sums are exact, so every form gives one row the same bits."""
    a, sa, w, sw = operands(400, 515, 1040, 77)
    full = run_gemm(lib, pkg, a, sa, w, sw, torch.float32)
    part = run_gemm(lib, pkg, a[:M].contiguous(), sa[:M].contiguous(), w, sw, torch.float32)
    assert torch.equal(part, full[:M])


def test_product_on_streams_and_in_a_graph(lib, pkg):
    """Two calls at once on streams of their own, then one captured and
    replayed with other work between: none shares anything with another."""
    ops = [operands(M, 1030, 2064, M) for M in (3, 260)]
    want = [run_gemm(lib, pkg, *o, torch.bfloat16).clone() for o in ops]
    outs = [torch.zeros_like(x) for x in want]
    streams = [torch.cuda.Stream() for _ in ops]
    torch.cuda.synchronize()
    for _ in range(5):
        for o, c, s in zip(ops, outs, streams):
            run_gemm(lib, pkg, *o, torch.bfloat16, stream=s.cuda_stream, C=c)
    torch.cuda.synchronize()
    for c, x in zip(outs, want):
        assert torch.equal(c, x)
    a, sa, w, sw = ops[1]
    x = torch.randn(260, 2064, device=DEV, generator=gen(1))
    q, s, c = torch.empty_like(a), torch.empty_like(sa), torch.empty_like(want[1])
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.graph(g, stream=side):
        h = torch.cuda.current_stream().cuda_stream
        lib.quant_i8_dev(q.data_ptr(), s.data_ptr(), x.data_ptr(), 0, 2064, 260, 2064, h)
        run_gemm(lib, pkg, q, s, w, sw, torch.bfloat16, stream=h, C=c)
    for i in range(4):
        x.copy_(torch.randn(260, 2064, device=DEV, generator=gen(10 + i)))
        g.replay()
        torch.cuda.synchronize()
        q2, s2 = quant(lib, x)
        assert torch.equal(q2, q) and torch.equal(s2, s)
        assert torch.equal(c, run_gemm(lib, pkg, q2, s2, w, sw, torch.bfloat16))


# ------------------------------------------------------- experts' product ----

def table_of(pkg, w, sw):
    """a device table of descriptors of w [E][N][K], sw [E][N]"""
    E, N, K = w.shape
    t = (pkg.QMat * E)(*[pkg.qmat(pkg.DSV4_WI8, w[e].data_ptr(), sw[e].data_ptr(), N, K, 1, K) for e in range(E)])
    return torch.frombuffer(bytearray(bytes(t)), dtype=torch.uint8).to(DEV)


def run_grouped(lib, pkg, a, sa, off, row_tok, n_rows, w, sw, dtype, table=None, E=None, stream=None):
    _, N, K = w.shape
    C = torch.full((n_rows + 2, N), 7.0, dtype=dtype, device=DEV)
    table = table_of(pkg, w, sw) if table is None else table
    lib.gemm_i8_grouped_dev(C[1:].data_ptr(), CODE[dtype], a.data_ptr(), sa.data_ptr(), a.shape[0],
                            None if row_tok is None else row_tok.data_ptr(), n_rows, off.data_ptr(), table.data_ptr(),
                            E or w.shape[0], N, K, stream)
    torch.cuda.synchronize()
    assert (C[0] == 7).all() and (C[-1] == 7).all()
    return C[1:-1]


def buckets(counts):
    off = torch.zeros(len(counts) + 1, dtype=torch.int32)
    off[1:] = torch.tensor(counts, dtype=torch.int32).cumsum(0)
    return off


GROUPS = [([0, 0, 1, 0], 40, 64), ([3, 0, 17, 5, 64, 1], 130, 272), ([65, 0, 128, 129], 257, 512), ([300], 100, 1040),
          ([0] * 70 + [2] + [0] * 60 + [1, 1, 40], 48, 128), ([1] * 256, 64, 4096), ([2, 1] * 500, 33, 48),
          ([700, 3, 0, 0, 40, 1], 515, 2048), ([0, 0], 16, 16), ([16, 15, 17, 33, 31, 32], 512, 144),
          ([100, 90, 110, 95] * 4, 1024, 640), ([1, 0, 3, 16, 2, 9, 40, 1] * 8, 1030, 1040),
          ([0, 7, 20, 1] * 16, 1024, 2064),
          ([40, 0, 30, 50, 65], 300, 272), ([100, 64, 140, 90], 4100, 4112), ([120, 128, 0, 131] * 16, 510, 1024), ([2500, 3, 0, 300], 2100, 8208),
          ([1, 0, 1200, 0, 60, 200, 1100] * 3, 781, 4112), ([1, 0, 2] * 341 + [4], 40, 2064),
          ([0] * 1023 + [70], 48, 512), ([5] + [0] * 64, 100, 528), ([0, 3] * 32, 513, 2064), ([40] * 1024, 300, 272)]


@pytest.mark.parametrize("case", range(len(GROUPS)))
@pytest.mark.parametrize("mapped", [True, False])
def test_experts_product(lib, pkg, case, mapped):
    counts, N, K = GROUPS[case]
    E, R = len(counts), sum(counts)
    dtype = TYPES[(case + mapped) % 3]
    extra = 5                                      # rows of dropped pairs behind the last bucket
    off = buckets(counts)
    n_a = max(1, R // 3 + 1) if mapped else R + extra
    a, sa, _, _ = operands(n_a, 1, K, case)
    _, _, w, sw = operands(1, E * N, K, case + 100)
    w, sw = w.view(E, N, K), sw.view(E, N)
    tok = torch.randint(0, n_a, (R + extra,), dtype=torch.int32, generator=torch.Generator().manual_seed(case))
    C = run_grouped(lib, pkg, a, sa, off.to(DEV), tok.to(DEV) if mapped else None, R + extra, w, sw, dtype)
    assert (C[R:] == 7).all()
    src = tok if mapped else torch.arange(R + extra)
    for e in range(E):
        lo, hi = int(off[e]), int(off[e + 1])
        if hi > lo:
            i = src[lo:hi].long().to(DEV)
            close(C[lo:hi], a[i], sa[i], w[e], sw[e])
    assert lib.status() == 0


def test_experts_product_reports_bad_rows_and_matrices(lib, pkg):
    E, N, K, R = 4, 70, 128, 50
    a, sa, _, _ = operands(20, 1, K, 1)
    _, _, w, sw = operands(1, E * N, K, 2)
    w, sw = w.view(E, N, K), sw.view(E, N)
    off = buckets([10, 15, 5, 20]).to(DEV)
    tok = torch.randint(0, 20, (R,), dtype=torch.int32).to(DEV)
    lib.status()
    want = run_grouped(lib, pkg, a, sa, off, tok, R, w, sw, torch.float32)
    bad = tok.clone()
    bad[3], bad[30], bad[49] = 20, -1, 1 << 30
    got = run_grouped(lib, pkg, a, sa, off, bad, R, w, sw, torch.float32)
    assert lib.status() == 1
    keep = torch.ones(R, dtype=torch.bool, device=DEV)
    keep[[3, 30, 49]] = False
    assert torch.isnan(got[~keep]).all() and torch.equal(got[keep], want[keep])
    for field, value in (("wdt", pkg.DSV4_WFP8), ("rows", N + 1), ("cols", K * 2), ("w", None), ("s", None)):
        ms = [pkg.qmat(pkg.DSV4_WI8, w[e].data_ptr(), sw[e].data_ptr(), N, K, 1, K) for e in range(E)]
        setattr(ms[1], field, value)
        t = torch.frombuffer(bytearray(bytes((pkg.QMat * E)(*ms))), dtype=torch.uint8).to(DEV)
        got = run_grouped(lib, pkg, a, sa, off, tok, R, w, sw, torch.float32, table=t)
        assert lib.status() == 2
        assert torch.isnan(got[10:25]).all()
        assert torch.equal(got[:10], want[:10]) and torch.equal(got[25:], want[25:])


def test_experts_product_stays_in_bounds_with_bad_offsets(lib, pkg):
    """Offsets beyond the rows, falling or negative: some rows are written,
    none outside C (the kernel clamps each to the rows there are)."""
    E, N, K, R = 5, 40, 64, 30
    a, sa, _, _ = operands(R, 1, K, 1)
    _, _, w, sw = operands(1, E * N, K, 2)
    w, sw = w.view(E, N, K), sw.view(E, N)
    for off in ([0, 10, 5, 1 << 30, 20, 25], [-50, -1, 3, 3, 2, 900], [30, 30, 30, 30, 30, 30]):
        run_grouped(lib, pkg, a, sa, torch.tensor(off, dtype=torch.int32, device=DEV), None, R, w, sw, torch.float32)
    lib.status()


def test_large_experts_product_stays_in_bounds_with_bad_offsets(lib, pkg):
    E, N, K, R = 5, 1701, 8208, 2900
    a, sa, _, _ = operands(R, 1, K, 1)
    _, _, w, sw = operands(1, E * N, K, 2)
    w, sw = w.view(E, N, K), sw.view(E, N)
    for off in ([0, 1000, 500, 1 << 30, 2000, 2500], [-50, -1, 300, 300, 200, 90000], [R, 0, R, 0, R, 0],
                [0, R, 0, R, 0, R], [-(1 << 31), (1 << 31) - 1, -(1 << 31), (1 << 31) - 1, 0, R]):
        run_grouped(lib, pkg, a, sa, torch.tensor(off, dtype=torch.int32, device=DEV), None, R, w, sw, torch.float32)
    lib.status()


# ------------------------------------------------------------- large sizes ----

def test_product_beyond_4_gib(lib, pkg):
    """Results, then tokens, of more than 2^32 bytes: the last rows are right."""
    M, N, K = 300001, 8192, 64
    a, sa, w, sw = operands(M, N, K, 1)
    C = torch.empty(M, N, dtype=torch.bfloat16, device=DEV)
    run_gemm(lib, pkg, a, sa, w, sw, torch.bfloat16, C=C)
    for r in (slice(0, 40), slice(262100, 262200), slice(M - 70, M)):
        close(C[r], a[r], sa[r], w, sw)
    del C
    M, N, K = 1100003, 24, 4096
    a, sa, w, sw = operands(M, N, K, 2)
    C = run_gemm(lib, pkg, a, sa, w, sw, torch.float32)
    for r in (slice(0, 40), slice(1048500, 1048700), slice(M - 70, M)):
        close(C[r], a[r], sa[r], w, sw)


def test_experts_product_beyond_4_gib(lib, pkg):
    R, N, K = 300001, 8192, 64
    a, sa, w, sw = operands(1000, 2 * N, K, 3)
    w, sw = w.view(2, N, K), sw.view(2, N)
    off = buckets([270000, R - 270000]).to(DEV)
    tok = torch.randint(0, 1000, (R,), dtype=torch.int32, device=DEV, generator=gen(4))
    C = run_grouped(lib, pkg, a, sa, off, tok, R, w, sw, torch.bfloat16)
    for e, r in ((0, slice(0, 40)), (0, slice(269900, 270000)), (1, slice(270000, 270100)), (1, slice(R - 70, R))):
        i = tok[r].long()
        close(C[r], a[i], sa[i], w[e], sw[e])


def test_rows_beyond_4_gib(lib):
    n, k = 300001, 8192
    x = torch.empty(n, k, dtype=torch.bfloat16, device=DEV).normal_(generator=gen(5))
    q, s = quant(lib, x)
    for r in (slice(0, 8), slice(262140, 262150), slice(n - 8, n)):
        check_rows(q[r], s[r], x[r].double())


def test_too_large_for_a_launch_is_refused(lib, pkg):
    """and leaves the library alive"""
    a, sa, w, sw = operands(2, 3, 16, 6)
    c = torch.empty(2, 3, device=DEV)
    d = pkg.qmat(pkg.DSV4_WI8, w.data_ptr(), sw.data_ptr(), 1 << 20, 16, 1, 16)
    for m in ((1 << 31) - 1, 1 << 28):
        with pytest.raises(pkg.Dsv4Error, match="too many"):
            lib.gemm_i8_dev(c.data_ptr(), 0, a.data_ptr(), sa.data_ptr(), m, d)
    with pytest.raises(pkg.Dsv4Error, match="too many"):
        lib.quant_i8_dev(a.data_ptr(), sa.data_ptr(), w.data_ptr(), 0, 16, 1 << 30, 16)
    close(run_gemm(lib, pkg, a, sa, w, sw, torch.float32), a, sa, w, sw)


def test_other_calls_refuse_int8_weights(lib, pkg):
    """fp32 tokens have no exact product with them: the drop-in matmul and the
    dequantizer know only the packed formats."""
    _, _, w, sw = operands(1, 128, 128, 7)
    x, y = torch.zeros(128, device=DEV), torch.zeros(128 * 128, device=DEV)
    d = pkg.qmat(pkg.DSV4_WI8, w.data_ptr(), sw.data_ptr(), 128, 128, 1, 128)
    for call in (lambda: lib.mmq_n_dev(y.data_ptr(), x.data_ptr(), d, 1), lambda: lib.dequant_dev(y.data_ptr(), d),
                 lambda: lib.gemm_fp8_dev(y.data_ptr(), False, x.data_ptr(), False, 1, d)):
        with pytest.raises(pkg.Dsv4Error):
            call()
