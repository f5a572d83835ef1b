# SPDX-License-Identifier: Apache-2.0
"""Every form of the int8 products, in every output type, at the sizes where a
form can go wrong: rows, features and blocks of K that end inside a tile, the
widest rows, code -128, results off 16-byte addresses, and the errors that the
device reports. tests/test_i8_choice.py holds each case to the form it names."""
import pytest
import torch

from test_gpu_i8 import DEV, TYPES, buckets, close, operands, run_gemm, run_grouped, table_of

pytestmark = pytest.mark.gpu

# form: (M, N, K), each with a remainder of rows, features and K
ONE = {"pair": [(13, 515, 2064), (14, 700, 8208)], "64x2": [(333, 515, 208), (213, 517, 336)],
       "64x2 deep": [(333, 515, 1040), (209, 1030, 4112)], "64x4": [(333, 2100, 1040), (520, 1030, 4112)],
       "128x4": [(520, 2100, 1040), (1000, 1030, 4112)], "128x8": [(1030, 2100, 1040), (2047, 1030, 4112)],
       "256x8": [(2047, 2100, 4112), (2047, 4001, 1040)]}

# the widest rows
WIDE = {"pair": (20, 500), "64x2": (200, 4104), "64x2 deep": (200, 248), "64x4": (520, 1030), "128x4": (520, 2100),
        "128x8": (1030, 2100), "256x8": (2050, 2100)}
KMAX = 131056

# rows of one product, by the form that their number takes
SLICES_N, SLICES_K = 4104, 1040
SLICES = {"pair": 1, "64x2 deep": 17, "64x4": 130, "64x2": 200, "128x4": 260, "128x8": 600, "256x8": 1000}

# rows that divide into 16-byte pieces
EVEN = {"pair": (13, 512, 1024), "64x2": (333, 520, 208), "64x2 deep": (333, 512, 1040), "64x4": (333, 2104, 1040),
        "128x4": (520, 2104, 1040), "128x8": (1030, 2104, 1040), "256x8": (2047, 2104, 4112)}

# form: (rows of each expert, N, K)
GROUPED = {"pair": ([9, 10, 0, 11, 10, 10, 5], 2100, 8208), "64x2": ([20, 0, 17, 19, 4], 2100, 8208),
           "128x4": ([25, 33, 0, 26, 24], 2100, 8208), "256x8": ([80, 175, 0, 130, 65], 2100, 8208)}
GROUPED_WIDE = {"pair": ([9, 10, 0, 6], 300, KMAX), "64x2": ([20, 0, 33, 17], 300, KMAX),
                "128x4": ([50, 65, 40, 16], 300, KMAX), "256x8": ([300, 0, 170, 260], 300, KMAX)}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form,i", [(f, i) for f in ONE for i in range(len(ONE[f]))])
def test_every_form_in_every_type(lib, pkg, form, i, dtype):
    M, N, K = ONE[form][i]
    a, sa, w, sw = operands(M, N, K, M + N + K, full=True)
    close(run_gemm(lib, pkg, a, sa, w, sw, dtype), a, sa, w, sw)


@pytest.mark.parametrize("form", WIDE)
def test_widest_rows_and_lowest_codes(lib, pkg, form):
    """-128 by -128 throughout, the largest sum there is, then codes of the
    whole range."""
    M, N = WIDE[form]
    a = torch.full((M, KMAX), -128, dtype=torch.int8, device=DEV)
    w = torch.full((N, KMAX), -128, dtype=torch.int8, device=DEV)
    w[1::2] = 127
    sa, sw = torch.ones(M, device=DEV), torch.ones(N, device=DEV)
    close(run_gemm(lib, pkg, a, sa, w, sw, torch.float32), a, sa, w, sw)
    a, sa, w, sw = operands(M, N, KMAX, M, full=True)
    close(run_gemm(lib, pkg, a, sa, w, sw, torch.float32), a, sa, w, sw)


@pytest.fixture(scope="module")
def whole(lib, pkg):
    ops = operands(1500, SLICES_N, SLICES_K, 77, full=True)
    return ops, run_gemm(lib, pkg, *ops, torch.float32).clone()


@pytest.mark.parametrize("form", SLICES)
def test_every_form_gives_one_row_the_same_bits(lib, pkg, whole, form):
    (a, sa, w, sw), full = whole
    M = SLICES[form]
    for lo in (0, 1500 - M):
        part = run_gemm(lib, pkg, a[lo:lo + M].contiguous(), sa[lo:lo + M].contiguous(), w, sw, torch.float32)
        assert torch.equal(part, full[lo:lo + M])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", EVEN)
def test_results_off_a_16_byte_address(lib, pkg, form, dtype):
    """C begins one element behind a boundary though its rows are whole pieces."""
    M, N, K = EVEN[form]
    a, sa, w, sw = operands(M, N, K, N)
    want = run_gemm(lib, pkg, a, sa, w, sw, dtype)
    for shift in (1, 16 // want.element_size() - 1):
        buf = torch.full((M * N + 64,), 7.0, dtype=dtype, device=DEV)
        C = buf[shift:shift + M * N].view(M, N)
        assert C.data_ptr() % 16
        run_gemm(lib, pkg, a, sa, w, sw, dtype, C=C)
        torch.cuda.synchronize()
        assert (buf[:shift] == 7).all() and (buf[shift + M * N:] == 7).all()
        assert torch.equal(C, want)


def experts(case, seed, n_a):
    counts, N, K = case
    E = len(counts)
    a, sa, _, _ = operands(n_a, 1, K, seed, full=True)
    _, _, w, sw = operands(1, E * N, K, seed + 1, full=True)
    return a, sa, w.view(E, N, K), sw.view(E, N)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("form", GROUPED)
@pytest.mark.parametrize("mapped", [True, False])
def test_every_form_of_the_experts_product(lib, pkg, form, mapped, dtype):
    counts, N, K = GROUPED[form]
    R, off = sum(counts), buckets(counts)
    n_a = R // 2 + 1 if mapped else R
    a, sa, w, sw = experts(GROUPED[form], R, n_a)
    tok = torch.randint(0, n_a, (R,), dtype=torch.int32, generator=torch.Generator().manual_seed(R))
    C = run_grouped(lib, pkg, a, sa, off.to(DEV), tok.to(DEV) if mapped else None, R, w, sw, dtype)
    src = (tok if mapped else torch.arange(R)).long().to(DEV)
    for e in range(len(counts)):
        i = src[int(off[e]):int(off[e + 1])]
        close(C[int(off[e]):int(off[e + 1])], a[i], sa[i], w[e], sw[e])
    assert lib.status() == 0


@pytest.mark.parametrize("form", GROUPED_WIDE)
def test_widest_rows_of_the_experts_product(lib, pkg, form):
    counts, N, K = GROUPED_WIDE[form]
    R, off = sum(counts), buckets(counts)
    a, sa, w, sw = experts(GROUPED_WIDE[form], R, R)
    a[0], w[0, ::2], w[0, 1::2] = -128, -128, 127
    C = run_grouped(lib, pkg, a, sa, off.to(DEV), None, R, w, sw, torch.float32)
    for e in range(len(counts)):
        r = slice(int(off[e]), int(off[e + 1]))
        close(C[r], a[r], sa[r], w[e], sw[e])
    assert lib.status() == 0


@pytest.mark.parametrize("form", GROUPED)
def test_every_form_reports_bad_rows_and_matrices(lib, pkg, form):
    counts, N, K = GROUPED[form]
    E, R, off = len(counts), sum(counts), buckets(counts)
    a, sa, w, sw = experts(GROUPED[form], 3, 20)
    tok = torch.randint(0, 20, (R,), dtype=torch.int32, generator=torch.Generator().manual_seed(3)).to(DEV)
    off_d, lo, hi = off.to(DEV), int(off[1]), int(off[2])
    b = 1 if hi > lo else 3                        # an expert that has rows
    lo, hi = int(off[b]), int(off[b + 1])
    lib.status()
    want = run_grouped(lib, pkg, a, sa, off_d, tok, R, w, sw, torch.float32)
    assert lib.status() == 0
    bad, at = tok.clone(), [0, R // 2, R - 1]
    bad[at[0]], bad[at[1]], bad[at[2]] = 20, -1, 1 << 30
    got = run_grouped(lib, pkg, a, sa, off_d, bad, R, w, sw, torch.float32)
    assert lib.status() == 1
    keep = torch.ones(R, dtype=torch.bool, device=DEV)
    keep[at] = False
    assert torch.isnan(got[~keep]).all() and torch.equal(got[keep], want[keep])
    for field, value in (("wdt", pkg.DSV4_WFP8), ("rows", N + 1), ("cols", K * 2), ("w", None), ("s", None),
                         ("w", w[b].data_ptr() + 8), ("s", sw[b].data_ptr() + 2)):
        ms = [pkg.qmat(pkg.DSV4_WI8, w[e].data_ptr(), sw[e].data_ptr(), N, K, 1, K) for e in range(E)]
        setattr(ms[b], field, value)
        t = torch.frombuffer(bytearray(bytes((pkg.QMat * E)(*ms))), dtype=torch.uint8).to(DEV)
        got = run_grouped(lib, pkg, a, sa, off_d, tok, R, w, sw, torch.float32, table=t)
        assert lib.status() == 2
        assert torch.isnan(got[lo:hi]).all()
        assert torch.equal(got[:lo], want[:lo]) and torch.equal(got[hi:], want[hi:])


@pytest.mark.parametrize("form", GROUPED)
def test_every_form_stays_in_bounds_with_bad_offsets(lib, pkg, form):
    counts, N, K = GROUPED[form]
    E, R = len(counts), sum(counts)
    a, sa, w, sw = experts(GROUPED[form], 5, R)
    table = table_of(pkg, w, sw)
    half, big = R // 2, (1 << 31) - 1
    for head in ([0, half, half // 2, 1 << 30, R], [-50, -1, half, 3, 90000], [R, 0, R, 0, R], [0, R, 0, R, 0],
                 [-big - 1, big, -big - 1, big, 0]):
        off = torch.tensor((head + [R] * E)[:E + 1], dtype=torch.int32, device=DEV)
        run_grouped(lib, pkg, a, sa, off, None, R, w, sw, torch.bfloat16, table=table)
    lib.status()
