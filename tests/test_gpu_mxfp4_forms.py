# SPDX-License-Identifier: Apache-2.0
"""Every form of the 4-bit experts' product (the rules that pick it are held to FAR
and BAD in test_mxfp4_forms.py) with tokens all over 2 GiB of codes, with table
entries that are no matrix of the product, and with tokens and offsets out of
range. Sums are exact as in test_gpu_mxfp4.py: products are multiples of 2^-4, and
their magnitudes add up to less than 2^20."""
import numpy as np
import pytest
import torch

from test_gpu_mxfp4 import DEV, gen, operand, table_of, values

pytestmark = pytest.mark.gpu

FAR = [([60], 40, 8192), ([9, 1, 0, 5, 2, 9, 3, 11], 4111, 8192), ([3, 0] * 50, 333, 1120), ([1] * 40, 4111, 8192),
       ([333], 2051, 8192), ([60, 33, 0, 1, 20, 40, 31, 15], 4111, 8192), ([1300], 4111, 8192), ([2100], 4111, 8192)]
BAD = [([30, 200, 0, 129, 70, 33], 130, 160), ([9, 1, 0, 5, 2, 9, 3, 11], 4111, 8192), ([20, 30, 25, 7, 41], 40, 160),
       ([5, 0, 9, 1, 12, 0, 3] * 9, 2051, 4128), ([200, 300, 250, 60], 300, 96), ([60, 33, 0, 1, 20, 40, 31, 15], 4111, 8192),
       ([400, 700, 130, 260, 500, 31], 1030, 160), ([300, 1000, 200, 129, 700, 513], 4111, 160)]


def offsets(counts):
    return torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device=DEV)


def experts(counts, N, K, seed):
    wq, ws = operand(len(counts) * N, K, seed)
    return wq.view(len(counts), N, -1), ws.view(len(counts), N, -1)


def want_rows(va, w, counts, tok):
    """fp64 products of the rows, expert by expert"""
    out = torch.zeros(len(tok), w[0].shape[1], dtype=torch.float64, device=DEV)
    r = 0
    for e, n in enumerate(counts):
        if n:
            vw = values(w[0][e], w[1][e]).t().contiguous()
            x = va[tok[r:r + n]]
            out[r:r + n] = x @ vw
            assert float((x.abs() @ vw.abs()).max()) < 2 ** 20
        r += n
    return out


@pytest.mark.parametrize("counts,N,K", FAR)
def test_tokens_all_over_2_gib(lib, pkg, counts, N, K):
    """the first, the middle and the last of as many tokens as a call takes"""
    R, n_a = sum(counts), (2 ** 32 - 1) // K
    q = torch.zeros(n_a, K // 2, dtype=torch.uint8, device=DEV)
    s = torch.full((n_a, K // 32), 127, dtype=torch.uint8, device=DEV)
    a = operand(3, K, 5)
    at = torch.tensor([0, n_a // 2, n_a - 1], device=DEV)
    q[at], s[at] = a[0], a[1]
    w = experts(counts, N, K, 6)
    pick = torch.randint(0, 3, (R,), device=DEV, generator=gen(R))
    tok, off, t = at[pick].to(torch.int32), offsets(counts), table_of(pkg, *w)
    c = torch.full((R + 1, N), 77.0, device=DEV)
    lib.status()
    lib.gemm_mxfp4q_grouped_dev(c.data_ptr(), 0, q.data_ptr(), s.data_ptr(), n_a, tok.data_ptr(), R, off.data_ptr(),
                                t.data_ptr(), len(counts), N, K)
    torch.cuda.synchronize()
    assert lib.status() == 0 and (c[R] == 77).all()
    assert torch.equal(c[:R].double(), want_rows(values(*a), w, counts, pick))


@pytest.mark.parametrize("counts,N,K", BAD)
def test_bad_descriptors(lib, pkg, counts, N, K):
    """Another type, size or block, no pointer or one off alignment: bit 1 and rows of NaN, the
    other experts' rows as they are."""
    E, R = len(counts), sum(counts)
    w, a = experts(counts, N, K, 3), operand(50, K, 10)
    good, off = table_of(pkg, *w), offsets(counts)
    tok = torch.randint(0, 50, (R,), device=DEV, generator=gen(1), dtype=torch.int32)
    want = want_rows(values(*a), w, counts, tok.long())
    one = 1 + int(np.argmax(counts[1:]))           # the largest bucket but for the first
    lo, hi = sum(counts[:one]), sum(counts[:one + 1])
    for field, value in ((2, 5 + (N << 32)), (2, 3 + ((N + 1) << 32)), (3, K + 32 + (1 << 32)), (3, K + (128 << 32)),
                         (4, 128), (0, 0), (1, 0), (0, int(good[one, 0]) + 8)):
        t = good.clone()
        t[one, field] = value
        c = torch.full((R + 1, N), 77.0, device=DEV)
        lib.status()
        lib.gemm_mxfp4q_grouped_dev(c.data_ptr(), 0, a[0].data_ptr(), a[1].data_ptr(), 50, tok.data_ptr(), R, off.data_ptr(),
                                    t.data_ptr(), E, N, K)
        torch.cuda.synchronize()
        assert lib.status() == 2
        assert torch.isnan(c[lo:hi]).all() and (c[R] == 77).all()
        assert torch.equal(c[:lo].double(), want[:lo]) and torch.equal(c[hi:R].double(), want[hi:])


@pytest.mark.parametrize("counts,N,K", BAD)
def test_tokens_and_offsets_out_of_range(lib, pkg, counts, N, K):
    """Tokens: bit 0 and a row of NaN each. Offsets that fall, lie below 0 or past the rows: nothing is
    written outside the rows."""
    E, R = len(counts), sum(counts)
    w, a = experts(counts, N, K, 3), operand(50, K, 10)
    t, off = table_of(pkg, *w), offsets(counts)
    tok = torch.randint(0, 50, (R,), device=DEV, generator=gen(1), dtype=torch.int32)
    want = want_rows(values(*a), w, counts, tok.long())
    nan = torch.zeros(R, dtype=torch.bool, device=DEV)
    for r, v in ((0, 50), (2, -1), (R // 2, 2 ** 31 - 1), (R - 1, -2 ** 31)):
        tok[r], nan[r] = v, True
    buf = torch.full((R + 16, N), 5.0, device=DEV)
    args = (0, a[0].data_ptr(), a[1].data_ptr(), 50, tok.data_ptr(), R)
    lib.status()
    lib.gemm_mxfp4q_grouped_dev(buf[8].data_ptr(), *args, off.data_ptr(), t.data_ptr(), E, N, K)
    torch.cuda.synchronize()
    assert lib.status() == 1
    c = buf[8:8 + R]
    assert torch.isnan(c[nan]).all() and torch.equal(c[~nan].double(), want[~nan])
    falls = [R if e % 2 else 0 for e in range(E + 1)]
    for bad in (falls, falls[::-1], [R + 900] + falls[1:], [-5] * E + [R], list(range(R, R - E - 1, -1)),
                [2 ** 31 - 1 if e % 2 else -2 ** 31 for e in range(E + 1)]):
        b = torch.tensor(bad, dtype=torch.int32, device=DEV)
        lib.gemm_mxfp4q_grouped_dev(buf[8].data_ptr(), *args, b.data_ptr(), t.data_ptr(), E, N, K)
        torch.cuda.synchronize()
        assert (buf[:8] == 5).all() and (buf[8 + R:] == 5).all()
    lib.status()
