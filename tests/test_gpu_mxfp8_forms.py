"""Every form of the MXFP8 products (q3_matmul_mxfp8_form) on the GPU: which one takes a call is a rule on its sizes, so
each case here names the form that it is for, and a test without a GPU holds the cases to it.

The inputs are those whose products and sums the matrix instruction forms exactly (tests/test_gpu_mxfp8.py): results are
the correctly rounded float64 ones, and in SwiGLU and behind an activation within the arithmetic after the sums.
"""
import ctypes

import pytest
import torch

from oracle import mxfp8 as M
from qwen3_5_vl_cuda_custom_amd import _lib
from qwen3_5_vl_cuda_custom_amd import kernels as K

from .test_gpu_mxfp8 import DEV, HALF, act_of, check_eight_bits, dev, exact_pair, rnd

ROWS, RING, T256, T128X256, T128, T128_BY_ROWS = range(6)

# (form, m, n, k): the row counts of each ring, odd and even numbers of stages of 128 k (and of 512), ends inside a stage
# (k no multiple of 128), inside four stages and at their end, remainders of m and n
PLAIN = [
    (ROWS, 5, 70, 96), (ROWS, 40, 333, 1056),
    (RING, 3, 70, 640), (RING, 12, 71, 128), (RING, 30, 200, 1152), (RING, 64, 130, 1664), (RING, 150, 301, 640),
    (T256, 3301, 4103, 160), (T256, 3301, 4103, 384), (T256, 3301, 4103, 512),
    (T128X256, 1301, 11003, 128), (T128X256, 1301, 11003, 160), (T128X256, 1301, 11003, 384),
    (T128X256, 1301, 11003, 512), (T128X256, 1301, 11003, 1152),
    (T128, 1030, 2101, 160), (T128, 700, 1501, 1056), (T128, 520, 2103, 96),
    (T128_BY_ROWS, 700, 1501, 640), (T128_BY_ROWS, 1000, 2301, 128), (T128_BY_ROWS, 401, 6003, 512),
]
SWIGLU = [
    (ROWS, 5, 70, 96), (ROWS, 40, 333, 1056),
    (RING, 3, 70, 640), (RING, 12, 71, 128), (RING, 30, 200, 1152), (RING, 64, 130, 1664), (RING, 150, 301, 640),
    (T256, 1601, 4403, 160), (T256, 1601, 4403, 384), (T256, 1601, 4403, 512),
    (T128X256, 600, 11003, 128), (T128X256, 600, 11003, 384), (T128X256, 600, 11003, 512), (T128X256, 401, 6003, 160),
    (T128X256, 401, 6003, 1152),
    (T128, 700, 1501, 160), (T128, 1030, 2101, 96), (T128, 520, 2103, 1056),
    (T128_BY_ROWS, 700, 1501, 640), (T128_BY_ROWS, 401, 6003, 512), (T128_BY_ROWS, 900, 1501, 128),
]


def cut(n):
    """The rows of the first of two weights side by side."""
    return n // 2 + 3


def form(m, ns, k, swiglu):
    return _lib.lib().q3_matmul_mxfp8_form(m, (ctypes.c_int64 * len(ns))(*ns), len(ns), k, swiglu)


def test_the_cases_take_the_forms_that_they_are_for():
    for swiglu, cases in enumerate((PLAIN, SWIGLU)):
        assert [form(m, [n], k, swiglu) for _, m, n, k in cases] == [f for f, *_ in cases]
        assert {f for f, *_ in cases} == set(range(6))
        # forms that keep several stages under way turn their slots over
        assert all(max(k for f, _, _, k in cases if f == g) > 3 * 128 for g in range(6))
    assert {form(m, [cut(n), n - cut(n)], k, 0) for _, m, n, k in PLAIN} == set(range(6))


def test_form_query_takes_any_sizes():
    assert form(0, [64], 64, 0) == -2 and form(4, [64], 48, 0) == -2 and form(4, [0], 64, 0) == -2
    assert form(4, [64] * 5, 64, 0) == -2 and form(4, [64], 1 << 23, 0) == -2
    assert _lib.lib().q3_matmul_mxfp8_form(4, None, 1, 64, 0) == -2
    for m in (1, 64, 65, 4096, (1 << 31) - 300):
        for n in (1, 300, 151936, (1 << 31) - 300):
            for k in (32, 128, 4096, (1 << 23) - 32):
                for s in (0, 1):
                    f = form(m, [n], k, s)
                    assert 0 <= f < 6 and (m > 64 or f == (k % 128 == 0))
                    work = _lib.lib().q3_matmul_mxfp8_workspace_bytes(m, (ctypes.c_int64 * 1)(n), 1, k, s)
                    assert (work == 0) == (f in (ROWS, RING, T128_BY_ROWS))


def values(pair):
    return M.values(*pair).to(DEV)


def head(pair, n):
    return pair[0][:n], pair[1][:n]


def within(y, want, err):
    """bf16 y against float64 `want`, off by `err` before its rounding."""
    assert y.dtype == torch.bfloat16 and y.shape == want.shape
    d, tol = (y.double() - want).abs(), HALF * (want.abs() + err) + err
    assert bool((d <= tol).all()), float((d / tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("f,m,n,k", PLAIN)
def test_products(f, m, n, k):
    x, w = exact_pair(m, k, 1), exact_pair(n, k, 2)
    b, r = rnd(n, seed=3).to(DEV), rnd(m, n, seed=4).to(DEV)
    xd, wd = dev(x), dev(w)
    a = values(x) @ values(w).T
    assert torch.equal(K.matmul_mxfp8(xd, wd), a.to(torch.bfloat16))
    out = r.clone()
    assert K.matmul_mxfp8(xd, wd, b, out, activation="silu", out=out) is out
    y, err = a + b.double(), 2.0 ** -23 * (a + b.double()).abs()
    z = act_of(y, "silu")
    err = 1.13 * err + 2.0 ** -20 * z.abs() + 2.0 ** -30
    within(out, z + r.double(), err + 2.0 ** -23 * (z.abs() + r.double().abs()))
    c = cut(n)
    y = K.matmul_segments_mxfp8(xd, [head(wd, c), (wd[0][c:], wd[1][c:])])
    assert torch.equal(y, a.to(torch.bfloat16))
    n -= n % 32
    codes, scales = K.matmul_mxfp8(xd, head(wd, n), quantize=True)
    want = K.mxfp8_quantize(a[:, :n].float().contiguous())  # exact sums, to the bit
    assert torch.equal(codes.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scales, want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("f,m,n,k", SWIGLU)
def test_swiglu(f, m, n, k):
    x, g, u = ((c, s - 5) for c, s in (exact_pair(r, k, i) for i, r in enumerate((m, n, n))))
    xd, gd, ud = dev(x), dev(g), dev(u)
    a, b = values(x) @ values(g).T, values(x) @ values(u).T
    want = a * torch.sigmoid(a) * b
    err = (2.0 ** -20 + 2.0 ** -22) * want.abs() + 2.0 ** -30
    within(K.matmul_swiglu_mxfp8(xd, gd, ud), want, err)
    n -= n % 32
    pair = K.matmul_swiglu_mxfp8(xd, head(gd, n), head(ud, n), quantize=True)
    check_eight_bits(pair, want[:, :n].cpu(), err[:, :n].cpu())


def with_nan(pair, *places):
    """The pair with NaN for the scales (rows, block) of `places`, and which rows have one."""
    scales = pair[1].clone()
    rows = torch.zeros(len(scales), dtype=torch.bool)
    for at, block in places:
        scales[at, block] = 255
        rows[at] = True
    return (pair[0], scales), rows.to(DEV)


def nan_exactly(y, rows, columns, want):
    """y is NaN in those rows and columns, and the correctly rounded `want` elsewhere."""
    bad = rows[:, None] | columns[None]
    assert torch.equal(torch.isnan(y), bad)
    assert torch.equal(y[~bad], want[~bad].to(torch.bfloat16))


def nan_x(m, k):
    return with_nan(exact_pair(m, k, 1), (slice(min(5, m - 1), None, 97), 0), (-1, -1))


@pytest.mark.gpu
@pytest.mark.parametrize("f,m,n,k", PLAIN)
def test_nan_scales_of_products_stay_where_they_are(f, m, n, k):
    """NaN in a row's first block, behind its neighbour's end, and in a matrix's last one; of two weights side by side in
    the rows that meet."""
    (x, rows), w = nan_x(m, k), exact_pair(n, k, 2)
    a = values(exact_pair(m, k, 1)) @ values(w).T
    v, columns = with_nan(w, (slice(7, None, 101), 0), (-1, -1))
    nan_exactly(K.matmul_mxfp8(dev(x), dev(v)), rows, columns, a)
    c = cut(n)
    v, columns = with_nan(w, (c - 1, -1), (c, 0), (-1, -1))
    vd = dev(v)
    y = K.matmul_segments_mxfp8(dev(x), [head(vd, c), (vd[0][c:], vd[1][c:])])
    nan_exactly(y, rows, columns, a)


@pytest.mark.gpu
@pytest.mark.parametrize("f,m,n,k", SWIGLU)
def test_nan_scales_of_swiglu_stay_where_they_are(f, m, n, k):
    """Gate's and up's in different rows; where neither has one the result is that of the weights without any."""
    (x, rows), g, u = nan_x(m, k), exact_pair(n, k, 2), exact_pair(n, k, 3)
    gv, gc = with_nan(g, (slice(7, None, 101), 0), (31, -1))
    uv, uc = with_nan(u, (slice(11, None, 103), -1), (32, 0), (-1, -1))
    want = K.matmul_swiglu_mxfp8(dev(exact_pair(m, k, 1)), dev(g), dev(u))
    nan_exactly(K.matmul_swiglu_mxfp8(dev(x), dev(gv), dev(uv)), rows, gc | uc, want)
    n -= n % 32
    codes, scales = K.matmul_swiglu_mxfp8(dev(x), head(dev(gv), n), head(dev(uv), n), quantize=True)
    blocks = rows[:, None] | (gc | uc)[:n].view(-1, 32).any(-1)[None]
    assert torch.equal(scales == 255, blocks)
