"""MXFP8 operators on the GPU against their definition in float64 (oracle/mxfp8.py).

Quantisation and its inverse are exact, so they must agree to the bit. The products are tested twice: on values whose
products and sums the matrix instruction forms exactly (products of at most 13 bits in a group of eight k, sums within
fp32), where the result must be the correctly rounded one; and on normal values, within the rounding (bf16 2^-8,
relative) of a sum that is off by what the instruction cuts and fp32 rounds (oracle.product's bound). An activation
passes an error on at most 1.13-fold (the largest slope of gelu_tanh; silu's is 1.1) and adds 2^-20 of its value for its
own arithmetic (the hardware exponential and reciprocal, 2^-22 each at most, a few operations). An output in eight
bits rounds by 2^-4 of a value or 2^-10 of its block's scale, whichever is more, from a value as far off as above; the
scale may come out one step apart where the largest value is that near a border.
"""
import math

import pytest
import torch

from oracle import mxfp8 as M
from qwen3_5_vl_cuda_custom_amd import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = 2.0 ** -8  # half a step of bf16, relative


def rnd(*shape, seed=0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype)


def dev(pair):
    return pair[0].to(DEV), pair[1].to(DEV)


def same_bits(a, b):
    a, b = a.cpu(), b.cpu()
    return a.dtype == b.dtype and torch.equal(torch.nan_to_num(a.double(), nan=12345.0),
                                              torch.nan_to_num(b.double(), nan=12345.0))


def same_pair(got, want):
    return (got[0].dtype == torch.float8_e4m3fn and got[0].shape == want[0].shape
            and torch.equal(got[0].cpu().view(torch.uint8), want[0].view(torch.uint8))
            and torch.equal(got[1].cpu(), want[1]))


# ------------------------------------------------------------------ rows
def special_rows(dtype):
    """Blocks at which quantisation can go wrong: zeros, one value, ties, borders of the scale, the smallest and largest."""
    t = torch.zeros(16, 32, dtype=torch.float64)
    t[1, 5] = -3.5
    t[2] = torch.linspace(-447.9, 447.9, 32)
    t[3, :16] = torch.tensor([448.0, 17, 19, 21, 1.0625, 1.1875, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, -17, -19, -1.0625,
                              -2.0 ** -10, 5 * 2.0 ** -10, 200.0, 216.0])
    t[4] = t[3] * 2.0 ** -120
    t[5] = t[3] * 2.0 ** 100
    t[6] = torch.arange(32) * 2.0 ** -131  # below the smallest scale's reach: subnormal inputs
    t[7, 0], t[7, 1:] = 3.0e38, 1e-3
    t[8, 3] = math.inf
    t[9, 31] = math.nan
    t[10, 0], t[10, 1] = -0.0, -1e-30
    t[10, 2] = 1.0
    t[11] = 2.0 ** -126 * torch.linspace(-1, 1, 32)
    t[12, 7], t[13, 7], t[14, 7] = 448.0, 450.0, 446.0  # bf16: 448, 450, 446 exactly
    t[15] = t[3] * 2.0 ** -127
    return t.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (257, 128), (64, 4096), (5, 1152)])
def test_quantize_and_back_match_the_definition(rows, cols, dtype):
    x = rnd(rows, cols, seed=rows, dtype=dtype) * torch.exp2(torch.randint(-20, 20, (rows, 1))).to(dtype)
    pair = K.mxfp8_quantize(x.to(DEV))
    want = M.quantize(x)
    assert same_pair(pair, want)
    for out in (torch.bfloat16, torch.float32):
        back = K.mxfp8_dequantize(*pair, out)
        assert back.dtype == out and same_bits(back.double(), M.values(*want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_special_blocks(dtype):
    x = special_rows(dtype)
    pair = K.mxfp8_quantize(x.to(DEV))
    assert same_pair(pair, M.quantize(x))
    back = K.mxfp8_dequantize(*pair).cpu()
    assert torch.isnan(back[8:10]).all() and torch.isfinite(back[:8]).all() and torch.isfinite(back[10:]).all()


def test_quantize_strided_and_empty_inputs():
    x = rnd(6, 7, 256, seed=3).to(DEV)
    for view in (x[:, :, 64:128], x[::2], x.transpose(0, 1), x[:, 1:, 8:200:2][..., :96], x[:0], x[..., :0], x[1, 2]):
        pair = K.mxfp8_quantize(view)
        assert pair[0].shape == view.shape and pair[1].shape == (*view.shape[:-1], view.shape[-1] // 32)
        if view.numel():
            assert same_pair(pair, M.quantize(view.cpu()))


def test_dequantize_every_code_and_scale():
    codes = torch.arange(256, dtype=torch.uint8).view(1, 8, 32).expand(256, 8, 32).contiguous().view(torch.float8_e4m3fn)
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1, 1).expand(256, 8, 1).contiguous()
    for out in (torch.bfloat16, torch.float32):  # the smallest scales reach below the types' range, the largest above
        want = M.values(codes, scales).to(out)
        assert same_bits(K.mxfp8_dequantize(codes.to(DEV), scales.to(DEV), out), want)


def test_dequantize_views():
    codes = torch.randint(0, 120, (3, 4, 50, 64), dtype=torch.uint8).view(torch.float8_e4m3fn)
    scales = torch.randint(100, 140, (3, 4, 50, 2), dtype=torch.uint8)
    c, s = codes.to(DEV), scales.to(DEV)
    for sl in ((slice(None), slice(None), slice(7, 30)), (slice(1, 3), slice(2, 3)), (slice(0, 0),), (2, 1, 5)):
        assert same_bits(K.mxfp8_dequantize(c[sl], s[sl]).double(), M.values(codes[sl], scales[sl]))


# ------------------------------------------------------------------ the norm
def check_eight_bits(pair, want, slack):
    """The pair against float64 values `want`, each off by `slack` (a tensor) before its rounding."""
    got = M.values(pair[0].cpu(), pair[1].cpu())
    top = (want.abs() + slack).unflatten(-1, (-1, 32)).amax(-1, keepdim=True)
    scale = torch.exp2(torch.ceil(torch.log2(top.clamp(min=2.0 ** -119) / 448)).clamp(min=-127) + 2.0 ** -40)
    step = torch.maximum((want.abs() + slack) / 16, (scale * 2.0 ** -10).expand(*top.shape[:-1], 32).flatten(-2))
    d = (got - want).abs()
    assert bool((d <= step + slack).all()), float((d / (step + slack)).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (2, 2048), (5, 2080), (33, 4096), (700, 1152), (2, 8192),
                                       (3, 12288), (2, 20000 // 32 * 32)])
def test_norm_matches_float64(rows, cols, residual, dtype):
    x, r = rnd(rows, cols, seed=rows, dtype=dtype) * 3, rnd(rows, cols, seed=1, dtype=dtype)
    w = 1 + 0.2 * rnd(cols, seed=2, dtype=dtype)
    h, codes, scales = K.add_rmsnorm_mxfp8(x.to(DEV), r.to(DEV) if residual else None, w.to(DEV), 1e-5)
    want_h = (x.float() + r.float()).to(dtype) if residual else x
    assert same_bits(h, want_h)
    hd = want_h.double()
    want = hd / torch.sqrt(hd.pow(2).mean(-1, keepdim=True) + 1e-5) * w.double()
    # the sum of squares: cols terms in fp32, each addition and product 2^-24 (half of it goes on through the root); the
    # root, two products
    check_eight_bits((codes, scales), want, (cols / 2 + 8) * 2.0 ** -24 * want.abs())


def test_norm_equals_its_parts():
    x, r, w = rnd(40, 4096, seed=1).to(DEV), rnd(40, 4096, seed=2).to(DEV), rnd(4096, seed=3).to(DEV)
    h, codes, scales = K.add_rmsnorm_mxfp8(x, r, w, 1e-6)
    assert torch.equal(h, K.residual_add(x, r))
    again = K.add_rmsnorm_mxfp8(h, None, w, 1e-6)
    assert again[0] is h and torch.equal(again[1].view(torch.uint8), codes.view(torch.uint8)) and torch.equal(again[2], scales)


def test_norm_special_rows():
    x = rnd(6, 128, seed=4, dtype=torch.float32)
    x[0] = 0
    x[1, 5], x[2, 5], x[3] = math.inf, math.nan, 1e-30
    x[4] = 1e25  # its squares pass fp32
    w = torch.ones(128)
    h, codes, scales = K.add_rmsnorm_mxfp8(x.to(DEV), None, w.to(DEV), 1e-6)
    back = K.mxfp8_dequantize(codes, scales, torch.float32).cpu()
    assert not back[0].any() and not torch.isfinite(back[2]).any() and torch.isfinite(back[3]).all()
    assert torch.isnan(back[1, :32]).all() and not back[1, 32:].any()  # 1 / infinity, and infinity times it
    assert not back[4].any() and torch.isfinite(back[5]).all()


def test_norm_strided_rows():
    wide, w = rnd(9, 3, 512, seed=5).to(DEV), rnd(128, seed=6).to(DEV)
    for view in (wide[..., 128:256], wide[:, 1, 64:192], wide[..., 4:132], wide.transpose(0, 1)[..., :128], wide[:0, :, :128]):
        h, codes, scales = K.add_rmsnorm_mxfp8(view, view, w, 1e-6)
        want = K.add_rmsnorm_mxfp8(view.contiguous(), view.contiguous(), w, 1e-6)
        assert torch.equal(h, want[0]) and torch.equal(codes.view(torch.uint8), want[1].view(torch.uint8))
        assert torch.equal(scales, want[2]) and h.shape == view.shape


# ------------------------------------------------------------------ products
def exact_pair(rows, k, seed):
    """Codes and scales whose products and sums the instruction forms exactly: values of 1, 1.25, 1.5, 1.75, 2 and their
    negatives, or zeros (three bits), scales of 1, 2 or 4 by blocks: products have six bits over 2^-4, of a group (one
    block) within 13 bits of its largest; a sum of k stays below 2^24 of its last bit for k up to 2^13."""
    g = torch.Generator().manual_seed(seed)
    v = torch.tensor([0.0, 1.0, 1.25, 1.5, 1.75, 2.0])[torch.randint(0, 6, (rows, k), generator=g)]
    v = v * (1 - 2 * torch.randint(0, 2, (rows, k), generator=g))
    return v.to(torch.float8_e4m3fn), torch.randint(127, 130, (rows, k // 32), generator=g).to(torch.uint8)


def normal_pair(rows, k, seed, size=1.0):
    return M.quantize(rnd(rows, k, seed=seed, dtype=torch.float32) * size)


def act_of(y, act):
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return y * torch.sigmoid(y) if act == "silu" else y


def reference(x, w, b=None, act=None, r=None):
    """(value, bound before the last rounding) in float64."""
    y, err = M.product(M.values(*x), M.values(*w))
    if b is not None:
        y = y + b.double()
        err = err + 2.0 ** -23 * y.abs()
    if act is not None:
        z = act_of(y, act)
        y, err = z, 1.13 * err + 2.0 ** -20 * z.abs() + 2.0 ** -30
    if r is not None:
        y = y + r.double()
        err = err + 2.0 ** -23 * y.abs()
    return y, err


def check(y, ref, err):
    assert y.dtype == torch.bfloat16 and y.shape == ref.shape
    d, tol = (y.double().cpu() - ref).abs(), HALF * (ref.abs() + err) + err
    assert bool((d <= tol).all()), float((d / tol).max())


ROWS = [1, 2, 16, 17, 33, 64, 65, 130, 300]
WEIGHTS = [(1, 32), (17, 96), (130, 160), (256, 4096), (1000, 1056), (33, 8192), (300, 128)]


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("n,k", WEIGHTS)
def test_matmul_of_exact_values(m, n, k):
    x, w = exact_pair(m, k, m), exact_pair(n, k, n + 1)
    y = K.matmul_mxfp8(dev(x), dev(w))
    assert torch.equal(y.cpu(), (M.values(*x) @ M.values(*w).T).to(torch.bfloat16))


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("n,k", [(17, 96), (130, 160), (256, 4096), (1000, 1056)])
def test_matmul_epilogues(m, n, k):
    x, w = normal_pair(m, k, m), normal_pair(n, k, n, 0.05)
    b, r = rnd(n, seed=1), rnd(m, n, seed=2)
    for bias, act, res in ((None, None, None), (b, None, r), (b, "gelu_tanh", None), (b, "silu", r), (None, "gelu_tanh", r)):
        y = K.matmul_mxfp8(dev(x), dev(w), None if bias is None else bias.to(DEV), None if res is None else res.to(DEV),
                           activation=act)
        check(y, *reference(x, w, bias, act, res))


@pytest.mark.parametrize("m,n,k", [(1100, 1000, 96), (520, 2100, 128), (700, 513, 2080), (257, 4304, 1152), (2050, 300, 640)])
def test_matmul_many_tiles(m, n, k):
    x, w = exact_pair(m, k, 1), exact_pair(n, k, 2)
    b, r = rnd(n, seed=1), rnd(m, n, seed=2)
    y = K.matmul_mxfp8(dev(x), dev(w))
    assert torch.equal(y.cpu(), (M.values(*x) @ M.values(*w).T).to(torch.bfloat16))
    y = K.matmul_mxfp8(dev(x), dev(w), b.to(DEV), r.to(DEV))
    exact = M.values(*x) @ M.values(*w).T
    want = exact + b.double() + r.double()
    tol = HALF * want.abs() + 2.0 ** -22 * (exact.abs() + b.double().abs() + r.double().abs())
    assert bool(((y.double().cpu() - want).abs() <= tol).all())


@pytest.mark.parametrize("m,n,k", [(5, 24, 131072), (80, 24, 66560), (300, 20, 32800), (129, 6000, 16384)])
def test_matmul_of_long_rows(m, n, k):
    """Rows past the lengths whose sums are exact: one value in sixteen is not zero."""
    x, w = exact_pair(m, k, 1), exact_pair(n, k, 2)
    x[0].view(torch.uint8)[torch.rand(m, k, generator=torch.Generator().manual_seed(3)) > 1 / 16] = 0
    want = (M.values(*x).float().to(DEV) @ M.values(*w).float().to(DEV).T).to(torch.bfloat16)
    assert torch.equal(K.matmul_mxfp8(dev(x), dev(w)), want)


def test_matmul_scales_of_every_size():
    """Scales far apart between rows, and between blocks of a row."""
    m, n, k = 70, 50, 256
    x, w = normal_pair(m, k, 1), normal_pair(n, k, 2)
    g = torch.Generator().manual_seed(3)
    x = x[0], torch.randint(60, 190, (m, 1), generator=g).expand(m, k // 32).contiguous().to(torch.uint8)
    w = w[0], torch.randint(100, 150, (n, k // 32), generator=g).to(torch.uint8)
    check(K.matmul_mxfp8(dev(x), dev(w)), *reference(x, w))


@pytest.mark.parametrize("m", [3, 64, 200])
def test_matmul_keeps_nan_in_its_rows_and_columns(m):
    x, w = exact_pair(m, 192, 1), exact_pair(70, 192, 2)
    xs, ws, wc = x[1].clone(), w[1].clone(), w[0].clone()
    xs[1, 3] = 255  # a row's block
    ws[5, 0] = 255  # a column's block
    wc.view(torch.uint8)[9, 100] = 0x7f  # one value
    y = K.matmul_mxfp8(dev((x[0], xs)), dev((wc, ws))).cpu()
    want = M.values(x[0], xs) @ M.values(wc, ws).T
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and int(torch.isnan(want).sum()) == 70 + 2 * (m - 1)
    assert same_bits(y, want.to(torch.bfloat16))


@pytest.mark.parametrize("m", [1, 30, 64, 65, 333])
@pytest.mark.parametrize("n,k", [(32, 96), (160, 512), (1056, 1024)])
def test_outputs_in_eight_bits(m, n, k):
    x, w, g = normal_pair(m, k, m), normal_pair(n, k, 1, 0.1), normal_pair(n, k, 2, 0.1)
    b, r = rnd(n, seed=1), rnd(m, n, seed=2)
    pair = K.matmul_mxfp8(dev(x), dev(w), b.to(DEV), r.to(DEV), activation="silu", quantize=True)
    check_eight_bits(pair, *reference(x, w, b, "silu", r))
    pair = K.matmul_swiglu_mxfp8(dev(x), dev(g), dev(w), quantize=True)
    check_eight_bits(pair, *swiglu_reference(x, g, w))


@pytest.mark.parametrize("m", [2, 70])
def test_outputs_in_eight_bits_of_exact_values(m):
    x, w = exact_pair(m, 512, m), exact_pair(96, 512, 1)
    assert same_pair(K.matmul_mxfp8(dev(x), dev(w), quantize=True), M.quantize(M.values(*x) @ M.values(*w).T))


def test_outputs_in_eight_bits_of_special_rows():
    x, w = exact_pair(70, 96, 1), exact_pair(64, 96, 2)
    x[0][3] = 0  # a row of zeros
    x[1][4, 1] = 255
    w[1][40, 0] = 255
    codes, scales = K.matmul_mxfp8(dev(x), dev(w), quantize=True)
    back = K.mxfp8_dequantize(codes, scales).cpu()
    assert not back[3, :32].any() and int(scales[3, 0]) == 0 and torch.isnan(back[4]).all()
    assert torch.isnan(back[:, 32:]).all() and torch.isfinite(back[[0, 1, 2, 5]][:, :32]).all()


def swiglu_reference(x, g, u):
    """(value, bound before the last rounding) in float64."""
    (a, ea), (b, eb) = (M.product(M.values(*x), M.values(*w)) for w in (g, u))
    s = a * torch.sigmoid(a)
    es = 1.1 * ea + 2.0 ** -20 * s.abs()
    return s * b, es * (b.abs() + eb) + s.abs() * eb + 2.0 ** -22 * (s * b).abs() + 2.0 ** -30


@pytest.mark.parametrize("m", ROWS)
@pytest.mark.parametrize("n,k", [(1, 32), (17, 96), (130, 160), (256, 4096), (1000, 1056), (300, 128)])
def test_swiglu_matches_float64(m, n, k):
    x, g, u = normal_pair(m, k, m), normal_pair(n, k, 1, 0.05), normal_pair(n, k, 2, 0.05)
    check(K.matmul_swiglu_mxfp8(dev(x), dev(g), dev(u)), *swiglu_reference(x, g, u))


@pytest.mark.parametrize("m", [1, 8, 40, 65, 300, 700])
@pytest.mark.parametrize("ns,k", [((64,), 96), ((512, 128, 128), 512), ((5, 300, 1, 77), 1056), ((33, 31), 32)])
def test_segments_of_exact_values(m, ns, k):
    x, ws = exact_pair(m, k, m), [exact_pair(n, k, n) for n in ns]
    y = K.matmul_segments_mxfp8(dev(x), [dev(w) for w in ws])
    want = [M.values(*x) @ M.values(*w).T for w in ws]
    assert torch.equal(y.cpu(), torch.cat(want, -1).to(torch.bfloat16))
    bs = [rnd(n, seed=n) if i != 1 else None for i, n in enumerate(ns)]
    y = K.matmul_segments_mxfp8(dev(x), [dev(w) for w in ws], [None if b is None else b.to(DEV) for b in bs])
    parts = [K.matmul_mxfp8(dev(x), dev(w), None if b is None else b.to(DEV)) for w, b in zip(ws, bs)]
    assert torch.equal(y, torch.cat(parts, -1))


@pytest.mark.parametrize("m,n,k", [(1030, 2100, 384), (1600, 4400, 256), (3300, 4100, 384), (2600, 6500, 160),
                                   (700, 1500, 640), (900, 2300, 1152)])
def test_tiles_of_every_size(m, n, k):
    """More rows and columns than 512 blocks of 64 by 64 cover: exact sums, one weight, two, and of SwiGLU."""
    x, g, u = ((c, s - 5) for c, s in (exact_pair(r, k, i) for i, r in enumerate((m, n, n))))
    xd, gd, ud = dev(x), dev(g), dev(u)
    a, b = (M.values(*x).float() @ M.values(*w).float().T for w in (g, u))  # exact in 24 bits
    r = rnd(m, n, seed=2)
    assert torch.equal(K.matmul_mxfp8(xd, gd).cpu(), a.to(torch.bfloat16))
    want, tol = a.double() + r.double(), 2.0 ** -22 * (a.double().abs() + r.double().abs())
    check(K.matmul_mxfp8(xd, gd, residual=r.to(DEV)), want, tol)
    cut = n // 2 + 3
    y = K.matmul_segments_mxfp8(xd, [(gd[0][:cut], gd[1][:cut]), (ud[0][cut:], ud[1][cut:])])
    assert torch.equal(y.cpu(), torch.cat([a[:, :cut], b[:, cut:]], -1).to(torch.bfloat16))
    s = a.double() * torch.sigmoid(a.double())
    want, err = s * b.double(), (2.0 ** -20 + 2.0 ** -22) * (s * b.double()).abs() + 2.0 ** -30
    check(K.matmul_swiglu_mxfp8(xd, gd, ud), want, err)
    n -= n % 32
    pair = K.matmul_swiglu_mxfp8(xd, (gd[0][:n], gd[1][:n]), (ud[0][:n], ud[1][:n]), quantize=True)
    check_eight_bits(pair, want[:, :n], err[:, :n])


@pytest.mark.parametrize("m,n,k", [(3, 70, 128), (8, 70, 640), (16, 70, 1152), (30, 200, 640), (64, 70, 640), (128, 300, 1152),
                                   (700, 2500, 640), (1600, 4400, 128), (3300, 4100, 384)])
def test_nan_scales_stay_in_their_rows_and_columns(m, n, k):
    """A row's first block is NaN: its neighbour's scales end right before it."""
    x, w = exact_pair(m, k, 1), exact_pair(n, k, 2)
    xs, ws = x[1].clone(), w[1].clone()
    r0 = min(5, m - 1)
    xs[r0::97, 0] = 255
    ws[7::101, 0] = 255
    y = torch.isnan(K.matmul_mxfp8(dev((x[0], xs)), dev((w[0], ws)))).cpu()
    want = torch.zeros(m, n, dtype=torch.bool)
    want[r0::97] = True
    want[:, 7::101] = True
    assert torch.equal(y, want)


@pytest.mark.parametrize("m", [65, 127, 129, 200])
@pytest.mark.parametrize("n,k", [(4, 128), (100, 640), (2000, 1152), (4096, 4224)])
def test_rows_in_parts_of_64(m, n, k):
    x, w, r = exact_pair(m, k, m), exact_pair(n, k, n), rnd(m, n, seed=3)
    want = M.values(*x).float() @ M.values(*w).float().T
    assert torch.equal(K.matmul_mxfp8(dev(x), dev(w)).cpu(), want.to(torch.bfloat16))
    want = want.double() + r.double()
    check(K.matmul_mxfp8(dev(x), dev(w), residual=r.to(DEV)), want, 2.0 ** -22 * ((want - r.double()).abs() + r.double().abs()))


def test_bf16_rows_are_quantised_first():
    x, w = rnd(2, 40, 256, seed=1).to(DEV), dev(normal_pair(64, 256, 2))
    pair = K.mxfp8_quantize(x)
    assert torch.equal(K.matmul_mxfp8(x, w), K.matmul_mxfp8(pair, w))
    assert torch.equal(K.matmul_segments_mxfp8(x, [w, w]), K.matmul_segments_mxfp8(pair, [w, w]))
    assert torch.equal(K.matmul_swiglu_mxfp8(x, w, w), K.matmul_swiglu_mxfp8(pair, w, w))
    view = x.transpose(0, 1)[3:, :, :]
    assert torch.equal(K.matmul_mxfp8(view, w), K.matmul_mxfp8(view.contiguous(), w))


@pytest.mark.parametrize("m", [5, 90])
def test_outputs_and_residuals_in_wider_buffers(m):
    x, w, r = dev(exact_pair(m, 128, 1)), dev(exact_pair(100, 128, 2)), rnd(m, 300, seed=3).to(DEV)
    want = K.matmul_mxfp8(x, w, residual=r[:, 7:107].contiguous())
    buf = torch.full((m, 400), 7.0, dtype=torch.bfloat16, device=DEV)
    out = K.matmul_mxfp8(x, w, residual=r[:, 7:107], out=buf[:, 33:133])
    assert out.data_ptr() == buf[:, 33:133].data_ptr() and torch.equal(buf[:, 33:133], want)
    assert bool((buf[:, :33] == 7).all()) and bool((buf[:, 133:] == 7).all())
    y = r[:, 7:107].contiguous()
    K.matmul_mxfp8(x, w, residual=y, out=y)  # onto the residual itself
    assert torch.equal(y, want)


def test_views_of_codes_and_scales():
    x, w = dev(exact_pair(12, 256, 1)), dev(exact_pair(80, 256, 2))
    want = K.matmul_mxfp8((x[0][::2].contiguous(), x[1][::2].contiguous()), (w[0][8:48].clone(), w[1][8:48].clone()))
    assert torch.equal(K.matmul_mxfp8((x[0][::2], x[1][::2]), (w[0][8:48], w[1][8:48])), want)
    half = K.matmul_mxfp8((x[0][:, :96], x[1][:, :3]), (w[0][:, 32:128], w[1][:, 1:4]))
    assert torch.equal(half, K.matmul_mxfp8((x[0][:, :96].contiguous(), x[1][:, :3].contiguous()),
                                            (w[0][:, 32:128].contiguous(), w[1][:, 1:4].contiguous())))
    odd = torch.empty(80 * 8 + 3, dtype=torch.uint8, device=DEV)  # scales at any byte
    odd[3:] = w[1].flatten()
    assert torch.equal(K.matmul_mxfp8(x, (w[0], odd[3:].view(80, 8))), K.matmul_mxfp8(x, w))


def test_empty_calls():
    w = dev(exact_pair(64, 96, 2))
    for shape in ((0, 96), (3, 0, 96)):
        x = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
        assert K.matmul_mxfp8(x, w).shape == (*shape[:-1], 64)
        assert K.matmul_segments_mxfp8(x, [w, w]).shape == (*shape[:-1], 128)
        assert K.matmul_swiglu_mxfp8(x, w, w, quantize=True)[1].shape == (*shape[:-1], 2)
        h, codes, scales = K.add_rmsnorm_mxfp8(x, x, torch.ones(96, dtype=torch.bfloat16, device=DEV))
        assert h.shape == codes.shape == shape and scales.shape == (*shape[:-1], 3)
    none = w[0][:0], w[1][:0]
    x = dev(exact_pair(5, 96, 1))
    assert K.matmul_mxfp8(x, none).shape == (5, 0)
    assert torch.equal(K.matmul_segments_mxfp8(x, [w, none, w])[:, :64], K.matmul_mxfp8(x, w))


def test_layer_half_in_a_row():
    """norm, gate and up into eight bits, down with the residual, as a layer calls them: the same as step by step."""
    m, h, i = 37, 512, 1056
    x, r, w = rnd(m, h, seed=1), rnd(m, h, seed=2), 1 + 0.1 * rnd(h, seed=3)
    g, u, d = normal_pair(i, h, 4, 0.05), normal_pair(i, h, 5, 0.05), normal_pair(h, i, 6, 0.05)
    hd, codes, scales = K.add_rmsnorm_mxfp8(x.to(DEV), r.to(DEV), w.to(DEV))
    act = K.matmul_swiglu_mxfp8((codes, scales), dev(g), dev(u), quantize=True)
    y = K.matmul_mxfp8(act, dev(d), residual=hd)
    cpu = tuple(t.cpu() for t in (codes, scales)), tuple(t.cpu() for t in act)
    check_eight_bits(act, *swiglu_reference(cpu[0], g, u))
    check(y, *reference(cpu[1], d, r=hd.cpu()))


# ------------------------------------------------------------------ offsets past 32 bits
def test_rows_past_two_to_the_31_values():
    """The norm, the quantisation and the way back over 2.4 thousand million values: 600 times the same rows."""
    x, w = rnd(1000, 4096, seed=1).to(DEV), torch.ones(4096, dtype=torch.bfloat16, device=DEV)
    big = x.repeat(600, 1)
    h, codes, scales = K.add_rmsnorm_mxfp8(big, big, w)
    h1, codes1, scales1 = K.add_rmsnorm_mxfp8(x, x, w)
    back, back1 = K.mxfp8_dequantize(codes, scales), K.mxfp8_dequantize(codes1, scales1)
    codes2, codes3 = K.mxfp8_quantize(big)[0], K.mxfp8_quantize(x)[0]
    for a, b in ((h, h1), (codes, codes1), (scales, scales1), (back, back1), (codes2, codes3)):
        a, b = (t.view(torch.uint8) for t in (a, b))
        assert bool((a.view(600, 1000, -1) == b).all())


@pytest.mark.parametrize("residual", [False, True])
def test_norm_of_more_rows_than_a_launch_has_blocks(residual):
    """2^24 rows of a block of 256 threads each would be 2^32 threads."""
    x, w = rnd(1021, 32, seed=1).to(DEV), rnd(32, seed=2).to(DEV)
    rows = (1 << 24) + 5
    of = torch.arange(rows, device=DEV) % 1021
    big = x[of]
    h, codes, scales = K.add_rmsnorm_mxfp8(big, big if residual else None, w)
    h1, codes1, scales1 = K.add_rmsnorm_mxfp8(x, x if residual else None, w)
    assert torch.equal(h, h1[of]) and torch.equal(scales, scales1[of])
    assert torch.equal(codes.view(torch.uint8), codes1.view(torch.uint8)[of])


@pytest.mark.parametrize("m", [2, 40, 700])
def test_weights_past_two_to_the_31_bytes(m):
    x, w = dev(exact_pair(m, 4096, 1)), dev(exact_pair(1000, 4096, 2))
    y = K.matmul_mxfp8(x, tuple(t.view(torch.uint8).repeat(600, 1).view(t.dtype) for t in w))
    assert bool((y.view(m, 600, 1000) == K.matmul_mxfp8(x, w)[:, None]).all())


@pytest.mark.parametrize("k", [128, 96])
def test_outputs_past_two_to_the_31_values(k):
    x, w = dev(exact_pair(250, k, 1)), dev(exact_pair(32768, k, 2))
    big = tuple(t.view(torch.uint8).repeat(280, 1).view(t.dtype) for t in x)
    want = K.matmul_mxfp8(x, w)
    assert bool((K.matmul_mxfp8(big, w).view(280, 250, -1) == want).all())
    r = want.repeat(280, 1)
    assert bool((K.matmul_mxfp8(big, w, residual=r, out=r).view(280, 250, -1) == K.matmul_mxfp8(x, w, residual=want)).all())
    codes, scales = K.matmul_mxfp8(big, w, quantize=True)
    codes1, scales1 = K.matmul_mxfp8(x, w, quantize=True)
    assert bool((codes.view(torch.uint8).view(280, 250, -1) == codes1.view(torch.uint8)).all())
    assert bool((scales.view(280, 250, -1) == scales1).all())


# ------------------------------------------------------------------ streams, graphs, refusals
@pytest.mark.parametrize("m", [8, 100, 1500])
def test_two_streams_at_once(m):
    """Products of the same weights on two streams, each with workspaces of its own."""
    w, xs = dev(exact_pair(4352, 1024, 1)), [dev(exact_pair(m, 1024, 2 + i)) for i in range(2)]
    want = [K.matmul_mxfp8(x, w) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(20):
        for s, x, out in zip(streams, xs, got):
            with torch.cuda.stream(s):
                out.append(K.matmul_mxfp8(x, w))
    torch.cuda.synchronize()
    for out, y in zip(got, want):
        assert all(torch.equal(o, y) for o in out)


def test_calls_follow_the_current_stream_and_replay_in_a_graph():
    m, n, k = 100, 1024, 4096
    x, r = rnd(m, k, seed=1).to(DEV), rnd(m, k, seed=2).to(DEV)
    w = torch.ones(k, dtype=torch.bfloat16, device=DEV)
    g, u, d = (dev(normal_pair(*s, i, 0.05)) for i, s in enumerate(((n, k), (n, k), (k, n))))

    def step():
        h, c, s = K.add_rmsnorm_mxfp8(x, r, w)
        return K.matmul_mxfp8(K.matmul_swiglu_mxfp8((c, s), g, u, quantize=True), d, residual=h)
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    side.synchronize()
    assert torch.equal(on_side, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        x.copy_(rnd(m, k, seed=10 + i))
        eager = step()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_refusals():
    x, w = dev(exact_pair(4, 96, 1)), dev(exact_pair(64, 96, 2))
    b = torch.zeros(64, dtype=torch.bfloat16, device=DEV)
    for bad in (lambda: K.matmul_mxfp8((x[0].cpu(), x[1].cpu()), w), lambda: K.matmul_mxfp8(x, (w[0].cpu(), w[1])),
                lambda: K.matmul_mxfp8(x, w, b.cpu()), lambda: K.mxfp8_quantize(torch.zeros(2, 32)),
                lambda: K.matmul_mxfp8(x, w, residual=torch.zeros(4, 64, dtype=torch.bfloat16))):
        with pytest.raises(RuntimeError):
            bad()
    for bad in (lambda: K.matmul_mxfp8((x[0].view(torch.uint8), x[1]), w), lambda: K.matmul_mxfp8(x, w, b.float()),
                lambda: K.matmul_mxfp8(torch.zeros(4, 96, device=DEV), w),
                lambda: K.matmul_mxfp8(x, w, out=torch.zeros(4, 64, device=DEV)),
                lambda: K.mxfp8_quantize(torch.zeros(2, 32, device=DEV, dtype=torch.float16)),
                lambda: K.add_rmsnorm_mxfp8(b[None], None, b.float())):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: K.matmul_mxfp8((x[0][:, :64], x[1]), w), lambda: K.matmul_mxfp8((x[0][:, :64], x[1][:, :2]), w),
                lambda: K.matmul_mxfp8(x, w, b[:5]), lambda: K.matmul_mxfp8(x, w, activation="relu"),
                lambda: K.matmul_mxfp8(x, (w[0][:40], w[1][:40]), quantize=True),
                lambda: K.matmul_mxfp8(x, w, residual=b), lambda: K.matmul_mxfp8(x, w, out=b[None].expand(4, 64)),
                lambda: K.matmul_mxfp8(x, w, quantize=True, out=torch.empty(4, 64, dtype=torch.bfloat16, device=DEV)),
                lambda: K.matmul_segments_mxfp8(x, []), lambda: K.matmul_segments_mxfp8(x, [w] * 5),
                lambda: K.matmul_segments_mxfp8(x, [w], [b, b]),
                lambda: K.matmul_swiglu_mxfp8(x, w, (w[0][:32], w[1][:32])),
                lambda: K.mxfp8_quantize(b[:40]), lambda: K.add_rmsnorm_mxfp8(b[None], b[None, :32], b),
                lambda: K.add_rmsnorm_mxfp8(b[None, :48], None, b[:48]), lambda: K.add_rmsnorm_mxfp8(b[None], None, b[:32])):
        with pytest.raises(ValueError):
            bad()
    with torch.enable_grad():
        p = torch.zeros(64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
        leaf = x[0].clone().requires_grad_(True)
        for bad in (lambda: K.matmul_mxfp8(x, w, p), lambda: K.mxfp8_quantize(p), lambda: K.add_rmsnorm_mxfp8(p, None, b),
                    lambda: K.matmul_mxfp8((leaf, x[1]), w), lambda: K.mxfp8_dequantize(leaf, x[1])):
            with pytest.raises(NotImplementedError):
                bad()
