"""MXFP4 operators on the GPU against their definition in float64 (oracle/mxfp4.py).

Quantisation and its inverse are exact, so they must agree to the bit. The products round once to bf16 (relative
2^-8 at most) after an fp32 sum of K terms (each addition 2^-24 of the magnitudes summed so far; twice that is
allowed). Attention adds the rounding of its weights to bf16 (2^-8 of each) and the fp32 error of a score s, which
its weight sees as a relative error: the dot product's D 2^-24 sum |q k|, and 2^-22 (1 + |s|) for the scaling and
the exponential.
"""
import math

import pytest
import torch

from oracle import mxfp4 as M
from qwen3_5_vl_cuda_custom_amd import _lib
from qwen3_5_vl_cuda_custom_amd import kernels as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = 2.0 ** -8  # half a step of bf16, relative


def rnd(*shape, seed=0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype)


def same_bits(a, b):
    a, b = a.cpu(), b.cpu()
    return a.dtype == b.dtype and torch.equal(torch.nan_to_num(a.double(), nan=12345.0),
                                              torch.nan_to_num(b.double(), nan=12345.0))


def special_rows(dtype):
    """Blocks at which quantisation can go wrong: zeros, one value, ties, saturation, the smallest and largest."""
    t = torch.zeros(12, 32, dtype=torch.float64)
    t[1, 5] = -3.5
    t[2] = torch.linspace(-7.9, 7.9, 32)
    t[3, :16] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0,
                              4.0])
    t[4] = t[3] * 2.0 ** -120
    t[5] = t[3] * 2.0 ** 100
    t[6] = torch.arange(32) * 2.0 ** -131  # below the smallest scale's reach: subnormal inputs
    t[7, 0], t[7, 1:] = 3.0e38, 1e-3
    t[8, 3] = math.inf
    t[9, 31] = math.nan
    t[10, 0], t[10, 1] = -0.0, -1e-30
    t[10, 2] = 1.0
    t[11] = 2.0 ** -126 * torch.linspace(-1, 1, 32)
    return t.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 96), (257, 128), (64, 4096), (5, 1152 * 2)])
def test_quantize_and_back_match_the_definition(rows, cols, dtype):
    x = rnd(rows, cols, seed=rows, dtype=dtype) * torch.exp2(torch.randint(-20, 20, (rows, 1))).to(dtype)
    codes, scales = K.mxfp4_quantize(x.to(DEV))
    want_c, want_s = M.quantize(x)
    assert torch.equal(scales.cpu(), want_s) and torch.equal(codes.cpu(), want_c)
    for out in (torch.bfloat16, torch.float32):
        back = K.mxfp4_dequantize(codes, scales, out)
        assert back.dtype == out and same_bits(back.double(), M.values(want_c, want_s))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_special_blocks(dtype):
    x = special_rows(dtype)
    codes, scales = K.mxfp4_quantize(x.to(DEV))
    want_c, want_s = M.quantize(x)
    assert torch.equal(scales.cpu(), want_s) and torch.equal(codes.cpu(), want_c)
    back = K.mxfp4_dequantize(codes, scales).cpu()
    assert torch.isnan(back[8:10]).all() and torch.isfinite(back[:8]).all()


def test_quantize_strided_and_empty_inputs():
    x = rnd(6, 7, 256, seed=3).to(DEV)
    for view in (x[:, :, 64:128], x[::2], x.transpose(0, 1), x[:, 1:, 8:200:2][..., :96], x[:0], x[..., :0]):
        codes, scales = K.mxfp4_quantize(view)
        assert codes.shape == (*view.shape[:-1], view.shape[-1] // 2)
        if view.numel():
            want_c, want_s = M.quantize(view.cpu())
            assert torch.equal(codes.cpu(), want_c) and torch.equal(scales.cpu(), want_s)


def test_dequantize_every_code_and_scale():
    codes = torch.arange(256, dtype=torch.uint8).view(1, 16, 16).expand(256, 16, 16).contiguous()
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1, 1).expand(256, 16, 1).contiguous()
    for out in (torch.bfloat16, torch.float32):  # scales 253 and 254 reach past the types' range: infinities
        want = M.values(codes, scales).to(out)
        assert bool((same_bits(K.mxfp4_dequantize(codes.to(DEV), scales.to(DEV), out), want)))
        assert torch.equal(want.double()[:253], M.values(codes, scales)[:253])


def test_dequantize_reads_cache_slices_in_place():
    codes = torch.randint(0, 256, (3, 4, 50, 64), dtype=torch.uint8)
    scales = torch.randint(100, 140, (3, 4, 50, 4), dtype=torch.uint8)
    c, s = codes.to(DEV), scales.to(DEV)
    for sl in ((slice(None), slice(None), slice(7, 30)), (slice(1, 3), slice(2, 3), slice(0, 1)),
               (slice(None), slice(None), slice(0, 50, 7)), (slice(0, 0),), (2, slice(1, 3), slice(5, 9))):
        assert same_bits(K.mxfp4_dequantize(c[sl], s[sl]).double(), M.values(codes[sl], scales[sl]))


# ------------------------------------------------------------------ products
def check_matmul(y, x, codes, scales, b=None, r=None):
    w, x = M.values(codes, scales), x.double()
    ref, mag = x @ w.T, x.abs() @ w.abs().T
    for t in (b, r):
        if t is not None:
            ref, mag = ref + t.double(), mag + t.double().abs()
    err = (x.shape[-1] + 2) * 2.0 ** -23 * mag
    tol = HALF * (ref.abs() + err) + err
    d = (y.double().cpu() - ref).abs()
    assert y.dtype == torch.bfloat16 and bool((d <= tol).all()), float((d / tol).max())


def weight(n, k, seed):
    return M.quantize(rnd(n, k, seed=seed, dtype=torch.float32) * 0.05)


@pytest.mark.parametrize("m", [1, 2, 4, 5, 16, 17, 32, 33, 64, 65, 130, 300])
@pytest.mark.parametrize("n,k", [(1, 32), (17, 96), (130, 160), (256, 4096), (1000, 1056), (64, 8224)])
def test_matmul_matches_float64(m, n, k):
    codes, scales = weight(n, k, seed=n)
    x = rnd(m, k, seed=m)
    y = K.matmul_mxfp4(x.to(DEV), codes.to(DEV), scales.to(DEV))
    check_matmul(y, x, codes, scales)


@pytest.mark.parametrize("m,n,k", [(1100, 8000, 96), (200, 66000, 64), (2500, 4100, 128), (900, 1001, 2080)])
def test_matmul_many_tiles_and_expanded_weights(m, n, k):
    codes, scales = weight(n, k, seed=n)
    x, b, r = rnd(m, k, seed=m), rnd(n, seed=1), rnd(m, n, seed=2)
    y = K.matmul_mxfp4(x.to(DEV), codes.to(DEV), scales.to(DEV), b.to(DEV), r.to(DEV))
    check_matmul(y, x, codes, scales, b, r)


# one to six 16-row groups per block, and more blocks than CUs
@pytest.mark.parametrize("m", [3, 4, 12, 31, 64])
@pytest.mark.parametrize("n,k", [(4001, 128), (6000, 640), (12003, 640), (16000, 1152), (24000, 512), (30001, 128)])
def test_matmul_few_rows_of_large_weights(m, n, k):
    codes, scales = weight(n, k, seed=n)
    x, b, r = rnd(m, k, seed=m), rnd(n, seed=1), rnd(m, n, seed=2)
    y = K.matmul_mxfp4(x.to(DEV), codes.to(DEV), scales.to(DEV), b.to(DEV), r.to(DEV))
    check_matmul(y, x, codes, scales, b, r)


# tiles of 32, 64 and 128 rows, their scales by words and by bytes, odd N, split k and not; expanded weights
@pytest.mark.parametrize("m,n,k", [(20, 4096, 12288), (20, 1001, 12320), (50, 1024, 8192), (50, 1003, 8224), (300, 4096, 8192),
                                   (300, 4001, 8224), (200, 40000, 640), (1500, 8192, 2048)])
def test_matmul_tiles_and_expansion(m, n, k):
    codes, scales = weight(n, k, seed=n)
    x, b, r = rnd(m, k, seed=m), rnd(n, seed=1), rnd(m, n, seed=2)
    dc, ds = codes.to(DEV), scales.to(DEV)
    check_matmul(K.matmul_mxfp4(x.to(DEV), dc, ds, b.to(DEV), r.to(DEV)), x, codes, scales, b, r)
    x[1, 7] = math.nan
    y = K.matmul_mxfp4(x.to(DEV), dc, ds).cpu()
    assert torch.isnan(y[1]).all() and torch.isfinite(y[[i for i in range(m) if i != 1]]).all()


@pytest.mark.parametrize("m", [65, 130, 300])
@pytest.mark.parametrize("n,k", [(1, 64), (37, 480), (300, 640), (4000, 96)])
def test_matmul_many_rows_of_small_weights(m, n, k):
    codes, scales = weight(n, k, seed=n)
    wide = rnd(m, k + 32, seed=m)
    x, b, r = wide[:, :k], rnd(n, seed=1), rnd(m, n, seed=2)
    y = K.matmul_mxfp4(wide.to(DEV)[:, :k], codes.to(DEV), scales.to(DEV), b.to(DEV), r.to(DEV))
    check_matmul(y, x, codes, scales, b, r)


@pytest.mark.parametrize("m", [2, 16, 32, 50])
def test_matmul_scales_at_odd_addresses_and_long_rows(m):
    n, k = 150, 9216 if m < 50 else 256
    codes, scales = weight(n, k, seed=15)
    odd = torch.empty(scales.numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(scales.shape)
    odd.copy_(scales)
    x = rnd(m, k, seed=m)
    for s in (odd, scales.to(DEV)):
        check_matmul(K.matmul_mxfp4(x.to(DEV), codes.to(DEV), s), x, codes, scales)


def normed(x, nw, eps):
    """x * nw / rms(x) in float64, and the sum of the magnitudes' share of the rounding of x * nw to bf16."""
    x = x.double()
    return x * nw.double() * (x.square().mean(-1, keepdim=True) + eps).rsqrt()


SEGMENTS = [((40,), 128), ((256, 64, 64), 512), ((1000, 96, 96), 1152), ((7, 9, 130, 33), 256), ((4096, 1024, 1024), 2048),
            ((30, 50), 96)]


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("m", [1, 4, 7, 16, 32, 40, 64, 70])
@pytest.mark.parametrize("ns,k", SEGMENTS)
def test_matmul_segments_matches_float64(ns, k, m, norm):
    ws = [weight(n, k, seed=n) for n in ns]
    bs = [rnd(n, seed=n + 1) if i != 1 else None for i, n in enumerate(ns)]
    x, nw, eps = rnd(m, k, seed=m), rnd(k, seed=3) * 0.2 + 1, 1e-5
    kw = dict(norm_weight=nw.to(DEV), eps=eps) if norm else {}
    y = K.matmul_segments_mxfp4(x.to(DEV).view(1, m, k), [(c.to(DEV), s.to(DEV)) for c, s in ws],
                                [b if b is None else b.to(DEV) for b in bs], **kw)
    assert y.shape == (1, m, sum(ns)) and y.dtype == torch.bfloat16
    at = 0
    xn = normed(x, nw, eps) if norm else x.double()
    for (c, s), b, n in zip(ws, bs, ns):
        w = M.values(c, s)
        ref, mag = xn @ w.T, xn.abs() @ w.abs().T
        # The norm adds one rounding to bf16 of each x, and fp32 errors of its own sum and square root.
        err = (k + 2) * 2.0 ** -23 * mag + (mag * (HALF + (k + 4) * 2.0 ** -23) if norm else 0)
        if b is not None:
            ref, err = ref + b.double(), err + 2.0 ** -23 * b.double().abs()
        tol = HALF * (ref.abs() + err) + err
        d = (y[0, :, at:at + n].double().cpu() - ref).abs()
        assert bool((d <= tol).all()), float((d / tol).max())
        at += n


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("m", [1, 4, 7, 16, 32, 40, 64, 70])
@pytest.mark.parametrize("n,k", [(40, 128), (1001, 640), (12288, 512), (15000, 128), (300, 4096), (64, 96)])
def test_matmul_swiglu_matches_float64(n, k, m, norm):
    (gc, gs), (uc, us) = weight(n, k, seed=n), weight(n, k, seed=n + 1)
    x, nw, eps = rnd(m, k, seed=m), rnd(k, seed=3) * 0.2 + 1, 1e-5
    kw = dict(norm_weight=nw.to(DEV), eps=eps) if norm else {}
    y = K.matmul_swiglu_mxfp4(x.to(DEV), (gc.to(DEV), gs.to(DEV)), (uc.to(DEV), us.to(DEV)), **kw)
    xn = normed(x, nw, eps) if norm else x.double()
    wg, wu = M.values(gc, gs), M.values(uc, us)
    g, u = xn @ wg.T, xn @ wu.T
    share = (k + 2) * 2.0 ** -23 + (HALF + (k + 4) * 2.0 ** -23 if norm else 0)
    if m > 64 or k % 128:  # two products, each rounded to bf16
        eg, eu = ((1 + HALF) * share * (xn.abs() @ w.abs().T) + HALF * t.abs() for w, t in ((wg, g), (wu, u)))
    else:
        eg, eu = (share * (xn.abs() @ w.abs().T) for w in (wg, wu))
    silu = torch.nn.functional.silu
    # |silu'| <= 1.1; fp32's exponential, sum, reciprocal and product: 2^-20 of the result (|g| <= 16 here).
    assert float(g.abs().max()) <= 16
    err = 1.1 * eg * (u.abs() + eu) + silu(g).abs() * eu + 2.0 ** -20 * (silu(g) * u).abs()
    ref = silu(g) * u
    tol = HALF * (ref.abs() + err) + err
    d = (y.double().cpu() - ref).abs()
    assert y.shape == (m, n) and bool((d <= tol).all()), float((d / tol).max())


def test_segments_and_swiglu_of_many_rows_over_expanded_weights():
    m, k, ns = 2100, 1024, (4096, 1024, 2048)
    ws = [weight(n, k, seed=n) for n in ns]
    dev = [(c.to(DEV), s.to(DEV)) for c, s in ws]
    x = rnd(m, k, seed=61)
    b = rnd(1024, seed=62)
    y = K.matmul_segments_mxfp4(x.to(DEV), dev, [None, b.to(DEV), None]).cpu()
    for i, at in enumerate((0, 4096, 5120)):
        check_matmul(y[:, at:at + ns[i]], x, *ws[i], b if i == 1 else None)
    gate, up = weight(8192, k, seed=63), weight(8192, k, seed=64)
    y = K.matmul_swiglu_mxfp4(x.to(DEV), *(tuple(t.to(DEV) for t in w) for w in (gate, up)))
    w = [M.values(*t) for t in (gate, up)]
    g, u = (x.double() @ t.T for t in w)
    eg, eu = ((k + 2) * 2.0 ** -23 * (x.double().abs() @ t.abs().T) for t in w)
    ref = torch.nn.functional.silu(g) * u
    # as in test_matmul_swiglu_matches_float64, in one epilogue
    err = 1.1 * eg * (u.abs() + eu) + torch.nn.functional.silu(g).abs() * eu + 2.0 ** -20 * ref.abs()
    assert float(g.abs().max()) <= 16
    assert bool(((y.double().cpu() - ref).abs() <= HALF * (ref.abs() + err) + err).all())


def test_few_rows_keep_nan_and_infinity_to_their_row_and_weight():
    k, m = 256, 7
    ws = [weight(n, k, seed=n) for n in (40, 24)]
    ws[1][1][3, 1] = 255
    x = rnd(m, k, seed=1)
    x[2, 5] = math.nan
    x[4, 200] = math.inf
    dev = [(c.to(DEV), s.to(DEV)) for c, s in ws]
    nw = torch.ones(k, dtype=torch.bfloat16, device=DEV)
    for kw in ({}, dict(norm_weight=nw, eps=1e-6)):
        y = K.matmul_segments_mxfp4(x.to(DEV), dev, **kw).cpu()
        assert torch.isnan(y[:, 43]).all() and torch.isnan(y[2]).all() and not torch.isfinite(y[4, :40]).any()
        keep = [i for i in range(m) if i not in (2, 4)]
        assert torch.isfinite(y[keep][:, [j for j in range(64) if j != 43]]).all()


@pytest.mark.parametrize("m", [1, 3, 20, 70])
def test_matmul_bias_residual_out_and_strides(m):
    n, k = 136, 320
    codes, scales = weight(n, k, seed=9)
    wide = rnd(m, k + 64, seed=1)
    x, b, r = wide[:, 32:32 + k], rnd(n, seed=2), rnd(m, n, seed=3)
    buf = torch.full((m, 3 * n), 7.0, dtype=torch.bfloat16, device=DEV)
    y = K.matmul_mxfp4(wide.to(DEV)[:, 32:32 + k], codes.to(DEV), scales.to(DEV), b.to(DEV), r.to(DEV),
                       out=buf[:, n:2 * n])
    assert y.data_ptr() == buf[:, n:].data_ptr()
    check_matmul(buf[:, n:2 * n], x, codes, scales, b, r)
    assert bool((buf[:, :n] == 7).all()) and bool((buf[:, 2 * n:] == 7).all())
    x3 = rnd(2, m, k, seed=4)
    y3 = K.matmul_mxfp4(x3.to(DEV), codes.to(DEV), scales.to(DEV), None, None)
    assert y3.shape == (2, m, n)
    check_matmul(y3.reshape(-1, n), x3.reshape(-1, k), codes, scales)
    assert K.matmul_mxfp4(x3.to(DEV)[:0], codes.to(DEV), scales.to(DEV)).shape == (0, m, n)


@pytest.mark.parametrize("m", [3, 20, 50, 70])
def test_matmul_keeps_a_rows_nan_and_infinity_to_itself(m):
    n, k = 96, 256
    codes, scales = weight(n, k, seed=11)
    scales[5, 2] = 255  # a weight row that could not be quantised
    x = rnd(m, k, seed=5)
    x[1, 7] = math.nan
    x[2, k - 1] = math.inf
    y = K.matmul_mxfp4(x.to(DEV), codes.to(DEV), scales.to(DEV)).cpu()
    assert torch.isnan(y[:, 5]).all() and torch.isnan(y[1]).all() and not torch.isfinite(y[2]).any()
    keep = [i for i in range(m) if i not in (1, 2)]
    ok = [j for j in range(n) if j != 5]
    check_matmul(y[keep][:, ok], x[keep], codes[ok], scales[ok])


# ------------------------------------------------------------------ the cache
class Cache:
    """A four-bit cache with random rows; rows at or past lens[b] + used hold NaN scales, which nothing may see."""

    def __init__(self, lens, hkv, cap, d, seed, used=0):
        B = len(lens)
        size = torch.exp(0.5 * rnd(d, seed=seed + 2, dtype=torch.float32))
        self.kc, self.ks = M.quantize((rnd(B, hkv, cap, d, seed=seed, dtype=torch.float32) * size))
        self.vc, self.vs = M.quantize((rnd(B, hkv, cap, d, seed=seed + 1, dtype=torch.float32) * size))
        self.lens = torch.tensor(lens, dtype=torch.int32)
        for b, n in enumerate(lens):
            self.ks[b, :, n + used:] = 255
            self.vs[b, :, n + used:] = 255

    def device(self):
        return tuple(t.to(DEV) for t in (self.kc, self.ks, self.vc, self.vs))

    def values(self):
        return M.values(self.kc, self.ks), M.values(self.vc, self.vs)


def check_attention(o, q, cache, seen, scale):
    """o, q (B, Hq, Sq, D) against float64 at the bound of the module's docstring."""
    k, v = cache.values()
    ref, spread = M.attention(q, k, v, seen, scale)
    D, rows = q.shape[-1], max(int(seen.max()), 1)
    G = q.shape[1] // k.shape[1]
    # sum |q k| of the largest score a query sees (rows behind hold NaN: left out)
    mag = torch.einsum("bhid,bhkd->bhik", q.double().abs(), k.abs().repeat_interleave(G, 1)).nan_to_num(0.0)
    for b in range(q.shape[0]):
        for i in range(q.shape[2]):
            mag[b, :, i, max(int(seen[b, i]), 0):] = 0
    mag = mag.amax(-1, keepdim=True) * scale
    weight_err = HALF + 2 * (D * 2.0 ** -24 * mag + 2.0 ** -22 * (1 + mag)) + rows * 2.0 ** -23
    tol = weight_err * spread * (1 + HALF) + HALF * ref.abs()
    d = (o.double().cpu() - ref).abs()
    assert bool((d <= tol).all()), float((d / tol.clamp(min=1e-300)).max())


LENS = [0, 1, 31, 32, 33, 257, 700]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hkv,groups", [(1, 1), (2, 3), (8, 4), (2, 8), (1, 16), (2, 20), (1, 33)])
def test_decode_matches_float64(hkv, groups, d):
    c = Cache(LENS, hkv, 700, d, seed=groups)
    q = rnd(len(LENS), hkv * groups, d, seed=4)
    lens = c.lens.to(DEV)
    o = K.decode_attention_mxfp4(q.to(DEV), *c.device(), lens, d ** -0.5)
    assert torch.equal(lens.cpu(), c.lens)
    check_attention(o.unsqueeze(2), q.unsqueeze(2), c, c.lens.view(-1, 1), d ** -0.5)
    assert bool((o[0] == 0).all())


# (lengths, KV heads, group, capacity): a block of four or of eight waves per pair, and units split between all waves
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lens,hkv,groups,cap", [([0, 1, 33, 300, 512], 8, 4, 512), ([1100, 0, 1200, 31] * 4, 8, 4, 1200),
                                                 ([1500, 700], 2, 4, 1500), ([5, 0, 600] * 10, 16, 1, 600),
                                                 ([1300, 64, 0], 40, 2, 1300), ([700] * 3, 90, 1, 700)])
def test_decode_by_pairs_and_split(lens, hkv, groups, cap, d):
    c = Cache(lens, hkv, cap, d, seed=51, used=0)
    q = rnd(len(lens), hkv * groups, d, seed=52)
    o = K.decode_attention_mxfp4(q.to(DEV), *c.device(), c.lens.to(DEV), d ** -0.5)
    check_attention(o.unsqueeze(2), q.unsqueeze(2), c, c.lens.view(-1, 1), d ** -0.5)


def test_decode_of_many_pairs_split_between_waves():
    """2160 pairs of one column: their records are merged by one wave each. Against float64 on the GPU: the weights'
    rounding to bf16 (2^-8 of each), an fp32 score's error (64 2^-24 sum |q k| scale < 2^-12 of a weight, as the sum stays
    below 64), the fp32 sums (700 2^-23) and the output's rounding."""
    B, H, cap, d = 24, 90, 700, 64
    g = torch.Generator().manual_seed(57)
    kc, vc = (torch.randint(0, 256, (B, H, cap, d // 2), generator=g, dtype=torch.uint8).to(DEV) for _ in range(2))
    ks, vs = (torch.randint(122, 127, (B, H, cap, d // 32), generator=g, dtype=torch.uint8).to(DEV) for _ in range(2))
    lens = torch.randint(0, cap + 1, (B,), generator=g, dtype=torch.int32).to(DEV)
    lens[0], lens[1] = 0, cap
    q = rnd(B, H, d, seed=58).to(DEV)
    o = K.decode_attention_mxfp4(q, kc, ks, vc, vs, lens, 0.1).double()
    k, v = K.mxfp4_dequantize(kc, ks).double(), K.mxfp4_dequantize(vc, vs).double()
    assert float((q.double().abs()[:, :, None] * k.abs()).sum(-1).max()) * 0.1 < 64
    sc = (q.double()[:, :, None] * k).sum(-1) * 0.1
    sc.masked_fill_(torch.arange(cap, device=DEV) >= lens[:, None, None], -math.inf)
    w = torch.softmax(sc, -1).nan_to_num(0.0)  # an empty sequence: zeros
    ref, spread = (w[..., None] * v).sum(2), (w[..., None] * v.abs()).sum(2)
    tol = (HALF + 2.0 ** -11 + 700 * 2.0 ** -23) * spread * (1 + HALF) + HALF * ref.abs()
    assert bool(((o - ref).abs() <= tol).all()) and not o[0].any()


@pytest.mark.parametrize("sq", [1, 3])
def test_nan_rows_where_units_are_split_between_waves(sq):
    """A value's NaN block reaches its block of the outputs that see it, a key's every output of its head, no other."""
    cap, n = 3000, [2500, 1700]
    c = Cache(n, 2, cap, 128, seed=55, used=sq)
    clean = Cache(n, 2, cap, 128, seed=55, used=sq)
    q = rnd(2, 8, sq, 128, seed=56)
    c.vs[0, 0, 1234, 2] = 255
    c.vs[1, 0, 1700 + sq - 1, 1] = 255  # the last token's own value
    c.ks[1, 1, 7, 0] = 255
    lens = c.lens.to(DEV)

    def run(k):
        if sq == 1:
            return K.decode_attention_mxfp4(q.to(DEV)[:, :, 0], *k.device(), lens, 0.1, append=True).unsqueeze(2).cpu()
        return K.flash_attention_cache_mxfp4(q.to(DEV), *k.device(), c.lens.to(DEV), 0.1, 4).cpu()

    o = run(c)
    lens.copy_(c.lens)
    ref = run(clean)
    bad = torch.zeros(o.shape, dtype=torch.bool)
    bad[0, :4, :, 64:96] = True
    bad[1, :4, -1:, 32:64] = True
    bad[1, 4:] = True
    assert torch.equal(torch.isnan(o), bad) and torch.isfinite(ref).all()
    assert torch.equal(o[~bad], ref[~bad])


@pytest.mark.parametrize("cap", [100, 1500])
def test_steps_advance_past_the_capacity_alike(cap):
    """Both forms attend to the rows up to the capacity and advance every length by one, the full ones too."""
    c = Cache([cap - 1, cap, 3], 1, cap, 128, seed=53, used=1)
    q, lens = rnd(3, 4, 128, seed=54), c.lens.to(DEV)
    o = K.decode_attention_mxfp4(q.to(DEV), *c.device(), lens, 0.1, append=True)
    assert lens.tolist() == [cap, cap + 1, 4]
    check_attention(o.unsqueeze(2), q.unsqueeze(2), c, (c.lens + 1).clamp(max=cap).view(-1, 1), 0.1)


def test_decode_one_long_sequence_and_large_scores():
    c = Cache([5003], 2, 5003, 128, seed=5)
    q = rnd(1, 8, 128, seed=6) * 6
    o = K.decode_attention_mxfp4(q.to(DEV), *c.device(), c.lens.to(DEV), 128 ** -0.5)
    check_attention(o.unsqueeze(2), q.unsqueeze(2), c, c.lens.view(-1, 1), 128 ** -0.5)


def test_decode_step_attends_to_the_new_row_and_advances():
    c = Cache(LENS[:-1] + [699], 2, 700, 128, seed=7, used=1)
    q, lens = rnd(len(LENS), 8, 128, seed=8), c.lens.to(DEV)
    out = torch.full((len(LENS), 3, 8, 128), 5.0, dtype=torch.bfloat16, device=DEV)
    o = K.decode_attention_mxfp4(q.to(DEV).unsqueeze(2), *c.device(), lens, 128 ** -0.5, append=True, out=out[:, 1])
    assert torch.equal(lens.cpu(), c.lens + 1)
    check_attention(o.unsqueeze(2), q.unsqueeze(2), c, (c.lens + 1).view(-1, 1), 128 ** -0.5)
    assert bool((out[:, 0] == 5).all()) and bool((out[:, 2] == 5).all())


def test_decode_reads_cache_slices_and_strided_queries():
    c = Cache([90, 0, 33, 128], 6, 128, 128, seed=9)
    kc, ks, vc, vs = (t[1:3, 2:5] for t in c.device())
    q = rnd(2, 128, 12, 2, seed=10)
    qd = q.to(DEV).permute(3, 2, 0, 1).reshape(2, 24, 128)[:, ::2]  # head rows two apart
    o = K.decode_attention_mxfp4(qd, kc, ks, vc, vs, c.lens.to(DEV)[1:3].contiguous(), 0.1)
    sub = Cache([1], 1, 1, 128, seed=0)
    sub.kc, sub.ks, sub.vc, sub.vs = (t[1:3, 2:5] for t in (c.kc, c.ks, c.vc, c.vs))
    check_attention(o.unsqueeze(2), qd.cpu().unsqueeze(2), sub, c.lens[1:3].view(-1, 1), 0.1)


def test_decode_nan_row_reaches_its_block_of_the_output_only():
    c = Cache([64, 64], 1, 64, 128, seed=11)
    c.vs[0, 0, 40, 2] = 255
    q = rnd(2, 4, 128, seed=12)
    o = K.decode_attention_mxfp4(q.to(DEV), *c.device(), c.lens.to(DEV), 0.1).cpu()
    assert torch.isnan(o[0, :, 64:96]).all() and torch.isfinite(o[0, :, :64]).all() and torch.isfinite(o[0, :, 96:]).all()
    assert torch.isfinite(o[1]).all()
    c.ks[0, 0, 3, 0] = 255  # a key of NaN: the sequence's softmax is NaN
    o = K.decode_attention_mxfp4(q.to(DEV), *c.device(), c.lens.to(DEV), 0.1).cpu()
    assert torch.isnan(o[0]).all() and torch.isfinite(o[1]).all()


# (KV heads, group, tokens): the last ones over the expanded cache
CHUNKS = [(1, 1, 2), (2, 4, 3), (1, 4, 4), (2, 4, 5), (2, 3, 40), (1, 8, 33), (2, 2, 100), (1, 1, 16), (1, 1, 17), (4, 8, 45), (9, 5, 75),
          (9, 5, 110), (13, 4, 92)]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hkv,groups,sq", CHUNKS)
def test_chunk_matches_float64(hkv, groups, sq, d):
    lens = [0, 1, 30, 63, 200]
    c = Cache(lens, hkv, 310, d, seed=sq, used=sq)
    q = rnd(len(lens), sq, hkv * groups, d, seed=13).transpose(1, 2)
    dl = c.lens.to(DEV)
    o = K.flash_attention_cache_mxfp4(q.to(DEV), *c.device(), dl, d ** -0.5, groups, advance=True,
                                      max_len=200 + sq)
    assert torch.equal(dl.cpu(), c.lens + sq)
    seen = c.lens.view(-1, 1) + 1 + torch.arange(sq)
    check_attention(o, q, c, seen, d ** -0.5)


def test_chunk_of_one_token_is_the_decode_step():
    c = Cache([0, 40, 99], 2, 100, 128, seed=14, used=1)
    q = rnd(3, 8, 1, 128, seed=15).to(DEV)
    a = K.flash_attention_cache_mxfp4(q, *c.device(), c.lens.to(DEV), 0.1, 4)
    b = K.decode_attention_mxfp4(q, *c.device(), c.lens.to(DEV), 0.1, append=True)
    assert torch.equal(a[:, :, 0], b)


@pytest.mark.parametrize("groups,sq", [(4, 4), (1, 3)])
def test_short_chunk_a_later_tokens_nan_is_masked(groups, sq):
    c = Cache([20, 31], 1, 64, 128, seed=16, used=sq)
    q = rnd(2, groups, sq, 128, seed=17)
    for b, n in enumerate((20, 31)):
        c.ks[b, :, n + sq - 1] = 255
        c.vs[b, :, n + sq - 1] = 255
    o = K.flash_attention_cache_mxfp4(q.to(DEV), *c.device(), c.lens.to(DEV), 0.1, groups).cpu()
    assert torch.isnan(o[:, :, -1]).all()
    seen = c.lens.view(-1, 1) + 1 + torch.arange(sq - 1)
    check_attention(o[:, :, :-1], q[:, :, :-1], c, seen, 0.1)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("advance", [False, True])
def test_long_chunk_a_nan_row_reaches_the_tokens_that_see_it(d, advance):
    """Past the streaming kernel's pairs, over expanded rows."""
    B, hkv, groups, sq = 2, 15, 8, 100
    assert B * hkv * groups * sq / 16 > 1400
    c = Cache([20, 31], hkv, 140, d, seed=26, used=sq)
    q = rnd(B, hkv * groups, sq, d, seed=27)
    c.vs[0, 0, 20 + 50, 1] = 255  # token 50's value
    c.vs[1, 3, 31 + 7, 0] = 255
    c.ks[1, 4, 31 + 60, 0] = 255  # token 60's key
    clean = Cache([20, 31], hkv, 140, d, seed=26, used=sq)
    lens = c.lens.to(DEV)
    o = K.flash_attention_cache_mxfp4(q.to(DEV), *c.device(), lens, 0.1, groups, advance=advance).cpu()
    ref = K.flash_attention_cache_mxfp4(q.to(DEV), *clean.device(), c.lens.to(DEV), 0.1, groups).cpu()
    bad = torch.zeros(o.shape, dtype=torch.bool)
    bad[0, :groups, 50:, 32:64] = True
    bad[1, 3 * groups:4 * groups, 7:, :32] = True
    bad[1, 4 * groups:5 * groups, 60:] = True
    assert torch.equal(torch.isnan(o), bad)
    # a masked row's weight is zero whatever it holds: the other outputs are the clean cache's to the bit
    assert torch.equal(o[~bad], ref[~bad]) and torch.isfinite(ref).all()
    assert torch.equal(lens.cpu(), c.lens + (sq if advance else 0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_append_writes_its_rows_and_no_other(d, dtype):
    B, S, H, cap = 4, 5, 3, 40
    lens = torch.tensor([0, 7, 36, 40], dtype=torch.int32)  # the last two run past the cap
    kv = rnd(B, S, 2 * H, d, seed=18, dtype=dtype)
    k, v = kv[:, :, :H], kv[:, :, H:]
    cache = [torch.full((B, H, cap, w), 0xA5, dtype=torch.uint8) for w in (d // 2, d // 32, d // 2, d // 32)]
    dev = [t.to(DEV) for t in cache]
    kvd = kv.to(DEV)
    K.kv_append_mxfp4(kvd[:, :, :H], kvd[:, :, H:], *dev, lens.to(DEV))
    for x, c, s in ((k, 0, 1), (v, 2, 3)):
        qc, qs = M.quantize(x)
        for b in range(B):
            for i in range(S):
                if int(lens[b]) + i < cap:
                    cache[c][b, :, int(lens[b]) + i] = qc[b, i]
                    cache[s][b, :, int(lens[b]) + i] = qs[b, i]
    for got, want in zip(dev, cache):
        assert torch.equal(got.cpu(), want)


def test_append_attend_chunk_and_steps_together_under_a_graph():
    """A chunk, then steps, as a layer runs them: eager and as a replayed graph, against float64."""
    B, H, G, D, cap = 2, 2, 4, 128, 80
    c = Cache([0, 0], H, cap, D, seed=19)
    cache, lens = c.device(), torch.tensor([3, 0], dtype=torch.int32, device=DEV)
    k0, v0, q0 = rnd(B, 20, H, D, seed=20), rnd(B, 20, H, D, seed=21), rnd(B, H * G, 20, D, seed=22)
    K.kv_append_mxfp4(k0.to(DEV)[:1, :3], v0.to(DEV)[:1, :3], *(t[:1] for t in cache),
                      torch.zeros(1, dtype=torch.int32, device=DEV))  # three rows of the first sequence
    K.kv_append_mxfp4(k0.to(DEV), v0.to(DEV), *cache, lens)
    o = K.flash_attention_cache_mxfp4(q0.to(DEV), *cache, lens, 0.1, G, advance=True)

    def host():
        c.kc, c.ks, c.vc, c.vs = (t.cpu() for t in cache)
        return c
    check_attention(o, q0, host(), torch.tensor([[3], [0]]) + 1 + torch.arange(20), 0.1)
    k, v, q = (torch.empty(B, 1, H, D, dtype=torch.bfloat16, device=DEV) for _ in range(3))
    q = torch.empty(B, H * G, D, dtype=torch.bfloat16, device=DEV)

    def step():
        K.kv_append_mxfp4(k, v, *cache, lens)
        return K.decode_attention_mxfp4(q, *cache, lens, 0.1, append=True)

    start = lens.clone()
    step()  # once eagerly
    lens.copy_(start)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        k.copy_(rnd(B, 1, H, D, seed=30 + i))
        v.copy_(rnd(B, 1, H, D, seed=40 + i))
        qi = rnd(B, H * G, D, seed=50 + i)
        q.copy_(qi)
        before = lens.cpu()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(lens.cpu(), before + 1)
        check_attention(out.unsqueeze(2), qi.unsqueeze(2), host(), (before + 1).view(-1, 1), 0.1)


def test_offsets_past_32_bits():
    """A cache whose last head starts over 4 GiB into the codes."""
    B, H, D, cap = 2, 4, 128, 9_000_000
    assert (B * H - 1) * cap * D // 2 > 2 ** 31
    cache = [torch.zeros(B, H, cap, w, dtype=torch.uint8, device=DEV) for w in (64, 4, 64, 4)]
    lens = torch.tensor([5, cap - 40], dtype=torch.int32, device=DEV)
    k, v = rnd(B, 40, H, D, seed=23), rnd(B, 40, H, D, seed=24)
    K.kv_append_mxfp4(k.to(DEV), v.to(DEV), *cache, lens)
    back = K.mxfp4_dequantize(cache[0][:, :, cap - 40:], cache[1][:, :, cap - 40:])
    assert same_bits(back[1].double(), M.values(*M.quantize(k))[1].transpose(0, 1))
    q = rnd(1, 4, D, seed=25)  # the last head over its last 40 rows alone
    o = K.decode_attention_mxfp4(q.to(DEV), *(t[1:, 3:, cap - 40:] for t in cache),
                                 torch.tensor([40], dtype=torch.int32, device=DEV), 0.1)
    sub = Cache([40], 1, 40, D, seed=0)
    sub.kc, sub.ks, sub.vc, sub.vs = (t[1:, 3:, cap - 40:].cpu() for t in cache)
    check_attention(o.unsqueeze(2), q.unsqueeze(2), sub, torch.tensor([[40]]), 0.1)
    # all rows but these 40 of the last head: zero values
    full = K.decode_attention_mxfp4(q.to(DEV).repeat(2, 4, 1), *cache, lens, 0.1)
    assert bool((full == 0).all())


# ------------------------------------------------------------------ refusals
def test_refusals():
    d = dict(device=DEV)
    x = torch.zeros(4, 64, dtype=torch.bfloat16, **d)
    u = lambda *s: torch.zeros(*s, dtype=torch.uint8, **d)  # noqa: E731
    lens = torch.zeros(2, dtype=torch.int32, **d)
    cache = (u(2, 2, 32, 64), u(2, 2, 32, 4), u(2, 2, 32, 64), u(2, 2, 32, 4))
    q = torch.zeros(2, 8, 128, dtype=torch.bfloat16, **d)
    kv = torch.zeros(2, 1, 2, 128, dtype=torch.bfloat16, **d)
    for bad, exc in [
        (lambda: K.mxfp4_quantize(x.cpu()), RuntimeError),
        (lambda: K.mxfp4_quantize(x[:, :48]), ValueError),
        (lambda: K.mxfp4_quantize(x.half()), TypeError),
        (lambda: K.mxfp4_dequantize(u(4, 32), u(4, 1)), ValueError),
        (lambda: K.mxfp4_dequantize(u(4, 32), u(3, 2)), ValueError),
        (lambda: K.mxfp4_dequantize(u(4, 32).int(), u(4, 2)), TypeError),
        (lambda: K.mxfp4_dequantize(u(4, 32), u(4, 2), torch.float16), TypeError),
        (lambda: K.matmul_mxfp4(x, u(8, 16), u(8, 1)), ValueError),
        (lambda: K.matmul_mxfp4(x.float(), u(8, 32), u(8, 2)), TypeError),
        (lambda: K.matmul_mxfp4(x, u(8, 32), u(8, 2), bias=x[0, :7]), ValueError),
        (lambda: K.matmul_mxfp4(x, u(8, 32), u(8, 2), residual=x[:, :7]), ValueError),
        (lambda: K.matmul_mxfp4(x, u(8, 32), u(8, 2), out=x[:, :7]), ValueError),
        (lambda: K.matmul_segments_mxfp4(x, []), ValueError),
        (lambda: K.matmul_segments_mxfp4(x, [(u(8, 32), u(8, 2))] * 5), ValueError),
        (lambda: K.matmul_segments_mxfp4(x, [(u(8, 16), u(8, 1))]), ValueError),
        (lambda: K.matmul_segments_mxfp4(x, [(u(8, 32), u(8, 1))]), ValueError),
        (lambda: K.matmul_segments_mxfp4(x, [(u(8, 32), u(8, 2))], [x[0, :7]]), ValueError),
        (lambda: K.matmul_segments_mxfp4(x.float(), [(u(8, 32), u(8, 2))]), TypeError),
        (lambda: K.matmul_segments_mxfp4(x, [(u(8, 32), u(8, 2))], norm_weight=x[0, :32], eps=1e-6), ValueError),
        (lambda: K.matmul_segments_mxfp4(x, [(u(8, 32).cpu(), u(8, 2))]), RuntimeError),
        (lambda: K.matmul_swiglu_mxfp4(x, (u(8, 32), u(8, 2)), (u(9, 32), u(9, 2))), ValueError),
        (lambda: K.matmul_swiglu_mxfp4(x, (u(8, 32), u(8, 2)), (u(8, 32).int(), u(8, 2))), TypeError),
        (lambda: K.kv_append_mxfp4(kv, kv[:, :, :1], *cache, lens), ValueError),
        (lambda: K.kv_append_mxfp4(kv, kv, *cache, lens.long()), ValueError),
        (lambda: K.kv_append_mxfp4(kv, kv, *cache[:3], u(2, 2, 31, 4), lens), ValueError),
        (lambda: K.kv_append_mxfp4(kv[:, :, :1], kv[:, :, :1], *cache, lens), ValueError),
        (lambda: K.decode_attention_mxfp4(q.float(), *cache, lens, 1.0), TypeError),
        (lambda: K.decode_attention_mxfp4(q[:, :7], *cache, lens, 1.0), ValueError),
        (lambda: K.decode_attention_mxfp4(q, *cache, lens[:1], 1.0), ValueError),
        (lambda: K.decode_attention_mxfp4(q[..., :64], *cache, lens, 1.0), ValueError),
        (lambda: K.decode_attention_mxfp4(q, *(t[:, :, ::2] for t in cache), lens, 1.0), ValueError),
        (lambda: K.flash_attention_cache_mxfp4(q.unsqueeze(2), *cache, lens, 1.0, 2), ValueError),
        (lambda: K.flash_attention_cache_mxfp4(q.unsqueeze(2), *cache, lens, 1.0, 4, max_len=33), ValueError),
        (lambda: K.flash_attention_cache_mxfp4(q.unsqueeze(2).expand(2, 8, 40, 128), *cache, lens, 1.0, 4),
         ValueError),  # more tokens than the cache has rows
        (lambda: K.decode_attention_mxfp4(q, *(t[:, :, :0] for t in cache), lens, 1.0), ValueError),
        (lambda: K.decode_attention_mxfp4(q, *cache, lens, 1.0, out=q.transpose(1, 2)), ValueError),
    ]:
        with pytest.raises(exc):
            bad()
    w = torch.zeros(4, 64, dtype=torch.bfloat16, requires_grad=True, **d)
    with torch.enable_grad(), pytest.raises(NotImplementedError):
        K.matmul_mxfp4(w, u(8, 32), u(8, 2))
    with pytest.raises(_lib.Q3Error):  # head dim 32: the cache can be written, not attended to
        K.decode_attention_mxfp4(q[..., :32], u(2, 2, 32, 16), u(2, 2, 32, 1), u(2, 2, 32, 16), u(2, 2, 32, 1), lens, 1.0)


def test_no_sequences_and_no_tokens():
    d = dict(device=DEV)
    u = lambda *s: torch.zeros(*s, dtype=torch.uint8, **d)  # noqa: E731
    for B in (0, 2):
        cache = (u(B, 2, 32, 64), u(B, 2, 32, 4), u(B, 2, 32, 64), u(B, 2, 32, 4))
        lens = torch.ones(B, dtype=torch.int32, **d)
        kv = torch.ones(B, 0, 2, 128, dtype=torch.bfloat16, **d)
        K.kv_append_mxfp4(kv, kv, *cache, lens)
        q = torch.zeros(B, 8, 0, 128, dtype=torch.bfloat16, **d)
        assert K.flash_attention_cache_mxfp4(q, *cache, lens, 1.0, 4, advance=True).shape == q.shape
        if B == 0:
            assert K.decode_attention_mxfp4(q.new_zeros(0, 8, 128), *cache, lens, 1.0, append=True).shape == (0, 8, 128)
        assert not any(t.any() for t in cache) and lens.tolist() == [1] * B
    x = torch.zeros(0, 64, dtype=torch.bfloat16, **d)
    assert K.matmul_mxfp4(x, u(8, 32), u(8, 2)).shape == (0, 8)
    assert K.matmul_segments_mxfp4(x, [(u(8, 32), u(8, 2))] * 2, norm_weight=x.new_ones(64)).shape == (0, 16)
    assert K.matmul_swiglu_mxfp4(x, (u(8, 32), u(8, 2)), (u(8, 32), u(8, 2))).shape == (0, 8)
    one = x.new_ones(1, 128)
    assert K.matmul_segments_mxfp4(one, [(u(8, 64), u(8, 4)), (u(0, 64), u(0, 4))]).tolist() == [[0.0] * 8]
    w = tuple(t.to(DEV) for t in weight(8, 128, seed=1))
    a = K.matmul_segments_mxfp4(2 * one, [w, (u(0, 64), u(0, 4))], norm_weight=one[0], eps=0.0)
    b = K.matmul_mxfp4(one, *w)  # rows of a constant normalise to ones
    assert torch.equal(a, b)
    assert [t.shape for t in K.mxfp4_quantize(x)] == [(0, 32), (0, 2)]


def test_two_streams_at_once():
    """Products, decode steps and chunks issued on two streams without waiting for each other: each call's workspace
    is its own."""
    g = torch.Generator().manual_seed(40)
    codes, scales = (t.to(DEV) for t in M.quantize(torch.randn(4096, 2048, generator=g).to(torch.bfloat16)))
    c = Cache([700, 40, 0], 2, 800, 128, seed=41, used=40)
    dev, lens = c.device(), c.lens.to(DEV)
    xs = [rnd(32, 2048, seed=42 + i).to(DEV) for i in range(2)]
    qs = [rnd(3, 8, 40, 128, seed=44 + i).to(DEV) for i in range(2)]

    def run(i):
        return (K.matmul_mxfp4(xs[i], codes, scales), K.decode_attention_mxfp4(qs[i][:, :, 0], *dev, lens, 0.1),
                K.flash_attention_cache_mxfp4(qs[i], *dev, lens, 0.1, 4))

    want = [run(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(run(i))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            for a, b in zip(r, want[i]):
                assert torch.equal(a, b)


@pytest.mark.parametrize("scale", [0.0, -0.1, math.inf, math.nan])
def test_attention_refuses_a_scale_that_is_not_positive(scale):
    """Masked scores are -inf before they are scaled, and the running maximum is that of the unscaled scores."""
    c = Cache([40, 7], 1, 64, 128, seed=60, used=3)
    q, lens = rnd(2, 4, 3, 128, seed=61).to(DEV), c.lens.to(DEV)
    for run in (lambda: K.decode_attention_mxfp4(q[:, :, 0], *c.device(), lens, scale, append=True),
                lambda: K.flash_attention_cache_mxfp4(q, *c.device(), lens, scale, 4, advance=True)):
        with pytest.raises(ValueError, match="scale"):
            run()
    assert torch.equal(lens.cpu(), c.lens)


@pytest.mark.parametrize("d", [96, 160, 192, 224])
def test_append_of_head_dims_with_an_odd_count_of_blocks(d):
    """Rows of 3, 5, 6 and 7 scales: no address of an allocation is a multiple of those, and none need be."""
    B, S, H, cap = 3, 4, 2, 20
    lens = torch.tensor([0, 7, 18], dtype=torch.int32)  # the last sequence runs past the cap
    k, v = rnd(B, S, H, d, seed=62), rnd(B, S, H, d, seed=63)
    for shift in (0, 1, 2, 3):
        cache = [torch.full((B, H, cap, w), 0xA5, dtype=torch.uint8) for w in (d // 2, d // 32, d // 2, d // 32)]
        dev = [t.to(DEV) for t in cache]
        for i in (1, 3):  # the scales at any byte
            dev[i] = torch.full((cache[i].numel() + shift,), 0xA5, dtype=torch.uint8, device=DEV)[shift:].view(cache[i].shape)
        K.kv_append_mxfp4(k.to(DEV), v.to(DEV), *dev, lens.to(DEV))
        for x, c, s in ((k, 0, 1), (v, 2, 3)):
            qc, qs = M.quantize(x)
            for b in range(B):
                for i in range(S):
                    if int(lens[b]) + i < cap:
                        cache[c][b, :, int(lens[b]) + i] = qc[b, i]
                        cache[s][b, :, int(lens[b]) + i] = qs[b, i]
        for got, want in zip(dev, cache):
            assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("d", [64, 128])
def test_append_writes_scales_at_any_byte_and_attention_refuses_them(d):
    B, H, cap = 2, 2, 16
    k, q = rnd(B, 1, H, d, seed=64).to(DEV), rnd(B, 4, d, seed=65).to(DEV)
    lens = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    even = [torch.zeros(B, H, cap, w, dtype=torch.uint8, device=DEV) for w in (d // 2, d // 32, d // 2, d // 32)]
    odd = [t if i % 2 == 0 else torch.zeros(t.numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(t.shape)
           for i, t in enumerate(t.clone() for t in even)]
    for cache in (even, odd):
        K.kv_append_mxfp4(k, k, *cache, lens)
    for a, b in zip(even, odd):
        assert torch.equal(a, b)
    pos = torch.zeros(3, B, 1, dtype=torch.int32, device=DEV)
    for cache in (even, odd):
        K.qk_norm_rope_mxfp4(q.unsqueeze(1), k, k, torch.empty_like(q.unsqueeze(1)), *cache, None, None, pos,
                             torch.ones(d // 2, device=DEV), (d // 2, 0, 0), 1e-6, lens + 1)
    for a, b in zip(even, odd):
        assert torch.equal(a, b)
    K.decode_attention_mxfp4(q, *even, lens, 0.1)
    for bad in (lambda: K.decode_attention_mxfp4(q, *odd, lens, 0.1),
                lambda: K.flash_attention_cache_mxfp4(q.unsqueeze(2), *odd, lens, 0.1, 2)):
        with pytest.raises(ValueError, match="scales"):
            bad()


@pytest.mark.parametrize("d", [32, 96, 160, 256])
def test_attention_refuses_head_dims_by_the_dim_alone(d):
    u = lambda w: torch.zeros(2, 1, 40, w, dtype=torch.uint8, device=DEV)  # noqa: E731
    q, lens = rnd(2, 2, 1, d).to(DEV), torch.ones(2, dtype=torch.int32, device=DEV)
    cache = (u(d // 2), u(d // 32), u(d // 2), u(d // 32))
    for shift in (0, 1):
        cache = (cache[0], torch.zeros(80 * (d // 32) + shift, dtype=torch.uint8, device=DEV)[shift:].view(2, 1, 40, d // 32),
                 *cache[2:])
        for bad in (lambda: K.decode_attention_mxfp4(q[:, :, 0], *cache, lens, 0.1),
                    lambda: K.flash_attention_cache_mxfp4(q, *cache, lens, 0.1, 2)):
            with pytest.raises(_lib.Q3Error, match="outside what"):
                bad()


# more than 1400 pairs of a KV head and 16 columns, with one to twelve column sets to a head: streamed all the same
@pytest.mark.parametrize("B,hkv,groups,sq,cap,d", [(180, 8, 4, 2, 90, 128), (40, 40, 1, 5, 200, 64), (90, 16, 8, 2, 60, 128),
                                                   (45, 16, 4, 8, 120, 128), (16, 8, 4, 48, 130, 64), (2, 720, 1, 3, 2100, 64)])
def test_chunks_of_few_columns_and_many_sequences(B, hkv, groups, sq, cap, d):
    """Against float64 on the GPU, at the bound of the module's docstring."""
    assert B * hkv * -(-groups * sq // 16) > 1400
    g = torch.Generator().manual_seed(66)
    kc, vc = (torch.randint(0, 256, (B, hkv, cap, d // 2), generator=g, dtype=torch.uint8).to(DEV) for _ in range(2))
    ks, vs = (torch.randint(122, 127, (B, hkv, cap, d // 32), generator=g, dtype=torch.uint8).to(DEV) for _ in range(2))
    lens = torch.randint(0, cap - sq + 1, (B,), generator=g, dtype=torch.int32).to(DEV)
    lens[0], lens[1] = 0, cap - sq
    row = torch.arange(cap, device=DEV)
    for t in (ks, vs):  # rows behind the chunk's: NaN
        t.masked_fill_((row >= (lens + sq)[:, None])[:, None, :, None], 255)
    q, scale, dl = rnd(B, hkv * groups, sq, d, seed=68).to(DEV), 0.1, lens.clone()
    o = K.flash_attention_cache_mxfp4(q, kc, ks, vc, vs, dl, scale, groups, advance=True)
    assert torch.equal(dl, lens + sq)
    k, v = (K.mxfp4_dequantize(*t).double().nan_to_num(0.0) for t in ((kc, ks), (vc, vs)))
    k, q2 = k.transpose(-1, -2).contiguous(), q.double().reshape(B, hkv, groups * sq, d)
    seen = (lens[:, None] + 1 + torch.arange(sq, device=DEV)).repeat(1, groups)[:, None, :, None]
    w = torch.softmax((q2 @ k * scale).masked_fill(row >= seen, -math.inf), -1)
    ref, spread = (w @ t for t in (v, v.abs()))
    mag = float((q2.abs() @ k.abs()).max()) * scale
    err = HALF + 2 * (d * 2.0 ** -24 * mag + 2.0 ** -22 * (1 + mag)) + cap * 2.0 ** -23
    tol = err * spread * (1 + HALF) + HALF * ref.abs()
    assert bool(((o.double().reshape(ref.shape) - ref).abs() <= tol).all())


def test_heads_that_start_past_32_bits():
    """The last head's codes start at 4.3e9 bytes, past 2^32. Everything but the written rows holds codes of 0x77 and
    scales of 255, so an offset cut to 32 bits, signed or not, would read those; the append must have written there."""
    B, H, G, D, cap, n = 2, 4, 4, 128, 9_600_000, 40
    assert (B * H - 1) * cap * (D // 2) > 2 ** 32
    cache = [torch.full((B, H, cap, w), 255 if w == 4 else 0x77, dtype=torch.uint8, device=DEV) for w in (64, 4, 64, 4)]
    assert cache[0][-1, -1].data_ptr() - cache[0].data_ptr() > 2 ** 32
    k, v = rnd(B, n, H, D, seed=69), rnd(B, n, H, D, seed=70)
    K.kv_append_mxfp4(k.to(DEV), v.to(DEV), *cache, torch.zeros(B, dtype=torch.int32, device=DEV))
    small = Cache([n] * B, H, n, D, seed=0)
    small.kc, small.ks = (t.transpose(1, 2).contiguous() for t in M.quantize(k))
    small.vc, small.vs = (t.transpose(1, 2).contiguous() for t in M.quantize(v))
    for big, want in zip(cache, (small.kc, small.ks, small.vc, small.vs)):
        assert torch.equal(big[:, :, :n].cpu(), want)
    assert int((cache[1] != 255).sum()) <= B * H * n * 4  # and nothing else was written
    lens = torch.full((B,), n, dtype=torch.int32, device=DEV)
    q = rnd(B, H * G, D, seed=71)
    o = K.decode_attention_mxfp4(q.to(DEV), *cache, lens, 0.1)
    check_attention(o.unsqueeze(2), q.unsqueeze(2), small, torch.full((B, 1), n), 0.1)
    for sq in (5, 32):
        q = rnd(B, H * G, sq, D, seed=72)
        o = K.flash_attention_cache_mxfp4(q.to(DEV), *cache, lens - sq, 0.1, G)
        check_attention(o, q, small, n - sq + 1 + torch.arange(sq).expand(B, sq), 0.1)
    y = K.mxfp4_dequantize(cache[0][:, :, :n], cache[1][:, :, :n])
    assert same_bits(y.double(), M.values(small.kc, small.ks))
    # the fused form's own addresses; at position 0 the rotation leaves the rows as they are
    rows = k.to(DEV)[:, :1]
    K.qk_norm_rope_mxfp4(rows, rows, v.to(DEV)[:, :1], torch.empty_like(rows), *cache, None, None,
                         torch.zeros(3, B, 1, dtype=torch.int32, device=DEV), torch.ones(D // 2, device=DEV),
                         (D // 2, 0, 0), 1e-6, lens)
    for i, want in enumerate((small.kc, small.ks, small.vc, small.vs)):
        assert torch.equal(cache[i][:, :, n].cpu(), want[:, :, 0])



def test_long_chunk_over_heads_that_start_past_32_bits():
    """Over expanded rows: to the bit what the same rows give in a cache that ends after them."""
    B, H, G, D, cap, sq, n = 2, 4, 16, 128, 9_600_000, 200, 230
    assert B * H * G * sq // 16 > 1400 and (B * H - 1) * cap * (D // 2) > 2 ** 32
    cache = [torch.full((B, H, cap, w), 255 if w == 4 else 0x77, dtype=torch.uint8, device=DEV) for w in (64, 4, 64, 4)]
    k, v, zero = rnd(B, n, H, D, seed=73).to(DEV), rnd(B, n, H, D, seed=74).to(DEV), torch.zeros(B, dtype=torch.int32, device=DEV)
    K.kv_append_mxfp4(k, v, *cache, zero)
    q, lens = rnd(B, H * G, sq, D, seed=75).to(DEV), torch.tensor([n - sq, 3], dtype=torch.int32, device=DEV)
    o = K.flash_attention_cache_mxfp4(q, *cache, lens, 0.1, G, max_len=n)
    ref = K.flash_attention_cache_mxfp4(q, *(t[:, :, :n].contiguous() for t in cache), lens, 0.1, G)
    assert torch.isfinite(o).all() and torch.equal(o, ref)


# Several weights and one, with the norm, whose rows come to three, four and six 16-row groups a block
@pytest.mark.parametrize("m", [1, 3, 7, 16, 20, 32])
@pytest.mark.parametrize("ns,k", [((8192, 1024, 1024), 256), ((9000, 3000, 1), 384), ((14000, 2384), 128), ((24000,), 128),
                                  ((12003,), 640)])
def test_matmul_segments_with_the_norm_of_many_output_rows(ns, k, m):
    ws = [weight(n, k, seed=n) for n in ns]
    x, nw, eps = rnd(m, k, seed=m), rnd(k, seed=3) * 0.2 + 1, 1e-5
    y = K.matmul_segments_mxfp4(x.to(DEV), [(c.to(DEV), s.to(DEV)) for c, s in ws], norm_weight=nw.to(DEV), eps=eps).cpu()
    xn, at = normed(x, nw, eps), 0
    for (c, s), n in zip(ws, ns):
        w = M.values(c, s)
        ref, mag = xn @ w.T, xn.abs() @ w.abs().T
        # as in test_matmul_segments_matches_float64: x * norm weight rounds to bf16, fp32 sums and square root
        err = (k + 2) * 2.0 ** -23 * mag + mag * (HALF + (k + 4) * 2.0 ** -23)
        tol = HALF * (ref.abs() + err) + err
        d = (y[:, at:at + n].double() - ref).abs()
        assert bool((d <= tol).all()), float((d / tol).max())
        at += n


# scales by bytes (K no multiple of 128, or their first byte at an odd address) with one to six 16-row groups a block
@pytest.mark.parametrize("m", [1, 4, 12, 16, 20, 32, 50])
@pytest.mark.parametrize("n,k", [(4001, 96), (6000, 160), (12003, 544), (16000, 96), (24000, 288), (30001, 32)])
def test_matmul_scales_by_bytes_of_many_weight_rows(n, k, m):
    codes, scales = weight(n, k, seed=n)
    x, b, r = rnd(m, k, seed=m), rnd(n, seed=1), rnd(m, n, seed=2)
    y = K.matmul_mxfp4(x.to(DEV), codes.to(DEV), scales.to(DEV), b.to(DEV), r.to(DEV))
    check_matmul(y, x, codes, scales, b, r)


@pytest.mark.parametrize("m", [2, 14, 30])
@pytest.mark.parametrize("n,k", [(6000, 256), (12003, 1024), (24000, 128)])
def test_matmul_scales_at_odd_addresses_of_many_weight_rows(n, k, m):
    codes, scales = weight(n, k, seed=n)
    odd = torch.empty(scales.numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(scales.shape)
    odd.copy_(scales)
    x = rnd(m, k, seed=m)
    check_matmul(K.matmul_mxfp4(x.to(DEV), codes.to(DEV), odd), x, codes, scales)


@pytest.mark.parametrize("m", [1, 20, 64, 200, 700])
def test_products_of_weights_below_the_normal_range(m):
    """Scale bytes 0 to 4: the smallest magnitudes are subnormal in bf16, and enter the products as they are."""
    n, k = (66000, 64) if m == 200 else (600, 1024)  # 200 rows: over the expanded weight
    g = torch.Generator().manual_seed(76)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(0, 5, (n, k // 32), generator=g, dtype=torch.uint8)
    x = rnd(m, k, seed=77, dtype=torch.float32).mul(2.0 ** 110).to(torch.bfloat16)
    y = K.matmul_mxfp4(x.to(DEV), codes.to(DEV), scales.to(DEV))
    check_matmul(y, x, codes, scales)
    if m <= 64:
        w = (codes[:64].to(DEV), scales[:64].to(DEV))
        check_matmul(K.matmul_segments_mxfp4(x.to(DEV), [w])[:, :64], x, codes[:64], scales[:64])


@pytest.mark.parametrize("sq,cap,groups", [(1, 90, 4), (1, 3000, 4), (5, 90, 4), (400, 420, 8)])
def test_attention_over_rows_below_the_normal_range(sq, cap, groups):
    """Keys and values of scale bytes 0 to 4, and queries large enough for scores of ordinary size."""
    B, hkv, d = 2, 16 if sq == 400 else 2, 128
    g = torch.Generator().manual_seed(78)
    kc, vc = (torch.randint(0, 256, (B, hkv, cap, d // 2), generator=g, dtype=torch.uint8).to(DEV) for _ in range(2))
    ks, vs = (torch.randint(0, 5, (B, hkv, cap, d // 32), generator=g, dtype=torch.uint8).to(DEV) for _ in range(2))
    lens = torch.full((B,), cap - sq, dtype=torch.int32, device=DEV)
    q, scale = rnd(B, hkv * groups, sq, d, seed=79, dtype=torch.float32).mul(2.0 ** 120).to(torch.bfloat16).to(DEV), 0.02
    o = K.flash_attention_cache_mxfp4(q, kc, ks, vc, vs, lens, scale, groups)
    k, v = (K.mxfp4_dequantize(*t).double() for t in ((kc, ks), (vc, vs)))
    k, q2 = k.transpose(-1, -2).contiguous(), q.double().reshape(B, hkv, groups * sq, d)
    seen = (lens[:, None] + 1 + torch.arange(sq, device=DEV)).repeat(1, groups)[:, None, :, None]
    w = torch.softmax((q2 @ k * scale).masked_fill(torch.arange(cap, device=DEV) >= seen, -math.inf), -1)
    ref, spread = (w @ t for t in (v, v.abs()))
    mag = float((q2.abs() @ k.abs()).max()) * scale
    assert 0.5 < mag < 64
    err = HALF + 2 * (d * 2.0 ** -24 * mag + 2.0 ** -22 * (1 + mag)) + cap * 2.0 ** -23
    # below 2^-126 bf16 has the step 2^-133, and fp32 (the sums) 2^-149
    tol = err * spread * (1 + HALF) + HALF * ref.abs() + 2.0 ** -134 + cap * 2.0 ** -149
    assert bool(((o.double().reshape(ref.shape) - ref).abs() <= tol).all())
    assert float(spread.max()) > 2.0 ** -128
