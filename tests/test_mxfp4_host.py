"""MXFP4 without a GPU: the float64 oracle against the format's definition, and the C entry points' refusals, which
come before any device work."""
import ctypes

import pytest
import torch

from oracle import mxfp4 as M
from qwen3_5_vl_cuda_custom_amd import _lib

FAKE = 0x100000  # a non-null, aligned address that validation never dereferences


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def test_oracle_rounds_to_the_nearest_code_ties_to_even():
    x = torch.zeros(1, 32, dtype=torch.float64)
    x[0, :15] = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.01, 7.9, -0.2, -0.26, -6.5, 1.0, 3.0])
    codes, scales = M.quantize(x)
    want = [4.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, 6.0, -0.0, -0.5, -6.0, 1.0, 3.0]
    assert int(scales) == 127 and M.values(codes, scales)[0, :15].tolist() == want
    again = M.quantize(M.values(codes, scales))  # what a code stands for keeps its code
    assert torch.equal(again[0], codes) and torch.equal(again[1], scales)


def test_oracle_scales():
    x = torch.zeros(6, 32, dtype=torch.float64)
    x[1, 3], x[2, 0], x[3, 9] = -2.0 ** 20, 2.0 ** -130, 1.999
    x[4, 1], x[5, 2] = float("inf"), float("nan")
    codes, scales = M.quantize(x)
    assert scales.flatten().tolist() == [0, 145, 0, 125, 255, 255]
    assert torch.isnan(M.values(codes, scales)[4:]).all() and not codes[4:].any()


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def test_quantize_refusals(L):
    q = L.q3_mxfp4_quantize
    assert q(None, FAKE, FAKE, 4, 64, 64, 1, None) == -1
    assert q(FAKE, FAKE, FAKE, 4, 48, 48, 1, None) == -2
    assert q(FAKE, FAKE, FAKE, 4, 64, 32, 1, None) == -2
    assert q(FAKE, FAKE, FAKE, 4, 64, 64, 2, None) == -3
    assert q(FAKE + 2, FAKE, FAKE, 4, 64, 64, 1, None) == -4
    assert q(FAKE, FAKE, FAKE, 4, 64, 68, 1, None) == -4
    assert q(FAKE, FAKE, FAKE, 0, 64, 64, 1, None) == 0
    d = L.q3_mxfp4_dequantize
    assert d(FAKE, FAKE, FAKE, 1, 1, 48, i64(0, 0, 0, 0), 1, None) == -2
    assert d(FAKE, FAKE, FAKE, 1, 1, 64, None, 1, None) == -1
    assert d(FAKE, FAKE, FAKE, 300, 300, 64, i64(0, 0, 0, 0), 1, None) == -5
    assert d(FAKE, FAKE, FAKE, 2, 1, 64, i64(33, 0, 0, 0), 1, None) == -4
    assert d(FAKE, FAKE, FAKE, 2, 1, 0, i64(0, 0, 0, 0), 1, None) == 0


def test_matmul_refusals(L):
    def mm(M_=4, N=64, K=64, x=FAKE, w=FAKE, ldx=64, ldw=32, lds=2, ldr=0, ldc=64, dt=1, ws=None, nws=0, res=None):
        return L.q3_matmul_mxfp4(x, w, FAKE, None, res, FAKE, M_, N, K, ldx, ldw, lds, ldr, ldc, dt, ws, nws, None)
    assert mm(x=None) == -1
    assert mm(K=48) == -2 and mm(K=0) == -2 and mm(ldw=16) == -2 and mm(lds=1) == -2 and mm(ldc=63) == -2
    assert mm(res=FAKE, ldr=60) == -2
    assert mm(dt=0) == -3
    assert mm(x=FAKE + 2) == -4 and mm(w=FAKE + 4) == -4 and mm(ldw=40) == -4
    big = dict(M_=5000, N=4096, K=12288, ldx=12288, ldw=6144, lds=384, ldc=4096)  # expands its weights
    need = L.q3_matmul_mxfp4_workspace_bytes(5000, 4096, 12288)
    assert need > 0 and mm(**big, ws=FAKE, nws=need - 1) == -6 and mm(**big) == -6
    assert mm(M_=0) == 0 and mm(N=0) == 0


def test_few_rows_refusals(L):
    def ptrs(*v):
        return (ctypes.c_void_p * len(v))(*v)

    def seg(x=FAKE, nw=None, c=ptrs(FAKE, FAKE), s=ptrs(FAKE, FAKE), n=i64(64, 32), nseg=2, M_=4, K=256, ldx=256,
            ldc=96, dt=1):
        return L.q3_matmul_segments_mxfp4(x, nw, 1e-6, c, s, None, n, nseg, FAKE, M_, K, ldx, ldc, dt, None)
    assert seg(x=None) == -1 and seg(c=ptrs(FAKE, None)) == -1 and seg(s=None) == -1
    assert seg(nseg=0) == -2 and seg(nseg=5) == -2 and seg(n=i64(64, 0)) == -2 and seg(ldc=95) == -2 and seg(ldx=128) == -2
    assert seg(K=48, ldx=48) == -2 and seg(dt=0) == -3
    assert seg(M_=65) == -5 and seg(K=96) == -5 and seg(nw=FAKE, K=8320, ldx=8320) == -5 and seg(nw=FAKE, M_=33) == -5
    assert seg(x=FAKE + 2) == -4 and seg(nw=FAKE + 8) == -4 and seg(ldx=260) == -4
    assert seg(c=ptrs(FAKE, FAKE + 8)) == -4 and seg(s=ptrs(FAKE + 1, FAKE)) == -4
    assert seg(M_=0) == 0

    def sw(g=FAKE, u=FAKE, M_=4, N=64, K=256, ldc=64):
        return L.q3_matmul_swiglu_mxfp4(FAKE, None, 0.0, g, FAKE, u, FAKE, FAKE, M_, N, K, K, ldc, 1, None)
    assert sw(g=None) == -1 and sw(ldc=63) == -2 and sw(M_=65) == -5 and sw(K=160) == -5 and sw(u=FAKE + 8) == -4
    assert sw(N=0) == 0 and sw(M_=0) == 0


def test_cache_refusals(L):
    st = i64(*([128] * 14))

    def append(k=FAKE, lens=FAKE, B=2, S=1, H=2, D=128, cap=32, s=st, dt=1):
        return L.q3_kv_append_mxfp4(k, FAKE, FAKE, FAKE, FAKE, FAKE, lens, B, S, H, D, cap, s, dt, None)
    assert append(k=None) == -1 and append(lens=None) == -1 and append(s=None) == -1
    assert append(B=-1) == -2 and append(H=0) == -2 and append(B=1 << 20, S=1 << 20) == -2
    assert append(dt=3) == -3
    assert append(D=48) == -5 and append(D=512) == -5
    assert append(k=FAKE + 4) == -4 and append(s=i64(4, *([128] * 13))) == -4
    assert append(B=0) == 0 and append(S=0) == 0

    def decode(q=FAKE, B=2, Hq=8, H=2, D=128, cap=32, s=st, dt=1, nws=1 << 30, ws=FAKE, kc=FAKE):
        return L.q3_decode_attention_mxfp4(q, kc, FAKE, FAKE, FAKE, FAKE, 0, FAKE, B, Hq, H, D, cap, s, 1.0, dt, ws,
                                           nws, None)
    assert decode(q=None) == -1 and decode(s=None) == -1
    assert decode(Hq=7) == -2 and decode(cap=-1) == -2
    assert decode(dt=0) == -3
    assert decode(kc=FAKE + 8) == -4 and decode(s=i64(4, *([128] * 13))) == -4
    assert decode(D=96) == -5 and decode(B=1025) == -5
    assert decode(cap=20000, nws=100) == -6 and decode(cap=20000, ws=None) == -6
    assert decode(cap=20000, ws=FAKE + 8) == -4
    assert L.q3_decode_attention_mxfp4_workspace_bytes(2, 8, 2, 128, 32) == 0  # a block per pair
    assert decode(B=0) == 0

    def chunk(Sq=64, ml=128, nws=1 << 30, ws=FAKE):
        return L.q3_flash_attention_cache_mxfp4(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 2, 8, 2, Sq, 128, ml, st,
                                                1.0, 0, 1, ws, nws, None)
    assert chunk(Sq=129) == -2 and chunk(ml=20000, nws=0) == -6 and chunk(ml=20000, ws=None) == -6
    assert chunk(Sq=0) == 0


def test_fused_append_refusals(L):
    st, sec = i64(*([128] * 20)), i64(24, 20, 20)

    def f(q=FAKE, w=FAKE, kw=FAKE, D=128, s=st, sec=sec, dt=1, B=2, S=1, kc=FAKE):
        return L.q3_qk_norm_rope_mxfp4(q, FAKE, FAKE, FAKE, kc, FAKE, FAKE, FAKE, w, kw, FAKE, FAKE, FAKE, 32, B, S, 8,
                                       2, D, sec, 1e-6, bytes(s), dt, None)
    assert f(q=None) == -1 and f(kw=None) == -1
    assert f(sec=i64(24, 20, 21)) == -2 and f(B=1 << 20, S=1 << 20) == -2
    assert f(dt=0) == -3
    assert f(D=96, sec=i64(16, 16, 16)) == -5
    assert f(q=FAKE + 8) == -4 and f(kc=FAKE + 2) == -4 and f(s=i64(4, *([128] * 19))) == -4
    assert f(B=0) == 0 and f(S=0) == 0


def test_cache_lengths_on_the_host():
    from qwen3_5_vl_cuda_custom_amd.modules import MXFP4KVCache
    c = MXFP4KVCache(3, 2, 40, 64, device="cpu")
    assert c.batch == 3 and c.empty and [t.shape[-1] for t in c.tensors] == [32, 2, 32, 2]
    c.set_lens([5, 0, 33])
    assert (c.min_len, c.max_len, c.lens.tolist()) == (0, 33, [5, 0, 33])
    c.reserve(7)
    with pytest.raises(ValueError, match="MXFP4KVCache overflow"):
        c.reserve(1)
    assert c.host_state() == (7, 40)
    for bad in (lambda: c.set_lens([41, 0, 0]), lambda: c.set_lens([1]), lambda: MXFP4KVCache(1, 1, 8, 96, device="cpu"),
                lambda: MXFP4KVCache(1025, 1, 8, 64, device="cpu"), lambda: c.gather(41),
                lambda: c.check_kernels(torch.float32, 2, 64), lambda: c.check_kernels(torch.bfloat16, 2, 128),
                lambda: c.check_kernels(torch.bfloat16, 4, 64)):
        with pytest.raises(ValueError):
            bad()
    c.check_kernels(torch.bfloat16, 2, 64)


@pytest.mark.parametrize("scale", [0.0, -1.0, float("inf"), float("nan")])
def test_attention_refuses_a_scale_that_is_not_positive(L, scale):
    st = i64(*([128] * 14))
    assert L.q3_decode_attention_mxfp4(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 0, FAKE, 2, 8, 2, 128, 32, st, scale, 1, None,
                                       0, None) == -2
    for Sq in (4, 1000):  # streamed, and over expanded rows
        assert L.q3_flash_attention_cache_mxfp4(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 2, 64, 8, Sq, 128, 1000, st, scale,
                                                0, 1, FAKE, 1 << 40, None) == -2


def test_chunks_of_few_columns_keep_to_the_four_bit_rows(L):
    """A chunk whose columns (tokens x query heads of a KV head) read a row only a few times streams the cache, however
    many sequences it has: its workspace is records, not the rows in bf16."""
    ws = L.q3_flash_attention_cache_mxfp4_workspace_bytes
    for B, Hq, Hkv, Sq in ((256, 32, 8, 2), (256, 32, 8, 4), (64, 128, 32, 3), (1024, 8, 8, 16), (256, 32, 8, 48)):
        sets = -(-Sq * (Hq // Hkv) // 16)
        for max_len in (300, 8192):
            assert ws(B, Hq, Hkv, Sq, 128, max_len) <= 8192 + (256 * 12 + B * Hkv * sets) * 16 * 130 * 4
    assert ws(256, 32, 8, 64, 128, 8192) == 4 * 256 * 8 * 8192 * 128  # 16 times: expanded
