"""MXFP8 without a GPU: the float64 oracle against the format's definition, and the C entry points' refusals, which
come before any device work."""
import ctypes

import pytest
import torch

from oracle import mxfp8 as M
from qwen3_5_vl_cuda_custom_amd import _lib

FAKE = 0x100000  # a non-null, aligned address that validation never dereferences


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def ptrs(*v):
    return (ctypes.c_void_p * len(v))(*v)


def test_oracle_values_are_the_type():
    codes = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn)
    v = M.values(codes, torch.full((8,), 127, dtype=torch.uint8))
    assert torch.equal(torch.nan_to_num(v, nan=-1.0), torch.nan_to_num(codes.double(), nan=-1.0))


def test_oracle_rounds_to_the_nearest_code_ties_to_even():
    x = torch.zeros(1, 32, dtype=torch.float64)
    given = [256.0, 17.0, 19.0, 21.0, 1.0625, 1.1875, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -9, -2.0 ** -11, 200.0, -441.0]
    x[0, :12] = torch.tensor(given)
    codes, scales = M.quantize(x)
    want = [256.0, 16.0, 20.0, 20.0, 1.0, 1.25, 2.0 ** -9, 0.0, 2.0 ** -8, -0.0, 192.0, -448.0]
    assert int(scales) == 127 and M.values(codes, scales)[0, :12].tolist() == want
    again = M.quantize(M.values(codes, scales))  # what a code stands for keeps its code
    assert torch.equal(again[0].view(torch.uint8), codes.view(torch.uint8)) and torch.equal(again[1], scales)


def test_oracle_scales():
    x = torch.zeros(9, 32, dtype=torch.float64)
    x[1, 3], x[2, 0], x[3, 9], x[4, 9] = -2.0 ** 20, 2.0 ** -130, 448.0, 448.5
    x[5, 1], x[6, 2], x[7, 2], x[8, 0] = float("inf"), float("nan"), 224.0, 3.4e38
    codes, scales = M.quantize(x)
    assert scales.flatten().tolist() == [0, 139, 0, 127, 128, 255, 255, 126, 247]
    assert torch.isnan(M.values(codes, scales)[5:7]).all() and not codes.view(torch.uint8)[5:7].any()


def test_quantize_refusals(L):
    q = L.q3_mxfp8_quantize
    assert q(None, FAKE, FAKE, 4, 64, 64, 1, None) == -1
    assert q(FAKE, FAKE, None, 4, 64, 64, 1, None) == -1
    assert q(FAKE, FAKE, FAKE, 4, 48, 48, 1, None) == -2 and q(FAKE, FAKE, FAKE, -1, 64, 64, 1, None) == -2
    assert q(FAKE, FAKE, FAKE, 4, 64, 32, 1, None) == -2
    assert q(FAKE, FAKE, FAKE, 4, 64, 64, 2, None) == -3
    assert q(FAKE + 2, FAKE, FAKE, 4, 64, 64, 1, None) == -4 and q(FAKE, FAKE + 4, FAKE, 4, 64, 64, 1, None) == -4
    assert q(FAKE, FAKE, FAKE, 4, 64, 68, 1, None) == -4
    assert q(FAKE, FAKE, FAKE, 0, 64, 64, 1, None) == 0
    d = L.q3_mxfp8_dequantize
    assert d(FAKE, FAKE, FAKE, 48, 1, None) == -2 and d(FAKE, None, FAKE, 64, 1, None) == -1
    assert d(FAKE, FAKE, FAKE, 64, 3, None) == -3 and d(FAKE, FAKE, FAKE + 8, 64, 1, None) == -4
    assert d(FAKE, FAKE, FAKE, 0, 1, None) == 0


def test_norm_refusals(L):
    def norm(x=FAKE, r=FAKE, w=FAKE, h=FAKE, c=FAKE, s=FAKE, rows=4, cols=64, ldx=64, ldr=64, dt=1):
        return L.q3_add_rmsnorm_mxfp8(x, r, w, h, c, s, rows, cols, ldx, ldr, 1e-6, dt, None)
    assert norm(x=None) == -1 and norm(w=None) == -1 and norm(s=None) == -1
    assert norm(h=None) == -1 and norm(r=None) == -1  # the sum goes with the residual
    assert norm(cols=48) == -2 and norm(cols=0) == -2 and norm(ldx=32) == -2 and norm(ldr=32) == -2
    assert norm(dt=2) == -3
    assert norm(x=FAKE + 2) == -4 and norm(ldx=68) == -4 and norm(w=FAKE + 8) == -4 and norm(c=FAKE + 4) == -4
    assert norm(cols=1 << 24, ldx=1 << 24, ldr=1 << 24) == -5
    assert norm(rows=0) == 0


def test_matmul_refusals(L):
    def mm(M_=4, N=64, K=64, x=FAKE, xs=FAKE, w=FAKE, ws=FAKE, res=None, y=FAKE, yc=None, ys=None, ldr=0, ldc=64, act=0):
        return L.q3_matmul_mxfp8(x, xs, w, ws, None, res, y, yc, ys, M_, N, K, ldr, ldc, act, None, 0, None)
    assert mm(x=None) == -1 and mm(xs=None) == -1 and mm(w=None) == -1 and mm(ws=None) == -1
    assert mm(y=None) == -1 and mm(yc=FAKE, ys=FAKE) == -1 and mm(y=None, yc=FAKE) == -1  # one output, whole
    assert mm(K=48) == -2 and mm(K=0) == -2 and mm(ldc=63) == -2 and mm(res=FAKE, ldr=60) == -2 and mm(M_=-1) == -2
    assert mm(y=None, yc=FAKE, ys=FAKE, N=48) == -2  # no whole blocks
    assert mm(x=FAKE + 8) == -4 and mm(w=FAKE + 4) == -4 and mm(y=None, yc=FAKE + 4, ys=FAKE) == -4
    assert mm(act=3) == -5 and mm(act=-1) == -5 and mm(K=1 << 23) == -5
    assert mm(M_=0) == 0 and mm(N=0) == 0


def test_segments_and_swiglu_refusals(L):
    def seg(x=FAKE, c=ptrs(FAKE, FAKE), s=ptrs(FAKE, FAKE), n=i64(64, 32), nseg=2, y=FAKE, M_=4, K=256, ldc=96):
        return L.q3_matmul_segments_mxfp8(x, FAKE, c, s, None, n, nseg, y, M_, K, ldc, None, 0, None)
    assert seg(x=None) == -1 and seg(c=ptrs(FAKE, None)) == -1 and seg(s=None) == -1 and seg(y=None) == -1
    assert seg(n=i64(64, 0)) == -2 and seg(nseg=5) == -2 and seg(nseg=0) == -2 and seg(ldc=95) == -2 and seg(K=40) == -2
    assert seg(c=ptrs(FAKE, FAKE + 4)) == -4
    assert seg(M_=0) == 0

    def sw(x=FAKE, g=FAKE, u=FAKE, us=FAKE, y=FAKE, yc=None, ys=None, M_=4, N=64, K=64, ldc=64):
        return L.q3_matmul_swiglu_mxfp8(x, FAKE, g, FAKE, u, us, y, yc, ys, M_, N, K, ldc, None, 0, None)
    assert sw(g=None) == -1 and sw(us=None) == -1 and sw(y=None) == -1
    assert sw(K=16) == -2 and sw(ldc=60) == -2 and sw(y=None, yc=FAKE, ys=FAKE, N=40) == -2
    assert sw(u=FAKE + 8) == -4
    assert sw(M_=0) == 0 and sw(N=0) == 0


def test_workspace_query_takes_any_sizes(L):
    q = L.q3_matmul_mxfp8_workspace_bytes
    assert q(0, i64(64), 1, 64, 0) == 0 and q(4, None, 1, 64, 0) == 0 and q(4, i64(64), 9, 64, 0) == 0
    assert q(4, i64(-5), 1, 64, 0) == 0 and q(4, i64(64), 1, 48, 0) == 0
    assert all(q(m, i64(n), 1, k, 0) >= 0 for m in (1, 65, 5000) for n in (1, 300, 20000) for k in (32, 4096, 65536))


def test_scales_and_workspaces_are_checked(L):
    def mm(M_=4, N=64, K=256, xs=FAKE, ws=FAKE, work=None, size=0):
        return L.q3_matmul_mxfp8(FAKE, xs, FAKE, ws, None, None, FAKE, None, None, M_, N, K, 0, N, 0, work, size, None)
    assert mm(xs=FAKE + 2) == -4 and mm(ws=FAKE + 1) == -4
    big = dict(M_=4096, N=4096, K=4096)
    need = L.q3_matmul_mxfp8_workspace_bytes(4096, i64(4096), 1, 4096, 0)
    assert need == 2 * 4096 * 4096 // 32  # the scales of both
    assert mm(**big) == -6 and mm(**big, work=FAKE, size=need - 1) == -6 and mm(**big, work=FAKE + 8, size=need) == -4
    assert mm(**big, size=need) == -6  # a size without memory
    q = L.q3_matmul_mxfp8_workspace_bytes
    assert all(q(m, i64(n), 1, k, s) == 0 for m in (1, 64) for n in (1, 200000) for k in (96, 4096) for s in (0, 1))
    assert q(1000, i64(4096), 1, 4096, 0) == 0 and q(1000, i64(4096), 1, 4128, 0) > 0  # scales by rows: whole words of them


@pytest.mark.parametrize("kind", ["CudaLinearMXFP4", "CudaLinearMXFP8"])
@pytest.mark.parametrize("name", ["gate_proj", "up_proj"])
def test_mlp_asks_no_bias_of_a_module_beside_a_quantised_projection(kind, name, monkeypatch):
    """A projection may be any module; the kernels are stubbed, only the way through the MLP is tested."""
    from qwen3_5_vl_cuda_custom_amd import modules
    from qwen3_5_vl_cuda_custom_amd.modules import mlp
    cls = getattr(modules, kind)
    monkeypatch.setattr(cls, "forward", lambda self, x, residual=None, out=None: x[..., :1].expand(*x.shape[:-1], 64) + 0)
    monkeypatch.setattr(mlp, "swiglu", lambda g, u: g * u)
    m = modules.CudaSwiGLUMLP(32, 64).requires_grad_(False)
    for n in ("gate_proj", "up_proj", "down_proj"):
        setattr(m, n, torch.nn.Identity() if n == name else cls(32, 64, bias=False))
    m.down_proj.forward = lambda x, residual=None: x + residual
    x = torch.full((2, 64), 3.0)
    assert torch.equal(m(x, residual=x), x * x + x)


def test_launches_of_2_to_the_32_threads_are_refused(L):
    """A launch has less than 2^32 threads along x: what would need more says so before any device work."""
    q, d = L.q3_mxfp8_quantize, L.q3_mxfp8_dequantize
    assert q(FAKE, FAKE, FAKE, 1 << 31, 32, 32, 1, None) == -5 and q(FAKE, FAKE, FAKE, 1 << 20, 1 << 16, 1 << 16, 0, None) == -5
    assert d(FAKE, FAKE, FAKE, 1 << 36, 1, None) == -5

    def mm(M_, N, K, work=FAKE, size=1 << 62):
        return L.q3_matmul_mxfp8(FAKE, FAKE, FAKE, FAKE, None, None, FAKE, None, None, M_, N, K, 0, N, 0, work, size, None)
    assert mm(1, 1 << 29, 32) == -5  # weight rows by 32, loads into registers
    assert mm(1, (1 << 31) - 300, 128) == -5  # by 96, through the ring
    assert mm((1 << 31) - 300, 600, 32) == -5  # tiles of any size

    def seg(M_, n, K):
        ns = i64(*n)
        return L.q3_matmul_segments_mxfp8(FAKE, FAKE, ptrs(*[FAKE] * len(n)), ptrs(*[FAKE] * len(n)), None, ns, len(n), FAKE,
                                          M_, K, sum(n), FAKE, 1 << 62, None)
    assert seg(1 << 29, (1, 1, 1, 1), 32) == -5
    sw = L.q3_matmul_swiglu_mxfp8
    assert sw(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None, None, 33, 1 << 29, 128, 1 << 29, None, 0, None) == -5


def test_products_of_few_rows_need_no_workspace(L):
    """Up to _FEW_ROWS rows the calls do not ask for its size."""
    from qwen3_5_vl_cuda_custom_amd.kernels.mxfp8 import _FEW_ROWS
    q = L.q3_matmul_mxfp8_workspace_bytes
    for m in (1, 16, _FEW_ROWS):
        for k in (32, 96, 128, 4096, 65536, (1 << 23) - 32):
            for ns in ((1,), (300,), (151936,), ((1 << 31) - 300,), (4096, 1024, 1024), (5, 300, 1, 77)):
                assert q(m, i64(*ns), len(ns), k, 0) == 0
                assert len(ns) > 1 or q(m, i64(*ns), 1, k, 1) == 0
