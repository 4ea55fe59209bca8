"""Microscaled 4-bit floating point (MXFP4): weights and KV caches at 4.25 bits a value (no reference counterpart;
the reference has bf16 and fp32 only).

A row is cut into blocks of 32 consecutive values, each value a 4-bit float (E2M1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and
their negatives), each block with one power-of-two scale held as its exponent (E8M0: byte s stands for 2^(s - 127),
255 for NaN). `codes` (..., K / 2) uint8 holds value 2j in the low and 2j + 1 in the high half of byte j, `scales`
(..., K / 32) uint8 the blocks' scales. Everything a code stands for is exact in bf16, so the products and the
attention below lose nothing beyond the quantisation itself and the bf16 arithmetic of their unquantised forms.

Inference only. All tensors of a call must be on the current device, whose current stream it uses. The kernels of a
decode step take a few microseconds each, so the checks here are written for their own time.
"""
from __future__ import annotations

import math
from functools import lru_cache
from struct import Struct

import torch

from .. import _lib
from ._common import mfma_operand, require_device, require_no_grad
from .elementwise import swiglu
from .matmul import matmul_segments, matmul_swiglu
from .norms import rmsnorm

MX_BLOCK = 32
MXFP4_FEW_ROWS, MXFP4_NORM_ROWS = 64, 32  # rows of the products over several weights in one launch, with the norm
_U8, _BF16, _F32 = torch.uint8, torch.bfloat16, torch.float32
_i64x4, _i64x14, _i64x20 = Struct("4q").pack, Struct("14q").pack, Struct("20q").pack


@lru_cache(maxsize=4096)
def _matmul_workspace(M: int, N: int, K: int) -> int:
    return _lib.lib().q3_matmul_mxfp4_workspace_bytes(M, N, K)


def _expands(M: int, N: int, K: int) -> bool:
    """Whether q3_matmul_mxfp4 would expand the weight to bf16: its workspace is then the weight (and not sums over
    ranges of k, which only fewer than 256 tiles of 128 x 256 need). Follows plan_of in csrc/mxfp4_matmul.hip."""
    return -(-M // 128) * -(-N // 256) > 256 and _matmul_workspace(M, N, K) == 2 * N * K


@lru_cache(maxsize=1024)
def _decode_workspace(B: int, Hq: int, Hkv: int, D: int, cap: int) -> int:
    return _lib.lib().q3_decode_attention_mxfp4_workspace_bytes(B, Hq, Hkv, D, cap)


def _off_device(op: str, *tensors: torch.Tensor | None) -> None:
    """Raise for tensors that are not all on the current device."""
    require_device(op, *tensors)
    raise RuntimeError(f"{op}: tensors must be on the current device (cuda:{torch.cuda.current_device()})")


def _pair_error(op: str, codes: torch.Tensor, scales: torch.Tensor) -> Exception:
    if codes.dtype != _U8 or scales.dtype != _U8:
        return TypeError(f"{op}: codes and scales must be uint8, got {codes.dtype} and {scales.dtype}")
    return ValueError(f"{op}: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} must be (..., K / 2) and "
                      "(..., K / 32)")


def mxfp4_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of bf16 or fp32 x (..., K), K a multiple of 32.

    A block's scale is 2^(floor(log2 t) - 2), t its largest magnitude (exponent -127 at least, also for a block of
    zeros); a value over the scale rounds to the nearest code, ties to the even one, and saturates at 6. A block
    that holds an infinity or a NaN reads back as NaN.
    """
    dev = x.get_device()
    if dev < 0 or dev != _lib.current_device():
        _off_device("mxfp4_quantize", x)
    if x.requires_grad:
        require_no_grad("mxfp4_quantize", x)
    dt = _lib.dtype_code(x.dtype)
    shape = x.shape
    if not shape or shape[-1] % MX_BLOCK:
        raise ValueError(f"mxfp4_quantize: the last dim of {tuple(shape)} must be a multiple of {MX_BLOCK}")
    K = shape[-1]
    codes = x.new_empty((*shape[:-1], K // 2), dtype=_U8)
    scales = codes.new_empty((*shape[:-1], K // MX_BLOCK))
    n = x.numel()
    if n == 0:
        return codes, scales
    ld = K
    if x.data_ptr() % 16 or not x.is_contiguous():
        x = x.reshape(-1, K)
        ld = x.stride(0) if n > K else K
        if x.stride(1) != 1 or ld < K or x.data_ptr() % 16 or ld * x.element_size() % 16:
            x, ld = x.clone(memory_format=torch.contiguous_format), K
    _lib.call("q3_mxfp4_quantize", x.data_ptr(), codes.data_ptr(), scales.data_ptr(), n // K, K, ld, dt,
              _lib.raw_stream(dev))
    return codes, scales


def mxfp4_dequantize(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values (..., K) in bf16 or fp32, both exact (blocks of scale 255: NaN; the scales past the type's range,
    which mxfp4_quantize never makes, give infinities). Contiguous tensors and (B, H, rows, ...) slices of a cache
    are read in place; other views are copied first."""
    op = "mxfp4_dequantize"
    dev = codes.get_device()
    if dev < 0 or dev != _lib.current_device() or scales.get_device() != dev:
        _off_device(op, codes, scales)
    dt = _lib.dtype_code(dtype)
    shape, sshape = codes.shape, scales.shape
    if (codes.dtype != _U8 or scales.dtype != _U8 or not shape or shape[:-1] != sshape[:-1]
            or shape[-1] != sshape[-1] * (MX_BLOCK // 2)):
        raise _pair_error(op, codes, scales)
    y = codes.new_empty((*shape[:-1], shape[-1] * 2), dtype=dtype)
    n = y.numel()
    if n == 0:
        return y
    n0, n1, st = 1, 1, (0, 0, 0, 0)
    if not (codes.is_contiguous() and scales.is_contiguous() and codes.data_ptr() % 4 == 0):
        cs = codes.stride()
        if (len(shape) >= 3 and shape[0] * shape[1] <= 65535 and codes.data_ptr() % 4 == 0 and cs[0] % 4 == 0
                and cs[1] % 4 == 0 and codes[0, 0].is_contiguous() and scales[0, 0].is_contiguous()):
            n0, n1, st = shape[0], shape[1], (*cs[:2], *scales.stride()[:2])
        else:
            codes, scales = (t.clone(memory_format=torch.contiguous_format) for t in (codes, scales))
    _lib.call("q3_mxfp4_dequantize", codes.data_ptr(), scales.data_ptr(), y.data_ptr(), n0, n1, n // (n0 * n1),
              _i64x4(*st), dt, _lib.raw_stream(dev))
    return y


def _rows(op: str, t: torch.Tensor, n: int) -> tuple[torch.Tensor, int]:
    """t (..., n) as rows of contiguous elements and their stride."""
    if t.is_contiguous():
        return t, n
    t = t.reshape(-1, n)
    if n > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < n:
        t = t.contiguous()
    return t, t.stride(0) if t.shape[0] > 1 else n


def matmul_mxfp4(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, bias: torch.Tensor | None = None,
                 residual: torch.Tensor | None = None, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """matmul with the weight (N, K) held in MXFP4: x·Wᵀ (+ bias) (+ residual), x (..., K) bf16, one rounding.

    Many rows run over the weight expanded to bf16, 2 * N * K bytes of workspace for the time of the call. `out`, when
    given: (..., N) whose rows have one stride and contiguous elements, written in place (a column
    slice of a wider buffer).
    """
    op = "matmul_mxfp4"
    dev = x.get_device()
    if dev < 0 or dev != _lib.current_device() or codes.get_device() != dev or scales.get_device() != dev:
        _off_device(op, x, codes, scales)
    for t in (bias, residual, out):
        if t is not None:
            if t.get_device() != dev:
                _off_device(op, t)
            if t.dtype != _BF16:
                raise TypeError(f"{op}: dtype mismatch ({t.dtype} vs {_BF16})")
            if t.requires_grad:
                require_no_grad(op, t)
    if x.requires_grad:
        require_no_grad(op, x)
    if x.dtype != _BF16:
        raise TypeError(f"{op}: x must be bfloat16, got {x.dtype}")
    xs, ws, ss = x.shape, codes.shape, scales.shape
    if (codes.dtype != _U8 or scales.dtype != _U8 or len(ws) != len(ss) or ws[:-1] != ss[:-1]
            or ws[-1] != ss[-1] * (MX_BLOCK // 2)):
        raise _pair_error(op, codes, scales)
    if len(ws) != 2 or not xs or ws[1] * 2 != xs[-1] or xs[-1] == 0:
        raise ValueError(f"{op}: codes {tuple(ws)} do not match x {tuple(xs)}")
    N, K = ws[0], xs[-1]
    shape = (*xs[:-1], N)
    if bias is not None and bias.shape != (N,):
        raise ValueError(f"{op}: bias {tuple(bias.shape)} != ({N},)")
    if residual is not None and residual.shape != shape:
        raise ValueError(f"{op}: residual {tuple(residual.shape)} != output {shape}")
    if out is None:
        same = residual is not None and residual.is_contiguous()
        y, ldy = torch.empty_like(residual) if same else x.new_empty(shape), N  # empty_like: 0.4 us less
    else:
        if out.shape != shape or (N > 1 and out.stride(-1) != 1):
            raise ValueError(f"{op}: out {tuple(out.shape)} must be {shape} with contiguous elements")
        y, ldy = out, N
        if not out.is_contiguous() and out.numel() > N:
            ldy = out.view(-1, N).stride(0)
            if ldy < N:
                raise ValueError(f"{op}: the rows of out overlap")
    M = x.numel() // K
    if M == 0 or N == 0:
        return y
    x2, ldx = _rows(op, x, K)
    if ldx >= 1 << 22 and K < 1 << 22:  # farther apart than the kernels address
        x2, ldx = x2.contiguous(), K
    if x2.data_ptr() % 16 or ldx % 8:
        x2, ldx = mfma_operand(op, x2.view(-1, K)), K
    r2, ldr = _rows(op, residual, N) if residual is not None else (None, 0)
    if not codes.is_contiguous() or codes.data_ptr() % 16:
        codes = codes.clone(memory_format=torch.contiguous_format)
    if not scales.is_contiguous():
        scales = scales.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    nws = _matmul_workspace(M, N, K)
    ws_ = codes.new_empty(nws) if nws else None
    _lib.call("q3_matmul_mxfp4", x2.data_ptr(), codes.data_ptr(), scales.data_ptr(), _lib.ptr(bias), _lib.ptr(r2),
              y.data_ptr(), M, N, K, ldx, K // 2, K // MX_BLOCK, ldr, ldy, _lib.Q3_BF16, _lib.ptr(ws_), nws,
              _lib.raw_stream(dev))
    return y


def _weight(op: str, K: int, codes: torch.Tensor, scales: torch.Tensor, dev: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The codes and scales of a weight (N, K), packed and aligned as the kernels of few rows read them."""
    if codes.get_device() != dev or scales.get_device() != dev:
        _off_device(op, codes, scales)
    if (codes.dtype != _U8 or scales.dtype != _U8 or codes.dim() != 2 or scales.dim() != 2
            or codes.shape[0] != scales.shape[0] or codes.shape[1] != scales.shape[1] * (MX_BLOCK // 2)):
        raise _pair_error(op, codes, scales)
    if codes.shape[1] * 2 != K:
        raise ValueError(f"{op}: codes {tuple(codes.shape)} do not match x (..., {K})")
    if not codes.is_contiguous() or codes.data_ptr() % 16:
        codes = codes.clone(memory_format=torch.contiguous_format)
    if not scales.is_contiguous() or scales.data_ptr() % 4:
        scales = scales.clone(memory_format=torch.contiguous_format)
    return codes, scales


def _few_rows(op: str, x: torch.Tensor, norm_weight: torch.Tensor | None, *others: torch.Tensor | None) -> tuple:
    """Checks x (..., K), the norm weight and the biases; returns the device, K, M, x as rows, their stride, and
    whether one launch takes the call."""
    dev = x.get_device()
    if dev < 0 or dev != _lib.current_device():
        _off_device(op, x)
    for t in (norm_weight, *others):
        if t is not None and t.get_device() != dev:
            _off_device(op, x, t)
    require_no_grad(op, x, norm_weight, *others)
    if x.dtype != _BF16:
        raise TypeError(f"{op}: x must be bfloat16, got {x.dtype}")
    for t in (norm_weight, *others):
        if t is not None and t.dtype != _BF16:
            raise TypeError(f"{op}: dtype mismatch ({t.dtype} vs {_BF16})")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"{op}: x {tuple(x.shape)} has no columns")
    K = x.shape[-1]
    if norm_weight is not None and norm_weight.shape != (K,):
        raise ValueError(f"{op}: norm weight {tuple(norm_weight.shape)} != ({K},)")
    M = x.numel() // K
    x2, ldx = _rows(op, x, K)
    if x2.data_ptr() % 16 or ldx % 8 or ldx >= 1 << 22:
        x2, ldx = x2.clone(memory_format=torch.contiguous_format), K
    fits = 0 < M <= MXFP4_FEW_ROWS and K % 128 == 0 and K < 1 << 22
    return dev, K, M, x2, ldx, fits


def matmul_segments_mxfp4(x: torch.Tensor, weights, biases=None, *, norm_weight: torch.Tensor | None = None,
                          eps: float = 0.0) -> torch.Tensor:
    """matmul_segments with the weights held in MXFP4: x·[W_0; W_1; ...]ᵀ (+ [b_0; b_1; ...]) over 1 to 4 weights,
    each a pair (codes, scales); returns (..., ΣN_i).

    With norm_weight the rows of x are RMS-normalised first (rmsnorm_matmul_segments). Up to 64 rows of K a multiple of
    128 are one launch (with the norm up to 32 of K at most 8192, else the norm is another); more rows, or another K, a
    product per weight, or where its weight would be expanded to bf16 (many rows), matmul_segments over the expanded
    weights, all of them at once: 2 * ΣN_i * K bytes for the time of the call.
    """
    op = "matmul_segments_mxfp4"
    weights = list(weights)
    biases = list(biases) if biases is not None else [None] * len(weights)
    if not 1 <= len(weights) <= 4 or len(biases) != len(weights):
        raise ValueError(f"{op}: 1 to 4 weights, one bias (or None) each")
    dev, K, M, x2, ldx, fits = _few_rows(op, x, norm_weight, *biases)
    ws = [_weight(op, K, c, s, dev) for c, s in weights]
    ns = [c.shape[0] for c, _ in ws]
    fits = fits and 0 not in ns
    if norm_weight is not None and M > 0 and (not fits or M > MXFP4_NORM_ROWS or K > 8192):
        x = x2 = rmsnorm(x, norm_weight, eps)
        norm_weight, ldx = None, K
    for b, n in zip(biases, ns):
        if b is not None and b.shape != (n,):
            raise ValueError(f"{op}: bias {tuple(b.shape)} != ({n},)")
    y = x.new_empty((*x.shape[:-1], sum(ns)))
    if not fits:
        if M == 0:
            return y
        if 0 not in ns and _expands(M, sum(ns), K):
            return matmul_segments(x, [mxfp4_dequantize(c, s) for c, s in ws], biases)
        at = 0
        for (c, s), b, n in zip(ws, biases, ns):
            matmul_mxfp4(x, c, s, b, out=y[..., at:at + n])
            at += n
        return y
    bs = [b.contiguous() if b is not None else None for b in biases]
    nw = None if norm_weight is None else _aligned(norm_weight)
    _lib.call("q3_matmul_segments_mxfp4", x2.data_ptr(), _lib.ptr(nw), eps, _lib.ptrs(*(c for c, _ in ws)),
              _lib.ptrs(*(s for _, s in ws)), _lib.ptrs(*bs) if any(b is not None for b in bs) else None,
              _lib.i64s(*ns), len(ns), y.data_ptr(), M, K, ldx, sum(ns), _lib.Q3_BF16, _lib.raw_stream(dev))
    return y


def matmul_swiglu_mxfp4(x: torch.Tensor, gate: tuple[torch.Tensor, torch.Tensor],
                        up: tuple[torch.Tensor, torch.Tensor], *, norm_weight: torch.Tensor | None = None,
                        eps: float = 0.0) -> torch.Tensor:
    """matmul_swiglu with the weights held in MXFP4: silu(x·W_gateᵀ)·(x·W_upᵀ), `gate` and `up` pairs (codes, scales)
    of (N, K).

    With norm_weight the rows of x are RMS-normalised first (rmsnorm_matmul_swiglu). Up to 64 rows of K a multiple of
    128 are one launch (with the norm up to 32 of K at most 8192, else the norm is another); more rows, or another K, two
    products and swiglu, or where their weights would be expanded to bf16 (many rows), matmul_swiglu over the expanded
    weights, both at once: 4 * N * K bytes for the time of the call (200 MB at N 12288, K 4096).
    """
    op = "matmul_swiglu_mxfp4"
    dev, K, M, x2, ldx, fits = _few_rows(op, x, norm_weight)
    if norm_weight is not None and M > 0 and (not fits or M > MXFP4_NORM_ROWS or K > 8192):
        x = x2 = rmsnorm(x, norm_weight, eps)
        norm_weight, ldx = None, K
    (gc, gs), (uc, us) = (_weight(op, K, c, s, dev) for c, s in (gate, up))
    if gc.shape != uc.shape:
        raise ValueError(f"{op}: gate {tuple(gc.shape)} and up {tuple(uc.shape)} codes must have one shape")
    N = gc.shape[0]
    if not fits or N == 0:
        if M == 0 or N == 0:
            return x.new_empty((*x.shape[:-1], N))
        if _expands(M, N, K):
            return matmul_swiglu(x, mxfp4_dequantize(gc, gs), mxfp4_dequantize(uc, us))
        return swiglu(matmul_mxfp4(x, gc, gs), matmul_mxfp4(x, uc, us))
    y = x.new_empty((*x.shape[:-1], N))
    nw = None if norm_weight is None else _aligned(norm_weight)
    _lib.call("q3_matmul_swiglu_mxfp4", x2.data_ptr(), _lib.ptr(nw), eps, gc.data_ptr(), gs.data_ptr(), uc.data_ptr(),
              us.data_ptr(), y.data_ptr(), M, N, K, ldx, N, _lib.Q3_BF16, _lib.raw_stream(dev))
    return y


def _aligned(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _check_cache(op: str, dev: int, k_codes, k_scales, v_codes, v_scales, kv_lens, B: int, D: int,
                 align: int = 1) -> tuple:
    """Checks a (B, Hkv, cap, D) cache in MXFP4 and its lengths; returns Hkv, cap and the strides [b, h] of the four
    tensors. align: bytes to which the kernel needs every row of scales aligned."""
    if dev < 0 or dev != _lib.current_device() or kv_lens.get_device() != dev:
        _off_device(op, kv_lens, k_codes)
    if kv_lens.dtype != torch.int32 or kv_lens.shape != (B,) or not kv_lens.is_contiguous():
        raise ValueError(f"{op}: kv_lens must be a contiguous int32 ({B},) device tensor")
    shape = k_codes.shape
    if len(shape) == 4:
        _, Hkv, cap, W = shape
        n = W // 16
        if (W * 2 == D and shape[0] == B and W == n * 16 and v_codes.shape == shape
                and k_scales.shape == v_scales.shape == (B, Hkv, cap, n)
                and k_codes.dtype == k_scales.dtype == v_codes.dtype == v_scales.dtype == _U8
                and k_codes.get_device() == k_scales.get_device() == v_codes.get_device() == v_scales.get_device() == dev
                and k_codes.is_contiguous() and k_scales.is_contiguous() and v_codes.is_contiguous()
                and v_scales.is_contiguous() and (k_codes.data_ptr() | v_codes.data_ptr()) % 16 == 0
                and (k_scales.data_ptr() | v_scales.data_ptr()) % align == 0):
            c, s = (Hkv * cap * W, cap * W), (Hkv * cap * n, cap * n)  # whole caches: the usual call
            return Hkv, cap, (*c, *s, *c, *s)
    st = []
    for c, s in ((k_codes, k_scales), (v_codes, v_scales)):
        if c.get_device() != dev or s.get_device() != dev:
            _off_device(op, c, s)
        cs, ss = c.shape, s.shape
        if (c.dtype != _U8 or s.dtype != _U8 or len(cs) != 4 or len(ss) != 4 or cs[:3] != ss[:3]
                or cs[3] != ss[3] * (MX_BLOCK // 2)):
            raise _pair_error(op, c, s)
        if cs != shape or cs[0] != B or cs[3] * 2 != D:
            raise ValueError(f"{op}: cache codes {tuple(k_codes.shape)} and {tuple(v_codes.shape)} must be "
                             f"({B}, Hkv, cap, {D // 2})")
        ct, s_t = c.stride(), s.stride()
        if cs[2] > 1 and (ct[2] != cs[3] or s_t[2] != ss[3]) or ct[3] != 1 or ss[3] > 1 and s_t[3] != 1:
            raise ValueError(f"{op}: the rows of a cache head must be packed")
        if c.data_ptr() % 16 or ct[0] % 16 or ct[1] % 16:
            raise ValueError(f"{op}: the cache codes must be 16-byte aligned")
        if s.data_ptr() % align or s_t[0] % align or s_t[1] % align:
            raise ValueError(f"{op}: the cache scales must be aligned to a row of them ({align} bytes)")
        st += (ct[0], ct[1], s_t[0], s_t[1])
    return shape[1], shape[2], st


def kv_append_mxfp4(k: torch.Tensor, v: torch.Tensor, k_codes: torch.Tensor, k_scales: torch.Tensor,
                    v_codes: torch.Tensor, v_scales: torch.Tensor, kv_lens: torch.Tensor) -> None:
    """Quantise new key / value rows into a four-bit cache.

    k, v (B, S, Hkv, D) bf16 or fp32, any strides with D contiguous; codes (B, Hkv, cap, D / 2) and scales (B, Hkv,
    cap, D / 32) of keys and values, D a multiple of 32 up to 256; kv_lens (B,) int32: row s of sequence b goes to
    cache row kv_lens[b] + s, and is dropped at or past cap. kv_lens is left as it is (the attention that follows
    advances it).
    """
    op = "kv_append_mxfp4"
    dev, shape = k.get_device(), k.shape
    if v.get_device() != dev:
        _off_device(op, k, v)
    if k.requires_grad or v.requires_grad:
        require_no_grad(op, k, v)
    dt = _lib.dtype_code(k.dtype)
    if k.dtype != v.dtype:
        raise TypeError(f"{op}: dtype mismatch ({v.dtype} vs {k.dtype})")
    if len(shape) != 4 or shape != v.shape:
        raise ValueError(f"{op}: k {tuple(shape)} and v {tuple(v.shape)} must be (B, S, Hkv, D)")
    B, S, Hkv, D = shape
    heads, cap, st = _check_cache(op, dev, k_codes, k_scales, v_codes, v_scales, kv_lens, B, D)
    if heads != Hkv:
        raise ValueError(f"{op}: {Hkv} KV heads for a cache of {heads}")
    if k.numel() == 0 or cap == 0:
        return
    unit = 16 // k.element_size()
    ks, vs = k.stride(), v.stride()
    if k.data_ptr() % 16 or ks[3] != 1 or ks[0] % unit or ks[1] % unit or ks[2] % unit:
        k = k.clone(memory_format=torch.contiguous_format)
        ks = k.stride()
    if v.data_ptr() % 16 or vs[3] != 1 or vs[0] % unit or vs[1] % unit or vs[2] % unit:
        v = v.clone(memory_format=torch.contiguous_format)
        vs = v.stride()
    _lib.call("q3_kv_append_mxfp4", k.data_ptr(), v.data_ptr(), k_codes.data_ptr(), k_scales.data_ptr(),
              v_codes.data_ptr(), v_scales.data_ptr(), kv_lens.data_ptr(), B, S, Hkv, D, cap,
              _i64x14(*ks[:3], *vs[:3], *st), dt, _lib.raw_stream(dev))


def qk_norm_rope_mxfp4(q_in: torch.Tensor, k_in: torch.Tensor, v_in: torch.Tensor, q_out: torch.Tensor,
                       k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor, v_scales: torch.Tensor,
                       q_weight: torch.Tensor | None, k_weight: torch.Tensor | None, positions: torch.Tensor,
                       inv_freq: torch.Tensor, mrope_section, eps: float, kv_lens: torch.Tensor) -> None:
    """qk_norm_rope with the k/v rows quantised into a four-bit cache at rows kv_lens[b] + s, in one launch.

    q_in, q_out (B, S, Hq, D), k_in, v_in (B, S, Hkv, D) bf16 views with 16-byte aligned rows (q_out may be q_in); D
    64, 128 or 256. The rows are rounded to bf16 first, so the cache equals qk_norm_rope followed by kv_append_mxfp4
    to the bit.
    """
    op = "qk_norm_rope_mxfp4"
    ts = (q_in, k_in, v_in, q_out)
    require_no_grad(op, *ts, q_weight, k_weight)
    if any(t.dim() != 4 for t in ts):
        raise ValueError(f"{op}: q, k and v must be (B, S, H, D)")
    B, S, Hq, D = q_in.shape
    dev = q_in.get_device()
    Hkv, cap, st = _check_cache(op, dev, k_codes, k_scales, v_codes, v_scales, kv_lens, B, D)
    if k_in.shape != (B, S, Hkv, D) or v_in.shape != k_in.shape or q_out.shape != q_in.shape:
        raise ValueError(f"{op}: q {tuple(q_in.shape)} -> {tuple(q_out.shape)}, k {tuple(k_in.shape)}, v "
                         f"{tuple(v_in.shape)} for a cache of {Hkv} heads")
    strides = []
    for t in ts:
        s = t.stride()
        if t.get_device() != dev:
            _off_device(op, t)
        if t.dtype != _BF16:
            raise TypeError(f"{op}: bfloat16 only, got {t.dtype}")
        if s[3] != 1 or t.data_ptr() % 16 or s[0] % 8 or s[1] % 8 or s[2] % 8:
            raise ValueError(f"{op}: every row must be 16-byte aligned with a contiguous head dim")
        strides += s[:3]
    if (q_weight is None) != (k_weight is None):
        raise ValueError(f"{op}: give both norm weights or none")
    for w in (q_weight, k_weight):
        if w is not None and (w.get_device() != dev or w.dtype != _BF16 or w.shape != (D,) or not w.is_contiguous()
                              or w.data_ptr() % 16):
            raise ValueError(f"{op}: norm weights must be contiguous, 16-byte aligned bfloat16 ({D},) device tensors")
    if (positions.dtype != torch.int32 or positions.get_device() != dev or positions.shape != (3, B, S)
            or not positions.is_contiguous()):
        raise ValueError(f"{op}: positions must be a contiguous int32 (3, {B}, {S}) device tensor")
    if (inv_freq.dtype != _F32 or inv_freq.get_device() != dev or inv_freq.numel() != D // 2
            or not inv_freq.is_contiguous()):
        raise ValueError(f"{op}: inv_freq must be a contiguous float32 ({D // 2},) device tensor")
    if len(mrope_section) != 3 or sum(mrope_section) * 2 != D:
        raise ValueError(f"{op}: mrope_section {list(mrope_section)} must be three counts that sum to D/2 = {D // 2}")
    if cap == 0:
        raise ValueError(f"{op}: the cache has no rows")
    if q_in.numel() == 0:
        return
    _lib.call("q3_qk_norm_rope_mxfp4", q_in.data_ptr(), k_in.data_ptr(), v_in.data_ptr(), q_out.data_ptr(),
              k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(), _lib.ptr(q_weight),
              _lib.ptr(k_weight), positions.data_ptr(), inv_freq.data_ptr(), kv_lens.data_ptr(), cap, B, S, Hq, Hkv, D,
              _lib.i64s(*mrope_section), eps, _i64x20(*strides, *st), _lib.Q3_BF16, _lib.raw_stream(dev))


def _query(op: str, q: torch.Tensor, out: torch.Tensor | None) -> tuple[torch.Tensor, torch.Tensor]:
    """q as the kernels read it, and the output."""
    if q.requires_grad or out is not None and out.requires_grad:
        require_no_grad(op, q, out)
    if q.dtype != _BF16:
        raise TypeError(f"{op}: q must be bfloat16, got {q.dtype}")
    packed = q.is_contiguous()
    if not packed or q.data_ptr() % 16:
        q = mfma_operand(op, q if q.stride(-1) == 1 else q.contiguous())
    if out is None:
        return q, torch.empty_like(q) if packed else q.new_empty(q.shape)
    if (out.get_device() != q.get_device() or out.shape != q.shape or out.dtype != _BF16 or out.data_ptr() % 16
            or out.stride(-1) != 1 or any(out.stride(i) % 8 for i in range(out.dim() - 1))):
        raise ValueError(f"{op}: out must be {tuple(q.shape)} {_BF16} on q's device with a contiguous head dim, 16-byte "
                         "aligned")
    return q, out


# Bytes of a row of scales, which the attention kernels load at once, by the head dims they take (the entry points
# refuse the others).
_SCALE_ROW = {64: 2, 128: 4}


def _scale(op: str, scale: float) -> float:
    scale = float(scale)
    if not 0 < scale < math.inf:
        raise ValueError(f"{op}: scale must be positive and finite, got {scale}")
    return scale


def decode_attention_mxfp4(q: torch.Tensor, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor,
                           v_scales: torch.Tensor, kv_lens: torch.Tensor, scale: float, *,
                           out: torch.Tensor | None = None, append: bool = False) -> torch.Tensor:
    """decode_attention over a four-bit cache, read in place.

    q (B, Hq, D) (or (B, Hq, 1, D)) bf16, D 64 or 128; codes (B, Hkv, cap, D / 2), scales (B, Hkv, cap, D / 32);
    sequence b attends to cache rows [0, kv_lens[b]). append=True is the decode step with the new token's row
    already written at kv_lens[b]: it is attended to as well, and kv_lens is then incremented in place. scale must be
    positive. Returns (B, Hq, D); an empty sequence gives zeros.
    """
    op = "decode_attention_mxfp4"
    if q.dim() == 4 and q.shape[2] == 1:
        q = q[:, :, 0]
    if q.dim() != 3:
        raise ValueError(f"{op}: q must be (B, Hq, D), got {tuple(q.shape)}")
    scale = _scale(op, scale)
    dev = q.get_device()
    B, Hq, D = q.shape
    Hkv, cap, st = _check_cache(op, dev, k_codes, k_scales, v_codes, v_scales, kv_lens, B, D, _SCALE_ROW.get(D, 1))
    if Hkv == 0 or Hq % Hkv:
        raise ValueError(f"{op}: {Hq} query heads for {Hkv} KV heads")
    if cap == 0:
        raise ValueError(f"{op}: the cache has no rows")
    q, o = _query(op, q, out)
    if B == 0:
        return o
    nws = _decode_workspace(B, Hq, Hkv, D, cap)
    ws = k_codes.new_empty(nws) if nws else None
    qs, os = q.stride(), o.stride()
    _lib.call("q3_decode_attention_mxfp4", q.data_ptr(), k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(),
              v_scales.data_ptr(), kv_lens.data_ptr(), 1 if append else 0, o.data_ptr(), B, Hq, Hkv, D, cap,
              _i64x14(qs[0], qs[1], 0, os[0], os[1], 0, *st), scale, _lib.Q3_BF16, _lib.ptr(ws), nws,
              _lib.raw_stream(dev))
    return o


def flash_attention_cache_mxfp4(q: torch.Tensor, k_codes: torch.Tensor, k_scales: torch.Tensor,
                                v_codes: torch.Tensor, v_scales: torch.Tensor, kv_lens: torch.Tensor, scale: float,
                                num_kv_groups: int = 1, *, out: torch.Tensor | None = None, advance: bool = False,
                                max_len: int | None = None) -> torch.Tensor:
    """flash_attention_cache over a four-bit cache: causal attention of a prefill chunk.

    q (B, Hq, Sq, D) bf16, D 64 or 128; the chunk's rows [kv_lens[b], kv_lens[b] + Sq) are already in the cache.
    Query i of sequence b attends to cache rows [0, kv_lens[b] + i]; advance=True adds Sq to kv_lens afterwards. scale
    must be positive. `max_len` bounds every kv_lens[b] + Sq (default: cap): rows past it are not read. It sizes the
    workspace of a chunk over expanded rows, 4 * B * Hkv * max_len * D bytes: one of more than 192 columns (tokens x
    query heads of a KV head) and of more than 1400 (sequence, KV head, 16 columns).
    """
    op = "flash_attention_cache_mxfp4"
    if q.dim() != 4:
        raise ValueError(f"{op}: q must be (B, Hq, Sq, D), got {tuple(q.shape)}")
    scale = _scale(op, scale)
    dev = q.get_device()
    B, Hq, Sq, D = q.shape
    Hkv, cap, st = _check_cache(op, dev, k_codes, k_scales, v_codes, v_scales, kv_lens, B, D, _SCALE_ROW.get(D, 1))
    if Hkv * num_kv_groups != Hq:
        raise ValueError(f"{op}: Hq={Hq} != Hkv={Hkv} * num_kv_groups={num_kv_groups}")
    ml = cap if max_len is None else int(max_len)
    if not Sq <= ml <= cap or cap == 0:
        raise ValueError(f"{op}: max_len {ml} must lie in [Sq, cap] = [{Sq}, {cap}]")
    q, o = _query(op, q, out)
    if q.numel() == 0:
        return o
    nws = _lib.lib().q3_flash_attention_cache_mxfp4_workspace_bytes(B, Hq, Hkv, Sq, D, ml)
    ws = k_codes.new_empty(nws) if nws else None
    qs, os = q.stride(), o.stride()
    _lib.call("q3_flash_attention_cache_mxfp4", q.data_ptr(), k_codes.data_ptr(), k_scales.data_ptr(),
              v_codes.data_ptr(), v_scales.data_ptr(), kv_lens.data_ptr(), o.data_ptr(), B, Hq, Hkv, Sq, D, ml,
              _i64x14(*qs[:3], *os[:3], *st), scale, 1 if advance else 0, _lib.Q3_BF16, _lib.ptr(ws), nws,
              _lib.raw_stream(dev))
    return o
