"""Microscaled 4-bit floating point (MXFP4): weights and KV caches at 4.25 bits a value (no reference counterpart;
the reference has bf16 and fp32 only).

A row is cut into blocks of 32 consecutive values, each value a 4-bit float (E2M1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and
their negatives), each block with one power-of-two scale held as its exponent (E8M0: byte s stands for 2^(s - 127),
255 for NaN). `codes` (..., K / 2) uint8 holds value 2j in the low and 2j + 1 in the high half of byte j, `scales`
(..., K / 32) uint8 the blocks' scales. Everything a code stands for is exact in bf16, so the products and the
attention below lose nothing beyond the quantisation itself and the bf16 arithmetic of their unquantised forms.
"""
from __future__ import annotations

import torch

from .. import _lib
from ._common import mfma_operand, require_device, require_no_grad, require_same_dtype

MX_BLOCK = 32


def _one_device(op: str, *tensors: torch.Tensor | None) -> None:
    """All on the current GPU, whose current stream the call uses."""
    ts = [t for t in tensors if t is not None]
    require_device(op, *ts)
    cur = torch.cuda.current_device()
    if any(t.device.index != cur for t in ts):
        raise RuntimeError(f"{op}: tensors must be on the current device (cuda:{cur})")


def _check(op: str, *tensors: torch.Tensor | None) -> None:
    ts = [t for t in tensors if t is not None]
    _one_device(op, *ts)
    require_no_grad(op, *ts)


def _check_pair(op: str, codes: torch.Tensor, scales: torch.Tensor) -> None:
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise TypeError(f"{op}: codes and scales must be uint8, got {codes.dtype} and {scales.dtype}")
    if (codes.dim() < 1 or codes.dim() != scales.dim() or codes.shape[:-1] != scales.shape[:-1]
            or codes.shape[-1] != scales.shape[-1] * (MX_BLOCK // 2)):
        raise ValueError(f"{op}: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} must be (..., K / 2) and "
                         "(..., K / 32)")


def mxfp4_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of bf16 or fp32 x (..., K), K a multiple of 32.

    A block's scale is 2^(floor(log2 t) - 2), t its largest magnitude (exponent -127 at least, also for a block of
    zeros); a value over the scale rounds to the nearest code, ties to the even one, and saturates at 6. A block
    that holds an infinity or a NaN reads back as NaN.
    """
    _check("mxfp4_quantize", x)
    dt = _lib.dtype_code(x.dtype)
    if x.dim() < 1 or x.shape[-1] % MX_BLOCK:
        raise ValueError(f"mxfp4_quantize: the last dim of {tuple(x.shape)} must be a multiple of {MX_BLOCK}")
    K = x.shape[-1]
    codes = torch.empty((*x.shape[:-1], K // 2), dtype=torch.uint8, device=x.device)
    scales = torch.empty((*x.shape[:-1], K // MX_BLOCK), dtype=torch.uint8, device=x.device)
    if x.numel() == 0:
        return codes, scales
    x2 = x.reshape(-1, K)
    if x2.stride(-1) != 1 or x2.data_ptr() % 16 or x2.stride(0) * x2.element_size() % 16:
        x2 = x2.clone(memory_format=torch.contiguous_format)
    _lib.call("q3_mxfp4_quantize", x2.data_ptr(), codes.data_ptr(), scales.data_ptr(), x2.shape[0], K,
              max(x2.stride(0), K), dt, _lib.stream())
    return codes, scales


def mxfp4_dequantize(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values (..., K) in bf16 or fp32, both exact (blocks of scale 255: NaN). Contiguous tensors
    and (B, H, rows, ...) slices of a cache are read in place; other views are copied first."""
    _check("mxfp4_dequantize", codes, scales)
    _check_pair("mxfp4_dequantize", codes, scales)
    dt = _lib.dtype_code(dtype)
    y = torch.empty((*codes.shape[:-1], codes.shape[-1] * 2), dtype=dtype, device=codes.device)
    if y.numel() == 0:
        return y
    n, st = (1, 1), (0, 0, 0, 0)
    if codes.is_contiguous() and scales.is_contiguous() and codes.data_ptr() % 4 == 0:
        pass
    elif (codes.dim() >= 3 and codes[0, 0].is_contiguous() and scales[0, 0].is_contiguous()
          and codes.shape[0] * codes.shape[1] <= 65535 and codes.data_ptr() % 4 == 0
          and codes.stride(0) % 4 == 0 and codes.stride(1) % 4 == 0):
        n, st = codes.shape[:2], (*codes.stride()[:2], *scales.stride()[:2])
    else:
        codes, scales = (t.clone(memory_format=torch.contiguous_format) for t in (codes, scales))
    _lib.call("q3_mxfp4_dequantize", codes.data_ptr(), scales.data_ptr(), y.data_ptr(), *n,
              y.numel() // (n[0] * n[1]), _lib.i64s(*st), dt, _lib.stream())
    return y


def matmul_mxfp4(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, bias: torch.Tensor | None = None,
                 residual: torch.Tensor | None = None, *, out: torch.Tensor | None = None) -> torch.Tensor:
    """matmul with the weight (N, K) held in MXFP4: x·Wᵀ (+ bias) (+ residual), x (..., K) bf16, one rounding.

    `out`, when given: (..., N) whose rows have one stride and contiguous elements, written in place (a column
    slice of a wider buffer). Inference only.
    """
    op = "matmul_mxfp4"
    _check(op, x, codes, scales, bias, residual, out)
    _check_pair(op, codes, scales)
    if x.dtype != torch.bfloat16:
        raise TypeError(f"{op}: x must be bfloat16, got {x.dtype}")
    require_same_dtype(op, x, bias, residual, out)
    if codes.dim() != 2 or x.dim() < 1 or codes.shape[1] * 2 != x.shape[-1] or x.shape[-1] == 0:
        raise ValueError(f"{op}: codes {tuple(codes.shape)} do not match x {tuple(x.shape)}")
    N, K = codes.shape[0], x.shape[-1]
    shape = (*x.shape[:-1], N)
    if bias is not None and bias.shape != (N,):
        raise ValueError(f"{op}: bias {tuple(bias.shape)} != ({N},)")
    if residual is not None and residual.shape != shape:
        raise ValueError(f"{op}: residual {tuple(residual.shape)} != output {shape}")
    if out is not None and (out.shape != shape or (N > 1 and out.stride(-1) != 1)):
        raise ValueError(f"{op}: out {tuple(out.shape)} must be {shape} with contiguous elements")
    y = out if out is not None else torch.empty(shape, dtype=x.dtype, device=x.device)
    if y.numel() == 0:
        return y
    x2 = x.reshape(-1, K)
    x2 = mfma_operand(op, x2 if x2.stride(-1) == 1 else x2.contiguous())
    y2 = y.view(-1, N)
    r2 = residual.reshape(-1, N) if residual is not None else None
    if r2 is not None and r2.stride(-1) != 1:
        r2 = r2.contiguous()
    M = x2.shape[0]
    if not codes.is_contiguous() or codes.data_ptr() % 16:
        codes = codes.clone(memory_format=torch.contiguous_format)
    scales = scales.contiguous()
    b = bias.contiguous() if bias is not None else None
    ws, nws = _lib.workspace(_lib.lib().q3_matmul_mxfp4_workspace_bytes(M, N, K), x.device)
    _lib.call("q3_matmul_mxfp4", x2.data_ptr(), codes.data_ptr(), scales.data_ptr(), _lib.ptr(b), _lib.ptr(r2),
              y2.data_ptr(), M, N, K, max(x2.stride(0), K), K // 2, K // MX_BLOCK,
              max(r2.stride(0), N) if r2 is not None else 0, max(y2.stride(0), N), _lib.Q3_BF16, _lib.ptr(ws), nws,
              _lib.stream())
    return y


def _check_cache(op: str, k_codes, k_scales, v_codes, v_scales, kv_lens, B: int, D: int) -> tuple[int, int]:
    """Checks a (B, Hkv, cap, D) cache in MXFP4 and its lengths; returns (Hkv, cap)."""
    for c, s in ((k_codes, k_scales), (v_codes, v_scales)):
        _check_pair(op, c, s)
        if c.dim() != 4 or c.shape[0] != B or c.shape[3] * 2 != D or c.shape != k_codes.shape:
            raise ValueError(f"{op}: cache codes {tuple(k_codes.shape)} and {tuple(v_codes.shape)} must be "
                             f"({B}, Hkv, cap, {D // 2})")
        for t in (c, s):
            if t.numel() and (t.stride(3) != 1 or (t.shape[2] > 1 and t.stride(2) != t.shape[3])):
                raise ValueError(f"{op}: the rows of a cache head must be packed")
        if c.numel() and (c.data_ptr() % 16 or c.stride(0) % 16 or c.stride(1) % 16):
            raise ValueError(f"{op}: the cache codes must be 16-byte aligned")
    if kv_lens.dtype != torch.int32 or kv_lens.shape != (B,) or not kv_lens.is_contiguous():
        raise ValueError(f"{op}: kv_lens must be a contiguous int32 ({B},) device tensor")
    return k_codes.shape[1], k_codes.shape[2]


def _cache_strides(*ts: torch.Tensor) -> list[int]:
    return [s for t in ts for s in (t.stride(0), t.stride(1))]


def kv_append_mxfp4(k: torch.Tensor, v: torch.Tensor, k_codes: torch.Tensor, k_scales: torch.Tensor,
                    v_codes: torch.Tensor, v_scales: torch.Tensor, kv_lens: torch.Tensor) -> None:
    """Quantise new key / value rows into a four-bit cache.

    k, v (B, S, Hkv, D) bf16 or fp32, any strides with D contiguous; codes (B, Hkv, cap, D / 2) and scales (B, Hkv,
    cap, D / 32) of keys and values; kv_lens (B,) int32: row s of sequence b goes to cache row kv_lens[b] + s, and is
    dropped at or past cap. kv_lens is left as it is (the attention that follows advances it).
    """
    op = "kv_append_mxfp4"
    _check(op, k, v, k_codes, k_scales, v_codes, v_scales, kv_lens)
    dt = _lib.dtype_code(k.dtype)
    require_same_dtype(op, k, v)
    if k.dim() != 4 or k.shape != v.shape:
        raise ValueError(f"{op}: k {tuple(k.shape)} and v {tuple(v.shape)} must be (B, S, Hkv, D)")
    B, S, Hkv, D = k.shape
    heads, cap = _check_cache(op, k_codes, k_scales, v_codes, v_scales, kv_lens, B, D)
    if heads != Hkv:
        raise ValueError(f"{op}: {Hkv} KV heads for a cache of {heads}")
    if k.numel() == 0 or cap == 0:
        return
    es = k.element_size()
    k, v = (t if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(t.stride(i) * es % 16 == 0 for i in range(3))
            else t.clone(memory_format=torch.contiguous_format) for t in (k, v))
    _lib.call("q3_kv_append_mxfp4", k.data_ptr(), v.data_ptr(), k_codes.data_ptr(), k_scales.data_ptr(),
              v_codes.data_ptr(), v_scales.data_ptr(), kv_lens.data_ptr(), B, S, Hkv, D, cap,
              _lib.i64s(*k.stride()[:3], *v.stride()[:3], *_cache_strides(k_codes, k_scales, v_codes, v_scales)), dt,
              _lib.stream())


def _query(op: str, q: torch.Tensor) -> torch.Tensor:
    if q.dtype != torch.bfloat16:
        raise TypeError(f"{op}: q must be bfloat16, got {q.dtype}")
    return mfma_operand(op, q if q.stride(-1) == 1 else q.contiguous())


def _output(op: str, q: torch.Tensor, out: torch.Tensor | None) -> torch.Tensor:
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if (out.shape != q.shape or out.dtype != q.dtype or out.data_ptr() % 16 or out.stride(-1) != 1
            or any(out.stride(i) % 8 for i in range(out.dim() - 1))):
        raise ValueError(f"{op}: out must be {tuple(q.shape)} {q.dtype} with a contiguous head dim, 16-byte aligned")
    return out


def decode_attention_mxfp4(q: torch.Tensor, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor,
                           v_scales: torch.Tensor, kv_lens: torch.Tensor, scale: float, *,
                           out: torch.Tensor | None = None, append: bool = False) -> torch.Tensor:
    """decode_attention over a four-bit cache, read in place.

    q (B, Hq, D) (or (B, Hq, 1, D)) bf16, D 64 or 128; codes (B, Hkv, cap, D / 2), scales (B, Hkv, cap, D / 32);
    sequence b attends to cache rows [0, kv_lens[b]). append=True is the decode step with the new token's row
    already written at kv_lens[b]: it is attended to as well, and kv_lens is then incremented in place. Returns (B,
    Hq, D); an empty sequence gives zeros.
    """
    op = "decode_attention_mxfp4"
    _check(op, q, k_codes, k_scales, v_codes, v_scales, kv_lens, out)
    if q.dim() == 4 and q.shape[2] == 1:
        q = q[:, :, 0]
    if q.dim() != 3:
        raise ValueError(f"{op}: q must be (B, Hq, D), got {tuple(q.shape)}")
    q = _query(op, q)
    B, Hq, D = q.shape
    Hkv, cap = _check_cache(op, k_codes, k_scales, v_codes, v_scales, kv_lens, B, D)
    if Hkv == 0 or Hq % Hkv:
        raise ValueError(f"{op}: {Hq} query heads for {Hkv} KV heads")
    o = _output(op, q, out)
    ws, nws = _lib.workspace(_lib.lib().q3_decode_attention_mxfp4_workspace_bytes(B, Hq, Hkv, D), q.device)
    _lib.call("q3_decode_attention_mxfp4", q.data_ptr(), k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(),
              v_scales.data_ptr(), kv_lens.data_ptr(), int(bool(append)), o.data_ptr(), B, Hq, Hkv, D, cap,
              _lib.i64s(q.stride(0), q.stride(1), 0, o.stride(0), o.stride(1), 0,
                        *_cache_strides(k_codes, k_scales, v_codes, v_scales)), float(scale), _lib.Q3_BF16,
              _lib.ptr(ws), nws, _lib.stream())
    return o


def flash_attention_cache_mxfp4(q: torch.Tensor, k_codes: torch.Tensor, k_scales: torch.Tensor,
                                v_codes: torch.Tensor, v_scales: torch.Tensor, kv_lens: torch.Tensor, scale: float,
                                num_kv_groups: int = 1, *, out: torch.Tensor | None = None, advance: bool = False,
                                max_len: int | None = None) -> torch.Tensor:
    """flash_attention_cache over a four-bit cache: causal attention of a prefill chunk.

    q (B, Hq, Sq, D) bf16, D 64 or 128; the chunk's rows [kv_lens[b], kv_lens[b] + Sq) are already in the cache.
    Query i of sequence b attends to cache rows [0, kv_lens[b] + i]; advance=True adds Sq to kv_lens afterwards.
    `max_len` bounds every kv_lens[b] + Sq (default: cap) and sizes the workspace of a longer chunk.
    """
    op = "flash_attention_cache_mxfp4"
    _check(op, q, k_codes, k_scales, v_codes, v_scales, kv_lens, out)
    if q.dim() != 4:
        raise ValueError(f"{op}: q must be (B, Hq, Sq, D), got {tuple(q.shape)}")
    q = _query(op, q)
    B, Hq, Sq, D = q.shape
    Hkv, cap = _check_cache(op, k_codes, k_scales, v_codes, v_scales, kv_lens, B, D)
    if Hkv * num_kv_groups != Hq:
        raise ValueError(f"{op}: Hq={Hq} != Hkv={Hkv} * num_kv_groups={num_kv_groups}")
    ml = cap if max_len is None else int(max_len)
    if not 0 <= ml <= cap:
        raise ValueError(f"{op}: max_len {ml} must lie in [0, {cap}]")
    o = _output(op, q, out)
    ws, nws = _lib.workspace(_lib.lib().q3_flash_attention_cache_mxfp4_workspace_bytes(B, Hq, Hkv, Sq, D, ml), q.device)
    _lib.call("q3_flash_attention_cache_mxfp4", q.data_ptr(), k_codes.data_ptr(), k_scales.data_ptr(),
              v_codes.data_ptr(), v_scales.data_ptr(), kv_lens.data_ptr(), o.data_ptr(), B, Hq, Hkv, Sq, D, ml,
              _lib.i64s(q.stride(0), q.stride(1), q.stride(2), o.stride(0), o.stride(1), o.stride(2),
                        *_cache_strides(k_codes, k_scales, v_codes, v_scales)), float(scale), int(bool(advance)),
              _lib.Q3_BF16, _lib.ptr(ws), nws, _lib.stream())
    return o
