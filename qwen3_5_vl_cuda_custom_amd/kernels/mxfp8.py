"""Microscaled 8-bit floating point (MXFP8): activations and weights at 8.25 bits a value, products on the 8-bit matrix
instructions (no reference counterpart; the reference has bf16 and fp32 only).

A row is cut into blocks of 32 consecutive values, each value an 8-bit float (E4M3, up to 448), each block with one
power-of-two scale held as its exponent (E8M0: byte s stands for 2^(s - 127), 255 for NaN). A tensor in eight bits is
a pair: `codes` (..., K) float8_e4m3fn and `scales` (..., K / 32) uint8.

add_rmsnorm_mxfp8 and the products with quantize=True write such pairs, the products take them; a product also takes
bf16 rows and quantises them first. Inference only. All tensors of a call must be on the current device, whose current
stream it uses. The kernels of a decode step take a few microseconds each, so the checks here are written for their own time.
"""
from __future__ import annotations

from functools import lru_cache
from struct import Struct

import torch

from .. import _lib
from ._common import require_device, require_no_grad

MX8_BLOCK = 32
_FEW_ROWS = 64  # up to which the products need no workspace (mx8_rows_takes, csrc/mxfp8_rows.hip)
_U8, _F8, _BF16 = torch.uint8, torch.float8_e4m3fn, torch.bfloat16
_i64s = [Struct(f"{n}q").pack for n in range(5)]  # C arrays of up to four numbers or addresses
_ACTS = {None: 0, "gelu_tanh": 1, "silu": 2}

Pair = tuple[torch.Tensor, torch.Tensor]


@lru_cache(maxsize=4096)
def _workspace(M: int, K: int, swiglu: int, *ns: int) -> int:
    return _lib.lib().q3_matmul_mxfp8_workspace_bytes(M, _i64s[len(ns)](*ns), len(ns), K, swiglu)


def _off_device(op: str, *tensors: torch.Tensor | None) -> None:
    """Raise for tensors that are not all on the current device."""
    require_device(op, *tensors)
    raise RuntimeError(f"{op}: tensors must be on the current device (cuda:{torch.cuda.current_device()})")


def _packed(op: str, codes: torch.Tensor, scales: torch.Tensor, dev: int) -> Pair:
    """The pair checked, packed and aligned as the kernels read it. (_weight asks the first condition too, in place: a
    change to one is a change to both.)"""
    cs, ss = codes.shape, scales.shape
    if (codes.dtype is _F8 and scales.dtype is _U8 and codes.get_device() == dev and scales.get_device() == dev
            and codes.is_contiguous() and scales.is_contiguous() and len(cs) == 2 and len(ss) == 2 and cs[0] == ss[0]
            and cs[1] == ss[1] * MX8_BLOCK and not (codes.data_ptr() % 16 or scales.data_ptr() % 4 or codes.requires_grad)):
        return codes, scales  # the usual call
    if codes.get_device() != dev or scales.get_device() != dev:
        _off_device(op, codes, scales)
    if codes.requires_grad:
        require_no_grad(op, codes)
    if codes.dtype != _F8 or scales.dtype != _U8:
        raise TypeError(f"{op}: codes must be float8_e4m3fn and scales uint8, got {codes.dtype} and {scales.dtype}")
    if not cs or len(cs) != len(ss) or cs[:-1] != ss[:-1] or cs[-1] != ss[-1] * MX8_BLOCK:
        raise ValueError(f"{op}: codes {tuple(cs)} and scales {tuple(ss)} must be (..., K) and (..., K / 32)")
    if not codes.is_contiguous() or codes.data_ptr() % 16:
        codes = codes.clone(memory_format=torch.contiguous_format)
    if not scales.is_contiguous() or scales.data_ptr() % 4:
        scales = scales.clone(memory_format=torch.contiguous_format)
    return codes, scales


def _device(op: str, t: torch.Tensor) -> int:
    dev = t.get_device()
    if dev < 0 or dev != _lib.current_device():
        _off_device(op, t)
    return dev


def _strided(x: torch.Tensor, K: int) -> tuple[torch.Tensor, int]:
    """x (..., K) as rows of contiguous elements, 16-byte aligned, and their stride."""
    if x.is_contiguous():
        return (x if x.data_ptr() % 16 == 0 else x.clone()), K
    x = x.reshape(-1, K)
    ld = x.stride(0) if x.shape[0] > 1 else K
    if x.stride(1) != 1 or ld < K or x.data_ptr() % 16 or ld * x.element_size() % 16:
        return x.clone(memory_format=torch.contiguous_format), K
    return x, ld


def mxfp8_quantize(x: torch.Tensor) -> Pair:
    """(codes, scales) of bf16 or fp32 x (..., K), K a multiple of 32.

    A block's scale is the smallest power of two, 2^-127 at least, that keeps its largest magnitude within 448; a value
    over the scale rounds to the nearest code, ties to even. A block that holds an infinity or a NaN reads back as NaN.
    """
    op = "mxfp8_quantize"
    dev = _device(op, x)
    if x.requires_grad:
        require_no_grad(op, x)
    dt = _lib.dtype_code(x.dtype)
    shape = x.shape
    if not shape or shape[-1] % MX8_BLOCK:
        raise ValueError(f"{op}: the last dim of {tuple(shape)} must be a multiple of {MX8_BLOCK}")
    K = shape[-1]
    packed = x.is_contiguous()
    codes = torch.empty_like(x, dtype=_F8) if packed else x.new_empty(shape, dtype=_F8)  # empty_like: 0.3 us less
    scales = codes.new_empty((*shape[:-1], K // MX8_BLOCK), dtype=_U8)
    n = x.numel()
    if n == 0:
        return codes, scales
    ld = K
    if not packed or x.data_ptr() % 16:
        x, ld = _strided(x, K)
    _lib.call("q3_mxfp8_quantize", x.data_ptr(), codes.data_ptr(), scales.data_ptr(), n // K, K, ld, dt,
              _lib.raw_stream(dev))
    return codes, scales


def mxfp8_dequantize(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values (..., K) in bf16 or fp32, exact in fp32 and, down to its smallest value, in bf16; blocks of scale
    255 are NaN. Views that are not contiguous are copied first."""
    op = "mxfp8_dequantize"
    dev = _device(op, codes)
    codes, scales = _packed(op, codes, scales, dev)
    dt = _lib.dtype_code(dtype)
    y = torch.empty_like(codes, dtype=dtype)
    n = y.numel()
    if n:
        _lib.call("q3_mxfp8_dequantize", codes.data_ptr(), scales.data_ptr(), y.data_ptr(), n, dt,
                  _lib.raw_stream(dev))
    return y


def add_rmsnorm_mxfp8(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor,
                      eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(h, codes, scales): h = x + residual as residual_add rounds it (x itself without a residual), and
    rmsnorm(h, weight, eps) in eight bits, quantised from fp32, in one launch. x (..., K) bf16 or fp32, K a multiple
    of 32."""
    op = "add_rmsnorm_mxfp8"
    dev = _device(op, x)
    shape, dtype = x.shape, x.dtype
    dt = _lib.dtype_code(dtype)
    for t in (residual, weight):
        if t is not None:
            if t.get_device() != dev:
                _off_device(op, t)
            if t.dtype != dtype:
                raise TypeError(f"{op}: dtype mismatch ({t.dtype} vs {dtype})")
            if t.requires_grad:
                require_no_grad(op, t)
    if x.requires_grad:
        require_no_grad(op, x)
    if not shape or shape[-1] % MX8_BLOCK or shape[-1] == 0:
        raise ValueError(f"{op}: the last dim of {tuple(shape)} must be a positive multiple of {MX8_BLOCK}")
    K = shape[-1]
    if weight.shape != (K,):
        raise ValueError(f"{op}: weight {tuple(weight.shape)} != ({K},)")
    if residual is not None and residual.shape != shape:
        raise ValueError(f"{op}: residual {tuple(residual.shape)} != x {tuple(shape)}")
    packed = x.is_contiguous()
    codes = torch.empty_like(x, dtype=_F8) if packed else x.new_empty(shape, dtype=_F8)
    scales = codes.new_empty((*shape[:-1], K // MX8_BLOCK), dtype=_U8)
    h = x if residual is None else torch.empty_like(x) if packed else x.new_empty(shape)
    n = x.numel()
    if n == 0:
        return h, codes, scales
    x2, ldx, r2, ldr = x, K, residual, K
    if not packed or x.data_ptr() % 16:
        x2, ldx = _strided(x, K)
    if residual is not None and (not residual.is_contiguous() or residual.data_ptr() % 16):
        r2, ldr = _strided(residual, K)
    if not weight.is_contiguous() or weight.data_ptr() % 16:
        weight = weight.clone(memory_format=torch.contiguous_format)
    _lib.call("q3_add_rmsnorm_mxfp8", x2.data_ptr(), _lib.ptr(r2), weight.data_ptr(),
              None if residual is None else h.data_ptr(), codes.data_ptr(), scales.data_ptr(), n // K, K, ldx, ldr,
              float(eps), dt, _lib.raw_stream(dev))
    return h, codes, scales


def _operand(op: str, x: torch.Tensor | Pair) -> tuple[int, torch.Tensor, torch.Tensor]:
    """The device, codes and scales of x, which may be bf16 rows."""
    if isinstance(x, torch.Tensor):
        if x.dtype != _BF16:
            raise TypeError(f"{op}: x must be bfloat16 or a pair (codes, scales), got {x.dtype}")
        if x.requires_grad:
            require_no_grad(op, x)
        dev = _device(op, x)
        codes, scales = mxfp8_quantize(x)
    else:
        codes, scales = x
        dev = codes.get_device()
        if dev < 0 or dev != _lib.current_device():
            _off_device(op, codes)
        codes, scales = _packed(op, codes, scales, dev)
    if codes.shape[-1] == 0:
        raise ValueError(f"{op}: x {tuple(codes.shape)} has no columns")
    return dev, codes, scales


def _weight(op: str, weight: Pair, K: int, dev: int) -> Pair:
    codes, scales = weight
    cs, ss = codes.shape, scales.shape
    if (codes.dtype is _F8 and scales.dtype is _U8 and codes.get_device() == dev and scales.get_device() == dev
            and codes.is_contiguous() and scales.is_contiguous() and len(cs) == 2 and len(ss) == 2 and cs[0] == ss[0]
            and cs[1] == K and ss[1] * MX8_BLOCK == K
            and not (codes.data_ptr() % 16 or scales.data_ptr() % 4 or codes.requires_grad)):
        return codes, scales  # the usual call: _packed's condition and the shape of x, without the calls below
    codes, scales = _packed(op, codes, scales, dev)
    if codes.dim() != 2 or codes.shape[1] != K:
        raise ValueError(f"{op}: weight codes {tuple(codes.shape)} do not match x (..., {K})")
    return codes, scales


def _vector(op: str, bias: torch.Tensor, n: int, dev: int) -> torch.Tensor:
    if bias.get_device() != dev:
        _off_device(op, bias)
    if bias.dtype != _BF16:
        raise TypeError(f"{op}: dtype mismatch ({bias.dtype} vs {_BF16})")
    if bias.requires_grad:
        require_no_grad(op, bias)
    if bias.shape != (n,):
        raise ValueError(f"{op}: bias {tuple(bias.shape)} != ({n},)")
    return bias if bias.is_contiguous() else bias.contiguous()


def _outputs(op: str, codes: torch.Tensor, shape: tuple, quantize: bool) -> tuple:
    """The output, and the pointers to it, its codes and its scales."""
    if not quantize:
        y = codes.new_empty(shape, dtype=_BF16)
        return y, y.data_ptr(), None, None
    if shape[-1] % MX8_BLOCK:
        raise ValueError(f"{op}: quantize=True needs outputs of a multiple of {MX8_BLOCK} columns, got {shape[-1]}")
    pair = codes.new_empty(shape), codes.new_empty((*shape[:-1], shape[-1] // MX8_BLOCK), dtype=_U8)
    return pair, None, pair[0].data_ptr(), pair[1].data_ptr()


def matmul_mxfp8(x: torch.Tensor | Pair, weight: Pair, bias: torch.Tensor | None = None,
                 residual: torch.Tensor | None = None, *, activation: str | None = None, quantize: bool = False,
                 out: torch.Tensor | None = None) -> torch.Tensor | Pair:
    """act(x·Wᵀ (+ bias)) (+ residual) with the weight (N, K) in eight bits and x (..., K) in eight bits or bf16 (then
    quantised first); fp32 accumulators, one rounding to bf16.

    activation: None, "gelu_tanh" or "silu". quantize=True returns the fp32 values in eight bits instead, a pair (N a multiple of
    32). `out`, when given: (..., N) bf16 whose rows have one stride and contiguous elements, written in place (a
    column slice of a wider buffer); it may be the residual itself, and must not overlap it otherwise.
    """
    op = "matmul_mxfp8"
    act = _ACTS.get(activation, -1)
    if act < 0:
        raise ValueError(f"{op}: activation must be None, 'gelu_tanh' or 'silu', got {activation!r}")
    dev, xc, xs = _operand(op, x)
    lead = xc.shape
    K = lead[-1]
    wc, ws = _weight(op, weight, K, dev)
    N = wc.shape[0]
    shape = (*lead[:-1], N)
    if bias is not None:
        bias = _vector(op, bias, N, dev)
    ldr, ldc, same = N, N, False
    if residual is not None:
        if residual.get_device() != dev:
            _off_device(op, residual)
        if residual.dtype != _BF16:
            raise TypeError(f"{op}: dtype mismatch ({residual.dtype} vs {_BF16})")
        if residual.requires_grad:
            require_no_grad(op, residual)
        if residual.shape != shape:
            raise ValueError(f"{op}: residual {tuple(residual.shape)} != output {shape}")
        same = residual.is_contiguous()
        if not same:
            residual = residual.reshape(-1, N)
            if N > 1 and residual.stride(1) != 1 or residual.shape[0] > 1 and residual.stride(0) < N:
                residual = residual.contiguous()
            ldr = residual.stride(0) if residual.shape[0] > 1 else N
    yc = ys = None
    if out is None:
        if same and not quantize:
            y = torch.empty_like(residual)
            yp = y.data_ptr()
        else:
            y, yp, yc, ys = _outputs(op, xc, shape, quantize)
    else:
        if quantize:
            raise ValueError(f"{op}: give either out or quantize=True")
        if out.get_device() != dev:
            _off_device(op, out)
        if out.dtype != _BF16:
            raise TypeError(f"{op}: dtype mismatch ({out.dtype} vs {_BF16})")
        if out.requires_grad:
            require_no_grad(op, out)
        if out.shape != shape or (N > 1 and out.stride(-1) != 1):
            raise ValueError(f"{op}: out {tuple(out.shape)} must be {shape} with contiguous elements")
        y, yp = out, out.data_ptr()
        if not out.is_contiguous() and out.numel() > N:
            ldc = out.view(-1, N).stride(0)
            if ldc < N:
                raise ValueError(f"{op}: the rows of out overlap")
    M = xc.numel() // K
    if M == 0 or N == 0:
        return y
    nws = 0 if M <= _FEW_ROWS else _workspace(M, K, 0, N)
    buf = xs.new_empty(nws) if nws else None
    _lib.call("q3_matmul_mxfp8", xc.data_ptr(), xs.data_ptr(), wc.data_ptr(), ws.data_ptr(), _lib.ptr(bias),
              _lib.ptr(residual), yp, yc, ys, M, N, K, ldr, ldc, act, _lib.ptr(buf), nws, _lib.raw_stream(dev))
    return y


def matmul_segments_mxfp8(x: torch.Tensor | Pair, weights, biases=None) -> torch.Tensor:
    """x·[W_0; W_1; ...]ᵀ (+ [b_0; b_1; ...]) over 1 to 4 weights in eight bits, each a pair of (N_i, K), in one launch;
    x as in matmul_mxfp8. Returns (..., ΣN_i) bf16."""
    op = "matmul_segments_mxfp8"
    weights = list(weights)
    given = [None] * len(weights) if biases is None else list(biases)
    if not 1 <= len(weights) <= 4 or len(given) != len(weights):
        raise ValueError(f"{op}: 1 to 4 weights, one bias (or None) each")
    dev, xc, xs = _operand(op, x)
    K = xc.shape[-1]
    ws = [_weight(op, w, K, dev) for w in weights]
    ns = [c.shape[0] for c, _ in ws]
    bs = [None if b is None else _vector(op, b, n, dev) for b, n in zip(given, ns)]
    N = sum(ns)
    y = xc.new_empty((*xc.shape[:-1], N), dtype=_BF16)
    M = xc.numel() // K
    if M == 0 or N == 0:
        return y
    if 0 in ns:
        ws, bs, ns = zip(*((w, b, n) for w, b, n in zip(ws, bs, ns) if n))
    array = _i64s[len(ns)]
    some = array(*(b.data_ptr() if b is not None else 0 for b in bs)) if biases is not None else None
    nws = 0 if M <= _FEW_ROWS else _workspace(M, K, 0, *ns)
    buf = xs.new_empty(nws) if nws else None
    _lib.call("q3_matmul_segments_mxfp8", xc.data_ptr(), xs.data_ptr(), array(*[c.data_ptr() for c, _ in ws]),
              array(*[t.data_ptr() for _, t in ws]), some, array(*ns), len(ns), y.data_ptr(), M, K, N, _lib.ptr(buf), nws,
              _lib.raw_stream(dev))
    return y


def matmul_swiglu_mxfp8(x: torch.Tensor | Pair, gate: Pair, up: Pair, *, quantize: bool = False) -> torch.Tensor | Pair:
    """silu(x·W_gateᵀ)·(x·W_upᵀ), `gate` and `up` pairs of (N, K), in one launch; x as in matmul_mxfp8. bf16, or with
    quantize=True a pair in eight bits (N a multiple of 32), as the down projection takes it."""
    op = "matmul_swiglu_mxfp8"
    dev, xc, xs = _operand(op, x)
    K = xc.shape[-1]
    gc, gs = _weight(op, gate, K, dev)
    uc, us = _weight(op, up, K, dev)
    if gc.shape != uc.shape:
        raise ValueError(f"{op}: gate {tuple(gc.shape)} and up {tuple(uc.shape)} must have one shape")
    N = gc.shape[0]
    y, yp, yc, ys = _outputs(op, xc, (*xc.shape[:-1], N), quantize)
    M = xc.numel() // K
    if M == 0 or N == 0:
        return y
    nws = 0 if M <= _FEW_ROWS else _workspace(M, K, 1, N)
    buf = xs.new_empty(nws) if nws else None
    _lib.call("q3_matmul_swiglu_mxfp8", xc.data_ptr(), xs.data_ptr(), gc.data_ptr(), gs.data_ptr(), uc.data_ptr(),
              us.data_ptr(), yp, yc, ys, M, N, K, N, _lib.ptr(buf), nws, _lib.raw_stream(dev))
    return y
