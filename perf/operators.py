"""Timed cases of the four-bit operators: microscaled 4-bit floating point (MXFP4) weights and KV caches.

The format: a row is cut into blocks of 32 consecutive values, each value a 4-bit float (E2M1: 0, 0.5, 1, 1.5, 2, 3,
4, 6 and their negatives), each block with one power-of-two scale held as its exponent (E8M0: byte s stands for
2^(s - 127), 255 for NaN). Byte j of a row of codes holds value 2j in its low and value 2j + 1 in its high half.

A case is a dict of plain values. `prepare` makes its inputs on the GPU, `run` is one pass: with `own` through the
package's public ops, else in elementary torch operations in 32 bits. `exact` is the same pass in float64, `work`
counts the bytes and floating-point operations that a pass cannot do without.

  round_trip   bf16 or fp32 rows to codes and scales, and back to bf16
  matmul       y = x w^T (+ bias) (+ residual) with 4-bit weights, bf16 x and y
  append_read  new key / value rows written into a 4-bit KV cache at each sequence's length, the cache read back
  decode       one query token per sequence over a ragged 4-bit cache
  chunk        a prefill chunk of several tokens per sequence, causal over a ragged 4-bit cache
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
BLOCK = 32


# ------------------------------------------------------------------ the cases
def listed() -> list[dict]:
    return [
        # The key rows of one decode step of 32 sequences: latency is all of it.
        {"name": "round_trip_256x128", "kind": "round_trip", "rows": 256, "cols": 128, "dtype": "bfloat16"},
        # A gate projection's fp32 master weight on its way into four bits, as when a model is loaded.
        {"name": "round_trip_12288x4096_fp32", "kind": "round_trip", "rows": 12288, "cols": 4096, "dtype": "float32"},
        # The output projection of one user's decode step.
        {"name": "matmul_m1_4096x4096", "kind": "matmul", "m": 1, "n": 4096, "k": 4096, "bias": False,
         "residual": True},
        # The down projection of a full decode batch.
        {"name": "matmul_m32_4096x12288", "kind": "matmul", "m": 32, "n": 4096, "k": 12288, "bias": False,
         "residual": True},
        # The gate projection of a prompt of odd length.
        {"name": "matmul_m777_12288x4096", "kind": "matmul", "m": 777, "n": 12288, "k": 4096, "bias": False,
         "residual": False},
        # The down projection of a long prompt.
        {"name": "matmul_m4096_4096x12288", "kind": "matmul", "m": 4096, "n": 4096, "k": 12288, "bias": False,
         "residual": True},
        # One token of one user, then the short cache read back.
        {"name": "append_read_b1_s1", "kind": "append_read", "batch": 1, "kv_heads": 8, "dim": 128, "cap": 500,
         "new": 1},
        # A prefill chunk of four ragged prompts, then their cache read back.
        {"name": "append_read_b4_s512", "kind": "append_read", "batch": 4, "kv_heads": 8, "dim": 128, "cap": 4096,
         "new": 512},
        # One user's chat turn: a single sequence, one token.
        {"name": "decode_b1_l1500", "kind": "decode", "batch": 1, "kv_heads": 8, "groups": 4, "dim": 128, "cap": 1500},
        # A full serving batch with ragged histories of up to 8k tokens.
        {"name": "decode_b32_l8192", "kind": "decode", "batch": 32, "kv_heads": 8, "groups": 4, "dim": 128,
         "cap": 8193},
        # A question of odd length asked in four chats with ragged histories.
        {"name": "chunk_b4_s37_l2000", "kind": "chunk", "batch": 4, "kv_heads": 4, "groups": 8, "dim": 128,
         "cap": 2000, "new": 37},
        # The last chunk of a long prompt that is prefilled piece by piece.
        {"name": "chunk_b1_s1024_l8192", "kind": "chunk", "batch": 1, "kv_heads": 8, "groups": 4, "dim": 128,
         "cap": 8192, "new": 1024},
    ]


def _log_int(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["round_trip", "matmul", "matmul", "append_read", "decode", "decode", "chunk"])
    if kind == "round_trip":
        cols = BLOCK * _log_int(rng, 1, 256)
        return {"kind": kind, "rows": _log_int(rng, 1, min(12288, 12288 * 4096 // cols)), "cols": cols,
                "dtype": rng.choice(["bfloat16", "float32"])}
    if kind == "matmul":
        k = BLOCK * _log_int(rng, 2, 384)
        n = _log_int(rng, 1, 12288)
        return {"kind": kind, "m": _log_int(rng, 1, min(4096, (1 << 37) // (n * k))), "n": n, "k": k,
                "bias": rng.random() < 0.5, "residual": rng.random() < 0.5}
    dim = rng.choice([64, 128, 128])
    batch, kv_heads, groups = _log_int(rng, 1, 32), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8, 16])
    if kind == "append_read":
        new = _log_int(rng, 1, 512)
        return {"kind": kind, "batch": min(batch, 8), "kv_heads": kv_heads, "dim": dim,
                "cap": new + _log_int(rng, 1, 2048), "new": new}
    if kind == "decode":
        return {"kind": kind, "batch": batch, "kv_heads": kv_heads, "groups": groups, "dim": dim,
                "cap": _log_int(rng, 1, 8192)}
    new = _log_int(rng, 2, 512)
    return {"kind": kind, "batch": min(batch, 4), "kv_heads": kv_heads, "groups": min(groups, 8), "dim": dim,
            "cap": new + _log_int(rng, 1, 2048), "new": new}


# ------------------------------------------------------------------ inputs
def _randn(g: torch.Generator, *shape, dtype=torch.bfloat16) -> torch.Tensor:
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def _kv_rows(g: torch.Generator, *shape) -> torch.Tensor:
    """Rows as keys and values are: channels of different size, a few of them large."""
    size = torch.exp(0.5 * torch.randn(shape[-1], generator=g, device=DEV))
    return (torch.randn(*shape, generator=g, device=DEV) * size).to(torch.bfloat16)


def _pack(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of x: what a program holds whose weights or cache are in four bits already."""
    code, s = _codes(x)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).contiguous(), s.contiguous()


def _lens(case: dict, g: torch.Generator) -> torch.Tensor:
    """Cache rows of each sequence before the call: from a tenth of the room to all of it, the longest filling it."""
    room = case["cap"] - case.get("new", 0)
    n = torch.randint(room // 10, room + 1, (case["batch"],), generator=g, device=DEV)
    n[0] = room
    return n.to(torch.int32)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    s = dict(case)
    if case["kind"] == "round_trip":
        s["x"] = _randn(g, case["rows"], case["cols"], dtype=getattr(torch, case["dtype"])) * 0.02
    elif case["kind"] == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        s["x"] = _randn(g, m, k)
        s["codes"], s["scales"] = _pack(_randn(g, n, k) * 0.02)
        s["b"] = _randn(g, n) if case["bias"] else None
        s["r"] = _randn(g, m, n) if case["residual"] else None
    else:
        B, H, D = case["batch"], case["kv_heads"], case["dim"]
        s["kc"], s["ks"] = _pack(_kv_rows(g, B, H, case["cap"], D))
        s["vc"], s["vs"] = _pack(_kv_rows(g, B, H, case["cap"], D))
        s["lens"] = _lens(case, g)
        if case["kind"] == "append_read":  # the (B, S, heads x D) projections of the new tokens
            s["k"], s["v"] = (_kv_rows(g, B, case["new"], H, D) for _ in range(2))
        elif case["kind"] == "decode":
            s["q"] = _randn(g, B, H * case["groups"], D)
        else:
            s["q"] = _randn(g, B, case["new"], H * case["groups"], D).transpose(1, 2)
    return s


# ------------------------------------------------------------------ the plain form
def _codes(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """One code per value (uint8, 0..15) and one scale byte per block. The scale's exponent is that of the block's
    largest magnitude less 2 (E2M1's largest exponent); values round to the nearest, ties to the even code."""
    y = x.float().unflatten(-1, (-1, BLOCK))
    top = y.abs().amax(-1)
    s = (torch.frexp(top)[1] + 124).clamp(min=0)
    s = torch.where(top == 0, 0, s)
    y = torch.ldexp(y, (127 - s).unsqueeze(-1))
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5))
    code = code + 8 * torch.signbit(y).to(torch.uint8)
    bad = ~torch.isfinite(top)
    return torch.where(bad.unsqueeze(-1), 0, code).flatten(-2), torch.where(bad, 255, s).to(torch.uint8)


def _values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """fp32 values of packed codes (..., K / 2) and scales (..., K / 32)."""
    v = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    table = torch.cat([v, -v])
    two = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    size = torch.where(scales == 255, math.nan, torch.ldexp(torch.ones_like(scales, dtype=torch.float32),
                                                            scales.int() - 127))
    return (table[two.int()].unflatten(-1, (-1, BLOCK)) * size.unsqueeze(-1)).flatten(-2)


def _attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, last: torch.Tensor, groups: int) -> torch.Tensor:
    """q (B, Hq, Sq, D), k / v (B, Hkv, rows, D); last (B, Sq): rows a query attends to. In q's type."""
    B, Hq, Sq, D = q.shape
    q = q.reshape(B, Hq // groups, groups * Sq, D)
    p = torch.matmul(q, k.transpose(-1, -2)) * D ** -0.5
    seen = torch.arange(k.shape[2], device=q.device) < last.repeat(1, groups)[:, None, :, None]
    p = torch.where(seen, p, -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True).clamp(min=-3e38))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total == 0, 1, total)
    return o.reshape(B, Hq, Sq, D)


def run(state: dict):
    s, kind = state, state["kind"]
    if own:
        from qwen3_5_vl_cuda_custom_amd import kernels as K
        if kind == "round_trip":
            return K.mxfp4_dequantize(*K.mxfp4_quantize(s["x"]))
        if kind == "matmul":
            return K.matmul_mxfp4(s["x"], s["codes"], s["scales"], s["b"], s["r"])
        cache = (s["kc"], s["ks"], s["vc"], s["vs"])
        if kind == "append_read":
            K.kv_append_mxfp4(s["k"], s["v"], *cache, s["lens"])
            return K.mxfp4_dequantize(s["kc"], s["ks"]), K.mxfp4_dequantize(s["vc"], s["vs"])
        if kind == "decode":
            return K.decode_attention_mxfp4(s["q"], *cache, s["lens"], s["dim"] ** -0.5)
        return K.flash_attention_cache_mxfp4(s["q"], *cache, s["lens"], s["dim"] ** -0.5, s["groups"])

    if kind == "round_trip":
        code, scale = _codes(s["x"])
        return _values(code[..., 0::2] | (code[..., 1::2] << 4), scale).to(torch.bfloat16)
    if kind == "matmul":
        y = torch.matmul(s["x"].float(), _values(s["codes"], s["scales"]).t())
        if s["b"] is not None:
            y = y + s["b"].float()
        if s["r"] is not None:
            y = y + s["r"].float()
        return y.to(torch.bfloat16)
    if kind == "append_read":
        B, new = s["k"].shape[:2]
        row = (s["lens"].long()[:, None] + torch.arange(new, device=DEV)).reshape(-1)
        at = torch.arange(B, device=DEV).repeat_interleave(new)
        for x, codes, scales in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
            c, sc = _pack(x)
            codes[at, :, row], scales[at, :, row] = c.flatten(0, 1), sc.flatten(0, 1)
        return tuple(_values(c, sc).to(torch.bfloat16) for c, sc in ((s["kc"], s["ks"]), (s["vc"], s["vs"])))
    k, v = _values(s["kc"], s["ks"]), _values(s["vc"], s["vs"])
    if kind == "decode":
        return _attend(s["q"].float().unsqueeze(2), k, v, s["lens"][:, None], s["groups"])[:, :, 0].to(torch.bfloat16)
    last = s["lens"][:, None] + torch.arange(1, s["new"] + 1, device=DEV)
    return _attend(s["q"].float(), k, v, last, s["groups"]).to(torch.bfloat16)


# ------------------------------------------------------------------ from the definition, in 64 bits
def _exact_rounded(x: torch.Tensor) -> torch.Tensor:
    """Every value of x as the nearest multiple of its step below 6 times the block's scale."""
    y = x.double().reshape(*x.shape[:-1], -1, BLOCK)
    top = y.abs().max(-1, keepdim=True).values
    scale = torch.exp2((torch.floor(torch.log2(top.clamp(min=2.0 ** -130))) - 2).clamp(min=-127))
    a = y.abs() / scale
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=1.0))).clamp(max=2.0) - 1)
    return (torch.sign(y) * torch.clamp(torch.round(a / step) * step, max=6.0) * scale).reshape(x.shape)


def _exact_values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """sign (1 + m / 2) 2^(e - 1), or m / 2 where e is 0, times 2^(scale - 127)."""
    c = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device=codes.device)
    for i in range(2):
        n = (codes >> (4 * i)) & 15
        e, m, sign = (n >> 1) & 3, (n & 1).double(), 1 - 2 * (n >> 3).double()
        c[..., i::2] = sign * torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2(e.double() - 1))
    return c * torch.exp2(scales.double() - 127).repeat_interleave(BLOCK, -1)


def _exact_attention(q, k, v, lens, groups: int) -> torch.Tensor:
    """Per sequence and key head: softmax over the rows a query sees, times the values. q (B, Hq, Sq, D)."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    B, Hq, Sq, D = q.shape
    for b in range(B):
        for h in range(Hq // groups):
            n = int(lens[b].max())
            if n == 0:
                continue
            kk, vv = _exact_values(*(t[b, h, :n] for t in k)), _exact_values(*(t[b, h, :n] for t in v))
            for j in range(h * groups, (h + 1) * groups):
                w = q[b, j].double() @ kk.T / math.sqrt(D)
                w.masked_fill_(torch.arange(n, device=q.device)[None, :] >= lens[b][:, None], -math.inf)
                out[b, j] = torch.softmax(w, -1).nan_to_num(0.0) @ vv
    return out


def exact(case: dict, seed: int):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "round_trip":
        return _exact_rounded(s["x"])
    if kind == "matmul":
        y = s["x"].double() @ _exact_values(s["codes"], s["scales"]).T
        for t in (s["b"], s["r"]):
            y = y if t is None else y + t.double()
        return y
    if kind == "append_read":
        both = []
        for x, codes, scales in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
            y = _exact_values(codes, scales)
            for b, n in enumerate(s["lens"].tolist()):
                y[b, :, n:n + case["new"]] = _exact_rounded(x[b]).transpose(0, 1)
            both.append(y)
        return tuple(both)
    k, v = (s["kc"], s["ks"]), (s["vc"], s["vs"])
    if kind == "decode":
        return _exact_attention(s["q"].unsqueeze(2), k, v, s["lens"][:, None], case["groups"])[:, :, 0]
    last = s["lens"][:, None] + torch.arange(1, case["new"] + 1, device=DEV)
    return _exact_attention(s["q"], k, v, last, case["groups"])


def work(case: dict) -> dict:
    """Bytes: inputs and outputs once each (a cache's rows in use: 11/20 of the room on average; the longest
    sequence fills it). Flops: two per multiply and add of the products."""
    kind = case["kind"]
    if kind == "round_trip":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (2 if case["dtype"] == "bfloat16" else 4) + 2 * n, "flops": 0}
    if kind == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        extra = (n if case["bias"] else 0) + (m * n if case["residual"] else 0)
        return {"bytes": n * k // 2 + n * k // BLOCK + 2 * (m * k + m * n + extra), "flops": 2 * m * n * k}
    B, H, D = case["batch"], case["kv_heads"], case["dim"]
    new, row = case.get("new", 0), D // 2 + D // BLOCK  # bytes of a key's or value's row
    if kind == "append_read":
        return {"bytes": 2 * B * H * (new * 2 * D + case["cap"] * (row + 2 * D)), "flops": 0}
    room = case["cap"] - new
    rows = room + (B - 1) * (room // 10 + room) / 2  # cached before the call, expected over the seeds
    Sq = max(new, 1)
    seen = Sq * rows + B * new * (new + 1) / 2
    return {"bytes": 2 * H * (rows + B * new) * row + 4 * B * H * case["groups"] * Sq * D,
            "flops": 4 * H * case["groups"] * D * seen}
