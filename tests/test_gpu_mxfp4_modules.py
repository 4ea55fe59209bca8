"""Four-bit weights and caches through the modules and models: the fused append, the attention module over an
MXFP4KVCache, generate(kv_format="mxfp4") and quantize_text_linears.

What the quantised forms compute is compared with the unquantised ops on the values the codes stand for, which are
exact in bf16: only the order of fp32 sums and the places of bf16 roundings differ. One rounding is 2^-8 of a value at
most, so a stage's output moves by at most 2^-8 of its norm (2-norm) per rounding that differs.
"""
import pytest
import torch

from oracle import mxfp4 as M
from qwen3_5_vl_cuda_custom_amd import kernels as K
from qwen3_5_vl_cuda_custom_amd import workloads as W
from qwen3_5_vl_cuda_custom_amd.configs import MoETextConfig, Qwen3VLConfig, TextConfig, VisionConfig
from qwen3_5_vl_cuda_custom_amd.models import CudaQwen3VLDenseModel, CudaQwen3VLMoeModel
from qwen3_5_vl_cuda_custom_amd.modules import (CudaLinear, CudaLinearMXFP4, MXFP4KVCache, StaticKVCache, StepGraph,
                                                quantize_text_linears)
from qwen3_5_vl_cuda_custom_amd.workloads import TextLayerConfig

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = 2.0 ** -8


def rnd(*shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def far(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


SECTIONS = {64: (12, 10, 10), 128: (24, 20, 20), 256: (48, 40, 40)}


@pytest.mark.parametrize("d,normed,S", [(64, True, 1), (128, True, 1), (128, False, 9), (256, True, 5), (128, True, 300)])
def test_fused_append_equals_norm_rotation_and_append(d, normed, S):
    B, Hq, Hkv, cap = 3, 8, 2, 40 + S
    lens = torch.tensor([0, 17, 41], dtype=torch.int32, device=DEV)  # the last sequence runs past the cap
    qkv = rnd(B, S, (Hq + 2 * Hkv) * d, seed=1)
    q, k, v = (t.view(B, S, -1, d) for t in qkv.split([Hq * d, Hkv * d, Hkv * d], -1))
    wq, wk = (rnd(d, seed=2) * 0.1 + 1, rnd(d, seed=3) * 0.1 + 1) if normed else (None, None)
    pos = torch.randint(0, 4000, (3, B, S), dtype=torch.int32, device=DEV)
    inv = W.make_rope(TextLayerConfig(256, 4, 2, d, 512, mrope_section=SECTIONS[d]), DEV).inv_freq
    shapes = [(B, Hkv, cap, w) for w in (d // 2, d // 32, d // 2, d // 32)]
    a, b = ([torch.full(s, 0x5A, dtype=torch.uint8, device=DEV) for s in shapes] for _ in range(2))
    qo = torch.empty_like(q, memory_format=torch.contiguous_format)
    K.qk_norm_rope_mxfp4(q, k, v, qo, *a, wq, wk, pos, inv, SECTIONS[d], 1e-6, lens)
    q2, k2 = torch.empty_like(qo), torch.empty(B, S, Hkv, d, dtype=torch.bfloat16, device=DEV)
    K.qk_norm_rope(q, k, None, q2, k2, None, wq, wk, pos, inv, SECTIONS[d], 1e-6)
    K.kv_append_mxfp4(k2, v, *b, lens)
    assert torch.equal(qo, q2)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    assert lens.tolist() == [0, 17, 41]


def _cfg(kv_heads=2, heads=8, d=128):
    return TextLayerConfig(hidden=512, heads=heads, kv_heads=kv_heads, head_dim=d, intermediate=1024,
                           mrope_section=SECTIONS[d])


def _pos(starts, n):
    p = torch.tensor(starts, device=DEV)[:, None] + torch.arange(n, device=DEV)
    return p.to(torch.int32).expand(3, len(starts), n).contiguous()


def _attention_on_values(attn, x, pos, rope, cache, before):
    """The attention module's step on the bf16 ops, over the rows the four-bit cache holds after it."""
    B, S, _ = x.shape
    Hq, Hkv, D = attn.num_heads, attn.num_kv_heads, attn.head_dim
    q, k, _ = (t.view(B, S, -1, D) for t in K.matmul_segments(
        x, [attn.q_proj.weight, attn.k_proj.weight, attn.v_proj.weight]).split([Hq * D, Hkv * D, Hkv * D], -1))
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    K.qk_norm_rope(q, k, None, qo, ko, None, attn.q_norm.weight, attn.k_norm.weight, pos, rope.inv_freq,
                   rope.mrope_section, attn.q_norm.eps)
    kc, vc = cache.gather(cache.capacity)
    o = K.flash_attention_cache(qo.transpose(1, 2), kc, vc, before, attn.scale, attn.num_kv_groups)
    return attn.o_proj(o.transpose(1, 2).reshape(B, S, Hq * D))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (6, 2), (4, 4)])
def test_attention_module_over_a_four_bit_cache(heads, kv_heads, d):
    cfg = _cfg(kv_heads, heads, d)
    attn, rope = W.make_text_layer(cfg, torch.bfloat16, DEV, seed=5).self_attn, W.make_rope(cfg, DEV)
    B, cap = 2, 200
    cache = MXFP4KVCache(B, kv_heads, cap, d, device=DEV)
    x = rnd(B, 60, cfg.hidden, seed=6)
    plain = StaticKVCache(B, kv_heads, cap, d, device=DEV)
    y = attn(x, rope.bind(_pos([0, 0], 60)), kv_cache=cache)[0]
    ref = attn(x, rope.bind(_pos([0, 0], 60)), kv_cache=plain)[0]
    # the first prefill attends to its unquantised rows, and stores them quantised. Two roundings differ (weights, output).
    assert far(y, ref) <= 3 * HALF
    want = MXFP4KVCache.from_static(plain)
    assert want.lens.tolist() == cache.lens.tolist() == [60, 60] and want.max_len == cache.max_len == 60
    for a, b in zip(cache.tensors, want.tensors):  # k's rotation differs in the order of a sum: few codes
        assert float((a[:, :, :60] != b[:, :, :60]).float().mean()) < 0.01
    cache.set_lens([60, 33])
    for starts, S in (([60, 33], 50), ([110, 83], 1), ([111, 84], 3), ([114, 87], 1)):
        before = cache.lens.clone()
        x = rnd(B, S, cfg.hidden, seed=7 + S)
        pos = _pos(starts, S)
        y, (kc, vc) = attn(x, rope.bind(pos), kv_cache=cache)
        assert kc is cache.k_codes and vc is cache.v_codes
        assert cache.lens.tolist() == [n + S for n in starts] and cache.max_len == starts[0] + S
        # roundings that may differ: the softmax weights, the attention's output, o_proj's
        assert far(y, _attention_on_values(attn, x, pos, rope, cache, before)) <= 4 * HALF


def test_attention_module_refuses_before_any_state_changes():
    cfg = _cfg()
    attn, rope = W.make_text_layer(cfg, torch.float32, DEV, seed=5).self_attn, W.make_rope(cfg, DEV)
    cache = MXFP4KVCache(2, 2, 32, 128, device=DEV)
    for x, c in ((rnd(2, 1, 512, dtype=torch.float32), cache),):
        with pytest.raises(ValueError):
            attn(x, rope.bind(_pos([0, 0], 1)), kv_cache=c)
    attn = attn.to(torch.bfloat16)
    x = rnd(2, 1, 512)
    for c in (MXFP4KVCache(2, 4, 32, 128, device=DEV), MXFP4KVCache(2, 2, 32, 64, device=DEV),
              MXFP4KVCache(3, 2, 32, 128, device=DEV)):
        with pytest.raises(ValueError):
            attn(x, rope.bind(_pos([0, 0], 1)), kv_cache=c)
        assert c.empty
    cache.set_lens([32, 1])
    with pytest.raises(ValueError, match="overflow"):
        attn(x, rope.bind(_pos([0, 0], 1)), kv_cache=cache)
    assert cache.lens.tolist() == [32, 1] and cache.max_len == 32


def test_captured_chunks_and_steps_of_two_caches_replayed_in_turn():
    """Two captured steps (one token, and three) over caches of their own, replayed in turn on another stream, give
    the eager results; a captured chunk's replays see the rows written since its capture."""
    cfg = _cfg()
    layer, rope = W.make_text_layer(cfg, torch.bfloat16, DEV, seed=8), W.make_rope(cfg, DEV)
    B = 2
    out = {}
    for mode in ("eager", "graph"):
        caches = {S: MXFP4KVCache(B, 2, 150, 128, device=DEV) for S in (1, 3)}
        x = {S: torch.zeros(B, S, cfg.hidden, dtype=torch.bfloat16, device=DEV) for S in caches}
        pos = {S: torch.zeros(3, B, S, dtype=torch.int32, device=DEV) for S in caches}
        graphs = {}
        for S, c in caches.items():
            layer(rnd(B, 90, cfg.hidden, seed=9), rope.bind(_pos([0, 0], 90)), kv_cache=c)
            c.set_lens([90, 40])
            bound = rope.bind(pos[S])

            def step(S=S, c=c, bound=bound):
                return layer(x[S], bound, kv_cache=c)[0]
            graphs[S] = StepGraph(step, warmup=0, caches=[c], tokens=S) if mode == "graph" else step
        side = torch.cuda.Stream()
        ys = []
        for i in range(5):
            for S, c in caches.items():
                x[S].copy_(rnd(B, S, cfg.hidden, seed=20 + i))
                pos[S].copy_(_pos(c.lens.tolist(), S))
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    y = graphs[S].replay() if mode == "graph" else graphs[S]()
                    y = y.clone()
                torch.cuda.current_stream().wait_stream(side)
                torch.cuda.synchronize()
                ys.append(y)
        out[mode] = ys
        assert caches[3].lens.tolist() == [105, 55] and caches[1].lens.tolist() == [95, 45]
    for a, b in zip(out["eager"], out["graph"]):
        assert torch.equal(a, b)


def _dense(seed=40, d=128):
    vc = VisionConfig(hidden_size=128, num_layers=1, num_heads=2, intermediate_size=256, patch_size=8,
                      num_position_embeddings=64, out_hidden_size=256, deepstack_layers=(0,))
    t = TextConfig(hidden_size=256, intermediate_size=544, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=d,
                   vocab_size=1000, rope_theta=1e4, mrope_section=list(SECTIONS[d]))
    m = CudaQwen3VLDenseModel(Qwen3VLConfig(family="dense", vision=vc, text=t)).to(DEV, torch.bfloat16)
    W.init_normal_(m, seed=seed, include_bias=True)
    m.embed_tokens.weight.normal_(0, 1.0, generator=torch.Generator(device=DEV).manual_seed(seed + 1))
    return m.eval().requires_grad_(False)


@pytest.mark.parametrize("four_bit_weights", [False, True])
def test_generate_over_a_four_bit_cache(four_bit_weights):
    m = _dense()
    if four_bit_weights:
        names = quantize_text_linears(m, lm_head=True)
        assert len(names) == 2 * 7 + 1 and isinstance(m.lm_head, CudaLinearMXFP4)
    ids = torch.randint(0, 1000, (3, 29), generator=torch.Generator().manual_seed(41)).to(DEV)
    lens = [29, 3, 17]
    a = m.generate(ids, max_new_tokens=20, prompt_lens=lens, kv_format="mxfp4")
    b = m.generate(ids, max_new_tokens=20, prompt_lens=lens, kv_format="mxfp4", use_graph=False)
    assert a.shape == (3, 49) and torch.equal(a, b)
    # the first new token comes from the unquantised prompt rows: the bf16 cache's
    assert torch.equal(a[:, 29], m.generate(ids, max_new_tokens=2, prompt_lens=lens)[:, 29])
    for bad in (dict(kv_format="int4"), dict(kv_format="mxfp4", page_rows=32)):
        with pytest.raises(ValueError):
            m.generate(ids, max_new_tokens=2, **bad)


def test_quantized_layers_equal_their_dequantized_weights():
    """A model with four-bit linears against the same model with the weights the codes stand for, in bf16. The
    roundings that may differ in a layer's branch (norm, q/k/v, q/k norm, softmax weights, attention, o; norm, gate,
    up, activation, down): at most 11, each 2^-8 of the branch, for prompt and decode shapes, over two layers."""
    m, ref = _dense(seed=50), _dense(seed=50)
    names = quantize_text_linears(m)
    assert names[0] == "layers.0.self_attn.q_proj" and len(names) == 14 and isinstance(m.lm_head, CudaLinear)
    for n in names:
        q = m.get_submodule(n)
        back = q.dequantize()
        want = M.values(*M.quantize(ref.get_submodule(n).weight.cpu()))
        assert torch.equal(back.double().cpu(), want)
        ref.get_submodule(n).weight.copy_(back)
    assert quantize_text_linears(m) == []  # nothing left
    for B, S in ((1, 1), (2, 20), (3, 100)):
        ids = torch.randint(0, 1000, (B, S), generator=torch.Generator().manual_seed(S)).to(DEV)
        assert far(m(ids), ref(ids)) <= 2 * 11 * HALF
    assert set(m.state_dict()) >= {"layers.1.mlp.down_proj.weight_codes", "layers.1.mlp.down_proj.weight_scales"}
    again = _dense(seed=51)
    quantize_text_linears(again)
    again.load_state_dict(m.state_dict())
    assert torch.equal(again(ids), m(ids))


def test_quantized_linear_with_bias_and_residual():
    lin = CudaLinear(96, 40, bias=True).to(DEV, torch.bfloat16).requires_grad_(False)
    q = CudaLinearMXFP4.from_linear(lin)
    x, r = rnd(2, 7, 96, seed=60), rnd(2, 7, 40, seed=61)
    w = M.values(*M.quantize(lin.weight.cpu()))
    y = q(x, residual=r)
    terms = x.double().cpu().abs() @ w.abs().T + lin.bias.double().cpu().abs() + r.double().cpu().abs()
    want = x.double().cpu() @ w.T + lin.bias.double().cpu() + r.double().cpu()
    err = 98 * 2.0 ** -23 * terms
    assert bool(((y.double().cpu() - want).abs() <= HALF * (want.abs() + err) + err).all())
    with pytest.raises(ValueError):
        CudaLinearMXFP4(100, 8)
    with torch.enable_grad(), pytest.raises(NotImplementedError):
        q(x.clone().requires_grad_(True))


def test_moe_model_with_four_bit_attention():
    vc = VisionConfig(hidden_size=128, num_layers=1, num_heads=2, intermediate_size=256, patch_size=8,
                      num_position_embeddings=64, out_hidden_size=256, deepstack_layers=(0,))
    t = MoETextConfig(hidden_size=256, intermediate_size=512, num_layers=2, num_heads=8, num_kv_heads=1, head_dim=128,
                      vocab_size=500, rope_theta=1e4, mrope_section=[24, 20, 20], num_experts=8, num_experts_per_tok=2,
                      moe_intermediate_size=128)
    m = CudaQwen3VLMoeModel(Qwen3VLConfig(family="moe", vision=vc, text=t)).to(DEV, torch.bfloat16)
    W.init_normal_(m, seed=70, include_bias=True)
    m = m.eval().requires_grad_(False)
    names = quantize_text_linears(m)
    assert len(names) == 8 and all("self_attn" in n for n in names)
    ids = torch.randint(0, 500, (2, 40), generator=torch.Generator().manual_seed(71)).to(DEV)
    a = m.generate(ids, max_new_tokens=12, kv_format="mxfp4")
    b = m.generate(ids, max_new_tokens=12, kv_format="mxfp4", use_graph=False)
    assert torch.equal(a, b)


def test_fused_append_refusals():
    B, S, Hq, Hkv, d, cap = 2, 1, 4, 2, 128, 16
    q, k = rnd(B, S, Hq, d), rnd(B, S, Hkv, d)
    cache = MXFP4KVCache(B, Hkv, cap, d, device=DEV)
    pos = torch.zeros(3, B, S, dtype=torch.int32, device=DEV)
    inv = torch.ones(d // 2, device=DEV)
    w = rnd(d)
    good = dict(q=q, k=k, v=k, qo=torch.empty_like(q), t=cache.tensors, wq=w, wk=w, pos=pos, inv=inv,
                sec=SECTIONS[d], lens=cache.lens)

    def call(**change):
        a = {**good, **change}
        K.qk_norm_rope_mxfp4(a["q"], a["k"], a["v"], a["qo"], *a["t"], a["wq"], a["wk"], a["pos"], a["inv"], a["sec"],
                             1e-6, a["lens"])
    for change, exc in [
        (dict(q=q.float()), TypeError), (dict(k=k[:, :, :1]), ValueError), (dict(v=k[:, :, :1]), ValueError),
        (dict(qo=torch.empty_like(q)[:, :, :3]), ValueError), (dict(wk=None), ValueError), (dict(wq=w[:64]), ValueError),
        (dict(pos=pos.long()), ValueError), (dict(pos=pos[:2]), ValueError), (dict(inv=inv.double()), ValueError),
        (dict(inv=torch.ones(d, device=DEV)[::2]), ValueError), (dict(sec=(24, 20, 19)), ValueError),
        (dict(lens=cache.lens.long()), ValueError), (dict(t=tuple(x[:, :, :0] for x in cache.tensors)), ValueError),
        (dict(q=q.cpu()), RuntimeError),
    ]:
        with pytest.raises(exc):
            call(**change)
    assert not cache.k_codes.any() and not cache.v_codes.any()
    call()
    assert cache.k_codes[:, :, 0].any() and not cache.k_codes[:, :, 1:].any()


def _plain(linear):
    """nn.Linear of the same weight (and bias)."""
    p = torch.nn.Linear(linear.in_features, linear.out_features, bias=linear.bias is not None, device=DEV,
                        dtype=linear.weight.dtype).requires_grad_(False)
    p.load_state_dict(linear.state_dict())
    return p


@pytest.mark.parametrize("S", [1, 40])
def test_projections_of_another_class_run_as_before(S):
    """q/k/v and gate/up as nn.Linear take the same fused products as CudaLinear, with and without the fused norm."""
    cfg = _cfg()
    x, pos = rnd(2, S, cfg.hidden, seed=80), _pos([0, 0], S)
    for names in (("q_proj",), ("q_proj", "k_proj", "v_proj")):
        layer = W.make_text_layer(cfg, torch.bfloat16, DEV, seed=81).requires_grad_(False)
        bound = W.make_rope(cfg, DEV).bind(pos)
        want = layer(x, bound)[0]
        for n in names:
            setattr(layer.self_attn, n, _plain(getattr(layer.self_attn, n)))
        layer.mlp.gate_proj = _plain(layer.mlp.gate_proj)
        if len(names) > 1:
            layer.mlp.up_proj = _plain(layer.mlp.up_proj)
        assert torch.equal(layer(x, bound)[0], want)
        cache = StaticKVCache(2, cfg.kv_heads, S, cfg.head_dim, device=DEV)
        layer(x, bound, kv_cache=cache)
        assert cache.max_len == S


@pytest.mark.parametrize("S", [1, 40])
def test_projections_of_another_class_beside_four_bit_ones(S):
    cfg = _cfg()
    x, pos = rnd(2, S, cfg.hidden, seed=82), _pos([0, 0], S)
    layer, bound = W.make_text_layer(cfg, torch.bfloat16, DEV, seed=83).requires_grad_(False), W.make_rope(cfg, DEV).bind(pos)
    for m, n in ((layer.self_attn, "k_proj"), (layer.mlp, "up_proj")):
        setattr(m, n, CudaLinearMXFP4.from_linear(getattr(m, n)))
    want = layer(x, bound)[0]
    layer.self_attn.q_proj = _plain(layer.self_attn.q_proj)
    assert torch.equal(layer(x, bound)[0], want)


def test_caches_go_by_the_type_of_a_head_of_another_class():
    m = _dense()
    m.lm_head = _plain(m.lm_head)
    m.norm.float()
    assert m.new_caches(1, 8)[0].k.dtype == torch.bfloat16
    assert len(m.new_caches(1, 8, kv_format="mxfp4")) == 2


def test_a_large_cache_is_quantised_whatever_its_size():
    """More values than 32 bits count in pieces of eight. The bf16 rows are views that repeat one sequence's or one
    row's values, so only the four-bit rows take memory (9 GB)."""
    B, H, cap, d = 1024, 8, 8200, 128
    assert B * cap * 2 * H * (d // 8) > 2 ** 31
    k, v = rnd(B, H, 1, d, seed=90), rnd(1, H, cap, d, seed=91)
    plain = StaticKVCache(1, 1, 1, d, device=DEV)
    plain.k, plain.v, plain.capacity = k.expand(B, H, cap, d), v.expand(B, H, cap, d), cap
    plain.lens = torch.full((B,), 5, dtype=torch.int32, device=DEV)
    plain.set_host_state((5, 5))
    c = MXFP4KVCache.from_static(plain)
    assert c.lens.tolist() == [5] * B and c.max_len == 5 and c.capacity == cap
    for x, codes, scales in ((k, c.k_codes, c.k_scales), (v, c.v_codes, c.v_scales)):
        qc, qs = K.mxfp4_quantize(x)
        for b in range(0, B, 128):
            s = slice(b, b + 128)
            assert bool((codes[s] == (qc[s] if qc.shape[0] > 1 else qc)).all())
            assert bool((scales[s] == (qs[s] if qs.shape[0] > 1 else qs)).all())
