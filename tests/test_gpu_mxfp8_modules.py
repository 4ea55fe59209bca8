"""Weights in eight bits through the modules and models: CudaLinearMXFP8, the MLP, the attention module, decoder layers,
generate and quantize_text_linears(weight_format="mxfp8").

What a module computes is compared bit for bit with its operators called one by one, and, on inputs and weights that
eight bits hold exactly, with the bf16 module; a whole model with its bf16 form by the size of the roundings.
"""
import pytest
import torch

from oracle import mxfp8 as M
from qwen3_5_vl_cuda_custom_amd import kernels as K
from qwen3_5_vl_cuda_custom_amd import workloads as W
from qwen3_5_vl_cuda_custom_amd.configs import MoETextConfig, Qwen3VLConfig, TextConfig, VisionConfig
from qwen3_5_vl_cuda_custom_amd.models import CudaQwen3VLDenseModel, CudaQwen3VLMoeModel
from qwen3_5_vl_cuda_custom_amd.modules import (CudaLinear, CudaLinearMXFP4, CudaLinearMXFP8, CudaRMSNorm, CudaSwiGLUMLP,
                                                MXFP4KVCache, PagedKVCache, StaticKVCache, quantize_text_linears)
from qwen3_5_vl_cuda_custom_amd.workloads import TextLayerConfig

pytestmark = pytest.mark.gpu
DEV = "cuda"
SECTIONS = {64: (12, 10, 10), 128: (24, 20, 20)}


@pytest.fixture(autouse=True)
def no_grad():
    with torch.no_grad():
        yield


def rnd(*shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


def small(*shape, seed=0):
    """Values of three bits and one size, which eight bits hold exactly, and whose products sum exactly."""
    g = torch.Generator().manual_seed(seed)
    v = torch.tensor([0.0, 1.0, 1.25, 1.5, 1.75])[torch.randint(0, 5, shape, generator=g)]
    return (v * (1 - 2 * torch.randint(0, 2, shape, generator=g))).to(torch.bfloat16).to(DEV)


def far(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def _cfg(kv_heads=2, heads=8, d=128):
    return TextLayerConfig(hidden=512, heads=heads, kv_heads=kv_heads, head_dim=d, intermediate=1024,
                           mrope_section=SECTIONS[d])


def _pos(starts, n):
    p = torch.tensor(starts, device=DEV)[:, None] + torch.arange(n, device=DEV)
    return p.to(torch.int32).expand(3, len(starts), n).contiguous()


# ------------------------------------------------------------------ the linear layer
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear(bias, dtype):
    lin = CudaLinear(96, 40, bias=bias).to(DEV, dtype)
    W.init_normal_(lin, seed=3, include_bias=True)
    q = CudaLinearMXFP8.from_linear(lin)
    codes, scales = M.quantize(lin.weight.cpu().to(torch.float32))
    assert torch.equal(q.weight_codes.view(torch.uint8).cpu(), codes.view(torch.uint8)) and torch.equal(q.weight_scales.cpu(), scales)
    assert torch.equal(q.dequantize().double().cpu(), M.values(codes, scales))
    x, r = rnd(2, 7, 96, seed=60), rnd(2, 7, 40, seed=61)
    b = lin.bias.to(torch.bfloat16) if bias else None
    want = K.matmul_mxfp8(x, q.pair, b, r)
    assert torch.equal(q(x, residual=r), want) and torch.equal(q(K.mxfp8_quantize(x), r), want)
    out = torch.empty(2, 7, 40, dtype=torch.bfloat16, device=DEV)
    assert q(x, residual=r, out=out) is out and torch.equal(out, want)


def test_linear_keeps_its_codes_through_conversions_and_state_dicts():
    q = CudaLinearMXFP8.from_linear(CudaLinear(64, 33, bias=True).to(DEV))
    before, x = q.weight_codes.clone(), rnd(3, 64)
    y = q(x)
    for move in (lambda: q.float(), lambda: q.half(), lambda: q.cpu(), lambda: q.to(DEV, torch.bfloat16)):
        move()
        assert q.weight_codes.dtype == torch.float8_e4m3fn and q.weight_scales.dtype == torch.uint8
    assert torch.equal(q.weight_codes.view(torch.uint8), before.view(torch.uint8)) and torch.equal(q(x), y)
    again = CudaLinearMXFP8(64, 33).to(DEV, torch.bfloat16)
    again.load_state_dict(q.state_dict())
    assert torch.equal(again(x), y) and set(q.state_dict()) == {"weight_codes", "weight_scales", "bias"}
    with pytest.raises(ValueError):
        CudaLinearMXFP8(100, 8)
    with torch.enable_grad(), pytest.raises(NotImplementedError):
        q(x.clone().requires_grad_(True))


# ------------------------------------------------------------------ the MLP
def _mlp(h, i, kinds, bias=False):
    m = CudaSwiGLUMLP(h, i, bias=bias).to(DEV, torch.bfloat16)
    W.init_normal_(m, seed=5, include_bias=True)
    for name, kind in zip(("gate_proj", "up_proj", "down_proj"), kinds):
        if kind is not None:
            setattr(m, name, kind.from_linear(getattr(m, name)))
    return m


@pytest.mark.parametrize("rows", [1, 40, 300])
@pytest.mark.parametrize("normed", [False, True])
def test_mlp_is_its_operators(rows, normed):
    h, i = 256, 544
    norm = CudaRMSNorm(h).to(DEV, torch.bfloat16)
    norm.weight.copy_(1 + 0.1 * rnd(h, seed=9))
    x, r = rnd(2, rows, h, seed=1), rnd(2, rows, h, seed=2)
    m = _mlp(h, i, [CudaLinearMXFP8] * 3)
    pair = K.add_rmsnorm_mxfp8(x, None, norm.weight, norm.eps)[1:] if normed else K.mxfp8_quantize(x)
    act = K.matmul_swiglu_mxfp8(pair, m.gate_proj.pair, m.up_proj.pair, quantize=True)
    want = K.matmul_mxfp8(act, m.down_proj.pair, residual=r)
    assert torch.equal(m(x, residual=r, input_norm=norm if normed else None), want)
    m = _mlp(h, i, [CudaLinearMXFP8, CudaLinearMXFP8, None])  # down in bf16 takes the activation in bf16
    act = K.matmul_swiglu_mxfp8(pair, m.gate_proj.pair, m.up_proj.pair)
    assert torch.equal(m(x, residual=r, input_norm=norm if normed else None), m.down_proj(act, residual=r))


@pytest.mark.parametrize("kinds,bias", [((CudaLinearMXFP8, None, None), False), ((None, CudaLinearMXFP8, CudaLinearMXFP8), False),
                                        ((CudaLinearMXFP8, CudaLinearMXFP4, CudaLinearMXFP4), False),
                                        ((CudaLinearMXFP8, CudaLinearMXFP8, CudaLinearMXFP8), True)])
def test_mlp_of_several_kinds_runs_each_by_itself(kinds, bias):
    m, norm, x = _mlp(256, 544, kinds, bias), CudaRMSNorm(256).to(DEV, torch.bfloat16), rnd(30, 256, seed=1)
    y = norm(x)
    want = m.down_proj(K.swiglu(m.gate_proj(y), m.up_proj(y)), residual=x)
    assert torch.equal(m(x, residual=x, input_norm=norm), want)


class _Plain(torch.nn.Module):
    """A projection that is no linear layer of this package: a weight, and no attribute `bias`."""

    def __init__(self, weight):
        super().__init__()
        self.weight = weight

    def forward(self, x):
        return K.matmul(x, self.weight)


@pytest.mark.parametrize("kind", [CudaLinearMXFP4, CudaLinearMXFP8])
@pytest.mark.parametrize("name", ["gate_proj", "up_proj"])
def test_mlp_takes_a_module_without_a_bias_beside_a_quantised_projection(kind, name):
    m, norm, x = _mlp(256, 544, [kind, kind, None]), CudaRMSNorm(256).to(DEV, torch.bfloat16), rnd(9, 256, seed=1)
    del m._modules[name]
    setattr(m, name, _Plain(torch.nn.Parameter(rnd(544, 256, seed=4), requires_grad=False)))
    y = norm(x)
    want = m.down_proj(K.swiglu(m.gate_proj(y), m.up_proj(y)), residual=x)
    assert torch.equal(m(x, residual=x, input_norm=norm), want)


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("cache_kind", [None, StaticKVCache, PagedKVCache, MXFP4KVCache])
@pytest.mark.parametrize("S", [1, 50])
def test_attention_on_exact_values_equals_bf16(cache_kind, S):
    """q, k and v of exact values are the bf16 module's to the bit, so is everything up to o_proj's input; o_proj takes
    that input in eight bits."""
    cfg = _cfg()
    attn, rope = W.make_text_layer(cfg, torch.bfloat16, DEV, seed=5).self_attn, W.make_rope(cfg, DEV)
    for i, p in enumerate((attn.q_proj, attn.k_proj, attn.v_proj)):
        p.weight.copy_(small(*p.weight.shape, seed=i) * 2.0 ** -6)

    def run(x):
        cache = None
        if cache_kind is PagedKVCache:
            cache = PagedKVCache(2, cfg.kv_heads, cfg.head_dim, num_pages=4, max_pages=2, device=DEV)
        elif cache_kind is not None:
            cache = cache_kind(2, cfg.kv_heads, 64, cfg.head_dim, device=DEV)
        ys = []
        for step in range(2):
            n = S if step == 0 else 1
            if step and cache is None:
                break
            pos = _pos([0, 0] if step == 0 else [S, S], n)
            ys.append(attn(x[:, :n], rope.bind(pos), kv_cache=cache, residual=x[:, :n])[0])
        return ys
    x = small(2, S, cfg.hidden, seed=9)
    want = run(x)
    for n in ("q_proj", "k_proj", "v_proj"):
        setattr(attn, n, CudaLinearMXFP8.from_linear(getattr(attn, n)))
    for a, b in zip(run(x), want):
        assert torch.equal(a, b)
    rows = []
    attn.o_proj = CudaLinearMXFP8.from_linear(attn.o_proj)
    attn.o_proj.register_forward_pre_hook(lambda m, args, kw: rows.append(args[0].clone()), with_kwargs=True)
    for y, o in zip(run(x), rows):
        assert torch.equal(y, K.matmul_mxfp8(o, attn.o_proj.pair, residual=x[:, :y.shape[1]]))


@pytest.mark.parametrize("kinds", [(CudaLinearMXFP8, None, None), (None, CudaLinearMXFP4, CudaLinearMXFP8)])
def test_attention_with_projections_of_several_kinds(kinds):
    cfg = _cfg()
    layer, x = W.make_text_layer(cfg, torch.bfloat16, DEV, seed=83), rnd(2, 20, cfg.hidden, seed=82)
    attn, bound = layer.self_attn, W.make_rope(cfg, DEV).bind(_pos([0, 0], 20))
    for n, kind in zip(("q_proj", "k_proj", "v_proj"), kinds):
        if kind is not None:
            setattr(attn, n, kind.from_linear(getattr(attn, n)))
    got = attn(x, bound, input_norm=layer.input_layernorm)[0]
    y = layer.input_layernorm(x)
    qkv = torch.cat([p(y) for p in (attn.q_proj, attn.k_proj, attn.v_proj)], -1)
    assert torch.equal(attn._project_apart(y, (attn.q_proj, attn.k_proj, attn.v_proj)), qkv)
    assert got.shape == x.shape and bool(torch.isfinite(got).all())


def test_other_types_are_refused():
    cfg = _cfg()
    layer = W.make_text_layer(cfg, torch.float32, DEV, seed=8)
    assert len(quantize_text_linears(layer, weight_format="mxfp8")) == 7
    bound = W.make_rope(cfg, DEV).bind(_pos([0], 4))
    for norm in (layer.input_layernorm, None):
        with pytest.raises(TypeError):
            layer.self_attn(rnd(1, 4, cfg.hidden, dtype=torch.float32), bound, input_norm=norm)
        with pytest.raises(TypeError):
            layer.mlp(rnd(4, cfg.hidden, dtype=torch.float32), input_norm=norm)
    with pytest.raises(ValueError):
        quantize_text_linears(layer, weight_format="int8")


# ------------------------------------------------------------------ models
def _dense(seed=40, d=128):
    vc = VisionConfig(hidden_size=128, num_layers=1, num_heads=2, intermediate_size=256, patch_size=8,
                      num_position_embeddings=64, out_hidden_size=256, deepstack_layers=(0,))
    t = TextConfig(hidden_size=256, intermediate_size=544, num_layers=2, num_heads=4, num_kv_heads=2, head_dim=d,
                   vocab_size=1000, rope_theta=1e4, mrope_section=list(SECTIONS[d]))
    m = CudaQwen3VLDenseModel(Qwen3VLConfig(family="dense", vision=vc, text=t)).to(DEV, torch.bfloat16)
    W.init_normal_(m, seed=seed, include_bias=True)
    m.embed_tokens.weight.normal_(0, 1.0, generator=torch.Generator(device=DEV).manual_seed(seed + 1))
    return m.eval().requires_grad_(False)


@pytest.mark.parametrize("options", [{}, {"kv_format": "mxfp4"}, {"page_rows": 32}])
def test_generate(options):
    m = _dense()
    assert len(quantize_text_linears(m, lm_head=True, weight_format="mxfp8")) == 15
    assert isinstance(m.lm_head, CudaLinearMXFP8)
    ids = torch.randint(0, 1000, (3, 29), generator=torch.Generator().manual_seed(41)).to(DEV)
    a = m.generate(ids, max_new_tokens=20, prompt_lens=[29, 3, 17], **options)
    b = m.generate(ids, max_new_tokens=20, prompt_lens=[29, 3, 17], use_graph=False, **options)
    assert a.shape == (3, 49) and torch.equal(a, b)


def test_quantized_model_is_near_its_bf16_form():
    """Against the model with the weights the codes stand for, in bf16. A quantised value is off by 2^-4 of itself at most
    (by the subnormal step, 2^-17 of its block's largest, below); a layer quantises four inputs (q/k/v's, o's, gate and
    up's, down's), each moving its branch by 2^-4 of its norm at most, where the bf16 roundings are 2^-8: two layers
    2 · 4 · 2^-4."""
    m, ref = _dense(seed=50), _dense(seed=50)
    names = quantize_text_linears(m, weight_format="mxfp8")
    assert names[0] == "layers.0.self_attn.q_proj" and len(names) == 14 and isinstance(m.lm_head, CudaLinear)
    for n in names:
        ref.get_submodule(n).weight.copy_(m.get_submodule(n).dequantize())
    assert quantize_text_linears(m, weight_format="mxfp8") == []  # nothing left
    for B, S in ((1, 1), (2, 20), (3, 100)):
        ids = torch.randint(0, 1000, (B, S), generator=torch.Generator().manual_seed(S)).to(DEV)
        assert far(m(ids), ref(ids)) <= 2 * 4 * 2.0 ** -4
    again = _dense(seed=51)
    quantize_text_linears(again, weight_format="mxfp8")
    again.load_state_dict(m.state_dict())
    assert torch.equal(again(ids), m(ids))


def test_moe_model_with_eight_bit_attention():
    vc = VisionConfig(hidden_size=128, num_layers=1, num_heads=2, intermediate_size=256, patch_size=8,
                      num_position_embeddings=64, out_hidden_size=256, deepstack_layers=(0,))
    t = MoETextConfig(hidden_size=256, intermediate_size=512, num_layers=2, num_heads=8, num_kv_heads=1, head_dim=128,
                      vocab_size=500, rope_theta=1e4, mrope_section=[24, 20, 20], num_experts=8, num_experts_per_tok=2,
                      moe_intermediate_size=128)
    m = CudaQwen3VLMoeModel(Qwen3VLConfig(family="moe", vision=vc, text=t)).to(DEV, torch.bfloat16)
    W.init_normal_(m, seed=70, include_bias=True)
    m = m.eval().requires_grad_(False)
    names = quantize_text_linears(m, weight_format="mxfp8")
    assert len(names) == 8 and all("self_attn" in n for n in names)
    ids = torch.randint(0, 500, (2, 40), generator=torch.Generator().manual_seed(71)).to(DEV)
    a = m.generate(ids, max_new_tokens=12)
    assert torch.equal(a, m.generate(ids, max_new_tokens=12, use_graph=False))


def test_two_layers_on_two_streams_and_replayed_graphs():
    """Two decoder layers captured into graphs that share a memory pool and replayed in turn, an eager layer on another
    stream between them: every result is the eager one."""
    cfg = _cfg()
    layers = [W.make_text_layer(cfg, torch.bfloat16, DEV, seed=s) for s in (90, 91)]
    for layer in layers:
        quantize_text_linears(layer, weight_format="mxfp8")
    bound = W.make_rope(cfg, DEV).bind(_pos([0], 130))
    xs = [rnd(1, 130, cfg.hidden, seed=s) for s in (1, 2)]
    graphs, outs, pool = [], [], torch.cuda.graph_pool_handle()
    for layer, x in zip(layers, xs):
        layer(x, bound)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(layer(x, bound)[0])
        graphs.append(g)
    side = torch.cuda.Stream()
    for i in range(3):
        for x in xs:
            x.copy_(rnd(*x.shape, seed=10 + i))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = layers[0](xs[0], bound)[0]
        want = [layer(x, bound)[0] for layer, x in zip(layers, xs)]
        for g, out, w in zip(graphs, outs, want):  # a replay may use what the other one's result lies in
            g.replay()
            assert torch.equal(out, w)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(eager, want[0])
