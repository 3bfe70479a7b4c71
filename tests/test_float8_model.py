"""8-bit weights in whole models: checkpoints that store them, engines that quantise when they are built, experts, refusals."""
import json
import os

import pytest
import torch

import plain_qwen3 as plain
from conftest import TEST_CONFIGS, rel_err

E4M3 = torch.float8_e4m3fn
DEV = "cuda:0"
BF16 = torch.bfloat16


def blocks(n):
    return -(-n // 128)


def cell_scales(w, tall):
    """The smallest 2^e (e >= -126) with which a block's largest magnitude is at most 448, for blocks of ``tall`` rows and 128
    columns: [row blocks, column blocks]."""
    n, k = w.shape
    pad = torch.zeros(-(-n // tall) * tall, blocks(k) * 128, dtype=torch.float64)
    pad[:n, :k] = w.to(torch.float64)
    top = pad.view(-1, tall, blocks(k), 128).abs().amax((1, 3))
    e = torch.ceil(torch.log2(top.clamp(min=1e-300) / 448.0)).clamp(min=-126.0)
    e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)
    e = torch.where((top <= 448.0 * torch.exp2(e - 1)) & (e > -126), e - 1, e)
    return torch.exp2(e).to(torch.float32)


def spread(scales, tall, n, k):
    return scales.repeat_interleave(tall, 0)[:n].repeat_interleave(128, 1)[:, :k]


def quantized(w, tall):
    """``w`` as its 8-bit form stands for (float32)."""
    s = spread(cell_scales(w, tall), tall, *w.shape)
    return (w.to(torch.float32) / s).to(E4M3).to(torch.float32) * s


def store_float8(folder, cfg_dict, seed, pe, general=True):
    """A model folder whose projections are stored in 8 bits with scales beside them; returns (config, weights as numbers)."""
    from safetensors.torch import load_file, save_file

    pe.write_random_model(folder, pe.Qwen3Config.from_dict(cfg_dict), seed=seed)
    path = os.path.join(folder, "model.safetensors")
    tensors = load_file(path)
    out, wide = {}, {}
    for name, t in tensors.items():
        wide[name] = t.to(torch.float32)
        out[name] = t
        if ".self_attn." in name and name.endswith("_proj.weight") or ".mlp." in name:
            s = cell_scales(t, 128)
            if general:          # scales as other programs make them: no powers of two
                s = s * 0.77
            v = (t.to(torch.float32) / spread(s, 128, *t.shape)).clamp(-448, 448).to(E4M3)
            out[name], out[name + "_scale_inv"] = v, s
            wide[name] = v.to(torch.float32) * spread(s, 128, *t.shape)
    save_file(out, path, metadata={"format": "pt"})
    return cfg_dict, wide


def make_folder(tmp_path, cfg_dict, seed, pe, **kw):
    folder = str(tmp_path / "m")
    return (folder, *store_float8(folder, cfg_dict, seed, pe, **kw))


# ---- on the CPU: loading and refusals --------------------------------------------------------------------------------------
def test_load(pe, tmp_path):
    folder, cfg, wide = make_folder(tmp_path, TEST_CONFIGS["B"], 3, pe)
    plan = pe.config.registry.architecture("Qwen3ForCausalLM").plan(pe.load_config(folder))
    got = pe.load_weights(folder, plan)
    for name, w in wide.items():
        t = got[name]
        if type(t) is pe.parts.float8.Float8Weight:
            assert t.values.dtype == E4M3 and t.scales.dtype == torch.float32
            t = t.dequantize()
        assert torch.equal(t.to(torch.float32), w), name
    assert set(got) == set(wide)


def test_load_refusals(pe, tmp_path):
    from safetensors.torch import load_file, save_file

    folder, cfg, _ = make_folder(tmp_path, TEST_CONFIGS["A"], 3, pe)
    plan = pe.config.registry.architecture("Qwen3ForCausalLM").plan(pe.load_config(folder))
    path = os.path.join(folder, "model.safetensors")
    whole = load_file(path)
    name = "model.layers.0.mlp.up_proj.weight"
    for change, text in (({name + "_scale_inv": None}, "missing"), ({name + "_scale_inv": torch.ones(3, 1)}, "wrong shapes"),
                         ({name + "_scale_inv": torch.ones(1, 1, dtype=torch.int32)}, "unusable dtypes"),
                         ({"model.norm.weight": whole["model.norm.weight"].to(E4M3)}, "unusable dtypes"),
                         ({"model.norm.weight_scale_inv": torch.ones(1, 1)}, "unexpected")):
        t = {**whole, **change}
        save_file({k: v for k, v in t.items() if v is not None}, path)
        with pytest.raises(pe.WeightError, match=text):
            pe.load_weights(folder, plan)


def test_weight_shapes(pe):
    f8 = pe.parts.float8
    v = torch.zeros(130, 200).to(E4M3)
    w = f8.Float8Weight(v, torch.ones(2, 2))
    assert tuple(w.shape) == (130, 200) and w.nbytes() == 130 * 200 + 16
    for bad in (lambda: f8.Float8Weight(v, torch.ones(1, 2)), lambda: f8.Float8Weight(v, torch.ones(2, 2, dtype=torch.float64)),
                lambda: f8.Float8Weight(torch.zeros(130, 200), torch.ones(2, 2)), lambda: f8.Float8Weight.cat_rows([w, w])):
        with pytest.raises(ValueError):
            bad()
    whole = f8.Float8Weight(torch.zeros(256, 200).to(E4M3), torch.ones(2, 2))
    cat = f8.Float8Weight.cat_rows([whole, w])
    assert tuple(cat.shape) == (386, 200) and tuple(cat.scales.shape) == (4, 2) and cat.values.stride(0) == 208
    assert torch.equal(cat.dequantize(), torch.zeros(386, 200))


def test_ops_refuse_cpu_tensors(pe):
    ops, f8 = pe.kernels.ops, pe.parts.float8
    x = torch.zeros(2, 128, dtype=BF16)
    w, s, out = torch.zeros(64, 128).to(E4M3), torch.ones(1, 1), torch.zeros(2, 64, dtype=BF16)
    if torch.cuda.is_available():
        return
    with pytest.raises(Exception):
        ops.linear_fp8(x, w, s, out, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(Exception):
        f8.Float8Rows.quantize(x)


# ---- refusals on the GPU -----------------------------------------------------------------------------------------------------
def test_sizes_refused(pe):
    """More rows than the tiles' 32-bit arithmetic holds: refused on the host, before anything is launched."""
    lib, p, big = pe.kernels.library(), 256, (1 << 30) + 1
    act = (0, 0, 0.0, 1.0, None)
    assert lib.pe_gemm_fp8(p, 128, p, big, p, 128, p, p, 64, big, 64, 128, *act, None, None, 0, p, None) == -1
    assert lib.pe_gemm_fp8_many(p, 128, p, big, p, 128, p, p, 64, None, 0, big, 64, 128, *act, None, None, 0, p, None) == -1
    assert lib.pe_quantize_rows_fp8(1, p, 128, None, None, p, 128, p, big, big, 128, big, p, None) == -1
    assert lib.pe_quantize_weight_fp8(1, p, 128, p, 128, p, big, 128, None) == -1


@pytest.mark.gpu
def test_op_refusals(pe):
    ops, f8 = pe.kernels.ops, pe.parts.float8
    pe.kernels.library()
    st = torch.zeros(4, dtype=torch.int32, device=DEV)
    x, out = torch.zeros(4, 256, dtype=BF16, device=DEV), torch.empty(4, 128, dtype=BF16, device=DEV)
    w = f8.Float8Weight.quantize(torch.ones(128, 256, device=DEV))
    r = f8.Float8Rows.quantize(x)
    call = dict(x=x, w=w.values, w_scales=w.scales, out=out, status=st)
    odd = torch.empty(128, 264, dtype=E4M3, device=DEV)[:, :256]                      # rows 264 bytes apart
    three = torch.zeros(3, dtype=torch.int32, device=DEV)
    for change in (dict(out=out[:3]), dict(out=out[:, :100]), dict(out=out.to(torch.float16)), dict(out=out.t().contiguous().t()), dict(w=odd),
                   dict(w=w.values[:, :128]), dict(w=w.values.to(BF16)), dict(w_scales=w.scales.double()), dict(w_scales=w.scales[:, :1]),
                   dict(w_scales=w.scales.expand(2, 2)), dict(w=w.values.cpu()), dict(x=x[:, ::2]), dict(x=x.half()), dict(offsets=three),
                   dict(row_weight=torch.ones(4, device=DEV)), dict(glu=("silu", 0.0, 1.0, torch.ones(3, device=DEV)), out=out[:, :64]),
                   dict(glu=("nothing", 0.0, 1.0, None), out=out[:, :64]), dict(out=torch.empty(4, 64, device=DEV), glu=()),
                   dict(row_map=torch.zeros(4, dtype=torch.int64, device=DEV))):
        with pytest.raises((pe.kernels.KernelError, KeyError)):
            ops.linear_fp8(**{**call, **change})
    for bad in (dict(x_scales=r.scales.t()), dict(x_scales=r.scales[:1]), dict(x_scales=r.scales.double()), dict(x=r.values[:, 8:], w=w.values[:, 8:])):
        with pytest.raises(pe.kernels.KernelError):
            ops.gemm_fp8(**{**dict(x=r.values, x_scales=r.scales, w=w.values, w_scales=w.scales, out=out, status=st), **bad})
    with pytest.raises(pe.kernels.KernelError):
        ops.quantize_rows_fp8(x, torch.empty(4, 256, dtype=torch.uint8, device=DEV), r.scales)
    with pytest.raises(pe.kernels.KernelError):
        ops.quantize_rows_fp8(x.half(), r.values, r.scales)
    with pytest.raises(pe.kernels.KernelError):
        ops.quantize_weight_fp8(torch.ones(128, 256, device=DEV), w.values, w.scales.t()[:1])
    with pytest.raises(pe.kernels.KernelError):
        ops.rmsnorm_residual_fp8(torch.zeros(4, 256, device=DEV), x.float(), torch.ones(256, device=DEV), r.values, r.scales, 1e-6)
    with pytest.raises(pe.kernels.KernelError):
        ops.rmsnorm_residual_fp8(torch.zeros(4, 255, device=DEV), None, torch.ones(255, device=DEV), r.values[:, :255], r.scales, 1e-6)
    assert st.tolist()[0] == 0


@pytest.mark.gpu
def test_engine_refusals(pe):
    cfg = pe.Qwen3Config.from_dict(TEST_CONFIGS["A"])
    for kw in (dict(weight_format="float4"), dict(weight_format="float8", dtype="float32")):
        with pytest.raises(ValueError, match="weight_format"):
            pe.Engine.from_random(cfg, 1, max_cache_tokens=256, max_batch=1, **kw)


# ---- whole models ------------------------------------------------------------------------------------------------------------
def plain_float8_forward(cfg, w, tokens, round_weights=True):
    """``plain.forward_logits`` in a bfloat16 run's roundings whose projections have 8-bit operands: rows in blocks of 128 features,
    and, with ``round_weights``, the stacked matrices q|k|v, o, gate|up and down in blocks of 128 x 128."""
    f = lambda name: w[name].to(torch.float32)
    st = lambda x: plain.stored(x, BF16)
    kv, d, nh = cfg["num_key_value_heads"], cfg["head_dim"], cfg["num_attention_heads"]
    eps = float(cfg["rms_norm_eps"])
    weight = (lambda ms: quantized(torch.cat(ms), 128)) if round_weights else torch.cat
    linear = lambda x, *ms: quantized(x, 1) @ weight([f(m) for m in ms]).T
    x = f("model.embed_tokens.weight")[torch.as_tensor(list(tokens))]
    S = x.shape[0]
    cos, sin = plain.rope_cos_sin(torch.arange(S), d, float(cfg["rope_theta"]))
    for i in range(cfg["num_hidden_layers"]):
        p = f"model.layers.{i}"
        n = st(plain.rms_norm(x, f(f"{p}.input_layernorm.weight"), eps))
        qkv = st(linear(n, *(f"{p}.self_attn.{c}_proj.weight" for c in "qkv")))
        q, k, v = qkv.split([nh * d, kv * d, kv * d], 1)
        q = plain.rms_norm(q.reshape(S, nh, d), f(f"{p}.self_attn.q_norm.weight"), eps)
        k = plain.rms_norm(k.reshape(S, kv, d), f(f"{p}.self_attn.k_norm.weight"), eps)
        q, k = (st(plain.rope_rotate_neox(t, cos, sin, d)) for t in (q, k))
        o = st(plain.causal_gqa_attention(q, k, v.reshape(S, kv, d), d ** -0.5, window=plain.layer_window(cfg, i)))
        x = x + st(linear(o.reshape(S, -1), f"{p}.self_attn.o_proj.weight"))
        n = st(plain.rms_norm(x, f(f"{p}.post_attention_layernorm.weight"), eps))
        g, u = linear(n, f"{p}.mlp.gate_proj.weight", f"{p}.mlp.up_proj.weight").chunk(2, 1)
        x = x + st(linear(st(g / (1 + torch.exp(-g)) * u), f"{p}.mlp.down_proj.weight"))
    n = st(plain.rms_norm(x, f("model.norm.weight"), eps))
    return n @ f("model.embed_tokens.weight" if cfg.get("tie_word_embeddings") else "lm_head.weight").T


# Two runs of one model whose activations differ by bfloat16's roundings (2^-8 of a value) fall on different sides of an e4m3
# rounding for up to 2 * 2^-8 / 2^-3 = 1/16 of the elements (its steps are 2^-3 of a value apart at the most), and differ there by a
# step: sqrt(1/16) * 2^-3 = 3.1 % of a product's inputs at the most in the 2-norm, as much of its outputs (random signs), and for
# the two or three layers here, whose outputs are a part of the stream, no more than twice that in the logits.
MODEL_TOL = 0.0625


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["A", "B", "D", "E"])
@pytest.mark.parametrize("graphs", [True, False])
def test_engine_quantizes(pe, tmp_path, name, graphs):
    """Prompts of one token to a few tiles, then single tokens, against the plain model with 8-bit operands."""
    cfg = TEST_CONFIGS[name]
    folder = str(tmp_path / "m")
    pe.write_random_model(folder, pe.Qwen3Config.from_dict(cfg), seed=5)
    pcfg, w = plain.load_folder(folder)
    eng = pe.Engine(folder, weight_format="float8", max_context_len=256, max_cache_tokens=64 * 16, max_batch=4, enable_cuda_graph=graphs)
    assert all(type(t) is pe.parts.float8.Float8Weight for b in eng.model.blocks for t in (b.mixer.qkv, b.mixer.o_proj, b.ffn.gate_up, b.ffn.down))
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, cfg["vocab_size"], (n,), generator=gen).tolist() for n in (1, 9, 70, 150)]
    slots = [eng.alloc_slot() for _ in prompts]
    got = eng.step([pe.StepEntry(s, p, tuple(range(len(p)))) for s, p in zip(slots, prompts)]).float().cpu()
    want = [plain_float8_forward(pcfg, w, p) for p in prompts]
    assert float((got - torch.cat(want)).norm() / torch.cat(want).norm()) < MODEL_TOL
    for t in range(3):
        step = eng.step([pe.StepEntry(s, (7 + t,), (0,)) for s in slots]).float().cpu()
        prompts = [p + [7 + t] for p in prompts]
        want = torch.stack([plain_float8_forward(pcfg, w, p)[-1] for p in prompts])
        assert float((step - want).norm() / want.norm()) < MODEL_TOL


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["A", "B", "E"])
def test_checkpoint(pe, tmp_path, name):
    """8-bit checkpoints: a bfloat16 run keeps what it can as it is stored, a float32 run computes with the numbers."""
    folder, cfg, wide = make_folder(tmp_path, TEST_CONFIGS[name], 4, pe)
    gen = torch.Generator().manual_seed(1)
    prompt = torch.randint(0, cfg["vocab_size"], (40,), generator=gen).tolist()
    exact = plain.forward_logits(cfg, wide, prompt)
    eng = pe.Engine(folder, dtype="float32", max_context_len=256, max_cache_tokens=64 * 8, max_batch=2)
    got = eng.step([pe.StepEntry(eng.alloc_slot(), prompt, tuple(range(40)))]).float().cpu()
    assert rel_err(got, exact) < 3e-5                         # the float32 run's usual bound
    eng = pe.Engine(folder, max_context_len=256, max_cache_tokens=64 * 8, max_batch=2)
    assert type(eng.model.blocks[0].mixer.o_proj) is pe.parts.float8.Float8Weight and type(eng.model.blocks[0].ffn.down) in (
        pe.parts.float8.Float8Weight, torch.Tensor)
    got = eng.step([pe.StepEntry(eng.alloc_slot(), prompt, tuple(range(40)))]).float().cpu()
    # its operands are e4m3 (or bfloat16): at most 2^-4 of a value off each, 2^-4 / sqrt(3) in the 2-norm, twice for the layers
    assert float((got - exact).norm() / exact.norm()) < 2 * 2.0 ** -4 / 3 ** 0.5


@pytest.mark.gpu
def test_generate(pe, tmp_path):
    """The whole loop with graphs: the same tokens as without, and a smaller model."""
    folder = str(tmp_path / "m")
    pe.write_random_model(folder, pe.Qwen3Config.from_dict(TEST_CONFIGS["E"]), seed=6)
    prompts = [[5, 17, 3], [9] * 70, [2]]
    runs = []
    for kw in (dict(), dict(enable_cuda_graph=False)):
        eng = pe.Engine(folder, weight_format="float8", max_context_len=256, max_cache_tokens=64 * 16, max_batch=4, **kw)
        runs.append([r.token_ids for r in eng.generate(prompts, pe.SamplingParams.greedy_params(max_tokens=8))])
    assert runs[0] == runs[1] and all(len(t) == 8 for t in runs[0])
    plain_eng = pe.Engine(folder, max_context_len=256, max_cache_tokens=64 * 16, max_batch=4)
    assert eng.model.weight_bytes() < 0.75 * plain_eng.model.weight_bytes()


@pytest.mark.gpu
@pytest.mark.parametrize("choice,n_identity,weight_on", [("softmax_all", 3, "output"), ("top_logits", 0, "input"), ("sigmoid_groups", 0, "output")])
@pytest.mark.parametrize("n", [1, 5, 300])
@pytest.mark.parametrize("stored", [False, True])
def test_routed_experts(pe, choice, n_identity, weight_on, n, stored):
    """The part against its formula with 8-bit operands, in 64 bits, with the choice that the part itself made."""
    from pytorch_engine_b200.parts.moe import RoutedExperts
    from pytorch_engine_b200.parts.runtime import Runtime

    f8 = pe.parts.float8
    rt = Runtime(DEV, BF16)
    rt.float8 = not stored
    hidden, inter, experts, top = 192, 128, 6, 2
    params = dict(hidden=hidden, n_experts=experts, n_identity=n_identity, top=top, intermediate=inter, choice=choice, weight_on=weight_on,
                  activation="silu")
    g = torch.Generator(device=DEV).manual_seed(n)
    weights = {}
    for name, decl in RoutedExperts.weight_decls(params).items():
        t = (torch.randn(decl.shape, generator=g, device=DEV) * 0.05).to(BF16)
        weights[name] = f8.Float8Weight.quantize(t) if stored and "." in name else t
    part = RoutedExperts(params, weights, rt)
    assert part.float8 and type(part.gate_up) is f8.Float8Weight
    kept = {}

    class Ctx:
        def buffer(self, name, shape, dtype):
            kept[name] = torch.empty(shape, dtype=dtype, device=DEV)
            return kept[name]

    x = (torch.randn(n, hidden, generator=g, device=DEV)).to(BF16)
    got = part.forward(x, Ctx()).to(torch.float64)
    rt.raise_on_status()
    chosen, weight = kept["moe.chosen"].cpu(), kept["moe.weight"].to(torch.float64).cpu()
    rows = f8.Float8Rows.quantize(x).dequantize(torch.float64)
    gate_up, down = part.gate_up.dequantize(torch.float64), part.down.dequantize(torch.float64)
    want = torch.zeros(n, hidden, dtype=torch.float64, device=DEV)
    for t in range(n):
        for j in range(top):
            e, s = int(chosen[t, j]), float(weight[t, j])
            if e >= experts:
                want[t] += s * x[t].to(torch.float64)
                continue
            a, u = (gate_up[e] @ rows[t] * (s if weight_on == "input" else 1.0)).chunk(2)
            h = (a * torch.sigmoid(a) * u).to(BF16)
            y = down[e] @ f8.Float8Rows.quantize(h[None]).dequantize(torch.float64)[0]
            want[t] += y if weight_on == "input" else s * y
    # an expert's output and the sum are rounded to bfloat16; an activation that falls on the other side of a rounding is a step
    # of e4m3 off, 2^-3 of its value at the most, one in a thousand of them (their sums differ by 2^-20, its roundings' span is 2^-8)
    assert float((got - want).norm() / want.norm()) < 2.0 ** -8 + 2.0 ** -8 + 2.0 ** -3 * 1e-3 ** 0.5


@pytest.mark.gpu
def test_command_line(pe, capsys):
    from pytorch_engine_b200 import cli

    assert cli.main(["--random", "tiny_b", "--prompt-ids", "1,2,3", "--max-tokens", "4", "--temperature", "0", "--weights", "float8", "--json"]) == 0
    assert len(json.loads(capsys.readouterr().out.strip().splitlines()[-1])["token_ids"]) <= 4
