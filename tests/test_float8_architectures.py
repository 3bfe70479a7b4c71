"""8-bit checkpoints and engines that quantise, for the models of every architecture: which parts keep 8-bit matrices, what a float32
run computes with, and that a bfloat16 run's 8-bit path leaves out nothing that the other one does."""
import importlib

import pytest
import torch

from conftest import TEST_CONFIGS, rel_err

E4M3 = torch.float8_e4m3fn
DEV = "cuda:0"
BF16 = torch.bfloat16
F32 = torch.float32
PLAIN = {"bobasun": "BobasunConfig", "burinex": "BurinexConfig", "lunadra": "LunadraConfig", "vabelorn": "VabelornConfig",
         "vemepel": "VemepelConfig", "zonevik": "ZonevikConfig"}
MODELS = [("qwen3", k) for k in "ABCDE"] + [("bobasun", k) for k in "ABCDE"] + [("burinex", k) for k in "ABCD"] + [
    ("lunadra", k) for k in "AB"] + [("vabelorn", k) for k in "PQR"] + [("vemepel", k) for k in "ABC"] + [("zonevik", k) for k in "ABCD"]


def describe(pe, arch, key):
    """(configuration, its plan, its plain dict, the plain module)"""
    if arch == "qwen3":
        d = TEST_CONFIGS[key]
        cfg = pe.Qwen3Config.from_dict(d)
        module = importlib.import_module("plain_qwen3")
    else:
        d = importlib.import_module(f"test_{arch}_gpu").CONFIGS[key]
        cfg = getattr(pe, PLAIN[arch]).from_dict(d)
        module = importlib.import_module(f"plain_{arch}")
    return cfg, pe.config.registry.architecture(cfg.architecture).plan(cfg), d, module


def weights_of(pe, arch, key, plan, d, module):
    if arch != "qwen3":
        return module.random_weights(d, 41)
    g = torch.Generator().manual_seed(41)
    return {name: (1.0 if decl.role == "norm" else 0.0) + 0.1 * torch.randn(decl.shape, generator=g) for name, decl in pe.weights.loader.expected_tensors(plan).items()}


def blocks(n):
    return -(-n // 128)


def stored(pe, decls, weights):
    """The weights with every matrix in 8 bits, with scales that are no powers of two; and the numbers that they stand for."""
    f8 = pe.parts.float8
    out, numbers = {}, {}
    for name, t in weights.items():
        out[name] = numbers[name] = t
        if name in decls and decls[name].role == "matrix" and t.dim() == 2:
            n, k = t.shape
            pad = torch.zeros(blocks(n) * 128, blocks(k) * 128, dtype=torch.float64)
            pad[:n, :k] = t
            s = (pad.view(blocks(n), 128, blocks(k), 128).abs().amax((1, 3)).clamp(min=1e-6) / 437.0).to(F32)
            whole = s.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
            v = (t.to(F32) / whole).clamp(-448, 448).to(E4M3)
            out[name] = f8.Float8Weight(v, s)
            numbers[name] = v.to(F32) * whole
    return out, numbers


def tensors_of(part):
    return {k: v for k, v in vars(part).items() if isinstance(v, torch.Tensor)}


# ---- on the CPU ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("arch,key", MODELS)
def test_a_float32_model_holds_the_numbers(pe, arch, key):
    """Every tensor of every part is what it is made from the numbers that the 8-bit matrices stand for, to the bit."""
    from pytorch_engine_b200.engine.model import DecoderModel
    from pytorch_engine_b200.parts.runtime import Runtime

    cfg, plan, d, module = describe(pe, arch, key)
    decls = pe.weights.loader.expected_tensors(plan)
    eight, numbers = stored(pe, decls, weights_of(pe, arch, key, plan, d, module))
    got, want = (DecoderModel(plan, w, Runtime("cpu", F32)) for w in (eight, numbers))
    pairs = [(got.embedding, want.embedding), (got.final_norm, want.final_norm), (got.head, want.head)]
    pairs += [(a[n], b[n]) for a, b in zip(got.block_parts, want.block_parts) for n in b]
    for a, b in pairs:
        a, b = tensors_of(a), tensors_of(b)
        assert set(a) == set(b)
        for n in b:
            assert a[n].dtype == b[n].dtype and torch.equal(a[n], b[n]), n


class OfWidth8:
    """What ``projection`` asks of a runtime, with 8-bit products."""
    device, dtype, float8 = torch.device("cpu"), BF16, False

    def takes_float8(self):
        return True


@pytest.mark.parametrize("rows", [(256, 128, 128, 6), (256, 128, 128, 8), (128, 128, 128, 1), (128, 128, 121), (127,), (128, 125)])
@pytest.mark.parametrize("k", [54, 144])
def test_a_padded_projection_stays_in_8_bits(pe, rows, k):
    """Stored matrices that end with a block of rows are put under each other as they are, with zeros behind the last."""
    from pytorch_engine_b200.parts.linear import projection

    f8 = pe.parts.float8
    g = torch.Generator().manual_seed(sum(rows))
    mats = [f8.Float8Weight(torch.randn(n, k, generator=g).mul(40).clamp(-448, 448).to(E4M3), torch.rand(blocks(n), blocks(k), generator=g)) for n in rows]
    got = projection(OfWidth8(), mats, 8)
    assert type(got) is f8.Float8Weight and got.shape == (-(-sum(rows) // 8) * 8, k)
    assert torch.equal(got.dequantize()[:sum(rows)], torch.cat([m.dequantize() for m in mats]))
    assert bool((got.dequantize()[sum(rows):] == 0).all()) and got.values.stride(0) % 16 == 0


def test_rows_that_end_inside_a_block(pe):
    """Then the matrices' numbers are used; and zeros are not put where they would begin a block."""
    from pytorch_engine_b200.parts.linear import projection

    f8 = pe.parts.float8
    mats = [f8.Float8Weight(torch.ones(n, 40).to(E4M3), torch.full((blocks(n), 1), 0.3)) for n in (100, 30)]
    got = projection(OfWidth8(), mats, 8)
    assert got.dtype == BF16 and got.shape == (136, 40)
    assert torch.equal(got[:130], torch.cat([m.dequantize(BF16) for m in mats])) and bool((got[130:] == 0).all())
    with pytest.raises(ValueError):
        f8.Float8Weight(torch.ones(128, 40).to(E4M3), torch.ones(1, 1)).with_zero_rows(1)


def test_weights_that_are_parameters(pe):
    """``torch.nn.Parameter``s are tensors: an attention of 16-bit weights joins a chain of products all the same."""
    from pytorch_engine_b200.engine.model import DecoderModel
    from pytorch_engine_b200.parts.runtime import Runtime

    cfg, plan, d, module = describe(pe, "qwen3", "D")
    weights = {n: t.to(BF16) for n, t in weights_of(pe, "qwen3", "D", plan, d, module).items()}
    models = [DecoderModel(plan, {n: kind(t) for n, t in weights.items()}, Runtime("cpu", BF16))
              for kind in (torch.clone, lambda t: torch.nn.Parameter(t, requires_grad=False))]
    assert type(models[1].blocks[0].mixer.o_proj) is torch.nn.Parameter
    assert [[b.mixer.chains(), b.ffn.chains()] for b in models[1].blocks] == [[b.mixer.chains(), b.ffn.chains()] for b in models[0].blocks]
    assert models[0].blocks[0].mixer.chains()


# ---- on the GPU ------------------------------------------------------------------------------------------------------------
def prompt_of(d, n, seed=3):
    vocab = d.get("vocab") or d["vocab_size"]
    return torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def on_gpu(weights):
    return {n: t.to(DEV) for n, t in weights.items()}


def run(pe, eng, prompts, more=2):
    """Logits of whole prompts, then of ``more`` single tokens of each: two tensors."""
    slots = [eng.alloc_slot() for _ in prompts]
    first = eng.step([pe.StepEntry(s, p, tuple(range(len(p)))) for s, p in zip(slots, prompts)]).float().cpu()
    steps = [eng.step([pe.StepEntry(s, (5 + t,), (0,)) for s in slots]).float().cpu() for t in range(more)]
    for s in slots:
        eng.free_slot(s)
    return first, torch.stack(steps)


@pytest.mark.gpu
@pytest.mark.parametrize("arch,key", [m for m in MODELS if m[0] != "qwen3"])
def test_a_float32_run_of_8_bit_matrices(pe, arch, key):
    """Against the plain model of the numbers, within the bound of that architecture's float32 runs."""
    cfg, plan, d, module = describe(pe, arch, key)
    eight, numbers = stored(pe, pe.weights.loader.expected_tensors(plan), weights_of(pe, arch, key, plan, d, module))
    eng = pe.Engine(None, config=cfg, weights=on_gpu(eight), dtype="float32", max_context_len=128, max_cache_tokens=64 * 8, max_batch=2)
    toks = prompt_of(d, 40)
    got = eng.step([pe.StepEntry(eng.alloc_slot(), toks, tuple(range(40)))]).float().cpu()
    assert rel_err(got, module.forward(d, numbers, toks).float()) < 3e-5


def eight_bit_parts(eng):
    """(kind, attribute) of the matrices that a model's parts keep in 8 bits, and of the others that could be."""
    f8 = type(eng).__module__.split(".")[0]
    Float8Weight = importlib.import_module(f8 + ".parts.float8").Float8Weight
    kept, other = [], []
    for built in eng.model.block_parts:
        for part in built.values():
            names = {"GQAttention": ("qkv", "o_proj"), "SwiGLU": ("gate_up", "down"), "RoutedExperts": ("gate_up", "down")}
            for n in names.get(type(part).__name__, ()):
                if type(part).__name__ == "RoutedExperts" and not part.n_experts:
                    continue
                (kept if type(getattr(part, n)) is Float8Weight else other).append((type(part).__name__, n))
    return kept, other


@pytest.mark.gpu
@pytest.mark.parametrize("arch,key", MODELS)
def test_every_part_that_can_quantizes(pe, arch, key):
    """``weight_format="float8"``: attention's, gated feed-forwards' and experts' matrices, in every arrangement; prompts and single
    tokens run, from graphs the same as without."""
    cfg, plan, d, module = describe(pe, arch, key)
    weights = on_gpu(weights_of(pe, arch, key, plan, d, module))
    prompts = [prompt_of(d, n, n) for n in (1, 9, 70)]
    got = []
    for graphs in (True, False):
        eng = pe.Engine(None, config=cfg, weights=weights, weight_format="float8", max_context_len=128, max_cache_tokens=64 * 12, max_batch=4,
                        enable_cuda_graph=graphs)
        kept, other = eight_bit_parts(eng)
        kinds = {s.kind for b in plan.blocks for _, s in b.parts.values()}
        assert not other and bool(kept) == bool(kinds & {"attention", "swiglu", "routed_experts"})
        report = eng.memory_report()
        assert (report["float8_mib"] > 0.0) == bool(kept) and report["float8_mib"] < report["weights_mib"]
        got.append(run(pe, eng, prompts))
    plain = pe.Engine(None, config=cfg, weights=weights, max_context_len=64, max_cache_tokens=64, max_batch=1)
    assert plain.memory_report()["float8_mib"] == 0.0
    assert all(bool(torch.isfinite(t).all()) for pair in got for t in pair)
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


@pytest.mark.gpu
@pytest.mark.parametrize("arch,key", [m for m in MODELS if m[0] in ("qwen3", "bobasun", "vabelorn")])
def test_as_a_bfloat16_run_with_8_bit_operands(pe, arch, key):
    """The same model in bfloat16, all its products taken over by one that rounds both operands to 8 bits and computes in float32:
    biases, gates, norms and the order of a block are those of the 16-bit path.

    The runs' activations differ by bfloat16's roundings, 2^-8 of a value, so up to 2 * 2^-8 / 2^-3 = 1/16 of a product's inputs fall
    on different sides of an e4m3 rounding and differ by its step, 2^-3 of a value at the most: 3.1 % in the 2-norm.  A sublayer is
    two products, a layer two sublayers: twice that of the stream if nothing else were in it, and the layers' errors add up like
    random ones."""
    f8 = pe.parts.float8
    cfg, plan, d, module = describe(pe, arch, key)
    weights = on_gpu(weights_of(pe, arch, key, plan, d, module))
    prompts = [prompt_of(d, n, n) for n in (1, 9, 70)]
    kw = dict(config=cfg, weights=weights, max_context_len=128, max_cache_tokens=64 * 12, max_batch=4, enable_cuda_graph=False)
    got = run(pe, pe.Engine(None, weight_format="float8", **kw), prompts)
    plain = pe.Engine(None, **kw)
    numbers = {}
    for built in plain.model.block_parts:
        for part in built.values():
            for n in {"GQAttention": ("qkv", "o_proj"), "SwiGLU": ("gate_up", "down")}.get(type(part).__name__, ()):
                w = getattr(part, n)
                numbers[w.data_ptr()] = f8.Float8Weight.quantize(w).dequantize()

    def product(x, weight, out, out_dtype):
        w = numbers.get(weight.data_ptr())
        if w is None:
            return None
        y = f8.Float8Rows.quantize(x).dequantize() @ w.t()
        return y.to(out_dtype or x.dtype) if out is None else out.copy_(y)

    rt = plain.runtime
    rt.gemm_backend, rt.own_small_gemm, rt.own_large_gemm = product, False, False
    want = run(pe, plain, prompts)
    bound = 0.0625 * len(plan.blocks) ** 0.5
    for a, b in zip(got, want):
        assert float((a - b).norm() / b.norm()) < bound
