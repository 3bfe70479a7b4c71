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
