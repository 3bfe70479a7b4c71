"""Files with 8-bit tensors that are no 8-bit matrices: refused with one error that names them, before any of them is read."""
import os

import pytest
import torch

from conftest import TEST_CONFIGS
from test_bobasun_gpu import CONFIGS as BOBASUN
from test_lunadra_gpu import CONFIGS as LUNADRA

E4M3 = torch.float8_e4m3fn


def written(pe, tmp_path, cfg):
    from safetensors.torch import load_file

    folder = str(tmp_path / "m")
    pe.write_random_model(folder, cfg, seed=1)
    plan = pe.config.registry.architecture(cfg.architecture).plan(cfg)
    # copies: the file that they are mapped from is written again
    return folder, plan, {n: t.clone() for n, t in load_file(os.path.join(folder, "model.safetensors")).items()}


def refused(pe, folder, plan, tensors):
    from safetensors.torch import save_file

    save_file({n: t.contiguous() for n, t in tensors.items()}, os.path.join(folder, "model.safetensors"))
    with pytest.raises(pe.WeightError) as e:
        pe.load_weights(folder, plan)
    return e.value


@pytest.mark.parametrize("arch", ["bobasun", "lunadra"])
def test_vectors_and_stacks(pe, tmp_path, arch):
    """Every tensor of another rank than two that is declared like a matrix, with a scale beside it and without."""
    cfg = pe.BobasunConfig.from_dict(BOBASUN["A"]) if arch == "bobasun" else pe.LunadraConfig.from_dict(LUNADRA["A"])
    folder, plan, whole = written(pe, tmp_path, cfg)
    names = [n for n, d in pe.weights.expected_tensors(plan).items() if d.role == "matrix" and len(d.shape) != 2]
    assert names
    for name in names[:6]:
        eight = {**whole, name: whole[name].to(E4M3)}
        assert [b[0] for b in refused(pe, folder, plan, eight).bad_dtype] == [name]
        scale = torch.ones([-(-d // 128) for d in whole[name].shape])
        e = refused(pe, folder, plan, {**eight, name + "_scale_inv": scale})
        assert [b[0] for b in e.bad_dtype] == [name] and e.unexpected == [name + "_scale_inv"]


def test_a_matrix_stored_as_something_else(pe, tmp_path):
    cfg = pe.Qwen3Config.from_dict(TEST_CONFIGS["A"])
    folder, plan, whole = written(pe, tmp_path, cfg)
    name = "model.layers.0.mlp.up_proj.weight"
    n, k = whole[name].shape
    for shape in ((n * k,), (1, n, k)):
        e = refused(pe, folder, plan, {**whole, name: whole[name].to(E4M3).reshape(shape), name + "_scale_inv": torch.ones(1, 1)})
        assert [w[0] for w in e.wrong_shape] == [name] and [b[0] for b in e.bad_dtype] == [name]


def test_a_duplicate_in_8_bits(pe, tmp_path):
    """A tied model whose file stores the head too, one or both in 8 bits."""
    cfg = pe.Qwen3Config.from_dict(TEST_CONFIGS["A"])
    folder, plan, whole = written(pe, tmp_path, cfg)
    name, head = "model.embed_tokens.weight", "lm_head.weight"
    eight = whole[name].to(E4M3)
    e = refused(pe, folder, plan, {**whole, name: eight, head: eight.clone()})
    assert [b[0] for b in e.bad_dtype] == [name] and e.conflicting == [(head, name)]
    assert refused(pe, folder, plan, {**whole, head: eight}).conflicting == [(head, name)]


# ---- what the command line and a checkpoint lead to ------------------------------------------------------------------------
@pytest.mark.parametrize("option,want", [([], None), (["--weights", "stored"], None), (["--weights", "float8"], "float8")])
def test_the_command_line_hands_the_format_on(pe, monkeypatch, option, want):
    from importlib import import_module

    cli, seen = import_module("pytorch-engine_b200.cli"), {}

    class Stop(Exception):
        pass

    class Engine:
        @staticmethod
        def from_random(cfg, seed, **kw):
            seen.update(kw)
            raise Stop

    monkeypatch.setattr(pe, "Engine", Engine)
    with pytest.raises(Stop):
        cli.main(["--random", "tiny_b", "--prompt-ids", "1,2,3", *option])
    assert seen["weight_format"] == want


@pytest.mark.gpu
@pytest.mark.parametrize("key", ["A", "B", "D", "E"])
def test_what_a_checkpoint_keeps(pe, tmp_path, key):
    """A projection stays in 8 bits where each of its stored matrices but the last ends with a block of 128 rows; a feed-forward
    where both of its do."""
    from test_float8_model import make_folder

    folder, cfg, _ = make_folder(tmp_path, TEST_CONFIGS[key], 4, pe)
    d = cfg["head_dim"]
    whole = lambda n: n % 128 == 0
    wants = {"qkv": whole(cfg["num_attention_heads"] * d) and whole(cfg["num_key_value_heads"] * d), "o_proj": True,
             "gate_up": whole(cfg["intermediate_size"]), "down": whole(cfg["intermediate_size"])}
    eng = pe.Engine(folder, max_context_len=128, max_cache_tokens=64 * 4, max_batch=1)
    for block in eng.model.blocks:
        for part, n in ((block.mixer, "qkv"), (block.mixer, "o_proj"), (block.ffn, "gate_up"), (block.ffn, "down")):
            assert (type(getattr(part, n)) is pe.parts.float8.Float8Weight) == wants[n], n


@pytest.mark.gpu
def test_cpu_tensors_are_refused(pe):
    """On a machine that has the kernels: by name, before anything is launched."""
    ops, dev = pe.kernels.ops, "cuda:0"
    pe.kernels.library()
    st = torch.zeros(4, dtype=torch.int32, device=dev)
    x, w = torch.zeros(2, 128, dtype=torch.bfloat16), torch.zeros(64, 128).to(E4M3)
    s, xs, out = torch.ones(1, 1), torch.ones(1, 2), torch.zeros(2, 64, dtype=torch.bfloat16)
    calls = [lambda: ops.linear_fp8(x, w, s, out, st), lambda: ops.linear_fp8(x, w.to(dev), s.to(dev), out.to(dev), st),
             lambda: ops.linear_fp8(x.to(dev), w.to(dev), s, out.to(dev), st), lambda: ops.linear_fp8(x.to(dev), w.to(dev), s.to(dev), out, st),
             lambda: ops.linear_fp8(x.to(dev), w.to(dev), s.to(dev), out.to(dev), st.cpu()),
             lambda: ops.gemm_fp8(x.to(E4M3), xs, w, s, out, st), lambda: ops.gemm_fp8(x.to(E4M3).to(dev), xs, w.to(dev), s.to(dev), out.to(dev), st),
             lambda: ops.quantize_weight_fp8(torch.zeros(64, 128), w, s), lambda: pe.parts.float8.Float8Weight.quantize(torch.zeros(64, 128)),
             lambda: ops.quantize_rows_fp8(x, x.to(E4M3), xs), lambda: pe.parts.float8.Float8Rows.quantize(x),
             lambda: ops.rmsnorm_residual_fp8(torch.zeros(2, 128), None, torch.ones(128), x.to(E4M3), xs, 1e-6)]
    for i, call in enumerate(calls):
        with pytest.raises(pe.kernels.KernelError):
            call()
            pytest.fail(f"call {i} was not refused")
    assert st.tolist()[0] == 0
