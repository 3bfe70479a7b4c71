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
