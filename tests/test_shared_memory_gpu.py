"""Launches whose dynamic shared memory, with the kernel's own static arrays, comes to the 48 KB that need no asking and just beyond.

A launch that has not asked is refused only until a larger one has: each kernel's first call in a process is made here, in a process
of its own (this file run as a program), with exactly the sizes that lie in between.  Results are held against the formulas in 64 bits.
"""
import json
import os
import subprocess
import sys

import pytest
import torch

DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8}        # a rounding is off by half a step


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def experts(ops, g, dtype, out_dtype):
    """moe_rows_gemm: 8 rows of 1,536 floats are 48 KB."""
    k, n = 1536, 40
    x, w = randn(g, 5, k).to(dtype), randn(g, 2, n, k).to(dtype)
    out = torch.empty(5, n, dtype=out_dtype, device=DEV)
    ops.moe_rows_gemm(x, None, torch.tensor([0, 2, 5], dtype=torch.int32, device=DEV), 2, 5, w, out)
    x64, w64 = x.to(F64), w.to(F64)
    want = torch.cat([x64[:2] @ w64[0].T, x64[2:] @ w64[1].T])
    size = torch.cat([x64[:2].abs() @ w64[0].T.abs(), x64[2:].abs() @ w64[1].T.abs()])
    return out, want, (k + 1) * 2.0 ** -24 * size + STEP[out_dtype] * want.abs()       # k products added in any order


CASES = {
    "experts float32": lambda ops, g: experts(ops, g, F32, F32),
    "experts bfloat16": lambda ops, g: experts(ops, g, BF16, BF16),
    "experts bfloat16 to float32": lambda ops, g: experts(ops, g, BF16, F32),
}


def main():
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    import importlib

    pe = importlib.import_module("pytorch-engine_b200")
    pe.kernels.library()
    found = {}
    for i, (name, case) in enumerate(CASES.items()):
        try:
            got, want, bound = case(pe.kernels.ops, torch.Generator(device=DEV).manual_seed(i))
            found[name] = float(((got.to(F64) - want).abs() / bound).max())
        except pe.kernels.KernelError as e:
            found[name] = str(e)
    print(json.dumps(found))


@pytest.fixture(scope="module")
def found():
    run = subprocess.run([sys.executable, os.path.abspath(__file__)], capture_output=True, text=True, timeout=600)
    assert run.returncode == 0, run.stderr[-2000:]
    return json.loads(run.stdout.strip().splitlines()[-1])


@pytest.mark.gpu
@pytest.mark.parametrize("name", CASES)
def test_first_call(found, name):
    assert not isinstance(found[name], str), found[name]
    assert found[name] <= 1.0


if __name__ == "__main__":
    main()
