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


def norm_bound(width, x64, w64, want, dtype):
    """A layer norm's: the mean is off by width * 2^-24 of the mean magnitude, so is every difference; the squares' sum by
    (width + 4) * 2^-24 of itself and by the differences' error; root, quotient, two products: 8 more roundings."""
    mean = x64.mean(1, keepdim=True)
    sigma = ((x64 - mean) ** 2).mean(1, keepdim=True).sqrt()
    e = (width + 2) * 2.0 ** -24 * x64.abs().mean(1, keepdim=True)
    return (2 * e / sigma + 8 * 2.0 ** -24 + (width + 4) * 2.0 ** -24) * (want.abs() + w64.abs()) + STEP[dtype] * want.abs()


def layer_norm(ops, g, dtype, width):
    x, w = randn(g, 3, width).to(dtype), randn(g, width)
    out = torch.empty_like(x)
    ops.layernorm(x, w, out, 1e-5)
    x64, w64 = x.to(F64), w.to(F64)
    d = x64 - x64.mean(1, keepdim=True)
    want = d / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5) * w64
    return out, want, norm_bound(width, x64, w64, want, dtype)


def streams(ops, g, dtype, s, width):
    """stream_mix: a row, and with nine streams the mix beside it."""
    x, w, read = randn(g, 2, s, width), randn(g, width), torch.rand(s, generator=g, device=DEV) + 0.5
    y, write = randn(g, 2, width).to(dtype), randn(g, s)
    mix = randn(g, s, s)
    out = torch.empty(2, width, dtype=dtype, device=DEV)
    before, y64 = x.to(F64), y.to(F64)
    ops.stream_mix(None, x, y, None, mix, write, read, "layer", w, 1e-5, out)
    now = torch.einsum("it,niw->ntw", mix.to(F64), before) + write.to(F64)[None, :, None] * y64[:, None]
    row = torch.einsum("i,niw->nw", read.to(F64), now)
    d = row - row.mean(1, keepdim=True)
    sigma = torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5)
    want = d / sigma * w.to(F64)
    # the row itself: s sums of s + 1 terms, each term a product
    size = torch.einsum("i,niw->nw", read.to(F64).abs(), torch.einsum("it,niw->ntw", mix.to(F64).abs(), before.abs())
                        + write.to(F64).abs()[None, :, None] * y64.abs()[:, None])
    bound = norm_bound(width, row, w.to(F64), want, dtype) + (2 * s + 4) * 2.0 ** -24 * size / sigma * w.to(F64).abs()
    return out, want, bound


def state_space(ops, g, n, dv, chunk):
    """ssd_recurrence: tokens of 32 staged at a time, beside their steps and decays."""
    heads, t = 2, 70
    xbc, dt = randn(g, t, heads * dv + 2 * n), randn(g, t, heads)
    bias, A_log, D = randn(g, heads), randn(g, heads) * 0.3, randn(g, heads)
    y, S = torch.empty(t, heads * dv, device=DEV), torch.zeros(1, heads, n, dv, device=DEV)
    chunks = -(-t // chunk) if chunk else 1
    scratch = torch.empty(ops.ssd_scratch_floats(1, heads, n, dv, chunks), device=DEV) if chunk else None
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
    status = i32(0, 0, 0, 0)
    ops.ssd_recurrence(xbc, dt, bias, A_log, D, y, S, i32(0), i32(0, t), 1, t, heads, 1, n, dv, status, chunk, chunks, scratch)
    assert status.tolist()[0] == 0
    x64, step = xbc.to(F64), torch.nn.functional.softplus(dt.to(F64) + bias.to(F64))
    B, C = x64[:, heads * dv:heads * dv + n], x64[:, heads * dv + n:]
    want, size = torch.zeros(t, heads * dv, dtype=F64, device=DEV), torch.zeros(t, heads * dv, dtype=F64, device=DEV)
    for h in range(heads):
        at = slice(h * dv, (h + 1) * dv)
        s = torch.zeros(n, dv, dtype=F64, device=DEV)
        a = s.clone()
        for i in range(t):
            f = torch.exp(-torch.exp(A_log[h].to(F64)) * step[i, h])
            s = f * s + step[i, h] * torch.outer(B[i], x64[i, at])
            a = f * a + step[i, h] * torch.outer(B[i].abs(), x64[i, at].abs())
            want[i, at] = s.T @ C[i] + D[h].to(F64) * x64[i, at]
            size[i, at] = a.T @ C[i].abs() + (D[h].to(F64) * x64[i, at]).abs()
    # a state's term has gone through at most t steps of 4 roundings (decay and step are functions good to 2^-20 of their value,
    # a decay's through its exponent of at most some 16), the output is a sum of n + 1
    return y, want, (t * (4 * 2.0 ** -24 + 16 * 2.0 ** -20) + (n + 2) * 2.0 ** -24) * size


CASES = {
    "experts float32": lambda ops, g: experts(ops, g, F32, F32),
    "experts bfloat16": lambda ops, g: experts(ops, g, BF16, BF16),
    "experts bfloat16 to float32": lambda ops, g: experts(ops, g, BF16, F32),
    "layer norm 12257 float32": lambda ops, g: layer_norm(ops, g, F32, 12257),
    "layer norm 12288 bfloat16": lambda ops, g: layer_norm(ops, g, BF16, 12288),
    "one stream 12260 bfloat16": lambda ops, g: streams(ops, g, BF16, 1, 12260),
    "two streams 12288 float32": lambda ops, g: streams(ops, g, F32, 2, 12288),
    "nine streams 12189 float32": lambda ops, g: streams(ops, g, F32, 9, 12189),
    "state space 64 x 240": lambda ops, g: state_space(ops, g, 64, 240, 0),
    "state space 64 x 240 in chunks": lambda ops, g: state_space(ops, g, 64, 240, 32),
    "state space 16 x 352": lambda ops, g: state_space(ops, g, 16, 352, 0),
    "state space 16 x 352 in chunks": lambda ops, g: state_space(ops, g, 16, 352, 32),
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
