"""Weights that go into a product right behind what writes them: conversions, copies, and copies by the caller with
``settle_weights`` behind them, eager and in graphs, with other contents every time."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32
E4M3 = torch.float8_e4m3fn
N, K = 1024, 4096


def matrices(g, n):
    return [torch.randn(N, K, generator=g, device=DEV).to(BF16) for _ in range(n)]


def eight(pe, mats):
    """Their 8-bit forms, long written."""
    out = [pe.parts.float8.Float8Weight.quantize(m) for m in mats]
    torch.cuda.synchronize()
    return out


def make(pe, how, mats, parts):
    """(the weight that was written last, the values it has to have, its scales)"""
    f8 = pe.parts.float8
    if how == "quantize":
        w = f8.Float8Weight.quantize(mats[0])
        return w, parts[0].values, parts[0].scales
    if how == "cat_rows":
        w = f8.Float8Weight.cat_rows(parts)
        return w, torch.cat([p.values.view(torch.uint8) for p in parts]).view(E4M3), torch.cat([p.scales for p in parts])
    if how == "stack":
        w = f8.Float8Weight.stack(parts)[len(parts) - 1]
        return w, parts[-1].values, parts[-1].scales
    if how == "to":                                       # rows off the 16-byte boundaries, which are copied
        odd = torch.empty(N, K + 8, dtype=E4M3, device=DEV)[:, :K]
        odd.copy_(parts[0].values)
        w = f8.Float8Weight(odd, parts[0].scales, True).to(DEV)
        return w, parts[0].values, parts[0].scales
    values, scales = torch.empty(N, K, dtype=E4M3, device=DEV), torch.empty_like(parts[0].scales)
    scales.copy_(parts[0].scales)
    values.copy_(parts[0].values)
    pe.kernels.ops.settle_weights(values)
    return f8.Float8Weight(values, scales), parts[0].values, parts[0].scales


@pytest.mark.parametrize("how", ["quantize", "cat_rows", "stack", "to", "settle_weights"])
@pytest.mark.parametrize("m", [1, 8, 40])
def test_right_behind(pe, how, m):
    ops, f8, st = pe.kernels.ops, pe.parts.float8, torch.zeros(4, dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(m)
    rows = f8.Float8Rows.quantize(torch.randn(m, K, generator=g, device=DEV).to(BF16))
    for turn in range(8):
        mats = matrices(g, 2)
        parts = eight(pe, mats)
        w, values, scales = make(pe, how, mats, parts)
        out = torch.empty(m, w.shape[0], dtype=F32, device=DEV)
        ops.gemm_fp8(rows.values, rows.scales, w.values, w.scales, out, st)
        torch.cuda.synchronize()
        want = torch.empty_like(out)
        ops.gemm_fp8(rows.values, rows.scales, values, scales, want, st)
        assert torch.equal(out, want)
        del w
    assert st.tolist()[0] == 0


@pytest.mark.parametrize("how", ["quantize", "settle_weights"])
def test_in_a_graph(pe, how):
    """Written and used in every replay."""
    ops, f8, st = pe.kernels.ops, pe.parts.float8, torch.zeros(4, dtype=torch.int32, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(7)
    rows = f8.Float8Rows.quantize(torch.randn(4, K, generator=g, device=DEV).to(BF16))
    src = matrices(g, 1)
    into = eight(pe, src)
    out = torch.empty(4, N, dtype=F32, device=DEV)

    def step():
        w, _, _ = make(pe, how, src, into)
        ops.gemm_fp8(rows.values, rows.scales, w.values, w.scales, out, st)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for _ in range(8):
        now = matrices(g, 1)
        src[0].copy_(now[0])
        fresh = eight(pe, now)[0]
        into[0].values.copy_(fresh.values)
        into[0].scales.copy_(fresh.scales)
        graph.replay()
        torch.cuda.synchronize()
        want = torch.empty_like(out)
        ops.gemm_fp8(rows.values, rows.scales, fresh.values, fresh.scales, want, st)
        assert torch.equal(out, want)
    assert st.tolist()[0] == 0


def test_settling_waits_and_counts(pe):
    """It is one launch, and leaves its weight and the device alone."""
    w = torch.arange(64, device=DEV, dtype=F32)
    before, device = pe.kernels.ops.launch_count(), torch.cuda.current_device()
    pe.kernels.ops.settle_weights(w)
    assert pe.kernels.ops.launch_count() == before + 1 and torch.cuda.current_device() == device
    assert torch.equal(w.cpu(), torch.arange(64, dtype=F32))
    pe.kernels.ops.settle_weights(torch.zeros(3))
    assert pe.kernels.ops.launch_count() == before + 1
