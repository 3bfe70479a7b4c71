"""Arguments of the 8-bit operators that would lead a kernel beyond its tensors: refused on the host.  What the checks themselves
say is tried on CPU tensors; the calls are made on a GPU, none of which launches anything."""
import pytest
import torch

E4M3 = torch.float8_e4m3fn
BF16, F32 = torch.bfloat16, torch.float32
DEV = "cuda:0"


def test_scales_that_share_memory(pe):
    """Rows of scales (one for a block of features) lie at least as far apart as there are rows."""
    ld, KernelError = pe.kernels.ops._fp8_scales_ld, pe.kernels.KernelError
    for good, want in ((torch.ones(3, 4), 4), (torch.ones(3, 9)[:, :4], 9), (torch.ones(1, 4), 4), (torch.ones(3, 1), 1), (torch.ones(3, 7)[:, :1], 7),
                       (torch.ones(1, 4).expand(1, 4), 4), (torch.ones(4, 1).t(), 4), (torch.ones(3, 0), 0), (torch.ones(1, 1).expand(1, 1), 1)):
        assert ld(good, *good.shape, "scales") >= want or good.shape[1] == 0
    for bad in (torch.ones(1, 4).expand(3, 4), torch.ones(1, 1).expand(3, 1), torch.ones(12).as_strided((3, 4), (2, 1)), torch.ones(4, 3).t(),
                torch.ones(1, 1).expand(3, 4)):
        with pytest.raises(KernelError):
            ld(bad, *bad.shape, "scales")


@pytest.mark.gpu
def test_calls_with_such_scales(pe):
    ops, f8, KernelError = pe.kernels.ops, pe.parts.float8, pe.kernels.KernelError
    st = torch.zeros(4, dtype=torch.int32, device=DEV)
    x = torch.ones(70, 384, dtype=BF16, device=DEV)
    r, w = f8.Float8Rows.quantize(x), f8.Float8Weight.quantize(torch.ones(128, 384, device=DEV))
    shared = torch.ones(1, 70, device=DEV).expand(3, 70)
    out = torch.empty(70, 128, dtype=BF16, device=DEV)
    before = ops.launch_count()
    for call in (lambda: ops.gemm_fp8(r.values, shared, w.values, w.scales, out, st), lambda: ops.quantize_rows_fp8(x, r.values, shared),
                 lambda: ops.rmsnorm_residual_fp8(x.float(), None, torch.ones(384, device=DEV), r.values, shared, 1e-6),
                 lambda: ops.gemm_fp8(r.values[:1], shared[:, :1], w.values, w.scales, out[:1], st)):
        with pytest.raises(KernelError):
            call()
    assert ops.launch_count() == before


@pytest.mark.gpu
def test_a_status_word_or_bias_elsewhere(pe):
    """Both are written or read by the kernels: they lie where the kernels run."""
    ops, f8, KernelError = pe.kernels.ops, pe.parts.float8, pe.kernels.KernelError
    st, there = torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros(4, dtype=torch.int32)
    x = torch.ones(4, 256, dtype=BF16, device=DEV)
    r, w = f8.Float8Rows.quantize(x), f8.Float8Weight.quantize(torch.ones(256, 256, device=DEV))
    pick = torch.zeros(4, dtype=torch.int32, device=DEV)
    out = torch.empty(4, 128, dtype=BF16, device=DEV)
    glu = ("silu", 0.0, 1.0, torch.zeros(256))
    before = ops.launch_count()
    for call in (lambda: ops.quantize_rows_fp8(x, r.values, r.scales, pick, None, there), lambda: ops.new_rows_fp8(x, pick, None, there),
                 lambda: ops.linear_fp8(x, w.values, w.scales, out, there, ()), lambda: ops.linear_fp8(x, w.values, w.scales, out, st, glu),
                 lambda: ops.gemm_fp8(r.values, r.scales, w.values, w.scales, out, there, ()),
                 lambda: ops.gemm_fp8(r.values, r.scales, w.values, w.scales, out, st, glu)):
        with pytest.raises(KernelError):
            call()
    assert ops.launch_count() == before


@pytest.mark.gpu
def test_8_bit_rows_and_a_16_bit_weight(pe):
    from pytorch_engine_b200.parts.runtime import Runtime

    rows = pe.parts.float8.Float8Rows.quantize(torch.ones(3, 128, dtype=BF16, device=DEV))
    with pytest.raises(pe.kernels.KernelError, match="8-bit weights"):
        Runtime(DEV, BF16).linear(rows, torch.ones(64, 128, dtype=BF16, device=DEV))
