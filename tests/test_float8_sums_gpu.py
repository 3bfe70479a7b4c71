"""How many bits the sums of 8-bit products are held in: the error that is left, against 64 bits, for sums whose terms all have one sign.

The tensor cores add 32 products (exact in 24 bits) to a float32 sum and cut the result to float32: an instruction's error is less
than one step of the sum, 2^-23 of its value, always towards zero, half of that on average.  A kernel that keeps its sums there over
all of K makes K / 32 such errors, each of a sum that is no larger than the whole: at most 2 K / 32 of 2^-24 of the sum, and K / 32 on
average (a sum's value lies anywhere between two powers of two).  A kernel that takes a block of 128 out adds four such errors of a
block's sum, 8 of 2^-24, and one rounding of 2^-24 for every block and every of up to eight parts of K.  Sums of two bits less
would be four times as far off."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
UNIT = 2.0 ** -24


def operands(pe, m, n, k):
    f8 = pe.parts.float8
    g = torch.Generator(device=DEV).manual_seed(k)
    x = torch.randn(m, k, generator=g, device=DEV).abs().to(BF16)
    w = torch.randn(n, k, generator=g, device=DEV).abs() * 0.02
    r, q = f8.Float8Rows.quantize(x), f8.Float8Weight.quantize(w)
    return r, q, r.dequantize(F64) @ q.dequantize(F64).t()


@pytest.mark.parametrize("k", [128, 1024, 4096, 12288])
def test_pairs(pe, k):
    """gemm_fp8_pair.cu: over all of K in the tensor cores (the kernel itself: products of short K go to another one)."""
    st = torch.zeros(4, dtype=torch.int32, device=DEV)
    m, n = 2048, 2048
    r, q, want = operands(pe, m, n, k)
    out = torch.empty(m, n, device=DEV)
    assert pe.kernels.library().pe_gemm_fp8_pair(
        r.values.data_ptr(), r.values.stride(0), r.scales.data_ptr(), m, q.values.data_ptr(), q.values.stride(0), q.scales.data_ptr(),
        out.data_ptr(), n, None, 0, m, n, k, 1, 0, 0.0, 1.0, None, None, None, 0, st.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    off = (out.to(F64) - want).abs() / want / UNIT
    steps = k / 32
    assert float(off.max()) <= 2 * steps and float(off.mean()) <= steps and st.tolist()[0] == 0


@pytest.mark.parametrize("m", [1, 8, 40, 100, 2048])
@pytest.mark.parametrize("k", [128, 1024, 4096, 12288])
def test_block_by_block(pe, m, k):
    """gemm_fp8.cu and gemm_fp8_many.cu: a block of 128 at a time."""
    ops, st = pe.kernels.ops, torch.zeros(4, dtype=torch.int32, device=DEV)
    n = 2048
    r, q, want = operands(pe, m, n, k)
    out = torch.empty(m, n, device=DEV)
    ops.gemm_fp8(r.values, r.scales, q.values, q.scales, out, st)
    off = (out.to(F64) - want).abs() / want / UNIT
    assert float(off.max()) <= 8 + k / 128 + 8 and st.tolist()[0] == 0
