"""Blocks of nothing but NaN: a NaN does not count for its block's maximum, so such a block has the scale of a block of zeros,
2^-126, whichever kernel converts it, and its values are NaN."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32 = torch.bfloat16, torch.float32
E4M3 = torch.float8_e4m3fn
LEAST = 2.0 ** -126
NAN = float("nan")


def check_rows(r, dead):
    """Rows ``dead`` are all NaN, the others have none."""
    nan = torch.isnan(r.values.to(F32))
    rows = torch.zeros(nan.shape[0], dtype=torch.bool, device=DEV)
    rows[dead] = True
    assert bool(nan[rows].all()) and not bool(nan[~rows].any())
    assert bool((r.scales[:, rows] == LEAST).all()) and bool((r.scales[:, ~rows] > LEAST).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,k", [(2, 128), (3, 200), (1, 1), (9, 1043), (700, 1300), (2048, 4096)])
def test_rows(pe, dtype, m, k):
    f8 = pe.parts.float8
    x = torch.randn(m, k, device=DEV).abs().add_(0.1).to(dtype)
    x[m // 2] = NAN
    check_rows(f8.Float8Rows.quantize(x), [m // 2])
    x[m // 2, :min(k, 128)] = 1.0                      # the other blocks of the row alone
    r = f8.Float8Rows.quantize(x)
    assert float(r.scales[0, m // 2]) == 2.0 ** -8 and bool((r.scales[1:, m // 2] == LEAST).all())     # 1 <= 448 * 2^-8 < 2


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_weight(pe, dtype):
    w = torch.ones(200, 300, dtype=dtype, device=DEV)
    w[:128, 128:256] = NAN
    got = pe.parts.float8.Float8Weight.quantize(w)
    assert float(got.scales[0, 1]) == LEAST and int((got.scales == 2.0 ** -8).sum()) == 5
    assert torch.equal(torch.isnan(got.values.to(F32)), torch.isnan(w))


@pytest.mark.parametrize("delta", [True, False])
@pytest.mark.parametrize("n,dim", [(3, 512), (70, 1000), (5, 4096)])
def test_norm(pe, n, dim, delta):
    """One NaN makes the whole normed row NaN."""
    ops, f8 = pe.kernels.ops, pe.parts.float8
    stream = torch.randn(n, dim, device=DEV)
    stream[1, 7] = NAN
    d = torch.randn(n, dim, device=DEV).to(BF16) if delta else None
    w = torch.rand(dim, device=DEV) + 0.5
    r = f8.Float8Rows.empty(n, dim, DEV)
    ops.rmsnorm_residual_fp8(stream, d, w, r.values, r.scales, 1e-6)
    check_rows(r, [1])


@pytest.mark.parametrize("m", [3, 40])
def test_product(pe, m):
    """Rows converted inside the product or in front of it, all NaN: only their outputs are."""
    f8, st = pe.parts.float8, torch.zeros(4, dtype=torch.int32, device=DEV)
    w = f8.Float8Weight.quantize(torch.randn(130, 300, device=DEV))
    x = torch.randn(m, 300, device=DEV).to(BF16)
    clean, dirty = (torch.empty(m, 130, dtype=BF16, device=DEV) for _ in range(2))
    pe.kernels.ops.linear_fp8(x, w.values, w.scales, clean, st)
    x[1] = NAN
    pe.kernels.ops.linear_fp8(x, w.values, w.scales, dirty, st)
    keep = torch.arange(m, device=DEV) != 1
    assert bool(torch.isnan(dirty[1]).all()) and torch.equal(clean[keep], dirty[keep]) and st.tolist()[0] == 0


@pytest.mark.parametrize("powers", [True, False])
def test_gated_output(pe, powers):
    """An activation that leaves the product quantised: the bits of its own conversion."""
    ops, f8, st = pe.kernels.ops, pe.parts.float8, torch.zeros(4, dtype=torch.int32, device=DEV)
    m, inter, k = 512, 4096, 512
    w = f8.Float8Weight.quantize(torch.randn(2 * inter, k, device=DEV))
    x = torch.randn(m, k, device=DEV).to(BF16)
    x[300, 11] = NAN
    r, got = f8.Float8Rows.quantize(x), f8.Float8Rows.empty(m, inter, DEV)
    assert ops.gemm_fp8_gated_supported(m, inter, k, 0, powers)
    ops.gemm_fp8_gated(r.values, r.scales, w.values, w.scales, got.values, got.scales, st, (), powers=powers)
    act = torch.empty(m, inter, dtype=BF16, device=DEV)
    ops.gemm_fp8(r.values, r.scales, w.values, w.scales, act, st, (), powers=powers)
    want = f8.Float8Rows.quantize(act)
    check_rows(got, [300])
    nan = torch.isnan(want.values.to(F32))
    assert torch.equal(got.scales, want.scales) and torch.equal(got.values.to(F32)[~nan], want.values.to(F32)[~nan]) and st.tolist()[0] == 0
