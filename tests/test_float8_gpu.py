"""8-bit weights: the kernels of csrc/quantize_fp8.cu and csrc/gemm_fp8.cu against their definitions in 64 bits.

Tolerances.  A conversion's result is defined to the bit (scales are powers of two, quotients exact, e4m3 to nearest with
ties to even), so it is compared for equality.  A product's operands are e4m3 (products of two are exact in float32); its float32
sums of K terms and K / 128 blocks are off by at most (K + 2 K / 128 + 8) * 2^-24 of the sum of the terms' magnitudes, whatever
their order, and a bfloat16 result by half a step, 2^-8 of its value, more.
"""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops(pe):
    pe.kernels.library()
    return pe.kernels.ops


@pytest.fixture(scope="module")
def f8(pe):
    return pe.parts.float8


@pytest.fixture()
def status():
    st = torch.zeros(4, dtype=torch.int32, device=DEV)
    yield st
    assert st.tolist()[0] == 0


def blocks(n):
    return -(-n // 128)


def plain_scales(a):
    """The smallest 2^e, e >= -126, with a <= 448 * 2^e, for 64-bit magnitudes: by trying every exponent."""
    e = torch.full_like(a, 121.0)
    for k in range(120, -127, -1):
        e = torch.where(a <= 448.0 * 2.0 ** k, torch.full_like(e, float(k)), e)
    return torch.exp2(e)


E4M3_VALUES = torch.arange(256, dtype=torch.uint8).view(E4M3).to(F64)


def plain_e4m3(x):
    """Nearest e4m3 value of 64-bit numbers, ties to the even code, by looking through all of them (CPU, small tensors)."""
    pos = E4M3_VALUES[:127]                          # 0 .. 448 in the order of their codes
    a = x.abs().cpu().clamp(max=448.0)
    hi = torch.searchsorted(pos, a.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = pos[hi] - a, a - pos[lo]
    take_lo = (down < up) | ((down == up) & (lo % 2 == 0))
    v = torch.where(take_lo, pos[lo], pos[hi])
    return torch.copysign(v, x.cpu()).to(x.device)


def plain_quantize(x, tall):
    """64-bit values and scales of ``x``; blocks of ``tall`` rows and 128 columns."""
    x = x.to(F64)
    n, k = x.shape
    scales = torch.empty(-(-n // tall), blocks(k), dtype=F64, device=x.device)
    q = torch.empty_like(x)
    for i, j in itertools.product(range(scales.shape[0]), range(scales.shape[1])):
        part = x[i * tall:(i + 1) * tall, j * 128:(j + 1) * 128]
        scales[i, j] = plain_scales(part.abs().max())
        q[i * tall:(i + 1) * tall, j * 128:(j + 1) * 128] = plain_e4m3(part / scales[i, j])
    return q, scales


def rows_of(n, k, dtype=BF16, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(n, k, generator=g, device=DEV) * torch.exp(2.0 * torch.randn(n, 1, generator=g, device=DEV))
    x[:, k // 2] *= 30.0
    return x.to(dtype)


def weight_of(f8, n, k, seed=0, groups=0):
    """An 8-bit weight with scales that are no powers of two."""
    g = torch.Generator(device=DEV).manual_seed(seed + 1000)
    shape = (groups, n, k) if groups else (n, k)
    ld = -(-k // 16) * 16
    values = torch.randn(*shape[:-1], ld, generator=g, device=DEV).mul_(60.0).clamp_(-448, 448).to(E4M3)[..., :k]
    scales = torch.rand(*shape[:-2], blocks(n), blocks(k), generator=g, device=DEV) * 0.01 + 1e-4
    return f8.Float8Weight(values, scales)


def wide(w):
    """A weight in 64 bits."""
    n, k = w.shape[-2:]
    s = w.scales.to(F64).repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]
    return w.values.to(F64) * s


def wide_rows(r):
    return r.values.to(F64) * r.scales.to(F64).t().repeat_interleave(128, 1)[:, :r.values.shape[1]]


def sum_error(x64, w64):
    """The bound on a product's float32 sums: see above."""
    k = x64.shape[1]
    return (k + 2 * blocks(k) + 8) * 2.0 ** -24 * (x64.abs() @ w64.abs().t())


def assert_within(got, want, bound):
    off = (got.to(F64) - want).abs()
    worst = (off - bound).max()
    assert bool((off <= bound).all()), f"off by {float(off.max())}, {float(worst)} more than allowed"


# ---- conversion ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,k", [(1, 1), (1, 128), (3, 127), (17, 129), (16, 8), (5, 1043), (33, 512), (2, 4097)])
def test_rows(ops, f8, dtype, n, k):
    x = rows_of(n, k, dtype)
    r = f8.Float8Rows.quantize(x)
    q, s = plain_quantize(x, 1)
    assert torch.equal(r.scales.to(F64), s.t())
    assert torch.equal(r.values.to(F64), q)
    assert torch.equal(r.dequantize(F64), (q * s.repeat_interleave(128, 1)[:, :k]))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (127, 129), (130, 40), (300, 1043)])
def test_weight(ops, f8, dtype, n, k):
    w = rows_of(n, k, dtype, 1)
    got = f8.Float8Weight.quantize(w)
    q, s = plain_quantize(w, 128)
    assert torch.equal(got.scales.to(F64), s)
    assert torch.equal(got.values.to(F64), q)


def test_many_rows_and_strides(ops, f8):
    """More rows than a tile, rows of a wider matrix that start off 16-byte boundaries, scales in a wider buffer."""
    base = rows_of(700, 1300, BF16, 3)
    for x in (base[:, 4:1028], base[:, 3:900], base[::2, :]):
        m, k = x.shape
        values = torch.empty(m, 1312, dtype=E4M3, device=DEV)[:, :k]
        scales = torch.full((blocks(k), m + 5), -1.0, device=DEV)
        ops.quantize_rows_fp8(x, values, scales[:, :m])
        whole = f8.Float8Rows.quantize(x.contiguous())
        assert torch.equal(values.to(F32), whole.values.to(F32)) and torch.equal(scales[:, :m], whole.scales)
        assert bool((scales[:, m:] == -1.0).all())


def test_every_bfloat16(ops, f8):
    """All finite bfloat16 values, each alone in a block of its own and in a block beside 448 times a power of two."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(BF16)
    v = bits[torch.isfinite(bits.to(F32))].to(DEV)
    x = torch.zeros(v.numel(), 256, dtype=BF16, device=DEV)
    x[:, 5] = v
    x[:, 130] = v
    x[:, 200] = 448.0 * 2.0 ** -20
    r = f8.Float8Rows.quantize(x)
    a = x.to(F64).abs()
    s = plain_scales(torch.stack([a[:, :128].amax(1), a[:, 128:].amax(1)], 1))
    assert torch.equal(r.scales.to(F64).t(), s)
    assert torch.equal(r.values[:, 5].to(F64), plain_e4m3(v.to(F64) / s[:, 0]))
    assert torch.equal(r.values[:, 130].to(F64), plain_e4m3(v.to(F64) / s[:, 1]))


def test_not_finite(ops, f8):
    """A NaN stays one and does not count for its block; an infinity becomes a NaN; other blocks do not notice."""
    x = rows_of(3, 384, BF16, 5)
    clean = f8.Float8Rows.quantize(x)
    x[0, 3] = float("nan")
    x[1, 200] = float("-inf")
    r = f8.Float8Rows.quantize(x)
    nan = torch.isnan(r.values.to(F32))
    assert bool(nan[0, 3]) and bool(nan[1, 200]) and int(nan.sum()) == 2
    same = torch.ones(3, 384, dtype=torch.bool, device=DEV)
    same[0, 3] = False
    same[1, 128:256] = False
    assert torch.equal(r.values.to(F32)[same], clean.values.to(F32)[same])
    assert float(r.scales[1, 1]) == 2.0 ** 120
    w = x.clone()
    got = f8.Float8Weight.quantize(w)
    assert bool(torch.isnan(got.values.to(F32))[1, 200])


def test_row_map(ops, f8, status):
    x = rows_of(9, 300, BF16, 6)
    pick = torch.tensor([8, 0, 0, 3, 7, 99], dtype=torch.int32, device=DEV)
    live = torch.tensor([5], dtype=torch.int32, device=DEV)      # the last one is not there: nobody looks at its index
    r = f8.Float8Rows.empty(6, 300, DEV)
    r.values.copy_(torch.full((6, 300), 7.0, device=DEV).to(E4M3))
    r.scales.fill_(7.0)
    ops.quantize_rows_fp8(x, r.values, r.scales, pick, live, status)
    whole = f8.Float8Rows.quantize(x)
    at = pick[:5].long()
    assert torch.equal(r.values[:5].to(F32), whole.values[at].to(F32)) and torch.equal(r.scales[:, :5], whole.scales[:, at])
    assert bool((r.values[5].to(F32) == 7.0).all()) and bool((r.scales[:, 5] == 7.0).all())


def test_row_map_outside(ops, f8):
    x = rows_of(4, 130, BF16, 7)
    st = torch.zeros(4, dtype=torch.int32, device=DEV)
    r = f8.Float8Rows.empty(2, 130, DEV)
    r.scales.fill_(7.0)
    ops.quantize_rows_fp8(x, r.values, r.scales, torch.tensor([1, 4], dtype=torch.int32, device=DEV), None, st)
    assert st.tolist() == [6, 1, 4, 4]
    assert bool((r.scales[:, 1] == 7.0).all())


@pytest.mark.parametrize("n,dim", [(1, 4), (3, 132), (2, 512), (5, 1000), (70, 2056), (3, 4096), (65, 4096)])
@pytest.mark.parametrize("delta", [True, False])
def test_norm(ops, f8, n, dim, delta):
    """The same bits as the norm's own kernel followed by the conversion's."""
    g = torch.Generator(device=DEV).manual_seed(n)
    stream = torch.randn(n, dim, generator=g, device=DEV) * 3
    d = torch.randn(n, dim, generator=g, device=DEV).to(BF16) if delta else None
    w = torch.randn(dim, generator=g, device=DEV)
    two, out = stream.clone(), torch.empty(n, dim, dtype=BF16, device=DEV)
    ops.rmsnorm_residual(two, d, w, out, 1e-6)
    want = f8.Float8Rows.quantize(out)
    r = f8.Float8Rows.empty(n, dim, DEV)
    ops.rmsnorm_residual_fp8(stream, d, w, r.values, r.scales, 1e-6)
    assert torch.equal(stream, two)
    assert torch.equal(r.values.to(F32), want.values.to(F32)) and torch.equal(r.scales, want.scales)


@pytest.mark.parametrize("n,dim", [(2, 12032), (3, 12256), (3, 12260), (70, 12288), (2, 12292), (1, 51200)])
def test_norm_wide(ops, f8, n, dim):
    """Rows about as wide as the shared memory that a kernel may have without asking, and the widest."""
    g = torch.Generator(device=DEV).manual_seed(n)
    stream, w = torch.randn(n, dim, generator=g, device=DEV) * 3, torch.randn(dim, generator=g, device=DEV)
    d = torch.randn(n, dim, generator=g, device=DEV).to(BF16)
    two, out = stream.clone(), torch.empty(n, dim, dtype=BF16, device=DEV)
    ops.rmsnorm_residual(two, d, w, out, 1e-6)
    want, r = f8.Float8Rows.quantize(out), f8.Float8Rows.empty(n, dim, DEV)
    ops.rmsnorm_residual_fp8(stream, d, w, r.values, r.scales, 1e-6)
    assert torch.equal(stream, two)
    assert torch.equal(r.values.to(F32), want.values.to(F32)) and torch.equal(r.scales, want.scales)
    x64 = two.to(F64)
    y64 = x64 * torch.rsqrt((x64 * x64).mean(1, keepdim=True) + 1e-6) * w.to(F64)
    # sums of squares: dim terms; the root, two products: 4 roundings; then bfloat16
    assert_within(out, y64, ((dim + 8) * 2.0 ** -24 + 2.0 ** -8) * y64.abs())


# ---- products --------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 128), (3, 129, 130), (16, 300, 1040), (17, 64, 2000), (33, 1111, 384),
                                   (65, 257, 640), (128, 128, 4096), (129, 130, 1043), (300, 384, 512), (8, 4096, 12288), (2, 6144, 4096)])
def test_product(ops, f8, status, m, n, k, out_dtype):
    rows, w = f8.Float8Rows.quantize(rows_of(m, k, BF16, m)), weight_of(f8, n, k, n)
    out = torch.empty(m, n, dtype=out_dtype, device=DEV)
    ops.gemm_fp8(rows.values, rows.scales, w.values, w.scales, out, status)
    x64, w64 = wide_rows(rows), wide(w)
    want = x64 @ w64.t()
    assert_within(out, want, sum_error(x64, w64) + (2.0 ** -8 * want.abs() if out_dtype == BF16 else 0.0))
    again = torch.empty_like(out)
    ops.gemm_fp8(rows.values, rows.scales, w.values, w.scales, again, status)
    assert torch.equal(out, again)


def plain_glu(kind, g, u, limit, alpha):
    """Activations of a gate and an up sum, in 64 bits."""
    if kind == "silu":
        return g * torch.sigmoid(g) * u
    if kind == "relu":
        return g.clamp(min=0) * u
    g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return g * torch.sigmoid(alpha * g) * (u + 1)


def glu_bound(kind, g, u, eg, eu, limit, alpha, want):
    """How far act(g, u) may be off for sums off by eg and eu: |d act / dg| <= 1.1 |u'|, |d act / du| <= |act(g)| <= |g| (silu's
    slope is at most 1.1, u' is u, or |u + 1| <= limit + 1); the exponential and the quotient are good to 2^-20, the result is
    rounded to bfloat16."""
    slope = 1.1 if kind != "clamped_swish" else 1.1
    up = u.abs() if kind != "clamped_swish" else u.clamp(-limit, limit).abs() + 1
    return slope * (up + eu) * eg + (g.abs() + eg) * eu + (2.0 ** -8 + 2.0 ** -20) * want.abs() + 1e-30


@pytest.mark.parametrize("kind,limit,alpha,bias", [("silu", 0.0, 1.0, False), ("relu", 0.0, 1.0, False), ("clamped_swish", 7.0, 1.7, True)])
@pytest.mark.parametrize("m,inter,k", [(1, 1, 16), (2, 64, 256), (7, 72, 1040), (20, 200, 512), (64, 96, 640), (130, 320, 384), (5, 12288, 4096)])
def test_gate(ops, f8, status, m, inter, k, kind, limit, alpha, bias):
    rows, w = f8.Float8Rows.quantize(rows_of(m, k, BF16, m) * 0.01), weight_of(f8, 2 * inter, k, inter)
    b = torch.randn(2 * inter, device=DEV) if bias else None
    out = torch.empty(m, inter, dtype=BF16, device=DEV)
    ops.gemm_fp8(rows.values, rows.scales, w.values, w.scales, out, status, glu=() if kind == "silu" else (kind, limit, alpha, b))
    x64, w64 = wide_rows(rows), wide(w)
    sums, err = x64 @ w64.t(), sum_error(x64, w64)
    if bias:
        sums = sums + b.to(F64)
        err = err + 2.0 ** -23 * sums.abs()
    g, u = sums[:, :inter], sums[:, inter:]
    want = plain_glu(kind, g, u, limit, alpha)
    assert_within(out, want, glu_bound(kind, g, u, err[:, :inter], err[:, inter:], limit, alpha, want))


# the rows of each expert: none, one, a tile's and beyond, all in one
@pytest.mark.parametrize("counts", [[0, 1, 0, 3], [5], [16, 17, 0, 33, 1], [0, 0, 200, 0], [0] * 40 + [2, 3] + [0] * 30, [130, 1, 140]])
@pytest.mark.parametrize("n,k", [(128, 128), (200, 400), (96, 1043)])
def test_experts_product(ops, f8, status, counts, n, k):
    live, groups = sum(counts), len(counts)
    m = live + 3                                       # rows that no expert has
    offsets = torch.tensor([sum(counts[:i]) for i in range(groups + 1)], dtype=torch.int32, device=DEV)
    rows, w = f8.Float8Rows.quantize(rows_of(m, k, BF16, m)), weight_of(f8, n, k, n, groups)
    out = torch.full((m, n), 5.0, device=DEV)
    ops.moe_rows_gemm_fp8(rows.values, rows.scales, offsets, w.values, w.scales, out, status)
    x64, w64 = wide_rows(rows), wide(w)
    for e, c in enumerate(counts):
        at = slice(int(offsets[e]), int(offsets[e]) + c)
        assert_within(out[at], x64[at] @ w64[e].t(), sum_error(x64[at], w64[e])) if c else None
    assert bool((out[live:] == 5.0).all())


@pytest.mark.parametrize("weighted", [False, True])
def test_experts_gate(ops, f8, status, weighted):
    counts, inter, k = [3, 0, 18, 1], 104, 272
    m, groups = sum(counts), len(counts)
    offsets = torch.tensor([0, 3, 3, 21, 22], dtype=torch.int32, device=DEV)
    rows, w = f8.Float8Rows.quantize(rows_of(m, k, BF16, 9) * 0.01), weight_of(f8, 2 * inter, k, 9, groups)
    rw = torch.rand(m, device=DEV) if weighted else None
    out = torch.empty(m, inter, dtype=BF16, device=DEV)
    ops.moe_rows_gemm_fp8(rows.values, rows.scales, offsets, w.values, w.scales, out, status, glu=(), row_weight=rw)
    x64, w64 = wide_rows(rows), wide(w)
    for e in range(groups):
        at = slice(int(offsets[e]), int(offsets[e + 1]))
        sums, err = x64[at] @ w64[e].t(), sum_error(x64[at], w64[e])
        if weighted:
            f = rw[at, None].to(F64)
            sums, err = sums * f, err * f + 2.0 ** -23 * (sums * f).abs()
        g, u = sums[:, :inter], sums[:, inter:]
        want = plain_glu("silu", g, u, 0, 1)
        if want.numel():
            assert_within(out[at], want, glu_bound("silu", g, u, err[:, :inter], err[:, inter:], 0, 1, want))


def test_offsets_outside_the_rows(ops, f8, status):
    """Offsets beyond the rows count as their number: nothing is written behind the output."""
    k, n = 128, 64
    rows, w = f8.Float8Rows.quantize(rows_of(6, k)), weight_of(f8, n, k, 0, 2)
    big = torch.full((40, n), 5.0, device=DEV)
    ops.moe_rows_gemm_fp8(rows.values, rows.scales, torch.tensor([-4, 2, 1000], dtype=torch.int32, device=DEV), w.values, w.scales,
                          big[:6], status)
    assert bool((big[6:] == 5.0).all())
    x64, w64 = wide_rows(rows), wide(w)
    assert_within(big[2:6], x64[2:] @ w64[1].t(), sum_error(x64[2:], w64[1]))


def test_product_strides(ops, f8, status):
    """Operands inside wider buffers, an output inside another, scales with room behind them."""
    m, n, k = 37, 190, 300
    wide_x = torch.empty(m, 640, dtype=E4M3, device=DEV)
    scales = torch.empty(blocks(k), 64, device=DEV)
    x = rows_of(m, k, BF16, 2)
    ops.quantize_rows_fp8(x, wide_x[:, 32:32 + k], scales[:, :m])
    w = weight_of(f8, n, k, 3)
    wide_w = torch.empty(n, 512, dtype=E4M3, device=DEV)
    wide_w[:, 48:48 + k] = w.values
    out = torch.full((m, 256), 5.0, dtype=BF16, device=DEV)
    ops.gemm_fp8(wide_x[:, 32:32 + k], scales[:, :m], wide_w[:, 48:48 + k], w.scales, out[:, 7:7 + n], status)
    plain = torch.empty(m, n, dtype=BF16, device=DEV)
    r = f8.Float8Rows.quantize(x)
    ops.gemm_fp8(r.values, r.scales, w.values, w.scales, plain, status)
    assert torch.equal(out[:, 7:7 + n], plain)
    assert bool((out[:, :7] == 5.0).all()) and bool((out[:, 7 + n:] == 5.0).all())


def test_empty(ops, f8, status):
    w = weight_of(f8, 64, 128)
    r = f8.Float8Rows.empty(0, 128, DEV)
    out = torch.empty(0, 64, dtype=BF16, device=DEV)
    ops.gemm_fp8(r.values, r.scales, w.values, w.scales, out, status)
    ops.quantize_rows_fp8(torch.empty(0, 128, dtype=BF16, device=DEV), r.values, r.scales)
    ops.rmsnorm_residual_fp8(torch.empty(0, 128, device=DEV), None, torch.ones(128, device=DEV), r.values, r.scales, 1e-6)


def test_a_nan_stays_in_its_row(ops, f8, status):
    x = rows_of(20, 300, BF16, 4)
    w = weight_of(f8, 130, 300)
    clean, dirty = (torch.empty(20, 130, dtype=BF16, device=DEV) for _ in range(2))
    r = f8.Float8Rows.quantize(x)
    ops.gemm_fp8(r.values, r.scales, w.values, w.scales, clean, status)
    x[7, 299] = float("inf")
    r = f8.Float8Rows.quantize(x)
    ops.gemm_fp8(r.values, r.scales, w.values, w.scales, dirty, status)
    assert bool(torch.isnan(dirty[7]).all())
    keep = torch.arange(20, device=DEV) != 7
    assert torch.equal(clean[keep], dirty[keep])


def test_own_stream_and_graph(ops, f8, status):
    """A run of them on another stream than the default, captured, and replayed on other inputs in the same buffers."""
    m, k, n = 9, 512, 640
    w = weight_of(f8, n, k)
    x = rows_of(m, k, BF16, 1)
    out = torch.empty(m, n, dtype=BF16, device=DEV)
    r = f8.Float8Rows.empty(m, k, DEV)

    def chain():
        ops.quantize_rows_fp8(x, r.values, r.scales)
        ops.gemm_fp8(r.values, r.scales, w.values, w.scales, out, status)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain()
    side.synchronize()
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        chain()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    x.copy_(rows_of(m, k, BF16, 2))
    graph.replay()
    torch.cuda.synchronize()
    replayed = out.clone()
    chain()
    assert torch.equal(out, replayed) and not torch.equal(out, first)


# ---- quantised on the way ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", [(1, 64, 128), (1, 6144, 4096), (5, 200, 1043), (8, 4096, 12288), (16, 333, 2000), (17, 64, 300), (70, 256, 512),
                                   (700, 2816, 2048)])
@pytest.mark.parametrize("gate", [False, True])
def test_linear(ops, f8, status, m, n, k, dtype, gate):
    """The same bits as conversion and product one after the other, whichever kernels take it."""
    if gate:
        n = n // 2 * 2
    x, w = rows_of(m, k, dtype, m) * 0.01, weight_of(f8, n, k, n)
    x = x.to(dtype)
    cols, glu = (n // 2, ()) if gate else (n, None)
    one, two = (torch.empty(m, cols, dtype=BF16, device=DEV) for _ in range(2))
    ops.linear_fp8(x, w.values, w.scales, one, status, glu)
    r = f8.Float8Rows.quantize(x)
    ops.gemm_fp8(r.values, r.scales, w.values, w.scales, two, status, glu)
    assert torch.equal(one, two)


def test_linear_of_rows_off_the_boundary(ops, f8, status):
    base, w = rows_of(9, 600, BF16, 1), weight_of(f8, 130, 500, 1)
    for x in (base[:, 3:503], base[:, 8:508], base.t()[:500].t()):
        assert x.stride(1) == 1
        one, two = (torch.empty(9, 130, dtype=BF16, device=DEV) for _ in range(2))
        ops.linear_fp8(x, w.values, w.scales, one, status)
        ops.linear_fp8(x.contiguous(), w.values, w.scales, two, status)
        assert torch.equal(one, two)


@pytest.mark.parametrize("counts", [[0, 1, 0, 3], [16, 17, 0, 33, 1], [1] * 40, [300, 0, 5]])
@pytest.mark.parametrize("mapped", [False, True])
def test_experts_linear(ops, f8, status, counts, mapped):
    """Grouped rows, taken from others by a map or not: as the grouped product of quantised rows."""
    k, n, m, groups = 400, 144, sum(counts), len(counts)
    offsets = torch.tensor([sum(counts[:i]) for i in range(groups + 1)], dtype=torch.int32, device=DEV)
    w = weight_of(f8, n, k, 2, groups)
    src = rows_of(50, k, BF16, 3)
    pick = torch.randint(0, 50, (m + 2,), device=DEV, dtype=torch.int32)
    pick[m:] = 12345                                    # rows that no expert has: nobody looks at their index
    x = src if mapped else src[pick[:m].long()]
    out = torch.full((m + 2 if mapped else m, n), 5.0, dtype=BF16, device=DEV)
    ops.linear_fp8(x, w.values, w.scales, out, status, offsets=offsets, row_map=pick if mapped else None)
    r = f8.Float8Rows.quantize(src[pick[:m].long()])
    want = torch.empty(m, n, dtype=BF16, device=DEV)
    ops.moe_rows_gemm_fp8(r.values, r.scales, offsets, w.values, w.scales, want, status)
    assert torch.equal(out[:m], want) and bool((out[m:] == 5.0).all())


def test_linear_nan_and_infinity(ops, f8, status):
    for m in (3, 40):
        x, w = rows_of(m, 300, BF16, 4), weight_of(f8, 130, 300)
        clean, dirty = (torch.empty(m, 130, dtype=BF16, device=DEV) for _ in range(2))
        ops.linear_fp8(x, w.values, w.scales, clean, status)
        x[1, 7], x[2, 299] = float("nan"), float("inf")
        ops.linear_fp8(x, w.values, w.scales, dirty, status)
        assert bool(torch.isnan(dirty[1:3]).all())
        keep = (torch.arange(m, device=DEV) < 1) | (torch.arange(m, device=DEV) > 2)
        assert torch.equal(clean[keep], dirty[keep])


@pytest.mark.parametrize("m,inter,k", [(513, 12288, 256), (700, 1408, 2048), (2100, 640, 1043)])
@pytest.mark.parametrize("kind", ["silu", "clamped_swish"])
def test_gate_quantized(ops, f8, status, m, inter, k, kind):
    """The same bits as the gated product and the conversion of what it gives; sizes that other tiles take are refused."""
    rows, w = f8.Float8Rows.quantize(rows_of(m, k, BF16, m) * 0.01), weight_of(f8, 2 * inter, k, inter)
    glu = () if kind == "silu" else (kind, 7.0, 1.7, torch.randn(2 * inter, device=DEV))
    out = torch.empty(m, inter, dtype=BF16, device=DEV)
    ops.gemm_fp8(rows.values, rows.scales, w.values, w.scales, out, status, glu=glu)
    want = f8.Float8Rows.quantize(out)
    got = f8.Float8Rows.empty(m, inter, DEV)
    if not ops.gemm_fp8_gated_supported(m, inter, k):
        with pytest.raises(RuntimeError, match="gemm_fp8_gated"):
            ops.gemm_fp8_gated(rows.values, rows.scales, w.values, w.scales, got.values, got.scales, status, glu)
        return
    ops.gemm_fp8_gated(rows.values, rows.scales, w.values, w.scales, got.values, got.scales, status, glu)
    assert torch.equal(got.scales, want.scales) and torch.equal(got.values.to(F32), want.values.to(F32))


@pytest.mark.parametrize("m", [1, 9, 64, 65, 600, 1030])
@pytest.mark.parametrize("hidden,inter", [(512, 1408), (256, 200)])
def test_feed_forward(pe, ops, f8, m, hidden, inter):
    """The run of them against the products one by one."""
    from pytorch_engine_b200.parts.runtime import Runtime

    rt = Runtime(DEV, BF16)
    x, gate_up, down = rows_of(m, hidden, BF16, m) * 0.01, weight_of(f8, 2 * inter, hidden, 1), weight_of(f8, hidden, inter, 2)
    out, act, want = (torch.empty(m, n, dtype=BF16, device=DEV) for n in (hidden, inter, hidden))
    rt.float8_feed_forward(x, gate_up, down, out)
    rows = f8.Float8Rows.quantize(x)
    ops.gemm_fp8(rows.values, rows.scales, gate_up.values, gate_up.scales, act, rt.status, glu=())
    r = f8.Float8Rows.quantize(act)
    ops.gemm_fp8(r.values, r.scales, down.values, down.scales, want, rt.status)
    assert torch.equal(out, want)
    again = torch.empty_like(out)
    rt.float8_feed_forward(rows, gate_up, down, again)
    assert torch.equal(out, again)
    rt.raise_on_status()


# many rows an expert: none, one tile, some, with a last tile of one row
@pytest.mark.parametrize("counts", [[0, 128, 300, 1], [700, 0, 0, 500], [129] * 5])
@pytest.mark.parametrize("weighted,inter,hidden", [(False, 256, 384), (True, 128, 272), (False, 200, 272)])
def test_experts_of_many_rows(pe, ops, f8, counts, weighted, inter, hidden):
    """The run of them, rows taken by a map, against each expert's feed-forward alone in 64 bits' definition of its two products."""
    from pytorch_engine_b200.parts.runtime import Runtime

    rt, groups, m = Runtime(DEV, BF16), len(counts), sum(counts)
    offsets = torch.tensor([sum(counts[:i]) for i in range(groups + 1)], dtype=torch.int32, device=DEV)
    src = rows_of(90, hidden, BF16, 1) * 0.01
    pick = torch.randint(0, 90, (m,), device=DEV, dtype=torch.int32)
    gate_up, down = weight_of(f8, 2 * inter, hidden, 1, groups), weight_of(f8, hidden, inter, 2, groups)
    rw = torch.rand(m, device=DEV) if weighted else None
    out = torch.full((m + 4, hidden), 5.0, dtype=BF16, device=DEV)
    row_weight = torch.cat([rw, rw[:4]]) if weighted else None
    rt.float8_experts(src, offsets, gate_up, down, out, row_weight=row_weight,
                      row_token=torch.cat([pick, torch.full((4,), 10 ** 6, dtype=torch.int32, device=DEV)]))
    rt.raise_on_status()
    assert bool((out[m:] == 5.0).all())
    x = f8.Float8Rows.quantize(src[pick.long()])
    act = torch.empty(m, inter, dtype=BF16, device=DEV)
    ops.moe_rows_gemm_fp8(x.values, x.scales, offsets, gate_up.values, gate_up.scales, act, rt.status, glu=(), row_weight=rw)
    x64, w64 = wide_rows(x), wide(gate_up)
    r = f8.Float8Rows.quantize(act)
    r64, d64 = wide_rows(r), wide(down)
    for e in range(groups):
        at = slice(int(offsets[e]), int(offsets[e + 1]))
        if counts[e] == 0:
            continue
        sums, err = x64[at] @ w64[e].t(), sum_error(x64[at], w64[e])
        if weighted:
            f = rw[at, None].to(F64)
            sums, err = sums * f, err * f + 2.0 ** -23 * (sums * f).abs()
        g, u = sums[:, :inter], sums[:, inter:]
        want = plain_glu("silu", g, u, 0, 1)
        assert_within(act[at], want, glu_bound("silu", g, u, err[:, :inter], err[:, inter:], 0, 1, want))
        want = r64[at] @ d64[e].t()
        assert_within(out[at], want, sum_error(r64[at], d64[e]) + 2.0 ** -8 * want.abs())


@pytest.mark.parametrize("counts", [[0, 3, 40, 1], [700, 0, 0, 500]])
def test_experts_of_quantized_rows(pe, ops, f8, counts):
    """Rows that are quantised already give the bits of the rows they come from; they cannot be taken by a map."""
    from pytorch_engine_b200.parts.runtime import KernelError, Runtime

    rt, groups, m, hidden, inter = Runtime(DEV, BF16), len(counts), sum(counts), 384, 256
    offsets = torch.tensor([sum(counts[:i]) for i in range(groups + 1)], dtype=torch.int32, device=DEV)
    x = rows_of(m, hidden, BF16, 1)
    gate_up, down = weight_of(f8, 2 * inter, hidden, 1, groups), weight_of(f8, hidden, inter, 2, groups)
    want, got = torch.empty(m, hidden, dtype=BF16, device=DEV), torch.empty(m, hidden, dtype=BF16, device=DEV)
    rt.float8_experts(x, offsets, gate_up, down, want)
    rows = f8.Float8Rows.quantize(x)
    rt.float8_experts(rows, offsets, gate_up, down, got)
    rt.raise_on_status()
    assert torch.equal(got, want)
    with pytest.raises(KernelError):
        rt.float8_experts(rows, offsets, gate_up, down, got, row_token=torch.arange(m, dtype=torch.int32, device=DEV))


def test_two_streams_at_once(pe, f8):
    """Feed-forwards of two streams and of their graphs share weights and a status word, and nothing else."""
    from pytorch_engine_b200.parts.runtime import Runtime

    rt, hidden, inter = Runtime(DEV, BF16), 512, 384
    gate_up, down = weight_of(f8, 2 * inter, hidden, 1), weight_of(f8, hidden, inter, 2)
    sizes = (5, 300)
    x = [rows_of(m, hidden, BF16, m) for m in sizes]
    want = [torch.empty(m, hidden, dtype=BF16, device=DEV) for m in sizes]
    for a, y in zip(x, want):
        rt.float8_feed_forward(a, gate_up, down, y)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sizes]
    out = [torch.zeros_like(y) for y in want]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, a, y in zip(streams, x, out):
            with torch.cuda.stream(s):
                rt.float8_feed_forward(a, gate_up, down, y)
    torch.cuda.synchronize()
    for y, w in zip(out, want):
        assert torch.equal(y, w)
        y.zero_()
    torch.cuda.synchronize()
    graphs = []
    for s, a, y in zip(streams, x, out):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            rt.float8_feed_forward(a, gate_up, down, y)
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for y, w in zip(out, want):
        assert torch.equal(y, w)
    rt.raise_on_status()


def test_weight_quantized_right_before(ops, f8, status):
    """A weight that the launch right in front of its product writes, in storage that held another."""
    m, k, n = 8, 4096, 6144
    x = rows_of(m, k, BF16, 1)
    r = f8.Float8Rows.quantize(x)
    mats = [rows_of(n, k, BF16, 2 + i) for i in range(3)]
    want = torch.empty(m, n, dtype=BF16, device=DEV)
    out, w = torch.empty_like(want), f8.Float8Weight.quantize(mats[0])
    for i in range(12):
        fresh = f8.Float8Weight.quantize(mats[i % 3])
        torch.cuda.synchronize()
        ops.gemm_fp8(r.values, r.scales, fresh.values, fresh.scales, want, status)
        ops.quantize_weight_fp8(mats[i % 3], w.values, w.scales)
        ops.gemm_fp8(r.values, r.scales, w.values, w.scales, out, status)
        assert torch.equal(out, want)


def test_shapes_refused(pe, ops, f8, status):
    from pytorch_engine_b200.parts.runtime import KernelError

    w, y = weight_of(f8, 64, 256), torch.empty(1, 64, dtype=BF16, device=DEV)
    with pytest.raises(KernelError):
        ops.linear_fp8(torch.zeros(256, dtype=BF16, device=DEV), w.values, w.scales, y, status)
    with pytest.raises(ValueError):
        f8.Float8Weight.quantize(torch.zeros(256, device=DEV))


# ---- scales that are powers of two -------------------------------------------------------------------------------------
def power_weight(f8, n, k, seed=0, groups=0):
    """A weight whose scales are powers of two, far apart."""
    w = weight_of(f8, n, k, seed, groups)
    g = torch.Generator(device=DEV).manual_seed(seed)
    scales = torch.exp2(torch.randint(-12, -3, tuple(w.scales.shape), generator=g, device=DEV).to(F32))
    return f8.Float8Weight(w.values, scales)


def pair_product(ops, rows, w, out, status, kind=0, scales=None, offsets=None, row_weight=None, bias=None):
    """The kernel for pairs of SMs whatever the sizes."""
    m, k = rows.shape
    lib, v, n = ops.library(), w.values, out.shape[1]
    p = lambda t: None if t is None else t.data_ptr()
    ld = lambda t, width: t.stride(0) if t.shape[0] > 1 else -(-width // 16) * 16
    assert lib.pe_gemm_fp8_pair(rows.values.data_ptr(), ld(rows.values, k), rows.scales.data_ptr(), m, v.data_ptr(), v.stride(-2), w.scales.data_ptr(),
                                out.data_ptr(), ld(out, n) if scales is not None else out.stride(0), p(scales), m if scales is not None else 0, m, n, k,
                                1 if out.dtype == F32 else 0, kind, 0.0, 1.0, p(bias), p(row_weight), p(offsets),
                                0 if offsets is None else w.shape[0], status.data_ptr(), ops._stream()) == 0


# one element to many tiles, one block of K to more than the stages and the slots of scales, odd sizes
@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (3, 130, 129), (127, 129, 128), (129, 257, 256), (256, 256, 384), (257, 300, 512), (300, 384, 640), (300, 1111, 1043),
                                   (513, 256, 2000), (64, 128, 4096), (1300, 4000, 1152), (40, 256, 12288)])
def test_pair_product(ops, f8, status, m, n, k, out_dtype):
    rows, w = f8.Float8Rows.quantize(rows_of(m, k, BF16, m)), power_weight(f8, n, k, n)
    out = torch.full((m + 1, n), 7.0, dtype=out_dtype, device=DEV)
    pair_product(ops, rows, w, out[:m], status)
    x64, w64 = wide_rows(rows), wide(w)
    want = x64 @ w64.t()
    assert_within(out[:m], want, sum_error(x64, w64) + (2.0 ** -8 * want.abs() if out_dtype == BF16 else 0.0))
    assert bool((out[m] == 7.0).all())
    again = torch.empty_like(out[:m])
    pair_product(ops, rows, w, again, status)
    assert torch.equal(out[:m], again)


@pytest.mark.parametrize("m,inter,k", [(5, 128, 300), (300, 256, 512), (700, 1408, 2048), (2100, 640, 1043)])
@pytest.mark.parametrize("kind", [1, 2])
@pytest.mark.parametrize("bias", [False, True])
def test_pair_gate(ops, f8, status, m, inter, k, kind, bias):
    rows, w = f8.Float8Rows.quantize(rows_of(m, k, BF16, m) * 0.01), power_weight(f8, 2 * inter, k, inter)
    b = torch.randn(2 * inter, device=DEV) if bias else None
    out = torch.empty(m, inter, dtype=BF16, device=DEV)
    pair_product(ops, rows, w, out, status, kind, bias=b)
    x64, w64 = wide_rows(rows), wide(w)
    sums, err = x64 @ w64.t(), sum_error(x64, w64)
    if bias:
        sums = sums + b.to(F64)
        err = err + 2.0 ** -24 * sums.abs()
    name = {v: n for n, v in ops.GLU_KINDS.items()}[kind]
    g, u = sums[:, :inter], sums[:, inter:]
    want = plain_glu(name, g, u, 0.0, 1.0)
    assert_within(out, want, glu_bound(name, g, u, err[:, :inter], err[:, inter:], 0.0, 1.0, want))
    # quantised on the way out: the same bits
    q, r = f8.Float8Rows.quantize(out), f8.Float8Rows.empty(m, inter, DEV)
    pair_product(ops, rows, w, r.values, status, kind, r.scales, bias=b)
    assert torch.equal(q.scales, r.scales) and torch.equal(q.values.to(F32), r.values.to(F32))


@pytest.mark.parametrize("counts", [[0, 128, 300, 1], [700, 0, 0, 500], [129] * 5, [0, 0], [257]])
@pytest.mark.parametrize("weighted", [False, True])
def test_pair_experts(ops, f8, status, counts, weighted):
    groups, m, n, k = len(counts), sum(counts) + 3, 256, 700
    offsets = torch.tensor([sum(counts[:i]) for i in range(groups + 1)], dtype=torch.int32, device=DEV)
    rows, w = f8.Float8Rows.quantize(rows_of(m, k, BF16, 1) * 0.01), power_weight(f8, 2 * n, k, 3, groups)
    rw = torch.rand(m, device=DEV) if weighted else None
    out = torch.full((m, n), 5.0, dtype=BF16, device=DEV)
    plain = torch.full((m, 2 * n), 5.0, dtype=F32, device=DEV)
    pair_product(ops, rows, w, out, status, 1, offsets=offsets, row_weight=rw)
    pair_product(ops, rows, w, plain, status, offsets=offsets)
    assert bool((out[sum(counts):] == 5.0).all()) and bool((plain[sum(counts):] == 5.0).all())
    x64, w64 = wide_rows(rows), wide(w)
    for e in range(groups):
        at = slice(int(offsets[e]), int(offsets[e + 1]))
        if counts[e] == 0:
            continue
        sums, err = x64[at] @ w64[e].t(), sum_error(x64[at], w64[e])
        assert_within(plain[at], sums, err)
        if weighted:
            f = rw[at, None].to(F64)
            sums, err = sums * f, err * f + 2.0 ** -23 * (sums * f).abs()
        g, u = sums[:, :n], sums[:, n:]
        want = plain_glu("silu", g, u, 0, 1)
        assert_within(out[at], want, glu_bound("silu", g, u, err[:, :n], err[:, n:], 0, 1, want))


def test_powers_are_known(f8):
    w = f8.Float8Weight.quantize(rows_of(300, 200, BF16, 1))
    assert w.powers is True and f8.Float8Rows.quantize(rows_of(3, 200, BF16, 1)).powers
    assert f8.Float8Weight(w.values, w.scales).powers is None
    assert f8.Float8Weight(w.values, w.scales).to(DEV).powers is True
    other = f8.Float8Weight(w.values, w.scales * 3).to(DEV)
    assert other.powers is False and f8.Float8Weight.stack([w, other]).powers is False
    assert f8.Float8Weight.stack([w, w]).powers is True and f8.Float8Weight.stack([w, w])[1].powers is True


@pytest.mark.parametrize("m,hidden,inter", [(1500, 512, 1408), (700, 4096, 2048), (2048, 1024, 200)])
def test_feed_forward_of_powers(pe, ops, f8, m, hidden, inter):
    """The run of them with weights whose scales are known to be powers of two, for rows quantised before too, within the rounding of its
    two products."""
    from pytorch_engine_b200.parts.runtime import Runtime

    rt = Runtime(DEV, BF16)
    x, gate_up, down = rows_of(m, hidden, BF16, m) * 0.01, power_weight(f8, 2 * inter, hidden, 1), power_weight(f8, hidden, inter, 2)
    out = torch.empty(m, hidden, dtype=BF16, device=DEV)
    rt.float8_feed_forward(x, gate_up.to(DEV), down.to(DEV), out)
    rows = f8.Float8Rows.quantize(x)
    again = torch.empty_like(out)
    rt.float8_feed_forward(rows, gate_up.to(DEV), down.to(DEV), again)
    assert torch.equal(out, again)
    act = torch.empty(m, inter, dtype=BF16, device=DEV)
    ops.gemm_fp8(rows.values, rows.scales, gate_up.values, gate_up.scales, act, rt.status, glu=(), powers=True)
    x64, w64 = wide_rows(rows), wide(gate_up)
    sums, err = x64 @ w64.t(), sum_error(x64, w64)
    g, u = sums[:, :inter], sums[:, inter:]
    want = plain_glu("silu", g, u, 0, 1)
    assert_within(act, want, glu_bound("silu", g, u, err[:, :inter], err[:, inter:], 0, 1, want))
    r = f8.Float8Rows.quantize(act)
    r64, d64 = wide_rows(r), wide(down)
    want = r64 @ d64.t()
    assert_within(out, want, sum_error(r64, d64) + 2.0 ** -8 * want.abs())
    rt.raise_on_status()


def test_more_than_two_to_the_31(ops, f8, status):
    """Outputs, rows and values that pass 2^31 elements and 2^32 bytes, in every kernel that writes many of them."""
    m, n, k = 66000, 33024, 128
    x = rows_of(m, k, BF16, 1)
    rows = f8.Float8Rows.quantize(x)
    picks = torch.tensor([0, 1, 32767, 32768, 65071, m - 129, m - 128, m - 1], device=DEV)
    x64 = wide_rows(f8.Float8Rows(rows.values[picks], rows.scales[:, picks].contiguous()))
    out = torch.empty(m, n, dtype=BF16, device=DEV)
    for w, powers in ((weight_of(f8, n, k, 1), False), (power_weight(f8, n, k, 1), True)):
        out.fill_(3.0)
        ops.gemm_fp8(rows.values, rows.scales, w.values, w.scales, out, status, powers=powers)
        w64 = wide(w)
        want = x64 @ w64.t()
        assert_within(out[picks], want, sum_error(x64, w64) + 2.0 ** -8 * want.abs())
    wide_row = f8.Float8Rows.quantize(out)              # [66000, 33024] again
    again = f8.Float8Rows.quantize(out[picks])
    assert torch.equal(wide_row.values[picks].to(F32), again.values.to(F32)) and torch.equal(wide_row.scales[:, picks], again.scales)
    rest = m % 128                                       # the last block of rows
    tall, last = f8.Float8Weight.quantize(out), f8.Float8Weight.quantize(out[-rest:])
    assert torch.equal(tall.values[-rest:].to(F32), last.values.to(F32)) and torch.equal(tall.scales[-1:], last.scales)


def test_pairs_on_two_streams(pe, f8):
    """Pairs of SMs for two streams at once, beside products of few rows, and their graphs."""
    from pytorch_engine_b200.parts.runtime import Runtime

    rt, hidden, inter = Runtime(DEV, BF16), 1024, 2816
    gate_up, down = power_weight(f8, 2 * inter, hidden, 1).to(DEV), power_weight(f8, hidden, inter, 2).to(DEV)
    sizes = (1500, 7, 2100)
    x = [rows_of(m, hidden, BF16, m) * 0.01 for m in sizes]
    want = [torch.empty(m, hidden, dtype=BF16, device=DEV) for m in sizes]
    for a, y in zip(x, want):
        rt.float8_feed_forward(a, gate_up, down, y)
    streams, out = [torch.cuda.Stream() for _ in sizes], [torch.zeros_like(y) for y in want]
    graphs = []
    torch.cuda.synchronize()
    for s, a, y in zip(streams, x, out):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=s):
            rt.float8_feed_forward(a, gate_up, down, y)
    for i in range(20):
        for s, a, y, g in zip(streams, x, out, graphs):
            with torch.cuda.stream(s):
                if i % 2:
                    rt.float8_feed_forward(a, gate_up, down, y)
                else:
                    g.replay()
    torch.cuda.synchronize()
    for y, w in zip(out, want):
        assert torch.equal(y, w)
    rt.raise_on_status()
