"""The operators of 8-bit weights, measured alone: rows and matrices to e4m3 in blocks of 128, matrix products of such
blocks, a gated feed-forward of two of them, and the same for rows grouped by expert.

A block has one scale, a power of two: with ``a`` the block's largest magnitude, ``s`` is the smallest ``2^e`` (``e >=
-126``) with ``a <= 448 * 2^e``, and its elements are kept as ``e4m3(x / s)`` (to nearest, ties to even).  A block is 128
neighbouring features of a row, or 128 x 128 elements of a weight matrix; the last blocks may be smaller.  Scales of rows
lie as ``[blocks, rows]``, those of a matrix as ``[row blocks, column blocks]``.  A product may be given any scales:

    y[m, n] = sum_b sx[b, m] * sw[n // 128, b] * sum_{k in block b} x[m, k] * w[n, k]

``own`` false: elementary torch operations in 32 bits.  ``own`` true: the calls of this package.  Sizes are those of this
repository's 8B preset (width 4,096, feed-forward 12,288, q|k|v 6,144) and of its small benchmark models (width 2,048).
"""
import math

import torch

own = False

DEVICE = "cuda:0"
BLOCK = 128
EPS = 1e-6
BF16 = torch.bfloat16
EXACT_FLOPS = 4.0e13        # above this a 64-bit run takes too long


# ---- the cases -----------------------------------------------------------------------------------------------------
def listed():
    return [
        # a decode step of eight sequences: the residual add, the norm and the q|k|v projection of what it gives
        dict(name="norm and linear 8", op="norm", rows=8, width=4096, out=6144, delta=True),
        # the first norm of a prompt whose length fits no tile, and the same projection
        dict(name="norm and linear 2011", op="norm", rows=2011, width=4096, out=6144, delta=False),
        # attention or feed-forward outputs of a prompt on their way into a product
        dict(name="rows 2048x12288", op="rows", rows=2048, width=12288, dtype="bfloat16"),
        # a model's largest matrix when its weights are converted at load
        dict(name="weight 24576x4096", op="weight", rows=24576, width=4096, dtype="bfloat16"),
        # a float32 matrix whose sizes are multiples of nothing
        dict(name="weight 1111x1043 f32", op="weight", rows=1111, width=1043, dtype="float32"),
        # one user's decode step: the q|k|v projection, where latency counts
        dict(name="linear 1x4096x6144", op="linear", rows=1, width=4096, out=6144, dtype="bfloat16"),
        # a small batch's down projection: a long sum and few outputs
        dict(name="linear 8x12288x4096", op="linear", rows=8, width=12288, out=4096, dtype="bfloat16"),
        # a float32 result of odd sizes (a router or a head), more rows than the few-row kernels of the package take
        dict(name="linear 37x2000x1111 f32", op="linear", rows=37, width=2000, out=1111, dtype="float32"),
        # a full server's decode step: the whole feed-forward of 64 sequences
        dict(name="feed forward 64", op="ffn", rows=64, width=4096, ff=12288),
        # the feed-forward of a prompt of 2,048 tokens
        dict(name="feed forward 2048", op="ffn", rows=2048, width=4096, ff=12288),
        # routed experts of a decode step: 8 sequences, 4 choices each, of 16 experts
        dict(name="experts 32 of 16", op="experts", rows=32, experts=16, width=2048, ff=1408, skew=0.5),
        # routed experts of a prompt, unevenly liked
        dict(name="experts 4096 of 16", op="experts", rows=4096, experts=16, width=2048, ff=1408, skew=1.0),
    ]


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(["norm", "rows", "weight", "linear", "linear", "linear", "ffn", "ffn", "experts", "experts"])
    if op == "norm":
        return dict(op=op, rows=spread(1, 2048), width=8 * spread(64, 1024), out=spread(500, 6144), delta=rng.random() < 0.7)
    if op == "rows":
        return dict(op=op, rows=spread(1, 2048), width=spread(100, 12288), dtype=rng.choice(["bfloat16", "float32"]))
    if op == "weight":
        return dict(op=op, rows=spread(1000, 24576), width=spread(500, 4096), dtype=rng.choice(["bfloat16", "float32"]))
    if op == "linear":
        return dict(op=op, rows=spread(1, 2048), width=spread(500, 12288), out=spread(500, 6144), dtype=rng.choice(["bfloat16", "bfloat16", "float32"]))
    if op == "ffn":
        return dict(op=op, rows=spread(1, 2048), width=8 * spread(64, 512), ff=8 * spread(128, 1536))
    return dict(op=op, rows=spread(1, 4096), experts=spread(2, 16), width=8 * spread(64, 256), ff=8 * spread(64, 176),
                skew=round(rng.uniform(0.0, 2.0), 2))


# ---- inputs --------------------------------------------------------------------------------------------------------
def _blocks(n):
    return -(-n // BLOCK)


def _activations(gen, rows, width, dtype=BF16):
    """What a norm hands to a product: normal values, some features many times as large as the rest, a row of zeros."""
    x = torch.randn(rows, width, generator=gen, device=DEVICE)
    gain = torch.exp(0.5 * torch.randn(width, generator=gen, device=DEVICE))
    gain[torch.randint(0, width, (max(1, width // 256),), generator=gen, device=DEVICE)] *= 20.0
    x = x * gain
    if rows > 4:
        x[rows // 2] = 0.0
    return x.to(dtype)


def _matrix(gen, groups, rows, width):
    """A checkpoint's matrices: e4m3 with scales that are no powers of two; rows start on 16-byte boundaries."""
    ld = -(-width // 16) * 16
    values = torch.empty(groups * rows, ld, dtype=torch.float8_e4m3fn, device=DEVICE)
    scales = torch.empty(groups, _blocks(rows), _blocks(width), device=DEVICE)
    for g in range(groups):
        w = torch.randn(rows, width, generator=gen, device=DEVICE) * 0.02
        w *= torch.exp(0.3 * torch.randn(rows, 1, generator=gen, device=DEVICE))
        padded = torch.zeros(_blocks(rows) * BLOCK, _blocks(width) * BLOCK, device=DEVICE)
        padded[:rows, :width] = w
        tiles = padded.view(_blocks(rows), BLOCK, _blocks(width), BLOCK)
        s = tiles.abs().amax((1, 3)) / 448.0
        values[g * rows:(g + 1) * rows, :width] = (tiles / s[:, None, :, None]).view_as(padded)[:rows, :width].to(torch.float8_e4m3fn)
        scales[g] = s
    values = values.view(groups, rows, ld)[:, :, :width]
    return (values, scales) if groups > 1 else (values[0], scales[0])


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed) * 1000003 + 17)
    op, s = case["op"], dict(case)
    dtype = getattr(torch, case.get("dtype", "bfloat16"))
    if op == "norm":
        s["stream"] = torch.randn(case["rows"], case["width"], generator=gen, device=DEVICE) * 3.0
        s["delta"] = _activations(gen, case["rows"], case["width"]) if case["delta"] else None
        s["weight"] = 1.0 + 0.1 * torch.randn(case["width"], generator=gen, device=DEVICE)
        s["work"] = torch.empty_like(s["stream"])
        s["w"], s["w_scales"] = _matrix(gen, 1, case["out"], case["width"])
        s["y"] = torch.empty(case["rows"], case["out"], dtype=BF16, device=DEVICE)
    elif op == "rows":
        s["x"] = _activations(gen, case["rows"], case["width"], dtype)
    elif op == "weight":
        w = torch.randn(case["rows"], case["width"], generator=gen, device=DEVICE) * 0.02
        w[:, case["width"] // 3] *= 9.0
        s["w"] = w.to(dtype)
    elif op == "linear":
        s["x"] = _activations(gen, case["rows"], case["width"])
        s["w"], s["w_scales"] = _matrix(gen, 1, case["out"], case["width"])
        s["y"] = torch.empty(case["rows"], case["out"], dtype=dtype, device=DEVICE)
    else:
        groups = case.get("experts", 1)
        s["x"] = _activations(gen, case["rows"], case["width"])
        s["gate_up"], s["gate_up_scales"] = _matrix(gen, groups, 2 * case["ff"], case["width"])
        s["down"], s["down_scales"] = _matrix(gen, groups, case["width"], case["ff"])
        s["y"] = torch.empty(case["rows"], case["width"], dtype=BF16, device=DEVICE)
        if groups > 1:
            s["expert"], s["place"], s["most"], s["offsets"] = _choices(gen, case["rows"], groups, case["skew"])
    return s


def _choices(gen, rows, groups, skew):
    """Rows in the order of their experts: each row's expert, its place among that expert's rows, the most rows that an
    expert has, and where each expert's rows begin."""
    like = torch.exp(skew * torch.randn(groups, generator=gen, device=DEVICE))
    expert = torch.multinomial(like, rows, replacement=True, generator=gen).sort().values
    counts = torch.bincount(expert, minlength=groups)
    offsets = torch.zeros(groups + 1, dtype=torch.int32, device=DEVICE)
    offsets[1:] = counts.cumsum(0)
    place = torch.arange(rows, device=DEVICE) - offsets[expert]
    return expert, place, int(counts.max()), offsets


# ---- one pass ------------------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


_RUNTIME = []


def _runtime():
    """What an engine has one of: device, run dtype, the kernels' status word."""
    if not _RUNTIME:
        from pytorch_engine_b200.parts.runtime import Runtime
        _RUNTIME.append(Runtime(DEVICE, BF16))
    return _RUNTIME[0]


def _run_own(s):
    from pytorch_engine_b200.kernels import ops
    from pytorch_engine_b200.parts.float8 import Float8Rows, Float8Weight
    op = s["op"]
    rt = _runtime()
    if op == "norm":
        stream = s["stream"]
        if s["delta"] is not None:        # the stream is changed in place
            stream = s["work"].copy_(stream)
        rows = Float8Rows.empty(s["rows"], s["width"], DEVICE)
        ops.rmsnorm_residual_fp8(stream, s["delta"], s["weight"], rows.values, rows.scales, EPS)
        return stream, rt.linear(rows, Float8Weight(s["w"], s["w_scales"]), out=s["y"])
    if op == "rows":
        rows = Float8Rows.quantize(s["x"])
        return rows.values, rows.scales
    if op == "weight":
        w = Float8Weight.quantize(s["w"])
        return w.values, w.scales
    if op == "linear":
        return rt.linear(s["x"], Float8Weight(s["w"], s["w_scales"]), out=s["y"], out_dtype=s["y"].dtype)
    gate_up, down = Float8Weight(s["gate_up"], s["gate_up_scales"]), Float8Weight(s["down"], s["down_scales"])
    if op == "ffn":
        return rt.float8_feed_forward(s["x"], gate_up, down, s["y"])
    return rt.float8_experts(s["x"], s["offsets"], gate_up, down, s["y"])


def _tiles(x, row_block):
    """``x`` cut into blocks of ``row_block`` rows and 128 columns, filled up with zeros: [row blocks, row_block, column blocks, 128]."""
    rows, width = x.shape
    x = torch.nn.functional.pad(x, (0, _blocks(width) * BLOCK - width, 0, -rows % row_block))
    return x.view(-(-rows // row_block), row_block, _blocks(width), BLOCK)


def _quantize(x, row_block):
    """The stored values (as 32-bit floats) and the scales of ``x`` in 32 bits, [row blocks, column blocks]."""
    rows, width = x.shape
    t = _tiles(x, row_block)
    m, e = torch.frexp(t.abs().amax((1, 3)))                        # a = m * 2^e, m in [0.5, 1): 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, e - 8, e - 9)
    e = torch.where(m == 0.0, torch.full_like(e, -126), e).clamp(min=-126)
    scales = ((e + 127) << 23).to(torch.int32).view(torch.float32)  # 2^e
    q = (t / scales[:, None, :, None]).to(torch.float8_e4m3fn).to(torch.float32)
    return q.reshape(t.shape[0] * row_block, -1)[:rows, :width], scales


def _dequantized(x):
    """Rows as the product sees them: quantised in blocks of 128 features, times their scales."""
    q, scales = _quantize(x.to(torch.float32), 1)
    return q * scales.repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def _weights(values, scales):
    """A matrix (or several) as 32-bit floats."""
    rows, width = values.shape[-2:]
    s = scales.repeat_interleave(BLOCK, -2)[..., :rows, :].repeat_interleave(BLOCK, -1)[..., :width]
    return values.to(torch.float32) * s


def _padded(s, x):
    """Rows grouped by expert as [experts, most rows, width], zeros where an expert has fewer."""
    out = torch.zeros(s["experts"], s["most"], x.shape[1], dtype=x.dtype, device=x.device)
    out[s["expert"], s["place"]] = x
    return out


def _run_plain(s):
    op = s["op"]
    if op == "norm":
        h = s["stream"] if s["delta"] is None else s["stream"] + s["delta"].to(torch.float32)
        # the normed row is rounded to bfloat16, as what any norm hands on
        x = (h * torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) * s["weight"]).to(BF16)
        return h, (_dequantized(x) @ _weights(s["w"], s["w_scales"]).t()).to(BF16)
    if op == "rows":
        q, scales = _quantize(s["x"].to(torch.float32), 1)
        return q.to(torch.float8_e4m3fn), scales.t()
    if op == "weight":
        q, scales = _quantize(s["w"].to(torch.float32), BLOCK)
        return q.to(torch.float8_e4m3fn), scales
    if op == "linear":
        return (_dequantized(s["x"]) @ _weights(s["w"], s["w_scales"]).t()).to(s["y"].dtype)
    gate_up, down = _weights(s["gate_up"], s["gate_up_scales"]), _weights(s["down"], s["down_scales"])
    x = _dequantized(s["x"])
    if op == "ffn":
        g, u = (x @ gate_up.t()).chunk(2, 1)
        h = (g * torch.sigmoid(g) * u).to(BF16)
        return (_dequantized(h) @ down.t()).to(BF16)
    at = (s["expert"], s["place"])
    g, u = torch.bmm(_padded(s, x), gate_up.transpose(1, 2))[at].chunk(2, 1)
    h = (g * torch.sigmoid(g) * u).to(BF16)
    return torch.bmm(_padded(s, _dequantized(h)), down.transpose(1, 2))[at].to(BF16)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    op, m, k = case["op"], case["rows"], case["width"]
    size = 4 if case.get("dtype") == "float32" else 2
    if op == "norm":
        stream = 4 + 2 + 4 if case["delta"] else 4
        return {"bytes": m * k * stream + 4 * k + case["out"] * k + 2 * m * case["out"], "flops": 2 * m * k * case["out"]}
    if op == "rows":
        return {"bytes": m * k * (size + 1) + 4 * m * _blocks(k), "flops": 3 * m * k}
    if op == "weight":
        return {"bytes": m * k * (size + 1) + 4 * _blocks(m) * _blocks(k), "flops": 3 * m * k}
    if op == "linear":
        n = case["out"]
        return {"bytes": n * k + 2 * m * k + size * m * n, "flops": 2 * m * n * k}
    ff = case["ff"]
    # every expert's weights are read where there are rows enough for all of them
    groups = min(case.get("experts", 1), m)
    return {"bytes": groups * 3 * ff * k + 4 * m * k, "flops": 6 * m * ff * k}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------
def _e4m3_64(x):
    """The nearest e4m3 value, ties to even, of 64-bit numbers of at most 448."""
    a = x.abs()
    exponent = torch.floor(torch.log2(torch.where(a > 0, a, torch.ones_like(a)))).clamp(min=-6.0)
    step = torch.exp2(exponent - 3.0)
    return torch.round(x / step) * step          # torch.round: half to even


def _blockwise_64(x, tall):
    """Stored values and scales of a 64-bit matrix, block by block; ``tall``: the rows of a block."""
    rows, width = x.shape
    big = x.new_zeros(-(-rows // tall) * tall, -(-width // BLOCK) * BLOCK)
    big[:rows, :width] = x
    cells = big.unfold(0, tall, tall).unfold(1, BLOCK, BLOCK)       # [row blocks, column blocks, tall, 128]
    top = cells.abs().flatten(2).max(2).values
    e = torch.ceil(torch.log2(torch.where(top > 0, top, torch.full_like(top, 1e-60)) / 448.0)).clamp(min=-126.0)
    e = torch.where(top > 448.0 * torch.exp2(e), e + 1.0, e)        # a logarithm may be off by its last bit
    e = torch.where((top <= 448.0 * torch.exp2(e - 1.0)) & (e > -126.0), e - 1.0, e)
    scales = torch.exp2(e)
    q = _e4m3_64(cells / scales[:, :, None, None])
    return q.permute(0, 2, 1, 3).reshape(big.shape)[:rows, :width], scales


def _rows_64(x):
    q, scales = _blockwise_64(x, 1)
    return q * scales.repeat_interleave(BLOCK, dim=1)[:, :x.shape[1]]


def _matrix_64(values, scales):
    """One matrix in 64 bits: every element times the scale of the block that it lies in."""
    row, col = (torch.arange(n, device=values.device) // BLOCK for n in values.shape)
    return values.to(torch.float64) * scales.to(torch.float64)[row][:, col]


def exact(case, seed):
    op = case["op"]
    if work(case)["flops"] > EXACT_FLOPS:
        return None
    s = prepare(case, seed)
    wide = torch.float64
    if op == "norm":
        h = s["stream"].to(wide)
        if s["delta"] is not None:
            h = h + s["delta"].to(wide)
        x = h / torch.sqrt((h * h).mean(1, keepdim=True) + EPS) * s["weight"].to(wide)
        return h, _rows_64(x.to(BF16).to(wide)) @ _matrix_64(s["w"], s["w_scales"]).t()
    if op == "rows":
        q, scales = _blockwise_64(s["x"].to(wide), 1)
        return q, scales.t()
    if op == "weight":
        return _blockwise_64(s["w"].to(wide), BLOCK)
    if op == "linear":
        return _rows_64(s["x"].to(wide)) @ _matrix_64(s["w"], s["w_scales"]).t()
    ff = case["ff"]
    x = _rows_64(s["x"].to(wide))
    y = torch.zeros_like(x)
    for g in range(case.get("experts", 1)):
        one = "experts" not in case
        mine = slice(None) if one else s["expert"] == g
        gate_up, down = (_matrix_64(*(t if one else t[g] for t in (s[n], s[n + "_scales"]))) for n in ("gate_up", "down"))
        both = x[mine] @ gate_up.t()
        h = both[:, :ff] / (1.0 + torch.exp(-both[:, :ff])) * both[:, ff:]
        y[mine] = (_rows_64(h.to(BF16).to(wide)) if h.shape[0] else h) @ down.t()
    return y
