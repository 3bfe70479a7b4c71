"""Weights and rows in 8-bit floating point, as the products of csrc/gemm_fp8.cu read them.

A matrix is kept as e4m3 values and a float32 scale for each 128 x 128 elements, rows on their way into a product as e4m3
values and a scale for each 128 features.  What this package quantises itself gets scales that are powers of two
(csrc/quantize_fp8.cu); a checkpoint's may be any.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from ..kernels import ops
from ..kernels.ops import FP8, FP8_BLOCK, fp8_blocks


def _padded_empty(shape, device) -> torch.Tensor:
    """Uninitialised e4m3 ``[..., K]`` whose rows start on 16-byte boundaries."""
    k = shape[-1]
    if k % 16 == 0:
        return torch.empty(*shape, dtype=FP8, device=device)
    strides = [1, (k + 15) // 16 * 16]
    for n in reversed(shape[1:-1]):
        strides.append(strides[-1] * n)
    return torch.empty_strided(shape, strides[::-1], dtype=FP8, device=device)


class Float8Rows:
    """``values [M, K]`` (e4m3) and ``scales [fp8_blocks(K), M]`` (float32).  ``powers``: the scales are powers of two, as this
    package's conversions make them (``empty`` and ``of_buffers`` are for those to fill)."""

    __slots__ = ("values", "scales", "powers")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor, powers: bool = False) -> None:
        self.values, self.scales, self.powers = values, scales, powers

    @property
    def shape(self) -> torch.Size:
        return self.values.shape

    @property
    def device(self) -> torch.device:
        return self.values.device

    @classmethod
    def empty(cls, rows: int, width: int, device) -> "Float8Rows":
        return cls(_padded_empty((rows, width), device), torch.empty(fp8_blocks(width), rows, dtype=torch.float32, device=device), True)

    @classmethod
    def of_buffers(cls, ctx, name: str, rows: int, width: int) -> "Float8Rows":
        """Rows in the step's buffers ``name`` (one name, one set of rows at a time)."""
        values = ctx.buffer(name + ".values", (rows, (width + 15) // 16 * 16), FP8)[:, :width]
        return cls(values, ctx.buffer(name + ".scales", (fp8_blocks(width), rows), torch.float32), True)

    @classmethod
    def quantize(cls, x: torch.Tensor, row_map: Optional[torch.Tensor] = None, live: Optional[torch.Tensor] = None,
                 status: Optional[torch.Tensor] = None) -> "Float8Rows":
        """``x [rows, K]`` in new storage (``row_map``, ``live``: see ``ops.quantize_rows_fp8``)."""
        return cls(*ops.new_rows_fp8(x, row_map, live, status), True)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        s = self.scales.repeat_interleave(FP8_BLOCK, 0)[:self.values.shape[1]].t()
        return (self.values.to(torch.float32) * s).to(dtype)


def _all_powers(weights) -> Optional[bool]:
    known = [w.powers for w in weights]
    return False if False in known else None if None in known else True


class Float8Weight:
    """``values [N, K]`` (e4m3) and ``scales [fp8_blocks(N), fp8_blocks(K)]`` (float32); or several such matrices stacked in
    front, ``[G, N, K]`` and ``[G, ...]``.  Rows start on 16-byte boundaries (``to`` makes it so).  ``powers``: whether all scales are
    powers of two, which makes products of many rows faster; None: not known (``to`` finds out).  What the methods here make can go
    into a product at once; for values written by other means see ``ops.settle_weights``."""

    __slots__ = ("values", "scales", "powers")
    dtype = FP8

    def __init__(self, values: torch.Tensor, scales: torch.Tensor, powers: Optional[bool] = None) -> None:
        shape = values.shape
        if values.dtype is not FP8 or scales.dtype is not torch.float32:
            raise ValueError(f"an 8-bit weight is float8_e4m3fn with float32 scales, got {values.dtype} and {scales.dtype}")
        want = (*shape[:-2], (shape[-2] + 127) >> 7, (shape[-1] + 127) >> 7)
        if scales.shape != want:
            raise ValueError(f"an 8-bit weight {list(values.shape)} has scales {list(want)}, got {list(scales.shape)}")
        self.values, self.scales, self.powers = values, scales, powers

    @property
    def shape(self) -> torch.Size:
        return self.values.shape

    @property
    def device(self) -> torch.device:
        return self.values.device

    def nbytes(self) -> int:
        return self.values.numel() + 4 * self.scales.numel()

    def __getitem__(self, i: int) -> "Float8Weight":
        """One of several stacked matrices."""
        return Float8Weight(self.values[i], self.scales[i], self.powers or None)

    @classmethod
    def quantize(cls, w: torch.Tensor) -> "Float8Weight":
        """A matrix ``[N, K]`` on a CUDA device, quantised into new storage."""
        if w.dim() != 2:
            raise ValueError(f"a matrix is quantised, got {list(w.shape)}")
        values = _padded_empty(w.shape, w.device)
        scales = torch.empty(fp8_blocks(w.shape[0]), fp8_blocks(w.shape[1]), dtype=torch.float32, device=w.device)
        ops.quantize_weight_fp8(w, values, scales)
        return cls(values, scales, True)

    @classmethod
    def _settled(cls, values: torch.Tensor, scales: torch.Tensor, powers: Optional[bool]) -> "Float8Weight":
        """A weight that copies in front of this call have written."""
        ops.settle_weights(values)
        return cls(values, scales, powers)

    @classmethod
    def stack(cls, weights: Sequence["Float8Weight"]) -> "Float8Weight":
        """Matrices of one shape as one weight ``[G, N, K]``."""
        first = weights[0]
        values = _padded_empty((len(weights), *first.shape), first.device)
        for i, w in enumerate(weights):
            values[i].copy_(w.values)
        return cls._settled(values, torch.stack([w.scales for w in weights]).contiguous(), _all_powers(weights))

    @staticmethod
    def stacks_rows(weights: Sequence["Float8Weight"]) -> bool:
        """Whether ``cat_rows`` keeps every element's block: all but the last must fill their blocks of rows."""
        return all(w.shape[0] % FP8_BLOCK == 0 for w in weights[:-1])

    @classmethod
    def cat_rows(cls, weights: Sequence["Float8Weight"]) -> "Float8Weight":
        """Matrices under each other (see ``stacks_rows``)."""
        if not cls.stacks_rows(weights):
            raise ValueError("8-bit weights whose rows end inside a block cannot be put under each other")
        values = _padded_empty((sum(w.shape[0] for w in weights), weights[0].shape[1]), weights[0].device)
        at = 0
        for w in weights:
            values[at:at + w.shape[0]].copy_(w.values)
            at += w.shape[0]
        return cls._settled(values, torch.cat([w.scales for w in weights]).contiguous(), _all_powers(weights))

    def with_zero_rows(self, rows: int) -> "Float8Weight":
        """The matrix with so many rows of zeros behind its last one, in whose block they must still lie."""
        if rows == 0:
            return self
        n, k = self.shape
        if fp8_blocks(n + rows) != fp8_blocks(n):
            raise ValueError(f"{rows} more rows do not fit the last block of an 8-bit weight {list(self.shape)}")
        values = _padded_empty((n + rows, k), self.device)
        values[:n].copy_(self.values)
        values[n:].view(torch.uint8).zero_()
        return self._settled(values, self.scales, self.powers)

    def to(self, device) -> "Float8Weight":
        """On ``device``, with rows on 16-byte boundaries, and ``powers`` known (for which the host waits for the device)."""
        values, scales = self.values, self.scales.to(device).contiguous()
        if values.device != torch.device(device) or values.stride(-2) % 16 or values.data_ptr() % 16:
            values = _padded_empty(self.shape, device)
            values.copy_(self.values)
        powers = self.powers
        if powers is None:
            bits = scales.view(torch.int32)
            powers = bool(((bits & 0x7fffff) == 0).logical_and_(bits > 0).logical_and_(bits != 0x7f800000).all())
        return self._settled(values, scales, powers)

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        n, k = self.shape[-2:]
        s = self.scales.repeat_interleave(FP8_BLOCK, -2)[..., :n, :].repeat_interleave(FP8_BLOCK, -1)[..., :k]
        return (self.values.to(torch.float32) * s).to(dtype)
