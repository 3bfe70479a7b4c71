"""Helpers for parts that own projection matrices."""
from __future__ import annotations

from typing import Iterable, Sequence, Union

import torch

from .float8 import Float8Weight


def fuse_rows(runtime, tensors: Sequence[torch.Tensor]) -> torch.Tensor:
    """Sibling projections stacked along the output features into one matrix, in the run dtype
    (q|k|v and gate|up, as the reference does: pygguf_engine/quant_kernels.py:1874-1893)."""
    parts = [t.to(device=runtime.device, dtype=runtime.dtype) for t in tensors]
    return torch.cat(parts, dim=0).contiguous()


def wide(tensor, dtype: torch.dtype) -> torch.Tensor:
    """A weight as numbers of 16 or 32 bits: a checkpoint's 8-bit matrix times its scales, in the run's ``dtype``; any other tensor
    as it is."""
    return tensor.dequantize(dtype) if type(tensor) is Float8Weight else tensor


def projection(runtime, tensors: Sequence, multiple: int = 1) -> Union[torch.Tensor, Float8Weight]:
    """A part's projection, the given matrices under each other and rows of zeros up to a multiple of ``multiple`` (of at most 128
    rows, a power of two): as ``fuse_rows`` makes it, or 8-bit.  A checkpoint's 8-bit matrices stay as they are where the run takes
    them (``runtime.takes_float8``) and each but the last ends with a block of rows; with ``runtime.float8`` everything else is
    quantised when the model is built."""
    stored = [type(t) is Float8Weight for t in tensors]
    zeros = -sum(t.shape[0] for t in tensors) % multiple
    if runtime.takes_float8() and all(stored) and Float8Weight.stacks_rows(tensors):
        mine = [t.to(runtime.device) for t in tensors]
        mine[-1] = mine[-1].with_zero_rows(zeros)
        return Float8Weight.cat_rows(mine) if len(mine) > 1 else mine[0]
    if len(tensors) == 1 and not stored[0] and not zeros and not (runtime.takes_float8() and runtime.float8):
        return runtime.adopt(tensors[0])
    parts = [wide(t, runtime.dtype) for t in tensors]
    if zeros:
        parts.append(torch.zeros((zeros, tensors[0].shape[1]), dtype=runtime.dtype, device=parts[0].device))
    whole = fuse_rows(runtime, parts)
    return Float8Weight.quantize(whole) if runtime.takes_float8() and runtime.float8 else whole


def quantized_stack(matrices: Iterable[torch.Tensor]) -> Float8Weight:
    """Matrices of one shape, each quantised (or 8-bit already), as one weight ``[G, N, K]``."""
    return Float8Weight.stack([m if type(m) is Float8Weight else Float8Weight.quantize(m) for m in matrices])
