"""Embedding of voxel labels: rows of a table by index, scaled, with the
gradient by sorted indices.  An addition: the reference has no such call (its
callers use torch's lookup).  It stands beside ``grid_sample_3d``, which reads
rows by coordinate."""
from typing import Optional

import torch

from .. import _native
from . import utils


def sparse_embedding(indices: torch.Tensor, table: torch.Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * table[indices]``.

    Args:
        indices: int32 or int64 of any shape, on the GPU, in [0, V).
        table: [V, C] float16, bfloat16 or float32 on the same GPU.
        scale: factor of every row (applied in float32, the result is rounded once).
        padding_idx: an index whose row gets no gradient.

    Returns:
        [*indices.shape, C] of the table's type.  Differentiable (once) in the table: the gradient is dense, the rows of an
        index are added in float32 in a fixed order, so it does not change from run to run.  An index outside [0, V) gives a row of
        zeros and no gradient, and raises from a later call, as every error that the device finds.
    """
    pad = -1 if padding_idx is None else padding_idx
    if padding_idx is None or (isinstance(padding_idx, int) and padding_idx >= 0):
        out = _native.ext().embedding(indices, table, scale, pad)
        if out is not None:
            return out
    assert table.dim() == 2, f"The table must be of shape [V, C], got {tuple(table.shape)}"
    if indices.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"indices must be int32 or int64, got {indices.dtype}")
    V, C = table.shape
    if V < 1 or V >= 2 ** 31 - 1 or C < 1 or C > 65536:
        raise ValueError(f"tables of 1 to 2^31 - 2 rows and 1 to 65536 channels are supported, got {V} x {C}")
    if padding_idx is not None and not 0 <= padding_idx < V:
        raise ValueError(f"padding_idx must be in [0, {V}), got {padding_idx}")
    if indices.numel() >= 2 ** 30:
        raise ValueError("at most 2^30 - 1 indices are supported")
    utils.check_feature_dtype(table)
    utils.require_cuda(table)
    if indices.device != table.device:
        raise ValueError("indices must be on the table's device")
    utils.refuse_tangents(table)
    if indices.numel() == 0:
        return utils.zeros_with_history((tuple(indices.shape) + (C,), table.dtype, table.device), table)
    out = _native.ext().embedding(indices.contiguous(), utils.kernel_layout(table), float(scale), pad)
    if out is None:
        raise ValueError("sparse_embedding: arguments that the kernels do not take")
    return out
