"""Products grouped by ragged row ranges: every sample, or every expert that rows
have been dealt to, has a matrix of its own.  An addition: the reference's only
products are the convolutions, whose kernels (tcgen05 tiles, fp32 accumulation,
``allow_tf32``) this one stands beside."""
from typing import Optional

import torch

from .. import _cabi, _native
from ..kernels import config
from . import utils


def sparse_grouped_linear(feats: torch.Tensor, offsets: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``feats[r] @ weight[g].T + bias[g]`` for the rows ``r`` of each group ``g``.

    Args:
        feats: [N, Ci] features (float16, bfloat16 or float32, CUDA), the rows of a group together.
        offsets: [G + 1] int32 or int64 on the GPU: group ``g`` has the rows ``offsets[g]`` to ``offsets[g + 1] - 1``
            (for samples, ``ops.utils.sample_offsets`` makes them from coordinates).  Groups may be empty.  Rows of no
            group come out as zeros, and so does their gradient, whatever they hold.
        weight: [G, Co, Ci] of the features' type; at most 2048 groups.
        bias: [G, Co] of the features' type, or None.

    Returns:
        [N, Co] of the features' type; sums are float32, the result is rounded once.  float32 follows
        ``kernels.config.allow_tf32`` at the time a pass runs: a product is off by 3 * 2^-16 of its value at most where it is set
        (a term of the bias gradient by 2^-16), by 2^-21 otherwise (an infinity among float32 inputs gives NaN).  Differentiable (once) in feats, weight and bias.  Offsets that do not
        ascend or leave the rows raise from a later call, as every error that the device finds.
    """
    out = _native.ext().grouped_linear(feats, offsets, weight, bias, config.allow_tf32)
    if out is not None:
        return out
    assert feats.dim() == 2, f"Features must be of shape [N, Ci], got {tuple(feats.shape)}"
    assert weight.dim() == 3, f"Weights must be of shape [G, Co, Ci], got {tuple(weight.shape)}"
    G, Co, Ci = weight.shape
    assert feats.shape[1] == Ci, f"Input channels ({feats.shape[1]}) should match weight channels ({Ci})"
    offsets = utils.check_offsets(offsets, feats)
    assert offsets.shape[0] == G + 1, f"Offsets must have an entry more than there are groups ({G}), got {offsets.shape[0]}"
    most = _cabi.lib().fgb_grouped_linear_max_groups()
    if not 1 <= G <= most:
        raise ValueError(f"1 to {most} groups are supported, got {G}")
    if not (1 <= Ci <= 65536 and 1 <= Co <= 65536):
        raise ValueError(f"1 to 65536 channels are supported, got {Ci} and {Co}")
    if feats.shape[0] >= 2 ** 31 - 256:
        raise ValueError("at most 2^31 - 257 rows are supported")
    utils.check_feature_dtype(feats)
    if weight.dtype != feats.dtype or (bias is not None and bias.dtype != feats.dtype):
        raise TypeError(f"weight and bias must be of the features' type ({feats.dtype})")
    if bias is not None:
        assert bias.shape == (G, Co), f"Bias must be of shape [{G}, {Co}], got {tuple(bias.shape)}"
    utils.require_cuda(feats)
    if weight.device != feats.device or (bias is not None and bias.device != feats.device):
        raise ValueError("weight and bias must be on the features' device")
    utils.refuse_tangents(feats, weight, bias)
    if feats.shape[0] == 0:
        return utils.zeros_with_history(((0, Co), feats.dtype, feats.device), feats, weight, bias)
    out = _native.ext().grouped_linear(utils.kernel_layout(feats), offsets, utils.kernel_layout(weight),
                                       bias.contiguous().resolve_neg() if bias is not None else None, config.allow_tf32)
    if out is None:
        raise ValueError("sparse_grouped_linear: arguments that the kernels do not take")
    return out
