"""Group norm with an activation on the rows of ragged samples, channels last:
what stands in front of a convolution in a residual block on sparse voxels.  An
addition: the reference has the convolutions only, and its callers loop over the
samples with torch's norm."""
from typing import Optional

import torch

from .. import _native
from . import utils

ACTIVATIONS = (None, "silu")


def sparse_group_norm(feats: torch.Tensor, offsets: Optional[torch.Tensor], num_groups: int, weight: Optional[torch.Tensor] = None,
                      bias: Optional[torch.Tensor] = None, eps: float = 1e-5, activation: Optional[str] = None) -> torch.Tensor:
    """``activation((x - mean) / sqrt(var + eps) * weight + bias)`` with the mean and the (biased) variance of each
    sample's rows over each group of ``C / num_groups`` neighbouring channels.

    Args:
        feats: [N, C] features (float16, bfloat16 or float32, CUDA), or with ``offsets`` None any [B, ..., C] whose leading
            entries are the samples ([N, C] is one sample then).
        offsets: [B + 1] int32 or int64 on the GPU: sample ``b`` has the rows ``offsets[b]`` to ``offsets[b + 1] - 1``
            (``ops.utils.sample_offsets`` makes them from coordinates).  Samples may be empty.  Rows of no sample come
            out as zeros, and so does their gradient, whatever they hold.
        num_groups: a divisor of C.
        weight, bias: [C] in the features' type or float32 (both in the same), or None.
        eps: added to the variance.
        activation: None or "silu".

    Returns:
        features of the shape and type of ``feats``; sums and statistics are float32 or wider, the result is rounded once.
        Differentiable (once) in feats, weight and bias.  Offsets that do not ascend or leave the rows raise from a later
        call, as every error that the device finds.
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f"Unsupported activation {activation!r}")
    silu = activation == "silu"
    out = _native.ext().group_norm(feats, offsets, num_groups, weight, bias, eps, silu)
    if out is not None:
        return out
    assert feats.dim() >= 2, f"Features must be of shape [N, C] or [B, ..., C], got {tuple(feats.shape)}"
    C = feats.shape[-1]
    if not isinstance(num_groups, int) or num_groups < 1 or C % num_groups != 0:
        raise ValueError(f"the number of groups ({num_groups}) must divide the channels ({C})")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if C < 1 or C > 65536:
        raise ValueError(f"1 to 65536 channels are supported, got {C}")
    if offsets is not None:
        assert feats.dim() == 2, f"Features must be of shape [N, C] where there are offsets, got {tuple(feats.shape)}"
        offsets = utils.check_offsets(offsets, feats)
    utils.check_feature_dtype(feats)
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None:
            assert p.shape == (C,), f"{name} must be of shape [{C}], got {tuple(p.shape)}"
            if p.dtype not in (feats.dtype, torch.float32):
                raise TypeError(f"{name} must be of the features' type or float32, got {p.dtype}")
            if p.device != feats.device:
                raise ValueError(f"{name} must be on the features' device")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight and bias must be of one type, got {weight.dtype} and {bias.dtype}")
    utils.require_cuda(feats)
    utils.refuse_tangents(feats, weight, bias)
    samples = offsets.shape[0] - 1 if offsets is not None else 1 if feats.dim() == 2 else feats.shape[0]
    if feats.numel() // C >= 2 ** 31 or samples >= 2 ** 24:
        raise ValueError("at most 2^31 - 1 rows and 2^24 - 1 samples are supported")
    if feats.numel() == 0:
        return utils.zeros_with_history((tuple(feats.shape), feats.dtype, feats.device), feats, weight, bias)
    out = _native.ext().group_norm(utils.kernel_layout(feats), offsets, num_groups, weight.contiguous().resolve_neg() if weight is not None else None,
                                   bias.contiguous().resolve_neg() if bias is not None else None, float(eps), silu)
    if out is None:
        raise ValueError("sparse_group_norm: arguments that the kernels do not take")
    return out
