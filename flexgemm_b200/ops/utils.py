"""Host helpers shared by the ops."""
from typing import Tuple

import torch

from .. import _cabi, _native


def hashmap_key_bits(spatial_size) -> int:
    """32-bit keys while B*W*H*D < 2^32, else 64-bit -- the rule of
    init_hashmap in the reference (flex_gemm/ops/utils.py:4-19)."""
    N, C, W, H, D = [int(s) for s in spatial_size]
    vol = N * W * H * D
    if vol < 2 ** 32:
        return 32
    if vol < 2 ** 64:
        return 64
    raise ValueError(f"The spatial size is too large to fit in a hashmap. Get volumn {vol} > 2^64.")


def init_hashmap(spatial_size, hashmap_size: int, device, with_values: bool = True):
    """The reference's table allocation (flex_gemm/ops/utils.py:4-19): keys of
    ``hashmap_size`` slots filled with all ones -- uint32 while B*W*H*D < 2^32,
    else uint64 -- and, with ``with_values``, an uninitialised uint32 value
    tensor.  Returns ``(hashmap_keys, hashmap_vals)`` or ``hashmap_keys``; these are
    what ``kernels.cuda.hashmap_insert*`` / ``hashmap_lookup*`` take."""
    dtype = torch.uint32 if hashmap_key_bits(spatial_size) == 32 else torch.uint64
    hashmap_keys = torch.full((int(hashmap_size),), torch.iinfo(dtype).max, dtype=dtype, device=device)
    if with_values:
        return hashmap_keys, torch.empty((int(hashmap_size),), dtype=torch.uint32, device=device)
    return hashmap_keys


def init_table(spatial_size, hashmap_size: int, device) -> Tuple[torch.Tensor, int]:
    """Storage for the library's own packed coordinate table of ``hashmap_size``
    slots, as the neighbour-map and grid-sample kernels use it: ``(table,
    key_bits)``.  One opaque buffer (key and row share a 64-bit slot for 32-bit
    keys); the kernels clear it themselves, and it never reaches the caller --
    the reference drops its table after the map is built as well
    (flex_gemm/ops/spconv/submanifold_conv3d.py:57-71)."""
    key_bits = hashmap_key_bits(spatial_size)
    nbytes = _cabi.check_size(_cabi.lib().fgb_hash_table_bytes(int(hashmap_size), key_bits), "fgb_hash_table_bytes")
    table = torch.empty((max(nbytes, 8) + 7) // 8, dtype=torch.int64, device=device)
    return table, key_bits


# --------------------------------------------------------------------------
# layers on ragged rows
# --------------------------------------------------------------------------
def sample_offsets(coords: torch.Tensor, batch: int) -> torch.Tensor:
    """Row ranges of the samples: int32 [batch + 1] on the GPU, sample ``b`` has the rows ``offsets[b]`` to
    ``offsets[b + 1] - 1``.  ``coords``: int32 [N, 4] rows (b, x, y, z) grouped by ascending ``b``, as the convolutions
    take and give them.  Nothing waits for the GPU; rows in another order raise from a later call."""
    assert coords.dim() == 2 and coords.shape[1] == 4, f"Coords must be of shape [N, 4], got {tuple(coords.shape)}"
    if not 1 <= batch < 2 ** 24:
        raise ValueError(f"1 to 2^24 - 1 samples are supported, got {batch}")
    if coords.shape[0] >= 2 ** 31:
        raise ValueError("at most 2^31 - 1 rows are supported")
    coords = _int32_coords(coords, batch)
    require_cuda(coords, "coords")
    out = _native.ext().sample_offsets(coords, batch)
    if out is None:
        out = _native.ext().sample_offsets(kernel_layout(coords), batch)
    return out


def _int32_coords(coords: torch.Tensor, batch: int) -> torch.Tensor:
    """Other integers are cut to the samples before they are cast: one of 2^32 must not come out as sample 0."""
    if coords.dtype == torch.int32:
        return coords
    if coords.dtype not in (torch.int64, torch.int16, torch.int8, torch.uint8):
        raise TypeError(f"unsupported coords dtype {coords.dtype}: expected int32")
    return (coords.clamp(-1, batch) if coords.dtype == torch.int64 else coords).int()


def require_cuda(t: torch.Tensor, name: str = "feats") -> None:
    if not t.is_cuda:
        raise NotImplementedError(f"{name} must be a CUDA tensor: flexgemm_b200 has no CPU implementation")


def check_feature_dtype(t: torch.Tensor) -> None:
    if t.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise TypeError(f"unsupported feature dtype {t.dtype}: expected float16, bfloat16 or float32")


def check_offsets(offsets: torch.Tensor, feats: torch.Tensor) -> torch.Tensor:
    """Offsets as the kernels take them."""
    assert offsets.dim() == 1 and offsets.shape[0] >= 2, f"Offsets must be of shape [B + 1], got {tuple(offsets.shape)}"
    if offsets.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"offsets must be int32 or int64, got {offsets.dtype}")
    if offsets.device != feats.device:
        raise ValueError("offsets must be on the features' device")
    return offsets.contiguous()


def refuse_tangents(*tensors) -> None:
    """Forward-mode derivatives do not exist: an input that carries a tangent is refused, not stripped of it."""
    for t in tensors:
        if t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("forward-mode derivatives are not supported")


def kernel_layout(t: torch.Tensor) -> torch.Tensor:
    """``t`` contiguous, at an address that 16-byte loads can take (a copy only where it is not)."""
    t = t.contiguous().resolve_neg()
    return t if t.numel() == 0 or t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


class _Zeros(torch.autograd.Function):
    @staticmethod
    def forward(ctx, like, *inputs):
        ctx.like = [(t.shape, t.dtype, t.device) if t is not None else None for t in inputs]
        shape, dtype, device = like
        return torch.zeros(shape, dtype=dtype, device=device)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, _):
        return (None, *(torch.zeros(k[0], dtype=k[1], device=k[2]) if k is not None and need else None
                        for k, need in zip(ctx.like, ctx.needs_input_grad[1:])))


def zeros_with_history(like, *inputs):
    """Zeros for a call without rows (``like``: shape, dtype, device), through which zero gradients reach the inputs."""
    return _Zeros.apply(like, *inputs)
