"""Species embedding: the rows of a table that an atomistic model starts from.

No counterpart in the reference, which ends at the neighbor list.
"""

from __future__ import annotations

from ctypes import c_float
from math import isfinite

import torch
from torch import Tensor

from ._extensions import check_device, load_torch_native

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def species_embedding(species: Tensor, weight: Tensor, *, scale: float = 1.0) -> Tensor:
    """``scale * weight[species]``, differentiable in ``weight``.

    ``species``: int32 or int64 of any shape, rows of ``weight`` (V, C), which is float32, bfloat16
    or float16.  The result has the shape ``(*species.shape, C)`` and the type of ``weight``.

    The gradient sums the rows of equal species after a stable sort, in 32 bits and in an order that
    the inputs alone fix, so that it is the same bits in every run.  A species outside the table gives
    a row of NaN (the call does not wait for the device to refuse it) and adds to no gradient.
    """
    for name, tensor in (("species", species), ("weight", weight)):
        if not isinstance(tensor, Tensor):
            raise TypeError(f"{name} must be a PyTorch tensor, not {type(tensor).__name__}")
    if species.dtype not in (torch.int32, torch.int64):
        raise ValueError("species must have dtype int32 or int64")
    if weight.ndim != 2 or weight.shape[1] == 0:
        raise ValueError("weight must have shape (V, C) with C > 0")
    if weight.dtype not in _TYPES:
        raise ValueError("weight must have dtype float32, bfloat16 or float16")
    if species.device != weight.device:
        raise ValueError("species and weight must be on the same device")
    scale = c_float(float(scale)).value  # as the kernels take it
    if not isfinite(scale):
        raise ValueError("scale must be finite in 32 bits")
    if not weight.is_cuda:
        raise RuntimeError("species_embedding runs on ROCm (HIP) devices; move the tensors to a GPU")
    check_device(weight.device.index)
    return load_torch_native().species_embedding(species, weight, scale)


__all__ = ["species_embedding"]
