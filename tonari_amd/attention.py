"""Attention over the atoms of a structure and along the pairs of a neighbor list.

For a query and a key at distance r, with x = scale q.k and a cap c,

    score = c tanh(x / c) - slopes[head] r        (x - slopes[head] r without a cap)

and the output is the softmax-weighted sum of the values.  ``structure_attention`` takes the batch
layout of ``neighbor_list`` (positions and batch_ptr) and attends to all atoms of the same structure;
``neighbor_attention`` attends along a list's pairs (i, j, d), whose distances may be those to periodic
images.  Both are differentiable in everything that is real; the gradient of d goes on through the
list to positions and cell.  Query heads may share key and value heads.

A gradient's own graph (``create_graph=True``, as training on forces takes) is built of torch operations
over all pairs of a query and a key: it holds several tensors of pairs x heads x dim floats (a structure
of 1,000 atoms with 8 heads of 64 has 2 GB in each), waits for the device to count the pairs, and its
sums are torch's, whose order may change from run to run.

No counterpart in the reference, which ends at the neighbor list.
"""

from __future__ import annotations

from ctypes import c_float
from math import isfinite, sqrt
from typing import NamedTuple

import torch
from torch import Tensor

from ._extensions import check_device, load_torch_native

_TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _check_tensors(**tensors: object) -> None:
    for name, tensor in tensors.items():
        if not isinstance(tensor, Tensor):
            raise TypeError(f"{name} must be a PyTorch tensor, not {type(tensor).__name__}")


def _check_heads(q: Tensor, k: Tensor, v: Tensor, slopes: Tensor) -> None:
    if q.ndim != 3 or k.ndim != 3:
        raise ValueError("q and k must have shape (N, heads, dim)")
    if v.shape != k.shape:
        raise ValueError("k and v must have the same shape")
    if q.dtype not in _TYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must have the same dtype: float32, bfloat16 or float16")
    if q.shape[2] != k.shape[2]:
        raise ValueError("q and k must have the same head dimension")
    if q.shape[2] % 8 != 0 or not 8 <= q.shape[2] <= 128:
        raise ValueError("the head dimension must be a multiple of 8, from 8 to 128")
    if q.shape[1] == 0 or k.shape[1] == 0 or q.shape[1] % k.shape[1] != 0:
        raise ValueError("the heads of q must be a multiple of those of k and v")
    if slopes.shape != (q.shape[1],) or slopes.dtype != torch.float32:
        raise ValueError("slopes must be float32 with shape (heads,)")


def _check_positions(name: str, positions: Tensor, n: int) -> None:
    if positions.shape != (n, 3) or positions.dtype not in (torch.float32, torch.float64):
        raise ValueError(f"{name} must be float32 or float64 with shape ({n}, 3)")


def _check_ptr(name: str, ptr: Tensor) -> None:
    if ptr.ndim != 1 or ptr.numel() == 0 or ptr.dtype != torch.int64:
        raise ValueError(f"{name} must be int64 with shape (B + 1,)")


def _score_rule(q: Tensor, scale: float | None, softcap: float | None) -> tuple[float, float]:
    # as the kernels take them: a cap that 32 bits round to 0 would be none
    scale = c_float(1.0 / sqrt(q.shape[2]) if scale is None else float(scale)).value
    if not isfinite(scale):
        raise ValueError("scale must be finite in 32 bits")
    if softcap is None:
        return scale, 0.0
    softcap = c_float(float(softcap)).value
    if not isfinite(softcap) or softcap <= 0.0:
        raise ValueError("softcap must be finite and positive in 32 bits")
    return scale, softcap


def _check_place(what: str, q: Tensor, **tensors: Tensor) -> None:
    for name, tensor in tensors.items():
        if tensor.device != q.device:
            raise ValueError(f"q and {name} must be on the same device")
    if not q.is_cuda:
        raise RuntimeError(f"{what} runs on ROCm (HIP) devices; move the tensors to a GPU")
    check_device(q.device.index)


def structure_attention(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    positions: Tensor,
    batch_ptr: Tensor,
    slopes: Tensor,
    *,
    softcap: float | None = None,
    scale: float | None = None,
    query_positions: Tensor | None = None,
    query_ptr: Tensor | None = None,
) -> Tensor:
    """Each atom attends to all atoms of its own structure (see the module for the scores).

    ``q`` (N, heads, dim), ``k`` and ``v`` (N, kv_heads, dim): float32, bfloat16 or float16, dim a
    multiple of 8 from 8 to 128, heads a multiple of kv_heads; ``positions`` (N, 3); ``batch_ptr``
    (B + 1,) int64 as in ``neighbor_list``; ``slopes`` (heads,) float32; ``scale`` is 1 / sqrt(dim)
    by default.  Distances are those of the positions as given, without periodic images, in 32 bits.

    With ``query_positions`` (M, 3) and ``query_ptr`` (B + 1,), q has M rows: queries of their own for
    each structure, such as the one atom of a trial move, that attend to the structure's N atoms.  A
    query whose structure has no atoms gives 0.

    Gradients reach q, k, v, positions, query_positions and slopes; those of positions and slopes are
    32 bits wide whatever the type of q.  Pointers that do not rise from 0 to the number of atoms
    give NaN throughout (the call does not wait for the device to refuse them).
    """
    _check_tensors(q=q, k=k, v=v, positions=positions, batch_ptr=batch_ptr, slopes=slopes)
    _check_heads(q, k, v, slopes)
    _check_positions("positions", positions, k.shape[0])
    _check_ptr("batch_ptr", batch_ptr)
    place = {"k": k, "v": v, "positions": positions, "batch_ptr": batch_ptr, "slopes": slopes}
    if (query_positions is None) != (query_ptr is None):
        raise ValueError("query_positions and query_ptr go together")
    if query_ptr is None:
        if q.shape[0] != k.shape[0]:
            raise ValueError("q must have a row for each atom, or query_positions and query_ptr")
    else:
        _check_tensors(query_positions=query_positions, query_ptr=query_ptr)
        _check_positions("query_positions", query_positions, q.shape[0])
        _check_ptr("query_ptr", query_ptr)
        if query_ptr.shape != batch_ptr.shape:
            raise ValueError("query_ptr and batch_ptr must have the same shape")
        place |= {"query_positions": query_positions, "query_ptr": query_ptr}
        query_positions = query_positions.to(torch.float32)
    scale, softcap = _score_rule(q, scale, softcap)
    _check_place("structure_attention", q, **place)
    return load_torch_native().structure_attention(
        q, k, v, positions.to(torch.float32), batch_ptr, slopes, query_positions, query_ptr, scale,
        softcap)


class NeighborRows(NamedTuple):
    """A neighbor list laid out for ``neighbor_attention`` (see ``neighbor_rows``)."""

    i: Tensor            # (E,) int64: sources
    j: Tensor            # (E,) int64: targets
    n_sources: int
    n_targets: int
    transpose: bool      # also by target: what the gradients need
    rows: Tensor         # device bytes, as the kernels read them


def neighbor_rows(
    i: Tensor, j: Tensor, n_sources: int, n_targets: int | None = None, *, transpose: bool = True
) -> NeighborRows:
    """The pairs (i, j) of a neighbor list by source, and by target for the gradients.

    Once for each list: all layers that attend along it, forward and backward, share the result.  Any
    list of ``neighbor_list`` or ``neighbor_graph`` serves, sorted or not, whole, half or cut out of
    one, as long as the pairs of a source lie together; ``transpose=False`` saves the order by target
    where no gradient is asked for.  ``n_targets`` is ``n_sources`` by default.

    A list whose sources do not lie together, or that names an atom that does not exist, makes every
    result along it NaN (the call does not wait for the device to refuse it).
    """
    _check_tensors(i=i, j=j)
    n_targets = n_sources if n_targets is None else n_targets
    for name, n in (("n_sources", n_sources), ("n_targets", n_targets)):
        if isinstance(n, bool) or not isinstance(n, int):
            raise TypeError(f"{name} must be an int")
        if n < 0:
            raise ValueError(f"{name} must not be negative")
    if not isinstance(transpose, bool):
        raise TypeError("transpose must be bool")
    if i.ndim != 1 or j.shape != i.shape or i.dtype != torch.int64 or j.dtype != torch.int64:
        raise ValueError("i and j must be int64 with the same shape (E,)")
    if i.device != j.device:
        raise ValueError("i and j must be on the same device")
    if not i.is_cuda:
        raise RuntimeError("neighbor_rows runs on ROCm (HIP) devices; move the tensors to a GPU")
    check_device(i.device.index)
    rows = load_torch_native().neighbor_rows(i, j, n_sources, n_targets, transpose)
    return NeighborRows(i, j, n_sources, n_targets, transpose, rows)


def neighbor_attention(
    q: Tensor,
    k: Tensor,
    v: Tensor,
    d: Tensor,
    rows: NeighborRows,
    slopes: Tensor,
    *,
    softcap: float | None = None,
    scale: float | None = None,
) -> Tensor:
    """Each source atom attends along its pairs in a list (see the module for the scores).

    ``q`` (n_sources, heads, dim), ``k`` and ``v`` (n_targets, kv_heads, dim) as in
    ``structure_attention``; ``d`` (E,) is the pairs' distances, in the order of the list that ``rows``
    was made from (``neighbor_rows``).  An atom without pairs gives 0.

    Gradients reach q, k, v, d and slopes; those of d and slopes are 32 bits wide whatever the type
    of q.
    """
    _check_tensors(q=q, k=k, v=v, d=d, slopes=slopes)
    if not isinstance(rows, NeighborRows):
        raise TypeError("rows must come from neighbor_rows")
    _check_tensors(i=rows.i, j=rows.j, rows=rows.rows)
    _check_heads(q, k, v, slopes)
    if q.shape[0] != rows.n_sources or k.shape[0] != rows.n_targets:
        raise ValueError("q needs a row for each source of the list, k and v one for each target")
    if rows.j.shape != rows.i.shape or d.shape != rows.i.shape or d.dtype not in (torch.float32, torch.float64):
        raise ValueError("d must be float32 or float64 with one value for each pair")
    scale, softcap = _score_rule(q, scale, softcap)
    _check_place("neighbor_attention", q, k=k, v=v, d=d, slopes=slopes, rows=rows.rows, i=rows.i,
                 j=rows.j)
    if not rows.transpose and torch.is_grad_enabled() and any(
            t.requires_grad for t in (q, k, v, d, slopes)):
        raise ValueError("gradients need rows with transpose=True")
    return load_torch_native().neighbor_attention(
        q, k, v, d.to(torch.float32), slopes, rows.rows, rows.i, rows.j, rows.transpose, scale,
        softcap)


__all__ = ["NeighborRows", "neighbor_attention", "neighbor_rows", "structure_attention"]
