"""Plain forms of the operators in float64 on the CPU, for their tests.

Tolerances are derived here once, from the types alone.  u is half the spacing of the type at 1
(2^-24, 2^-11, 2^-8).  An output is a sum of products of values of that type, each product's weight
rounded to it once (16-bit types) and the sum rounded once; float32 outputs of 16-bit inputs are
summed in 32 bits throughout.  Errors are taken relative to the largest value of the output (a
gradient is a difference of sums, so that single values may be small):

    16-bit outputs   8 u     (two roundings, and a margin of four for the cancellation in gradients)
    32-bit outputs   2e-5    (scores up to about 2^6 carry 2^-24 2^6 = 4e-6 into the weights; five
                              times that for the sums' own rounding)
"""

from __future__ import annotations

import torch

HALF_SPACING = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def tolerance(dtype: torch.dtype) -> float:
    return 2e-5 if dtype in (torch.float32, torch.float64) else 8 * HALF_SPACING[dtype]


def assert_near(actual: torch.Tensor, expected: torch.Tensor, what: str = "") -> None:
    a, e = actual.detach().double().cpu(), expected.detach().double().cpu()
    assert a.shape == e.shape, (what, a.shape, e.shape)
    if a.numel() == 0:
        return
    assert torch.equal(torch.isfinite(a), torch.isfinite(e)), what
    scale = float(e.abs().max())
    err = float((a - e).abs().max())
    assert err <= tolerance(actual.dtype) * scale + 1e-30, f"{what}: {err:.3e} over {scale:.3e}"


def double(*tensors):
    """Float64 copies on the CPU, leaves where the originals need a gradient."""
    return [None if t is None else
            t.detach().cpu().double().requires_grad_(t.requires_grad) for t in tensors]


def attend(q, k, v, r, slopes, source, target, scale, softcap):
    """Attention along the pairs (source, target) at distances r, by its definition."""
    N, H, D = q.shape
    group = H // k.shape[1]
    head = torch.arange(H) // group
    x = scale * (q[source] * k[target][:, head]).sum(-1)
    s = (softcap * torch.tanh(x / softcap) if softcap else x) - slopes * r[:, None]
    top = torch.full((N, H), -torch.inf, dtype=s.dtype).scatter_reduce(
        0, source[:, None].expand(-1, H), s.detach(), "amax")
    e = torch.exp(s - top[source])
    total = torch.zeros(N, H, dtype=s.dtype).index_add(0, source, e)
    p = e / total[source]
    return torch.zeros_like(q).index_add(0, source, p[:, :, None] * v[target][:, head])


def structure_pairs(query_ptr, key_ptr):
    source, target = [], []
    for b in range(len(key_ptr) - 1):
        qs = torch.arange(query_ptr[b], query_ptr[b + 1])
        ks = torch.arange(key_ptr[b], key_ptr[b + 1])
        source.append(qs.repeat_interleave(len(ks)))
        target.append(ks.repeat(len(qs)))
    return torch.cat(source), torch.cat(target)


def distances(x, y):
    """|x - y| by rows, whose gradient at 0 is 0."""
    t = x - y
    r2 = (t * t).sum(-1)
    apart = r2 > 0
    return torch.where(apart, torch.sqrt(torch.where(apart, r2, 1.0)), 0.0)


def pointer(lengths) -> torch.Tensor:
    return torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int64)
