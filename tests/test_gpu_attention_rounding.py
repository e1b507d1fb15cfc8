"""GPU: structure attention in 16 bits, rounded once.

Inputs and results are 16-bit; between them everything has 32 bits, or two pieces of 16 whose rest is
rounded itself.  So a result lies within its own rounding, u |result|, and 2e-5 + u^2 of the sum of the
magnitudes that make it (u is half the type's spacing at 1; 2e-5 as in tests/_operators.py).  Those sums
are taken in float64 over all pairs:

    output   sum p |v|                     grad_v   sum p |do|
    grad_q   sum scale p (a + sum p a) |k|  grad_k   sum scale p (a + sum p a) |q|,  a = sum |do| |v|
"""

from __future__ import annotations

import math

import pytest
import torch

from tests._operators import HALF_SPACING, double, structure_pairs
from tests.test_gpu_structure_attention import DTYPES, IDS, call, expected, make

pytestmark = pytest.mark.gpu


def sums_of_magnitudes(c, softcap):
    """The magnitudes that make out, grad_q, grad_k and grad_v."""
    q, k, v, x, slopes, y = double(*(c[n] for n in ("q", "k", "v", "positions", "slopes",
                                                    "query_positions")))
    up = c["upstream"].double().cpu().abs()
    kp = c["batch_ptr"].tolist()
    source, target = structure_pairs(kp if c["query_ptr"] is None else c["query_ptr"].tolist(), kp)
    heads, dim, group = q.shape[1], q.shape[2], q.shape[1] // k.shape[1]
    of = torch.arange(heads) // group
    qs, ks, vs, us = (t[at] for t, at in ((q, source), (k[:, of], target), (v[:, of], target),
                                          (up, source)))
    r = torch.linalg.vector_norm((x if y is None else y)[source] - x[target], dim=1)
    s = (qs * ks).sum(-1) / dim**0.5
    s = (softcap * torch.tanh(s / softcap) if softcap else s) - slopes * r[:, None]
    rows = torch.zeros(q.shape[0], heads, dtype=torch.float64)
    e = torch.exp(s - rows.scatter_reduce(0, source[:, None].expand(-1, heads), s, "amax",
                                          include_self=False)[source])
    p = e / rows.index_add(0, source, e)[source]
    a = (us * vs.abs()).sum(-1)
    ds = p * (a + rows.index_add(0, source, p * a)[source]) / dim**0.5

    def summed(pairs, at, like):
        full = torch.zeros(like.shape[0], heads, dim, dtype=torch.float64).index_add(0, at, pairs)
        return full.view(like.shape[0], like.shape[1], -1, dim).sum(2)

    with torch.no_grad():
        return {"out": summed(p[:, :, None] * vs.abs(), source, q),
                "q": summed(ds[:, :, None] * ks.abs(), source, q),
                "k": summed(ds[:, :, None] * qs.abs(), target, k),
                "v": summed(p[:, :, None] * us, target, v)}


def assert_rounded_once(c, softcap, names):
    out = call(c, softcap)
    ref, leaves = expected(c, softcap)
    found = {"out": (out.detach(), ref.detach())}
    for n, a, e in zip("qkv", torch.autograd.grad(out, [c[n] for n in "qkv"], c["upstream"]),
                       torch.autograd.grad(ref, leaves[:3], c["upstream"].double().cpu())):
        found[n] = (a, e)
    size, u = sums_of_magnitudes(c, softcap), HALF_SPACING[c["q"].dtype]
    for n in names:
        a, e = found[n]
        # (values near the type's smallest are rounded to multiples of it)
        most = u * e.abs() + (2e-5 + u * u) * size[n] + (2.0**-24 if u == 2.0**-11 else 0.0)
        worst = float(((a.double().cpu() - e).abs() / most).max())
        assert worst <= 1.0, (n, worst)


CASES = [
    ([700], None, 4, 2, 40),
    ([90, 33, 120, 64, 77], None, 3, 3, 32),
    ([300, 1, 2], None, 8, 2, 64),
    ([260], None, 2, 1, 128),
    ([1500, 1400], [40, 33], 2, 2, 64),       # keys split over workgroups
    ([200], [1900], 2, 1, 32),                # rows split in the keys' gradients
]


def biased(c, mean):
    """Keys and values with a component in common, as linear layers make them."""
    for n in "kv":
        c[n] = (c[n].detach().float() + mean).to(c[n].dtype).requires_grad_()
    return c


def case_of(lengths, queries, heads, kv_heads, dim, dtype, mean):
    c = make(lengths, heads, kv_heads, dim, dtype, queries=queries, seed=40)
    return biased(c, mean)


@pytest.mark.parametrize("dtype", DTYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("lengths,queries,heads,kv_heads,dim", CASES)
def test_output(dtype, lengths, queries, heads, kv_heads, dim):
    assert_rounded_once(case_of(lengths, queries, heads, kv_heads, dim, dtype, 0.0), 8.0, ["out"])


@pytest.mark.parametrize("dtype", DTYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("lengths,queries,heads,kv_heads,dim", CASES)
def test_gradients_of_keys_and_values(dtype, lengths, queries, heads, kv_heads, dim):
    assert_rounded_once(case_of(lengths, queries, heads, kv_heads, dim, dtype, 0.0), 8.0, "kv")


@pytest.mark.parametrize("dtype", DTYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("mean", [0.0, 3.0])
@pytest.mark.parametrize("lengths,queries,heads,kv_heads,dim", CASES)
def test_gradient_of_queries(dtype, mean, lengths, queries, heads, kv_heads, dim):
    assert_rounded_once(case_of(lengths, queries, heads, kv_heads, dim, dtype, mean), None, "q")


def test_many_keys_that_weigh_little():
    # one near key and 20,000 far ones, whose weights of 2^-26 add up to 3e-4 of the row
    n, dim = 20_000, 16
    c = make([n], 1, 1, dim, torch.float16, queries=[1], grad=False, seed=41)
    c["q"], c["k"] = torch.zeros_like(c["q"]), torch.zeros_like(c["k"])
    x = torch.zeros(n, 3, device="cuda")
    x[1:, 0] = 26 * math.log(2.0)
    c |= {"positions": x, "query_positions": torch.zeros(1, 3, device="cuda"),
          "slopes": torch.ones(1, device="cuda")}
    v = torch.zeros(n, 1, dim, dtype=torch.float16, device="cuda")
    v[1:] = 2.0
    c["v"] = v
    want = 2.0 * (n - 1) * 2.0**-26 / (1 + (n - 1) * 2.0**-26)
    out = call(c)
    assert bool(((out.double() - want).abs() <= (2.0**-11 + 2e-5) * want + 2.0**-24).all())


@pytest.mark.parametrize("opposite", [False, True])
@pytest.mark.parametrize("scale", [0.9, 0.9e-3])
@pytest.mark.parametrize("lengths,queries", [([2], None), ([40], None), ([2], [600]), ([600], [2])])
def test_large_values(lengths, queries, scale, opposite):
    # sums over 64 channels of values of 3,000 lie far beyond float16, the gradients within it
    c = make(lengths, 1, 1, 64, torch.float16, queries=queries, seed=28)
    sign = torch.where(torch.arange(sum(lengths), device="cuda") % 2 == 0, 1.0, -1.0)
    with torch.no_grad():
        c["v"].copy_(3000.0 * sign[:, None, None].expand_as(c["v"]))
        c["q"].mul_(0.01)
        c["k"].mul_(0.01)
        c["slopes"].zero_()
        c["upstream"] = torch.full_like(c["upstream"], scale)
        if opposite:
            c["upstream"][1::2] *= -1
    assert_rounded_once(c, None, "qkv")


def test_small_gradients_beside_large_ones():
    # rows whose upstream gradient is 2^-12 of the others', and scores that spread over 2^20
    c = make([70], 2, 2, 32, torch.float16, seed=29)
    with torch.no_grad():
        c["upstream"][::3] *= 2.0**-12
        c["v"].mul_(64.0)
        c["q"].mul_(4.0)
    assert_rounded_once(c, None, "qkv")
