"""GPU: the species embedding and its gradient against sums in float64.

The forward is one product, rounded once: exact to the last bit against the same in 32 bits.  A
gradient is a sum of up to 65,536 rows in 32 bits, rounded once: within 2^-24 sqrt(n) of the sum of
absolute values, doubled, and half a spacing of the type.
"""

from __future__ import annotations

import pytest
import torch

from tests._operators import HALF_SPACING
from tonari_amd.embedding import species_embedding

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["float32", "bfloat16", "float16"]


def make(shape, rows, channels, dtype, seed=1, index=torch.int64, skew=3.0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.rand(shape, generator=g) ** skew * rows).to(index).clamp_(max=max(rows - 1, 0))
    w = torch.randn(rows, channels, generator=g).to(dtype)
    up = torch.randn(*z.shape, channels, generator=g).to(dtype)
    return z.to(DEV), w.to(DEV).requires_grad_(), up.to(DEV)


def check(z, w, up, scale):
    out = species_embedding(z, w, scale=scale)
    assert out.shape == (*z.shape, w.shape[1]) and out.dtype == w.dtype
    flat = z.reshape(-1).long()
    scale32 = torch.tensor(scale, dtype=torch.float32, device=DEV)
    assert torch.equal(out.reshape(-1, w.shape[1]), (w.detach().float()[flat] * scale32).to(w.dtype))
    (got,) = torch.autograd.grad(out, w, up)
    rows = up.reshape(-1, w.shape[1]).double()
    want = torch.zeros(w.shape, dtype=torch.float64, device=DEV).index_add_(0, flat, rows) * scale
    size = torch.zeros_like(want).index_add_(0, flat, rows.abs()) * abs(scale)
    most = 2 * 2.0**-24 * len(flat) ** 0.5 * size + HALF_SPACING[w.dtype] * 1.01 * want.abs() + 2.0**-24
    assert bool(((got.double() - want).abs() <= most).all())
    return got


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape,rows,channels", [
    ((1,), 1, 1), ((7,), 3, 5), ((64,), 119, 8), ((2047,), 4, 36), ((2049,), 119, 64),
    ((70, 30), 11, 128), ((5000,), 1023, 20), ((5000,), 1024, 24), ((9000,), 3000, 257),
    ((65_536,), 95, 130), ((30_000,), 1, 48),
])
def test_rows_and_gradient(dtype, shape, rows, channels):
    z, w, up = make(shape, rows, channels, dtype)
    check(z, w, up, 1.5)


def test_int32_and_empty_species():
    z, w, up = make((4000,), 500, 40, torch.float32, index=torch.int32, skew=12.0)
    got = check(z, w, up, -0.25)
    unused = torch.ones(500, dtype=torch.bool, device=DEV)
    unused[z.long()] = False
    assert bool(unused.any()) and bool((got[unused] == 0).all())


def test_many_species():
    # two passes of the sort, and three
    for rows in (70_000, 1_200_000):
        z, w, up = make((20_000,), rows, 8, torch.float32, skew=1.0)
        check(z, w, up, 1.0)


def test_no_atoms_and_no_species():
    z, w, up = make((0,), 6, 8, torch.float32)
    assert bool((check(z, w, up, 1.0) == 0).all())
    z, w, up = make((0,), 0, 8, torch.float32)
    check(z, w, up, 1.0)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_species_outside_the_table(index):
    z, w, up = make((3000,), 10, 16, torch.float32, index=index)
    clean = species_embedding(z, w)
    bad = z.clone()
    bad[5], bad[77], bad[2999] = -1, 10, 2_000_000_000
    out = species_embedding(bad, w)
    keep = torch.ones(3000, dtype=torch.bool, device=DEV)
    keep[[5, 77, 2999]] = False
    assert torch.equal(out[keep], clean[keep]) and bool(torch.isnan(out[~keep]).all())
    (got,) = torch.autograd.grad(out, w, up)
    want = torch.zeros(10, 16, dtype=torch.float64, device=DEV).index_add_(
        0, z[keep].long(), up[keep].double())
    assert float((got.double() - want).abs().max()) <= 1e-3


def test_nan_reaches_its_species_only():
    z, w, up = make((5000,), 20, 16, torch.float32)
    up[123] = float("nan")
    (got,) = torch.autograd.grad(species_embedding(z, w), w, up)
    nan = torch.isnan(got).all(1)
    assert int(nan.sum()) == 1 and bool(nan[int(z[123])])


def test_strides_and_alignment():
    z, w, up = make((3000,), 33, 24, torch.bfloat16)
    want = check(z, w, up, 2.0)
    wide = torch.zeros(33, 48, dtype=torch.bfloat16, device=DEV)
    wide[:, 3:27] = w.detach()
    v = wide[:, 3:27].requires_grad_()
    spread = torch.zeros(3000, 24, 2, dtype=torch.bfloat16, device=DEV)
    spread[..., 0] = up
    out = species_embedding(torch.stack([z, z], 1)[:, 1], v, scale=2.0)
    assert torch.equal(out, species_embedding(z, w, scale=2.0))
    assert torch.equal(torch.autograd.grad(out, v, spread[..., 0])[0], want)
    # a broadcast upstream gradient
    out = species_embedding(z, w, scale=2.0)
    one = torch.ones((), dtype=torch.bfloat16, device=DEV).expand_as(out)
    check(z, w, one, 2.0)


def test_repeats_are_equal_bits():
    z, w, up = make((40_000,), 119, 64, torch.float32)
    first = check(z, w, up, 1.0)
    for _ in range(3):
        assert torch.equal(torch.autograd.grad(species_embedding(z, w), w, up)[0], first)


def test_gradient_of_the_gradient():
    z, w, up = make((50,), 6, 8, torch.float32)
    z[4] = -1
    up.requires_grad_()
    (gw,) = torch.autograd.grad(species_embedding(z, w, scale=3.0), w, up, create_graph=True)
    (gu,) = torch.autograd.grad((gw * gw).sum(), up)
    want = 2 * 3.0 * gw.detach()[z.clamp(min=0)]
    want[4] = 0
    assert torch.allclose(gu, want, rtol=1e-5, atol=1e-5)


def test_graph_has_the_same_bits():
    z, w, up = make((40_000,), 119, 64, torch.bfloat16)
    z[7], z[40] = -1, 119
    out = species_embedding(z, w, scale=0.5)
    (want,) = torch.autograd.grad(out, w, up, retain_graph=True)
    up.requires_grad_()
    for _ in range(2):
        (got,) = torch.autograd.grad(out, w, up, create_graph=True)
        assert torch.equal(got, want)
    # and on: a sum of cubes of the gradient, twice in the upstream gradient
    (first,) = torch.autograd.grad((got.float() ** 3).sum(), up, create_graph=True)
    assert bool((first[[7, 40]] == 0).all())
    (second,) = torch.autograd.grad(first.float().sum(), up)
    assert bool(torch.isfinite(second).all()) and bool((second[[7, 40]] == 0).all())


def test_graph_of_an_empty_table():
    z, w, up = make((9,), 0, 8, torch.float32)
    up.requires_grad_()
    out = species_embedding(z, w)
    assert bool(torch.isnan(out).all())
    (got,) = torch.autograd.grad(out, w, up, create_graph=True)
    assert got.shape == (0, 8)
    assert bool((torch.autograd.grad(got.sum(), up)[0] == 0).all())
