"""GPU: what the operators would lose without a word is refused: forward-mode tangents and traces."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from tests import test_gpu_neighbor_attention as neighbor
from tests import test_gpu_structure_attention as structure
from tonari_amd.attention import neighbor_attention, neighbor_rows
from tonari_amd.embedding import species_embedding

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def calls():
    """Each operator as a function of one of its real inputs, and that input."""
    z = torch.tensor([0, 2, 1], device=DEV)
    s = structure.make([9], 2, 1, 16, torch.float32, grad=False)
    i, j = neighbor.random_list(9, 9, 4, seed=1)
    n = neighbor.make(i, j, 9, 9, 2, 1, 16, torch.float32, grad=False)
    rows = neighbor_rows(n["i"], n["j"], 9)

    def along(c):
        return neighbor_attention(c["q"], c["k"], c["v"], c["d"], rows, c["slopes"])

    return [
        (lambda w: species_embedding(z, w), torch.randn(3, 8, device=DEV)),
        *((lambda t, x=x: structure.call(dict(s, **{x: t})), s[x]) for x in ("q", "positions", "slopes")),
        *((lambda t, x=x: along(dict(n, **{x: t})), n[x]) for x in ("k", "d")),
    ]


@pytest.mark.parametrize("which", range(6))
@pytest.mark.parametrize("leaf", [False, True])
def test_forward_mode(which, leaf):
    f, x = calls()[which]
    f(x)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x.clone().requires_grad_(leaf), torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(dual)


@pytest.mark.parametrize("which", range(6))
def test_forward_mode_through_the_backward(which):
    f, x = calls()[which]
    x = x.clone().requires_grad_()
    out = f(x)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.autograd.grad(out, x, dual)


@pytest.mark.parametrize("which", range(6))
def test_trace(which):
    f, x = calls()[which]
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(f, x, check_trace=False)


def test_trace_of_the_layout():
    i = torch.tensor([0, 0, 1], device=DEV)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda j: neighbor_rows(i, j, 2).rows, i, check_trace=False)
