"""GPU: the example model runs the operators together, learns, and its forces are its energy's slope."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("dtype,forces", [(torch.float32, True), (torch.float32, False),
                                          (torch.bfloat16, False)])
def test_it_learns(dtype, forces):
    from examples.atom_transformer import train

    _, losses = train(25, device=DEV, dtype=dtype, forces=forces)
    assert losses[-1] < 0.6 * losses[0]


def test_forces_are_the_slope_of_the_energy():
    from examples.atom_transformer import AtomTransformer, crystals, predict

    torch.manual_seed(3)
    model = AtomTransformer().to(DEV)
    data = crystals(6, 4, DEV)
    energy, forces = predict(model, data, training=False)
    graph = predict(model, data, training=True)[1]
    # the kernels' forces and those of the expression behind create_graph
    assert float((forces - graph).norm()) <= 1e-3 * float(graph.norm())
    way = torch.randn(data["positions"].shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    way /= way.norm()
    # central differences, averaged over steps: pairs that enter or leave at the cutoff make the
    # energy step (their weight is not 0 there), so the smallest difference is the one to take
    best = 1.0
    along = -float((forces.double() * way).sum())
    for step in (2.0**-7, 2.0**-8, 2.0**-9):
        with torch.no_grad():
            up, down = (float(model(data["species"], data["positions"] + s * way, data["cell"],
                                    data["pbc"], data["batch_ptr"]).double().sum())
                        for s in (step, -step))
        best = min(best, abs((up - down) / (2 * step) - along))
    assert best <= 0.05 * max(1.0, float(forces.norm()))
