"""A small atomistic transformer on neighbor lists: energies and forces, trained and then used.

Species are embedded, atoms attend along their neighbor list (periodic images included) and then to
all atoms of their own structure; the energy of a structure is the sum over its atoms.  Forces are the
gradient of the energy through both attentions and the list's distances.

    python examples/atom_transformer.py [--steps 20] [--dtype bfloat16]

trains on a synthetic pair potential over small periodic crystals, then asks for the energies and
forces of new ones.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import Tensor, nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from tonari_amd import neighbor_list  # noqa: E402
from tonari_amd.attention import neighbor_attention, neighbor_rows, structure_attention  # noqa: E402
from tonari_amd.embedding import species_embedding  # noqa: E402

CUTOFF = 4.0


class Layer(nn.Module):
    """Pre-norm attention and a two-layer network, both with residuals."""

    def __init__(self, width: int, heads: int, kv_heads: int):
        super().__init__()
        dim = width // heads
        self.heads, self.kv_heads = heads, kv_heads
        self.norm, self.norm2 = nn.LayerNorm(width), nn.LayerNorm(width)
        self.qkv = nn.Linear(width, (heads + 2 * kv_heads) * dim, bias=False)
        self.out = nn.Linear(width, width, bias=False)
        self.mlp = nn.Sequential(nn.Linear(width, 2 * width), nn.SiLU(), nn.Linear(2 * width, width))
        # how fast a head's attention falls with distance, 1 / Angstrom
        self.slopes = nn.Parameter(torch.logspace(0, -1, heads, base=4.0))

    def forward(self, x: Tensor, attend, dtype: torch.dtype) -> Tensor:
        n, h = x.shape[0], self.heads
        t = self.qkv(self.norm(x)).to(dtype).view(n, h + 2 * self.kv_heads, -1)
        q, k, v = t.split([h, self.kv_heads, self.kv_heads], 1)
        x = x + self.out(attend(q, k, v, self.slopes).reshape(n, -1).to(x.dtype))
        return x + self.mlp(self.norm2(x))


class AtomTransformer(nn.Module):
    def __init__(self, species: int = 8, width: int = 64, heads: int = 4, kv_heads: int = 2,
                 dtype: torch.dtype = torch.float32):
        super().__init__()
        self.dtype = dtype
        self.table = nn.Parameter(torch.randn(species, width) / width**0.5)
        self.local = Layer(width, heads, kv_heads)
        self.whole = Layer(width, heads, kv_heads)
        self.energy = nn.Sequential(nn.LayerNorm(width), nn.Linear(width, 1))

    def forward(self, species: Tensor, positions: Tensor, cell: Tensor, pbc: Tensor,
                batch_ptr: Tensor) -> Tensor:
        """Energies of the structures, differentiable in positions and cell."""
        i, j, d = neighbor_list("ijd", positions, cell, pbc, CUTOFF, batch_ptr)
        # one layout of the list serves every layer and both passes
        rows = neighbor_rows(i, j, positions.shape[0])
        x = species_embedding(species, self.table, scale=self.table.shape[1] ** 0.5)
        x = self.local(x, lambda q, k, v, m: neighbor_attention(q, k, v, d, rows, m, softcap=20.0),
                       self.dtype)
        x = self.whole(x, lambda q, k, v, m: structure_attention(q, k, v, positions, batch_ptr, m,
                                                                 softcap=20.0), self.dtype)
        atoms = self.energy(x).squeeze(1)
        b = torch.bucketize(torch.arange(len(atoms), device=atoms.device), batch_ptr[1:], right=True)
        return torch.zeros(batch_ptr.numel() - 1, device=atoms.device).index_add(0, b, atoms)


def crystals(count: int, seed: int, device: str) -> dict[str, Tensor]:
    """Random periodic crystals of 4 to 24 atoms."""
    g = torch.Generator().manual_seed(seed)
    lengths = torch.randint(4, 25, (count,), generator=g)
    edge = (lengths.float() * 12.0) ** (1.0 / 3.0)
    n = int(lengths.sum())
    data = {
        "species": torch.randint(0, 8, (n,), generator=g),
        "positions": torch.rand(n, 3, generator=g) * edge.repeat_interleave(lengths)[:, None],
        "cell": edge[:, None, None] * torch.eye(3),
        "pbc": torch.ones(count, 3, dtype=torch.bool),
        "batch_ptr": torch.cat([torch.zeros(1, dtype=torch.int64), lengths.cumsum(0)]),
    }
    return {name: t.to(device) for name, t in data.items()}


def target(data: dict[str, Tensor]) -> tuple[Tensor, Tensor]:
    """Energies and forces of a smooth pair potential whose strength depends on the species."""
    x = data["positions"].clone().requires_grad_()
    i, j, d = neighbor_list("ijd", x, data["cell"], data["pbc"], CUTOFF, data["batch_ptr"])
    z = 0.2 + 0.1 * data["species"].float()
    pair = z[i] * z[j] * (1.0 - d / CUTOFF) ** 2 * torch.cos(2.0 * d)
    b = torch.bucketize(i, data["batch_ptr"][1:], right=True)
    energy = torch.zeros(data["pbc"].shape[0], device=d.device).index_add(0, b, pair)
    return energy.detach(), -torch.autograd.grad(energy.sum(), x)[0]


def predict(model: AtomTransformer, data: dict[str, Tensor], *, training: bool):
    x = data["positions"].clone().requires_grad_()
    energy = model(data["species"], x, data["cell"], data["pbc"], data["batch_ptr"])
    # training on forces needs the gradient's own graph
    forces = -torch.autograd.grad(energy.sum(), x, create_graph=training)[0]
    return energy, forces


def train(steps: int, *, batch: int = 16, device: str = "cuda", dtype: torch.dtype = torch.float32,
          forces: bool = True, seed: int = 0) -> tuple[AtomTransformer, list[float]]:
    torch.manual_seed(seed)
    model = AtomTransformer(dtype=dtype).to(device)
    optimizer = torch.optim.Adam(model.parameters(), lr=3e-3)
    data = crystals(batch, seed, device)
    energy0, forces0 = target(data)
    losses = []
    for _ in range(steps):
        if forces:
            energy, found = predict(model, data, training=True)
            loss = (energy - energy0).square().mean() + 4.0 * (found - forces0).square().mean()
        else:
            energy = model(data["species"], data["positions"], data["cell"], data["pbc"],
                           data["batch_ptr"])
            loss = (energy - energy0).square().mean()
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
    return model, losses


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    parser.add_argument("--steps", type=int, default=20)
    parser.add_argument("--dtype", choices=["float32", "bfloat16", "float16"], default="float32")
    args = parser.parse_args()
    model, losses = train(args.steps, dtype=getattr(torch, args.dtype))
    print(f"loss: {losses[0]:.4f} -> {losses[-1]:.4f} in {len(losses)} steps")
    data = crystals(4, 1000, "cuda")
    energy, forces = predict(model, data, training=False)
    print("energies of new crystals:", [round(e, 3) for e in energy.detach().tolist()])
    print(f"largest force: {float(forces.detach().norm(dim=1).max()):.3f}")


if __name__ == "__main__":
    main()
