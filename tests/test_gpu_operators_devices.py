"""GPU: the operators on a device that is not the current one."""

from __future__ import annotations

import pytest
import torch

from tests import test_gpu_neighbor_attention as neighbor
from tests import test_gpu_species_embedding as embedding
from tests import test_gpu_structure_attention as structure

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")]


def test_tensors_of_another_device(monkeypatch):
    for m in (embedding, neighbor, structure):
        monkeypatch.setattr(m, "DEV", "cuda:1")
    assert torch.cuda.current_device() == 0
    embedding.check(*embedding.make((500,), 20, 16, torch.float32), 1.0)
    structure.check(structure.make([40, 9], 2, 1, 16, torch.bfloat16), 5.0)
    i, j = neighbor.random_list(30, 30, 10, seed=1)
    neighbor.check(neighbor.make(i, j, 30, 30, 2, 1, 16, torch.float32), 5.0)
    assert torch.cuda.current_device() == 0
