"""The operators without a GPU: what they refuse, and the C ABI's checks before any launch."""

from __future__ import annotations

import ctypes
import os
import re

import pytest
import torch

from tests.test_abi import lib  # noqa: F401
from tonari_amd import _extensions as ext
from tonari_amd.attention import NeighborRows, neighbor_attention, neighbor_rows, structure_attention
from tonari_amd.embedding import species_embedding

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "tonari_operators.h")


def declared() -> list[str]:
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    return re.findall(r"^\s*[A-Za-z_][\w\s\*]*?\b(tnr_\w+)\s*\(", text, flags=re.M)


def test_header_and_library(lib):  # noqa: F811
    assert sorted(declared()) == sorted(ext.OPERATOR_EXPORTS)
    for name in declared():
        assert hasattr(lib, name), name
    version = int(re.search(r"#define\s+TNR_OPERATORS_VERSION\s+(\d+)", open(HEADER).read()).group(1))
    assert lib.tnr_operators_version() == version == ext.OPERATORS_VERSION


# ------------------------------------------------------------------- Python


def attention_arguments(**changed):
    a = {"q": torch.zeros(6, 4, 16), "k": torch.zeros(6, 2, 16), "v": torch.zeros(6, 2, 16),
         "positions": torch.zeros(6, 3), "batch_ptr": torch.tensor([0, 2, 6]),
         "slopes": torch.zeros(4)}
    return a | changed


@pytest.mark.parametrize("changed,kind,message", [
    ({"q": None}, TypeError, "q must be a PyTorch tensor"),
    ({"slopes": [1.0]}, TypeError, "slopes must be a PyTorch tensor"),
    ({"q": torch.zeros(6, 64)}, ValueError, r"shape \(N, heads, dim\)"),
    ({"v": torch.zeros(6, 1, 16)}, ValueError, "k and v must have the same shape"),
    ({"q": torch.zeros(6, 4, 16, dtype=torch.float64)}, ValueError, "the same dtype"),
    ({"k": torch.zeros(6, 2, 16).half()}, ValueError, "the same dtype"),
    ({"q": torch.zeros(6, 4, 24)}, ValueError, "same head dimension"),
    ({"q": torch.zeros(6, 3, 16), "slopes": torch.zeros(3)}, ValueError, "must be a multiple of"),
    ({"slopes": torch.zeros(2)}, ValueError, "slopes must be float32"),
    ({"slopes": torch.zeros(4).double()}, ValueError, "slopes must be float32"),
    ({"positions": torch.zeros(5, 3)}, ValueError, "positions must be float32 or float64"),
    ({"positions": torch.zeros(6, 3).half()}, ValueError, "positions must be float32 or float64"),
    ({"batch_ptr": torch.tensor([0, 6], dtype=torch.int32)}, ValueError, "batch_ptr must be int64"),
    ({"q": torch.zeros(7, 4, 16)}, ValueError, "q must have a row for each atom"),
    ({"query_ptr": torch.tensor([0, 2, 6])}, ValueError, "go together"),
    ({"query_ptr": torch.tensor([0, 6]), "query_positions": torch.zeros(6, 3)}, ValueError,
     "the same shape"),
    ({"query_ptr": torch.tensor([0, 2, 6]), "query_positions": torch.zeros(5, 3)}, ValueError,
     "query_positions must be"),
    ({"softcap": 0.0}, ValueError, "softcap must be finite and positive"),
    ({"softcap": float("inf")}, ValueError, "softcap must be finite and positive"),
    ({"scale": float("nan")}, ValueError, "scale must be finite"),
    ({}, RuntimeError, "runs on ROCm"),
])
def test_structure_attention_refuses(changed, kind, message):
    with pytest.raises(kind, match=message):
        structure_attention(**attention_arguments(**changed))


@pytest.mark.parametrize("dim", [4, 12, 136])
def test_head_dimensions(dim):
    with pytest.raises(ValueError, match="multiple of 8, from 8 to 128"):
        structure_attention(**attention_arguments(q=torch.zeros(6, 4, dim), k=torch.zeros(6, 2, dim),
                                                  v=torch.zeros(6, 2, dim)))


@pytest.mark.parametrize("changed,kind,message", [
    ({"i": [0]}, TypeError, "i must be a PyTorch tensor"),
    ({"i": torch.zeros(3, dtype=torch.int32)}, ValueError, "must be int64"),
    ({"j": torch.zeros(2, dtype=torch.int64)}, ValueError, "must be int64"),
    ({"n_sources": 2.0}, TypeError, "n_sources must be an int"),
    ({"n_targets": -1}, ValueError, "must not be negative"),
    ({"transpose": 1}, TypeError, "transpose must be bool"),
    ({}, RuntimeError, "runs on ROCm"),
])
def test_neighbor_rows_refuses(changed, kind, message):
    a = {"i": torch.zeros(3, dtype=torch.int64), "j": torch.zeros(3, dtype=torch.int64),
         "n_sources": 4} | changed
    with pytest.raises(kind, match=message):
        neighbor_rows(**a)


@pytest.mark.parametrize("changed,kind,message", [
    ({"rows": None}, TypeError, "neighbor_rows"),
    ({"d": torch.zeros(2)}, ValueError, "one value for each pair"),
    ({"d": torch.zeros(3).half()}, ValueError, "one value for each pair"),
    ({"q": torch.zeros(5, 4, 16)}, ValueError, "a row for each source"),
    ({"k": torch.zeros(5, 2, 16), "v": torch.zeros(5, 2, 16)}, ValueError, "one for each target"),
    ({}, RuntimeError, "runs on ROCm"),
])
def test_neighbor_attention_refuses(changed, kind, message):
    three = torch.zeros(3, dtype=torch.int64)
    a = {"q": torch.zeros(6, 4, 16), "k": torch.zeros(6, 2, 16), "v": torch.zeros(6, 2, 16),
         "d": torch.zeros(3), "slopes": torch.zeros(4),
         "rows": NeighborRows(three, three, 6, 6, True, torch.zeros(1, dtype=torch.uint8))} | changed
    with pytest.raises(kind, match=message):
        neighbor_attention(**a)


@pytest.mark.parametrize("changed,kind,message", [
    ({"species": [1]}, TypeError, "species must be a PyTorch tensor"),
    ({"species": torch.zeros(3)}, ValueError, "int32 or int64"),
    ({"weight": torch.zeros(4)}, ValueError, r"shape \(V, C\)"),
    ({"weight": torch.zeros(4, 0)}, ValueError, r"shape \(V, C\)"),
    ({"weight": torch.zeros(4, 8, dtype=torch.float64)}, ValueError, "float32, bfloat16 or float16"),
    ({"scale": float("inf")}, ValueError, "scale must be finite"),
    ({}, RuntimeError, "runs on ROCm"),
])
def test_species_embedding_refuses(changed, kind, message):
    a = {"species": torch.zeros(3, dtype=torch.int64), "weight": torch.zeros(4, 8)} | changed
    with pytest.raises(kind, match=message):
        species_embedding(**a)


# -------------------------------------------------------------------- C ABI

PTR = 1 << 20  # never dereferenced: every call here returns before a launch


def refused(f, req, *more):
    err = ctypes.create_string_buffer(256)
    code = f(req if req is None else ctypes.byref(req), *more, None, err, len(err))
    return code, err.value.decode()


def embedding(**kw):
    return ext.Embedding(**(dict(dtype=0, index_bytes=8, n_atoms=10, n_species=5, channels=8,
                                 species=PTR, weight=PTR, scale=1.0, out=PTR, grad_out=PTR,
                                 grad_weight=PTR) | kw))


def test_embedding_requests(lib):  # noqa: F811
    bad = [(None, "request is null"), (embedding(dtype=1), "dtype must be"),
           (embedding(index_bytes=2), "int32 or int64"), (embedding(n_atoms=-1), "invalid sizes"),
           (embedding(channels=0), "invalid sizes"), (embedding(species=None), "pointers are null")]
    for req, message in bad:
        code, said = refused(lib.tnr_embedding_forward, req)
        assert code == ext.TNR_INPUT_ERROR and message in said
        code, said = refused(lib.tnr_embedding_backward, req, PTR, 1 << 30)
        assert code == ext.TNR_INPUT_ERROR and message in said
    assert refused(lib.tnr_embedding_forward, embedding(n_atoms=0))[0] == ext.TNR_OK
    need = lib.tnr_embedding_workspace_size(ctypes.byref(embedding()))
    for space, size in ((None, need), (PTR, need - 1), (PTR + 8, need)):
        code, said = refused(lib.tnr_embedding_backward, embedding(), space, size)
        assert code == ext.TNR_INPUT_ERROR and "workspace" in said


def structure(**kw):
    two = ctypes.c_int64 * 2
    return ext.StructureAttention(**(dict(
        dtype=2, heads=4, kv_heads=2, dim=32, n_structures=3, n_queries=50, n_keys=50, query_ptr=PTR,
        key_ptr=PTR, q=PTR, k=PTR, v=PTR, q_stride=two(128, 32), k_stride=two(64, 32),
        v_stride=two(64, 32), query_positions=None, positions=PTR, slopes=PTR, scale=0.2, softcap=0.0,
        tiles=PTR, out=PTR, lse=PTR, grad_out=PTR, grad_q=PTR, grad_k=PTR, grad_v=PTR,
        grad_query_positions=None, grad_positions=PTR, grad_slopes=PTR) | kw))


def test_structure_requests(lib):  # noqa: F811
    two = ctypes.c_int64 * 2
    bad = [(None, "request is null"), (structure(dtype=1), "dtype must be"),
           (structure(heads=3), "multiple of the key"), (structure(kv_heads=0), "multiple of the key"),
           (structure(dim=20), "head dimension"), (structure(dim=136), "head dimension"),
           (structure(scale=float("nan")), "scale"), (structure(softcap=-1.0), "softcap"),
           (structure(n_keys=-1), "invalid sizes"), (structure(n_structures=0), "invalid sizes"),
           (structure(n_queries=49), "positions of their own"),
           (structure(n_queries=1 << 30, n_keys=1 << 30), "too many atoms"),
           (structure(tiles=None), "tiles"), (structure(tiles=PTR + 16), "tiles"),
           (structure(q=None), "pointers are null"), (structure(key_ptr=None), "pointers are null"),
           (structure(k=PTR + 8), "aligned"), (structure(v_stride=two(64, 12)), "aligned"),
           (structure(q_stride=two(1 << 25, 32)), "aligned")]
    for req, message in bad:
        for f in (lib.tnr_structure_forward, lib.tnr_structure_backward):
            code, said = refused(f, req, PTR, 1 << 40)
            assert code == ext.TNR_INPUT_ERROR and message in said, (message, said)
    for req, message in [(structure(grad_q=None), "pointers are null"),
                         (structure(lse=None), "pointers are null"),
                         (structure(grad_out=PTR + 2), "aligned"),
                         (structure(grad_query_positions=PTR), "the keys'")]:
        code, said = refused(lib.tnr_structure_backward, req, PTR, 1 << 40)
        assert code == ext.TNR_INPUT_ERROR and message in said
    need = lib.tnr_structure_backward_workspace_size(ctypes.byref(structure()))
    assert need > 0 and lib.tnr_structure_tiles_size(ctypes.byref(structure())) > 0
    code, said = refused(lib.tnr_structure_backward, structure(), PTR, need - 1)
    assert code == ext.TNR_INPUT_ERROR and "workspace" in said


def listing(**kw):
    return ext.NeighborList(**(dict(n_pairs=30, n_sources=10, n_targets=10, sources=PTR, targets=PTR,
                                    transpose=1, rows=PTR) | kw))


def neighbor(list_=None, **kw):
    two = ctypes.c_int64 * 2
    return ext.NeighborAttention(**(dict(
        dtype=0, heads=4, kv_heads=4, dim=16, list=list_ or listing(), q=PTR, k=PTR, v=PTR,
        q_stride=two(64, 16), k_stride=two(64, 16), v_stride=two(64, 16), distances=PTR, slopes=PTR,
        scale=0.25, softcap=0.0, out=PTR, out32=None, lse=PTR, grad_out=PTR, grad_q=PTR, grad_k=PTR,
        grad_v=PTR, grad_distances=PTR, grad_slopes=PTR) | kw))


def test_neighbor_requests(lib):  # noqa: F811
    lists = [(listing(n_pairs=-1), "invalid sizes"), (listing(n_sources=0), "sources and targets"),
             (listing(n_pairs=1 << 31), "too many"), (listing(n_targets=1 << 26), "too many"),
             (listing(rows=None), "rows"), (listing(rows=PTR + 4), "rows")]
    for l, message in [(None, "list is null"), (listing(sources=None), "pointers are null"), *lists]:
        code, said = refused(lib.tnr_neighbor_rows, l, PTR, 1 << 40)
        assert code == ext.TNR_INPUT_ERROR and message in said
    need = lib.tnr_neighbor_rows_workspace_size(ctypes.byref(listing()))
    assert lib.tnr_neighbor_rows_size(ctypes.byref(listing())) > 0
    code, said = refused(lib.tnr_neighbor_rows, listing(), PTR, need - 1)
    assert code == ext.TNR_INPUT_ERROR and "workspace" in said
    bad = [(None, "request is null"), (neighbor(dim=20), "head dimension"),
           (neighbor(distances=None), "pointers are null"), (neighbor(k=PTR + 4), "aligned"),
           *((neighbor(l), message) for l, message in lists)]
    for req, message in bad:
        code, said = refused(lib.tnr_neighbor_forward, req)
        assert code == ext.TNR_INPUT_ERROR and message in said
        code, said = refused(lib.tnr_neighbor_backward, req, PTR, 1 << 40)
        assert code == ext.TNR_INPUT_ERROR and message in said
    for req, message in [(neighbor(listing(transpose=0)), "by target"),
                         (neighbor(grad_distances=None), "pointers are null"),
                         (neighbor(dtype=2), "pointers are null"),
                         (neighbor(grad_v=PTR + 8), "aligned")]:
        code, said = refused(lib.tnr_neighbor_backward, req, PTR, 1 << 40)
        assert code == ext.TNR_INPUT_ERROR and message in said
    code, said = refused(lib.tnr_neighbor_backward, neighbor(), PTR, 64)
    assert code == ext.TNR_INPUT_ERROR and "workspace" in said


def test_sizes_beyond_a_launch(lib):  # noqa: F811
    for req in (embedding(n_species=1 << 24), embedding(channels=1 << 19),
                embedding(n_atoms=(1 << 31) - 1)):
        code, said = refused(lib.tnr_embedding_backward, req, PTR, 1 << 40)
        assert code == ext.TNR_INPUT_ERROR and "too many" in said
    code, said = refused(lib.tnr_neighbor_rows, listing(n_pairs=(1 << 31) - 100), PTR, 1 << 40)
    assert code == ext.TNR_INPUT_ERROR and "too many" in said
    code, said = refused(lib.tnr_structure_forward,
                         structure(heads=1, kv_heads=1, n_queries=1 << 30, n_keys=1 << 30), PTR,
                         1 << 40)
    assert code == ext.TNR_INPUT_ERROR and "too many atoms" in said


def test_structure_backward_needs_the_wide_output(lib):  # noqa: F811
    need = lib.tnr_structure_backward_workspace_size(ctypes.byref(structure()))
    code, said = refused(lib.tnr_structure_backward, structure(out32=None), PTR, need)
    assert code == ext.TNR_INPUT_ERROR and "pointers are null" in said
    code, said = refused(lib.tnr_structure_backward, structure(out32=PTR + 4), PTR, need)
    assert code == ext.TNR_INPUT_ERROR and "aligned" in said


def test_no_queries_need_no_positions(lib):  # noqa: F811
    # (the workspace is refused, which comes after the sizes)
    code, said = refused(lib.tnr_structure_backward, structure(n_queries=0), None, 0)
    assert code == ext.TNR_INPUT_ERROR and "workspace" in said


@pytest.mark.parametrize("changed,message", [
    ({"softcap": 1e-46}, "softcap must be finite and positive"),
    ({"softcap": 1e39}, "softcap must be finite and positive"),
    ({"scale": -1e39}, "scale must be finite"),
])
def test_scores_beyond_32_bits(changed, message):
    with pytest.raises(ValueError, match=message):
        structure_attention(**attention_arguments(**changed))
    if "scale" in changed:
        with pytest.raises(ValueError, match=message):
            species_embedding(torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8), **changed)


def test_score_rules_beyond_32_bits(lib):  # noqa: F811
    for rule in (dict(scale=0.25, softcap=1e-40), dict(scale=3e38), dict(softcap=3e38)):
        for req, forward in ((structure(**rule), lambda r: refused(lib.tnr_structure_forward, r, PTR, 1 << 40)),
                             (neighbor(**rule), lambda r: refused(lib.tnr_neighbor_forward, r))):
            code, said = forward(req)
            assert code == ext.TNR_INPUT_ERROR and "too large for 32 bits" in said


def test_sizes_at_the_edge_of_a_launch(lib):  # noqa: F811
    # 2^32 threads are one too many; (the workspace is refused after the sizes)
    most = (1 << 26) - 4
    for n, word in ((most, "workspace"), (most + 1, "too many")):
        code, said = refused(lib.tnr_neighbor_rows, listing(n_targets=n), None, 0)
        assert code == ext.TNR_INPUT_ERROR and word in said
        code, said = refused(lib.tnr_neighbor_backward,
                             neighbor(listing(n_sources=n), heads=1, kv_heads=1), None, 0)
        assert code == ext.TNR_INPUT_ERROR and word in said
    code, said = refused(lib.tnr_embedding_backward, embedding(n_species=1 << 58), PTR, 1 << 40)
    assert code == ext.TNR_INPUT_ERROR and "too many" in said
    for n, word in ((700_000_000, "workspace"), (720_000_000, "too many")):
        code, said = refused(lib.tnr_structure_backward,
                             structure(heads=1, kv_heads=1, n_queries=n, n_keys=n), None, 0)
        assert code == ext.TNR_INPUT_ERROR and word in said, said
