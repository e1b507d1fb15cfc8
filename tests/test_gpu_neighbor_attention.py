"""GPU: attention along a neighbor list against its definition in float64 on the CPU.

Lists of this package's own search (periodic, with images and self pairs), sorted and in bin order,
and lists made by hand: atoms without pairs, long rows, one pair.  Gradients by the formula's own, by
differences, and through the list to positions and cell.  Tolerances: tests/_operators.py.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from tests._operators import assert_near, attend, double
from tonari_amd import neighbor_list
from tonari_amd.attention import neighbor_attention, neighbor_rows

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["float32", "bfloat16", "float16"]
LEAVES = ("q", "k", "v", "d", "slopes")


def random_list(n, m, mean, seed, longest=0):
    """Rows of random lengths, some empty; the first takes `longest` pairs."""
    rng = np.random.default_rng(seed)
    counts = rng.poisson(mean, n)
    counts[rng.random(n) < 0.2] = 0
    if longest:
        counts[0] = longest
    i = torch.as_tensor(np.repeat(np.arange(n), counts))
    return i, torch.as_tensor(rng.integers(0, m, len(i)))


def make(i, j, n, m, heads, kv_heads, dim, dtype, seed=1, grad=True):
    g = torch.Generator().manual_seed(seed)
    c = {"q": torch.randn(n, heads, dim, generator=g).to(dtype),
         "k": torch.randn(m, kv_heads, dim, generator=g).to(dtype),
         "v": torch.randn(m, kv_heads, dim, generator=g).to(dtype),
         "d": 1.0 + 5.0 * torch.rand(len(i), generator=g),
         "slopes": torch.rand(heads, generator=g) - 0.2}
    c = {name: t.to(DEV).requires_grad_(grad) for name, t in c.items()}
    c |= {"i": i.to(DEV), "j": j.to(DEV),
          "upstream": torch.randn(n, heads, dim, generator=g).to(dtype).to(DEV)}
    return c


def call(c, softcap=None, scale=None, transpose=True):
    rows = neighbor_rows(c["i"], c["j"], c["q"].shape[0], c["k"].shape[0], transpose=transpose)
    return neighbor_attention(c["q"], c["k"], c["v"], c["d"], rows, c["slopes"], softcap=softcap,
                              scale=scale)


def expected(c, softcap=None, scale=None):
    leaves = double(*(c[n] for n in LEAVES))
    q, k, v, d, slopes = leaves
    scale = q.shape[2] ** -0.5 if scale is None else scale
    return attend(q, k, v, d, slopes, c["i"].cpu(), c["j"].cpu(), scale, softcap), leaves


def check(c, softcap=None, scale=None):
    out = call(c, softcap, scale)
    ref, leaves = expected(c, softcap, scale)
    assert_near(out, ref, "out")
    grads = torch.autograd.grad(out, [c[n] for n in LEAVES], c["upstream"])
    refs = torch.autograd.grad(ref, leaves, c["upstream"].double().cpu())
    for name, a, e in zip(LEAVES, grads, refs):
        assert_near(a, e, f"gradient of {name}")
    return out, grads


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("softcap", [None, 3.0])
@pytest.mark.parametrize("heads,kv_heads,dim", [
    (1, 1, 8), (2, 1, 16), (3, 3, 24), (4, 1, 32), (8, 2, 40), (6, 2, 48), (2, 2, 64), (12, 3, 72),
    (16, 4, 56), (4, 4, 96), (3, 1, 128), (32, 8, 48),
])
def test_heads_and_widths(dtype, softcap, heads, kv_heads, dim):
    i, j = random_list(60, 50, 20, seed=heads + dim)
    check(make(i, j, 60, 50, heads, kv_heads, dim, dtype), softcap)


@pytest.mark.parametrize("n,m,mean,longest", [
    (1, 1, 0, 1), (5, 3, 1, 0), (400, 400, 3, 0), (7, 2000, 90, 1500), (1100, 9, 30, 0),
    (3, 70_000, 400, 2000),
])
def test_shapes_of_lists(n, m, mean, longest):
    i, j = random_list(n, m, mean, seed=n, longest=longest)
    check(make(i, j, n, m, 4, 2, 16, torch.float32))


@pytest.mark.parametrize("sorted", [False, True])
@pytest.mark.parametrize("half_list", [False, True])
def test_lists_of_the_search(sorted, half_list):
    g = torch.Generator().manual_seed(3)
    edge = 13.0
    x = (torch.rand(500, 3, generator=g) * edge).to(DEV)
    i, j, d = neighbor_list("ijd", x, edge * torch.eye(3, device=DEV),
                            torch.ones(3, dtype=torch.bool, device=DEV), 4.0,
                            algorithm="cell_list", sorted=sorted, half_list=half_list)
    c = make(i.cpu(), j.cpu(), 500, 500, 4, 2, 32, torch.bfloat16)
    c["d"] = d.detach().requires_grad_()
    check(c, 10.0)


def test_images_and_self_pairs():
    # a cell smaller than the cutoff: many pairs of the same two atoms, and of an atom with itself
    x = torch.tensor([[0.1, 0.2, 0.3], [1.0, 1.5, 0.7]], device=DEV)
    i, j, d = neighbor_list("ijd", x, 2.5 * torch.eye(3, device=DEV),
                            torch.ones(3, dtype=torch.bool, device=DEV), 6.0, include_self=True)
    c = make(i.cpu(), j.cpu(), 2, 2, 2, 2, 16, torch.float32)
    c["d"] = d.detach().requires_grad_()
    assert len(i) > 200
    check(c)


def test_forces_and_stress():
    # the gradient of d goes on through the list
    g = torch.Generator().manual_seed(5)
    x = (torch.rand(60, 3, generator=g) * 7.0).to(DEV).requires_grad_()
    cell = (7.0 * torch.eye(3)).to(DEV).requires_grad_()
    pbc = torch.ones(3, dtype=torch.bool, device=DEV)
    i, j, S, d = neighbor_list("ijSd", x, cell, pbc, 3.5)
    c = make(i.cpu(), j.cpu(), 60, 60, 2, 1, 16, torch.float32)
    c["d"] = d
    got = torch.autograd.grad(call(c, 4.0), (x, cell), c["upstream"])

    q, k, v, slopes = double(*(c[n] for n in ("q", "k", "v", "slopes")))
    y, box = double(x, cell)
    ic, jc = i.cpu(), j.cpu()
    r = torch.linalg.vector_norm(y[jc] - y[ic] + S.cpu().double() @ box, dim=1)
    ref = attend(q, k, v, r, slopes, ic, jc, 16**-0.5, 4.0)
    want = torch.autograd.grad(ref, (y, box), c["upstream"].double().cpu())
    for a, e in zip(got, want):
        # the list's own backward is tested to 1e-4 (float atomics)
        err = float((a.double().cpu() - e).abs().max())
        assert err <= 1e-4 * max(1.0, float(e.abs().max()))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_negative_scale_under_the_cap(dtype):
    i, j = random_list(40, 40, 20, seed=13)
    check(make(i, j, 40, 40, 4, 1, 32, dtype, seed=2), 0.5, scale=-0.5)


def test_pairs_that_weigh_nothing():
    i, j = random_list(40, 40, 15, seed=2)
    c = make(i, j, 40, 40, 2, 2, 16, torch.float32, grad=False)
    c["slopes"] = torch.ones(2, device=DEV)
    far = c["d"].clone()
    far[c["i"] == int(c["i"][0])] = float("inf")     # a row at infinite distances
    far[-1] = float("inf")                           # one pair of a row
    c["d"] = far
    for n in ("q", "k", "v"):
        c[n] = c[n].requires_grad_()
    out = call(c)
    grads = torch.autograd.grad(out, [c[n] for n in ("q", "k", "v")], c["upstream"])
    assert bool((out[int(c["i"][0])] == 0).all())
    assert all(bool(torch.isfinite(t).all()) for t in (out, *grads))
    keep = torch.isfinite(far)
    d = dict(c, i=c["i"][keep], j=c["j"][keep], d=far[keep])
    assert_near(out, call(d))


def test_nan_stays_in_its_rows():
    i, j = random_list(50, 50, 12, seed=4)
    c = make(i, j, 50, 50, 4, 2, 24, torch.bfloat16, grad=False)
    clean = call(c)
    for name in ("k", "v"):
        bad = dict(c, **{name: c[name].clone()})
        bad[name][9, 1] = float("nan")
        out = call(bad)
        touched = torch.zeros(50, dtype=torch.bool, device=DEV)
        touched[c["i"][c["j"] == 9]] = True
        assert torch.equal(out[~touched], clean[~touched])
        assert torch.equal(out[:, :2], clean[:, :2])          # the other key head
        assert not bool(torch.isfinite(out[touched][:, 2:]).all())


def test_rows_are_shared_and_repeats_equal():
    i, j = random_list(300, 300, 40, seed=6)
    c = make(i, j, 300, 300, 8, 2, 32, torch.float16)
    rows = neighbor_rows(c["i"], c["j"], 300)
    outs = []
    for _ in range(3):
        out = neighbor_attention(c["q"], c["k"], c["v"], c["d"], rows, c["slopes"])
        outs.append((out, *torch.autograd.grad(out, [c[n] for n in LEAVES], c["upstream"])))
    for again in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], again))
    plain = neighbor_rows(c["i"], c["j"], 300, transpose=False)
    with torch.no_grad():
        assert torch.equal(neighbor_attention(c["q"], c["k"], c["v"], c["d"], plain, c["slopes"]),
                           outs[0][0])
    with pytest.raises(ValueError, match="transpose=True"):
        neighbor_attention(c["q"], c["k"], c["v"], c["d"], plain, c["slopes"])


def test_strides():
    i, j = random_list(64, 64, 25, seed=7)
    c = make(i, j, 64, 64, 4, 4, 24, torch.bfloat16)
    out, grads = check(c)
    packed = torch.stack([c["q"], c["k"], c["v"]], 1).detach()
    d = dict(c, q=packed[:, 0].requires_grad_(), k=packed[:, 1].requires_grad_(),
             v=packed[:, 2].requires_grad_())
    again = call(d)
    assert torch.equal(again, out)
    for a, e in zip(torch.autograd.grad(again, [d[n] for n in LEAVES], c["upstream"]), grads):
        assert torch.equal(a, e)


def test_by_differences():
    i, j = random_list(30, 30, 10, seed=8)
    c = make(i, j, 30, 30, 2, 1, 16, torch.float32)
    w = c["upstream"]
    grads = dict(zip(LEAVES, torch.autograd.grad(call(c, 4.0), [c[n] for n in LEAVES], w)))
    g = torch.Generator().manual_seed(5)
    for name in LEAVES:
        way = torch.randn(c[name].shape, generator=g).to(DEV)
        way /= way.norm()
        step = 2.0**-6
        with torch.no_grad():
            up = (call(dict(c, **{name: c[name] + step * way}), 4.0).double() * w).sum()
            down = (call(dict(c, **{name: c[name] - step * way}), 4.0).double() * w).sum()
        along = float((grads[name].double() * way).sum())
        assert abs(float(up - down) / (2 * step) - along) <= 2e-3 * max(
            1.0, float(grads[name].norm())), name


def test_gradient_of_the_gradient():
    i, j = random_list(20, 20, 6, seed=9)
    c = make(i, j, 20, 20, 2, 1, 16, torch.float32)

    def second(out, d, leaves, w):
        first = torch.autograd.grad(out, d, w, create_graph=True)[0]
        return torch.autograd.grad((first * first).sum(), leaves)

    got = second(call(c, 4.0), c["d"], [c[n] for n in LEAVES], c["upstream"])
    ref, leaves = expected(c, 4.0)
    want = second(ref, leaves[3], leaves, c["upstream"].double().cpu())
    for name, a, e in zip(LEAVES, got, want):
        assert_near(a, e, name)


def test_inputs_that_depend_on_each_other():
    # q and d of one tensor: the graph's gradient takes each path once
    i, j = random_list(20, 20, 6, seed=9)
    c = make(i, j, 20, 20, 2, 1, 16, torch.float32, grad=False)
    found = []
    for graph in (False, True):
        x = c["d"].detach().clone().requires_grad_()
        d = dict(c, d=x, q=c["q"] * x.sum() * 0.01, v=c["v"] * x.mean())
        found.append(torch.autograd.grad(call(d, 5.0), x, c["upstream"], create_graph=graph)[0])
    assert_near(found[1], found[0])


@pytest.mark.parametrize("i,j", [
    ([0, 1, 0], [1, 0, 2]),          # the pairs of 0 do not lie together
    ([0, 0, 3], [1, 2, 0]),          # no such source
    ([0, -1, 1], [1, 2, 0]),
    ([0, 0, 1], [1, 3, 0]),          # no such target
    ([0, 0, 1], [1, -2, 0]),
])
def test_wrong_lists_are_nan(i, j):
    c = make(torch.tensor(i), torch.tensor(j), 3, 3, 2, 2, 16, torch.float32)
    out = call(c)
    assert bool(torch.isnan(out).all())
    for t in torch.autograd.grad(out, [c[n] for n in LEAVES], c["upstream"]):
        assert bool(torch.isnan(t).all())


def test_empty():
    none = torch.empty(0, dtype=torch.int64)
    for n, m in ((0, 0), (4, 0), (4, 6), (0, 6)):
        c = make(none, none, n, m, 2, 1, 16, torch.float32)
        out = call(c)
        assert out.shape == (n, 2, 16) and bool((out == 0).all())
        for name, t in zip(LEAVES, torch.autograd.grad(out, [c[x] for x in LEAVES], c["upstream"])):
            assert t.shape == c[name].shape and bool((t == 0).all())


def test_in_a_graph():
    i, j = random_list(90, 90, 20, seed=10)
    c = make(i, j, 90, 90, 4, 4, 16, torch.float32, grad=False)
    fixed = {n: c[n].clone() for n in ("q", "d")}
    d = dict(c, **fixed)
    for _ in range(2):
        call(d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(d)
    for seed in range(4):
        other = make(i, j, 90, 90, 4, 4, 16, torch.float32, grad=False, seed=20 + seed)
        for n in fixed:
            fixed[n].copy_(other[n])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call(dict(c, **{n: other[n] for n in fixed})))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 8), (4, 4, 16), (4, 1, 32), (2, 1, 128)])
def test_first_pairs_far_below_the_rest(dtype, heads, kv_heads, dim):
    # the first 20 pairs of a row score below -200, where exp has nothing left
    i, j = random_list(30, 30, 40, seed=14)
    c = make(i, j, 30, 30, heads, kv_heads, dim, dtype, seed=4)
    with torch.no_grad():
        c["slopes"].fill_(1.0)
        first = torch.searchsorted(c["i"], torch.arange(30, device=DEV))
        place = torch.arange(len(i), device=DEV) - first[c["i"]]
        c["d"] += torch.where(place < 20, 250.0, 0.0)
    out = call(c)
    ref, leaves = expected(c)
    assert_near(out, ref, "out")
    grads = torch.autograd.grad(out, [c[n] for n in LEAVES], c["upstream"])
    refs = torch.autograd.grad(ref, leaves, c["upstream"].double().cpu())
    for name, a, e in list(zip(LEAVES, grads, refs))[:4]:
        assert_near(a, e, f"gradient of {name}")


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 8), (1, 1, 16), (2, 2, 8), (2, 1, 8),
                                                (4, 1, 8)])
@pytest.mark.parametrize("pairs", [64, 65, 90, 128, 150, 300])
def test_long_rows_of_narrow_heads(dtype, heads, kv_heads, dim, pairs):
    # a pair takes a lane or two, so that a wave takes all 64 pairs of a chunk in a step or less
    i = torch.arange(3).repeat_interleave(torch.tensor([pairs, 0, pairs + 1]))
    j = torch.randint(0, 40, (len(i),), generator=torch.Generator().manual_seed(pairs))
    check(make(i, j, 3, 40, heads, kv_heads, dim, dtype, seed=3), 4.0)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 8), (4, 4, 16), (4, 1, 32), (2, 1, 128)])
def test_slopes_of_rows_whose_first_pairs_are_far(dtype, heads, kv_heads, dim):
    # distances near 250, which weigh nothing, before those that carry the row
    i, j = random_list(30, 30, 40, seed=14)
    c = make(i, j, 30, 30, heads, kv_heads, dim, dtype, seed=4)
    with torch.no_grad():
        c["slopes"].fill_(1.0)
        first = torch.searchsorted(c["i"], torch.arange(30, device=DEV))
        place = torch.arange(len(i), device=DEV) - first[c["i"]]
        c["d"] += torch.where(place < 20, 250.0, 0.0)
    check(c)


def test_rows_of_another_list():
    # a tuple altered by hand is refused by its size, or read no further than its head
    def given(i, j, n, m):
        c = make(i, j, n, m, 2, 1, 16, torch.float32)
        return c, neighbor_rows(c["i"], c["j"], n, m)

    def attend_along(c, rows):
        return neighbor_attention(c["q"], c["k"], c["v"], c["d"], rows, c["slopes"])

    c, rows = given(*random_list(10, 12, 4, seed=1), 10, 12)
    plain = neighbor_rows(c["i"], c["j"], 10, 12, transpose=False)
    with pytest.raises(ValueError, match="not those of this list"):
        attend_along(c, plain._replace(transpose=True))
    with pytest.raises(ValueError, match="not those of this list"):
        attend_along(c, rows._replace(rows=rows.rows[:256]))
    fewer = make(c["i"].cpu()[:-1], c["j"].cpu()[:-1], 10, 12, 2, 1, 16, torch.float32)
    for other, altered in (
            (dict(c, k=c["k"][:11], v=c["v"][:11]), rows._replace(n_targets=11)),
            (dict(c, q=c["q"][:9], upstream=c["upstream"][:9]), rows._replace(n_sources=9)),
            (dict(fewer), rows._replace(i=fewer["i"], j=fewer["j"]))):
        for n in ("q", "k", "v"):
            other[n] = other[n].detach().requires_grad_()
        out = attend_along(other, altered)
        assert bool(torch.isnan(out).all())
        for t in torch.autograd.grad(out, [other[n] for n in LEAVES], other["upstream"]):
            assert bool(torch.isnan(t).all())
    assert bool(torch.isfinite(attend_along(c, rows)).all())


@pytest.mark.parametrize("i,j", [
    ([0, 1, 0], [1, 0, 2]), ([0, 0, 3], [1, 2, 0]), ([0, -1, 1], [1, 2, 0]), ([0, 0, 1], [1, 3, 0]),
    ([0, 0, 1], [1, -2, 0]), ([0, 0, 1], [1, 1 << 40, 0]),
])
def test_graphs_of_wrong_lists_are_nan(i, j):
    c = make(torch.tensor(i), torch.tensor(j), 3, 3, 2, 2, 16, torch.float32)
    grads = torch.autograd.grad(call(c), [c[n] for n in LEAVES], c["upstream"], create_graph=True)
    again = torch.autograd.grad(sum(t.sum() for t in grads), [c[n] for n in LEAVES])
    for t in (*grads, *again):
        assert bool(torch.isnan(t).all())


def test_graph_of_pairs_that_weigh_nothing():
    i, j = random_list(40, 40, 15, seed=2)
    c = make(i, j, 40, 40, 2, 2, 16, torch.float32, grad=False)
    c["slopes"] = torch.ones(2, device=DEV)
    c["d"] = torch.where(c["i"] == c["i"][0], float("inf"), c["d"])     # a row, and a pair of another
    c["d"][-1] = float("inf")
    leaves = [c[n].requires_grad_() for n in ("q", "k", "v")]
    out = call(c)
    plain = torch.autograd.grad(out, leaves, c["upstream"], retain_graph=True)
    graph = torch.autograd.grad(out, leaves, c["upstream"], create_graph=True)
    for a, e in zip(graph, plain):
        assert_near(a, e)
    for t in torch.autograd.grad(sum((t * t).sum() for t in graph), leaves):
        assert bool(torch.isfinite(t).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 2, 16), (2, 2, 24), (3, 1, 40), (4, 1, 48)])
def test_keys_at_minus_infinity(dtype, heads, kv_heads, dim):
    # keys that are masked by a channel of -inf leave their pairs without weight, also where a
    # head's channels do not fill its lanes
    i, j = random_list(30, 30, 12, seed=15)
    c = make(i, j, 30, 30, heads, kv_heads, dim, dtype, seed=5, grad=False)
    c["q"] = c["q"].abs() + 0.1
    c["k"][7, :, 0] = c["k"][11, :, dim - 1] = float("-inf")
    keep = (c["j"] != 7) & (c["j"] != 11)
    assert_near(call(c), call(dict(c, i=c["i"][keep], j=c["j"][keep], d=c["d"][keep])))
