"""GPU: attention within structures against its definition in float64 on the CPU.

Lengths from one atom to several tiles, structures without atoms or queries, shared key heads, head
widths that fill no tile, strided and misaligned tensors, splits of long rows, gradients by the
formula's own (float64 autograd of the definition) and by differences.  Tolerances: tests/_operators.py.
"""

from __future__ import annotations

import pytest
import torch

from tests._operators import HALF_SPACING, assert_near, attend, distances, double, pointer, structure_pairs
from tests._operators import tolerance
from tonari_amd.attention import structure_attention

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def make(lengths, heads, kv_heads, dim, dtype, *, queries=None, seed=1, grad=True, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    n = sum(lengths)
    m = n if queries is None else sum(queries)
    c = {"q": spread * torch.randn(m, heads, dim, generator=g),
         "k": torch.randn(n, kv_heads, dim, generator=g),
         "v": torch.randn(n, kv_heads, dim, generator=g)}
    c = {name: t.to(dtype) for name, t in c.items()}
    c["positions"] = 4.0 * torch.randn(n, 3, generator=g)
    c["slopes"] = torch.rand(heads, generator=g) * 0.6 - 0.1
    c["query_positions"] = 4.0 * torch.randn(m, 3, generator=g) if queries is not None else None
    for name, t in c.items():
        if t is not None:
            c[name] = t.to(DEV).requires_grad_(grad)
    c["batch_ptr"] = pointer(lengths).to(DEV)
    c["query_ptr"] = pointer(queries).to(DEV) if queries is not None else None
    c["upstream"] = torch.randn(m, heads, dim, generator=g).to(dtype).to(DEV)
    return c


LEAVES = ("q", "k", "v", "positions", "slopes", "query_positions")


def call(c, softcap=None, scale=None):
    return structure_attention(c["q"], c["k"], c["v"], c["positions"], c["batch_ptr"], c["slopes"],
                               softcap=softcap, scale=scale, query_positions=c["query_positions"],
                               query_ptr=c["query_ptr"])


def expected(c, softcap=None, scale=None):
    q, k, v, x, slopes, y = double(*(c[n] for n in LEAVES))
    kp = c["batch_ptr"].tolist()
    qp = kp if c["query_ptr"] is None else c["query_ptr"].tolist()
    source, target = structure_pairs(qp, kp)
    r = distances((x if y is None else y)[source], x[target])
    scale = q.shape[2] ** -0.5 if scale is None else scale
    out = attend(q, k, v, r, slopes, source, target, scale, softcap)
    return out, [t for t in (q, k, v, x, slopes, y) if t is not None]


def check(c, softcap=None, scale=None):
    out = call(c, softcap, scale)
    ref, leaves = expected(c, softcap, scale)
    assert_near(out, ref, "out")
    given = [c[n] for n in LEAVES if c[n] is not None]
    names = [n for n in LEAVES if c[n] is not None]
    grads = torch.autograd.grad(out, given, c["upstream"])
    refs = torch.autograd.grad(ref, leaves, c["upstream"].double().cpu())
    for name, a, e in zip(names, grads, refs):
        assert_near(a, e, f"gradient of {name}")
    return out, grads


DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["float32", "bfloat16", "float16"]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("softcap", [None, 5.0])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim", [
    ([1], 1, 1, 8),
    ([2, 1, 3], 2, 1, 16),
    ([31, 32, 33], 4, 4, 32),
    ([0, 64, 0, 65, 127, 0], 4, 2, 40),
    ([129, 1, 20], 3, 1, 64),
    ([70, 200], 2, 2, 72),
    ([97], 8, 2, 96),
    ([45, 150], 2, 1, 128),
])
def test_self_attention(dtype, softcap, lengths, heads, kv_heads, dim):
    check(make(lengths, heads, kv_heads, dim, dtype), softcap)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("lengths,queries,heads,kv_heads,dim", [
    ([40, 700, 3], [1, 1, 1], 8, 2, 64),
    ([0, 50, 600], [2, 0, 5], 4, 4, 24),       # queries without keys, keys without queries
    ([2500], [1], 4, 1, 32),                   # keys split over workgroups
    ([1, 1], [300, 40], 2, 2, 16),             # rows split in the keys' gradients
    ([3], [2100], 4, 1, 48),
])
def test_queries_of_their_own(dtype, lengths, queries, heads, kv_heads, dim):
    c = make(lengths, heads, kv_heads, dim, dtype, queries=queries)
    out, _ = check(c, 8.0)
    for b, n in enumerate(lengths):
        if n == 0:
            rows = out[c["query_ptr"][b]:c["query_ptr"][b + 1]]
            assert bool((rows == 0).all())


@pytest.mark.parametrize("dtype", DTYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("lengths,queries,heads,kv_heads,dim", [
    ([4000, 3973, 4500], [1, 1, 1], 2, 2, 40),  # keys split over workgroups
    ([700, 40], [7, 3], 4, 1, 64),
    ([550, 600, 3], [2, 2, 2], 8, 1, 128),
    ([20, 5, 1, 32], None, 3, 3, 32),
])
def test_few_rows_round_once(dtype, lengths, queries, heads, kv_heads, dim):
    # Few rows: the output's rounding, u |out|, is the only one to its type.  The weights' remainder
    # after their rounding is rounded itself, u^2 of the weights, and 32-bit sums and scores add 2e-5
    # of them, each times the values' magnitude.
    c = make(lengths, heads, kv_heads, dim, dtype, queries=queries, grad=False)
    out = call(c, 8.0).double().cpu()
    ref, _ = expected(c, 8.0)
    size, _ = expected({**c, "v": c["v"].abs()}, 8.0)
    u = HALF_SPACING[dtype]
    assert bool(((out - ref).abs() <= u * ref.abs() + (2e-5 + u * u) * size).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_long_structure(dtype):
    check(make([1300], 4, 2, 32, dtype, seed=3), 20.0)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_many_small_structures(dtype):
    g = torch.Generator().manual_seed(9)
    lengths = torch.randint(0, 40, (300,), generator=g).tolist()
    check(make(lengths, 2, 1, 16, dtype, seed=4))


def test_large_scores_and_negative_scale():
    # scores far apart: one key takes all the weight, and the maximum moves from tile to tile
    c = make([150], 2, 2, 32, torch.float32, spread=20.0)
    check(c)
    check(c, scale=-0.3)
    check(c, 50.0)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_negative_scale_under_the_cap(dtype):
    # products far beyond the cap on either side
    check(make([70, 33], 2, 1, 32, dtype, seed=24, spread=4.0), 2.0, scale=-0.5)


def test_far_atoms():
    # far atoms weigh nothing; a lone far atom still attends to itself
    c = make([60], 2, 2, 32, torch.float32, grad=False)
    x = c["positions"].clone()
    x[7] += 1.0e4
    c["positions"] = x.requires_grad_()
    c["slopes"] = torch.tensor([1.0, 2.0], device=DEV, requires_grad=True)
    for n in ("q", "k", "v"):
        c[n] = c[n].requires_grad_()
    out, _ = check(c)
    assert torch.allclose(out[7], c["v"][7], atol=1e-5)


def test_coincident_atoms():
    # the distance's gradient at 0 is 0, not NaN
    c = make([5, 9], 2, 2, 16, torch.float32)
    with torch.no_grad():
        c["positions"][3] = c["positions"][2]
        c["positions"][8:11] = 0.5
    check(c)


def test_other_structures_do_not_reach_in():
    # NaN and infinities in one structure stay there, also where a tile crosses its end
    c = make([20, 33, 50], 2, 2, 32, torch.bfloat16, grad=False)
    clean = call(c)
    for name, bad in (("k", float("nan")), ("v", float("inf")), ("q", float("-inf")),
                      ("positions", float("nan"))):
        d = dict(c)
        d[name] = c[name].clone()
        d[name][20:53] = bad
        out = call(d)
        assert torch.equal(out[:20], clean[:20]) and torch.equal(out[53:], clean[53:])
        assert not bool(torch.isfinite(out[20:53]).all())


def test_infinite_distance_leaves_nothing():
    # every key at an infinite distance: the row has no weight, and no gradient
    c = make([4], 2, 2, 16, torch.float32, queries=[2], grad=False)
    y = c["query_positions"].clone()
    y[1] = float("inf")
    c["query_positions"] = y
    c["slopes"] = torch.ones(2, device=DEV)
    for n in ("q", "k", "v"):
        c[n] = c[n].requires_grad_()
    out = call(c)
    assert bool((out[1] == 0).all()) and bool(torch.isfinite(out[0]).all())
    gq, gk, gv = torch.autograd.grad(out, [c[n] for n in ("q", "k", "v")], c["upstream"])
    assert bool((gq[1] == 0).all())
    assert all(bool(torch.isfinite(t).all()) for t in (gq, gk, gv))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_strides_and_alignment(dtype):
    c = make([37, 66], 4, 2, 40, dtype, seed=6)
    base, grads = check(c, 10.0)
    n = 103

    def same(d):
        out = call(d, 10.0)
        assert torch.equal(out, base)
        got = torch.autograd.grad(out, [d[x] for x in LEAVES if d[x] is not None], c["upstream"])
        for a, e in zip(got, grads):
            assert torch.equal(a, e)

    # one tensor of q, k and v side by side; heads before atoms; off 16 bytes; channels apart
    packed = torch.cat([c["q"], c["k"], c["v"]], 1).detach()
    d = dict(c, q=packed[:, :4], k=packed[:, 4:6], v=packed[:, 6:])
    for x in ("q", "k", "v"):
        d[x] = d[x].detach().requires_grad_()
    assert not d["q"].is_contiguous()
    same(d)
    same(dict(c, k=c["k"].detach().transpose(0, 1).contiguous().transpose(0, 1).requires_grad_()))
    flat = torch.empty(n * 2 * 40 + 1, dtype=dtype, device=DEV)
    flat[1:] = c["v"].detach().reshape(-1)
    same(dict(c, v=flat[1:].view(n, 2, 40).requires_grad_()))
    wide = torch.empty(n, 4, 80, dtype=dtype, device=DEV)
    wide[:, :, ::2] = c["q"].detach()
    same(dict(c, q=wide[:, :, ::2].requires_grad_()))


def test_expanded_inputs():
    # one set of keys for all heads, broadcast: its gradient is summed over them
    c = make([50], 4, 1, 32, torch.float32, seed=8)
    k = c["k"].detach().requires_grad_()
    out = structure_attention(c["q"], k.expand(50, 4, 32), c["v"].detach().expand(50, 4, 32),
                              c["positions"], c["batch_ptr"], c["slopes"])
    shared = structure_attention(c["q"], c["k"], c["v"], c["positions"], c["batch_ptr"], c["slopes"])
    assert_near(out, shared)
    assert_near(torch.autograd.grad(out, k, c["upstream"])[0],
                torch.autograd.grad(shared, c["k"], c["upstream"])[0])


def test_by_differences():
    # central differences of the float64 definition would only check autograd: take them of the
    # operator itself, float32, step 2^-6, error of third order plus rounding over the step
    c = make([25, 12], 2, 1, 16, torch.float32, seed=12)
    w = c["upstream"]
    out = call(c, 6.0)
    grads = dict(zip(LEAVES, torch.autograd.grad(out, [c[n] for n in LEAVES if c[n] is not None], w)))
    g = torch.Generator().manual_seed(5)
    for name in ("q", "k", "v", "positions", "slopes"):
        way = torch.randn(c[name].shape, generator=g).to(DEV)
        way /= way.norm()
        step = 2.0**-6
        with torch.no_grad():
            up = (call(dict(c, **{name: c[name] + step * way}), 6.0).double() * w).sum()
            down = (call(dict(c, **{name: c[name] - step * way}), 6.0).double() * w).sum()
        slope = float(up - down) / (2 * step)
        along = float((grads[name].double() * way).sum())
        assert abs(slope - along) <= 2e-3 * max(1.0, float(grads[name].norm())), name


def test_small_float16_gradients():
    # upstream gradients near the type's smallest values keep their digits
    c = make([90], 2, 2, 32, torch.float16, seed=14)
    c["upstream"] = (c["upstream"].float() * 2.0**-12).half()
    out = call(c)
    ref, leaves = expected(c)
    grads = torch.autograd.grad(out, [c[n] for n in ("q", "k", "v")], c["upstream"])
    refs = torch.autograd.grad(ref, leaves[:3], c["upstream"].double().cpu())
    for a, e in zip(grads, refs):
        # outputs near 2^-14 are rounded to multiples of 2^-24
        err = float((a.double().cpu() - e).abs().max())
        assert err <= 8 * 2.0**-11 * float(e.abs().max()) + 2.0**-24


def test_large_float16_gradients():
    c = make([90, 40], 2, 2, 32, torch.float16, seed=15)
    c["upstream"] = (c["upstream"].float() * 2.0**10).half()
    check(c)


def test_repeats_are_equal_bits():
    c = make([333, 80], 4, 2, 32, torch.bfloat16, seed=16)
    first = check(c, 9.0)
    for _ in range(3):
        out = call(c, 9.0)
        got = torch.autograd.grad(out, [c[n] for n in LEAVES if c[n] is not None], c["upstream"])
        assert torch.equal(out, first[0])
        assert all(torch.equal(a, b) for a, b in zip(got, first[1]))


def test_only_what_needs_a_gradient():
    c = make([60, 41], 2, 2, 32, torch.float32, seed=17)
    out, grads = check(c)
    d = dict(c, positions=c["positions"].detach(), slopes=c["slopes"].detach())
    got = torch.autograd.grad(call(d), [d[n] for n in ("q", "k", "v")], c["upstream"])
    for a, e in zip(got, grads):
        assert torch.equal(a, e)
    with torch.no_grad():
        assert torch.equal(call(c), out)
    # queries at the atoms' own positions, which stay fixed: only the keys' share
    fixed = dict(c, query_positions=c["positions"].detach(), query_ptr=c["batch_ptr"])
    moving = torch.autograd.grad(call(fixed), c["positions"], c["upstream"])[0]
    ref, leaves = expected(fixed)
    assert_near(moving, torch.autograd.grad(ref, leaves[3], c["upstream"].double().cpu())[0])


def test_gradient_of_the_gradient():
    c = make([9, 0, 14], 2, 1, 16, torch.float32, seed=18)

    def second(out, x, leaves, w):
        force = torch.autograd.grad(out, x, w, create_graph=True)[0]
        return force, torch.autograd.grad((force * force).sum(), leaves)

    out = call(c, 5.0)
    names = ("q", "k", "v", "positions", "slopes")
    force, got = second(out, c["positions"], [c[n] for n in names], c["upstream"])
    ref, leaves = expected(c, 5.0)
    ref_force, want = second(ref, leaves[3], leaves, c["upstream"].double().cpu())
    assert_near(force, ref_force)
    for name, a, e in zip(names, got, want):
        assert_near(a, e, name)


def test_inputs_that_depend_on_each_other():
    # q, k and v of the positions: the graph's gradient takes each path once
    c = make([9, 0, 14], 2, 1, 16, torch.float32, seed=19, grad=False)
    g = torch.Generator().manual_seed(2)
    mix = [torch.randn(3, h * 16, generator=g).to(DEV) * 0.3 for h in (2, 1, 1)]
    found = []
    for graph in (False, True):
        x = c["positions"].detach().clone().requires_grad_()
        d = dict(c, positions=x, **{n: (x @ m).view(23, -1, 16) for n, m in zip("qkv", mix)})
        found.append(torch.autograd.grad(call(d, 5.0), x, c["upstream"], create_graph=graph)[0])
    assert_near(found[1], found[0])


@pytest.mark.parametrize("ptr", [[0, 5, 3, 10], [1, 5, 7, 10], [0, 5, 7, 9], [0, 5, 7, 11]])
def test_wrong_pointers_are_nan(ptr):
    c = make([10], 2, 2, 16, torch.float32, grad=False)
    c["batch_ptr"] = torch.tensor(ptr, dtype=torch.int64, device=DEV)
    c["q"] = c["q"].requires_grad_()
    c["k"] = c["k"].requires_grad_()
    c["positions"] = c["positions"].requires_grad_()
    out = call(c)
    assert bool(torch.isnan(out).all())
    for t in torch.autograd.grad(out, (c["q"], c["k"], c["positions"]), c["upstream"]):
        assert bool(torch.isnan(t).all())


def test_empty():
    for lengths in ([], [0], [0, 0]):
        c = make(lengths, 2, 1, 16, torch.float32)
        out = call(c)
        assert out.shape == (0, 2, 16)
        torch.autograd.grad(out.sum(), c["q"])


def test_float64_positions():
    c = make([30], 2, 2, 16, torch.float32, seed=21)
    d = dict(c, positions=c["positions"].detach().double().requires_grad_())
    out = call(d)
    assert torch.equal(out, call(c))
    assert torch.autograd.grad(out, d["positions"], c["upstream"])[0].dtype == torch.float64


def test_on_another_stream():
    c = make([120, 44], 4, 2, 32, torch.bfloat16, seed=22)
    want, grads = check(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = call(c)
        got = torch.autograd.grad(out, [c[n] for n in LEAVES if c[n] is not None], c["upstream"])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)
    assert all(torch.equal(a, b) for a, b in zip(got, grads))


def test_in_a_graph():
    c = make([70, 33], 4, 2, 32, torch.bfloat16, grad=False, seed=23)
    fixed = {n: c[n].clone() for n in ("q", "k", "v")}
    d = dict(c, **fixed)
    for _ in range(2):
        call(d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(d)
    for seed in range(4):
        other = make([70, 33], 4, 2, 32, torch.bfloat16, grad=False, seed=30 + seed)
        for n in ("q", "k", "v"):
            fixed[n].copy_(other[n])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call(dict(c, **{n: other[n] for n in ("q", "k", "v")})))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("where", [40, 70, 250])
def test_lone_atom_of_a_later_tile(dtype, where):
    # every key of the first tiles scores far below what exp holds; the atom's own key comes later
    c = make([256], 2, 1, 32, dtype, seed=25)
    with torch.no_grad():
        c["positions"][where] += 300.0
        c["slopes"].copy_(torch.tensor([0.5, 2.0]))
    check(c)


def check_scores(c, score):
    """check() where the scores that carry weight go up to `score`: 32 bits hold these to 2^-24 of it,
    so that the tolerance of scores up to 2^6 grows with it."""
    out = call(c)
    ref, leaves = expected(c)
    given = [n for n in LEAVES if c[n] is not None]
    grads = torch.autograd.grad(out, [c[n] for n in given], c["upstream"])
    refs = torch.autograd.grad(ref, leaves, c["upstream"].double().cpu())
    for name, a, e in zip(["out", *given], (out, *grads), (ref, *refs)):
        a, most = a.detach().double().cpu(), max(tolerance(a.dtype), 2e-5 * score / 64)
        assert bool(((a - e).abs() <= most * e.abs().max()).all()), name


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_far_keys_before_near_ones(dtype):
    # an ordered slab, split over workgroups: whole splits lie hundreds of lengths away, and the
    # nearest key of the last query 1,100
    c = make([5000], 2, 2, 16, dtype, queries=[3], seed=26)
    with torch.no_grad():
        c["positions"][:, 0] = torch.linspace(-900.0, 900.0, 5000, device=DEV)
        c["query_positions"][:, 0] = torch.tensor([890.0, 0.0, -2000.0], device=DEV)
        c["slopes"].fill_(1.0)
    check_scores(c, 1100.0)


def test_scores_far_below_zero():
    # q.k of -8 8 32 / sqrt(32)
    c = make([150], 2, 2, 32, torch.float32, seed=27)
    g = torch.Generator().manual_seed(3)
    with torch.no_grad():
        c["q"].fill_(8.0)
        c["k"].copy_(-8.0 + 0.05 * torch.randn(c["k"].shape, generator=g))
    check_scores(c, 362.0)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 16), (4, 1, 32), (2, 1, 128)])
def test_slopes_where_the_middle_atom_is_far(dtype, heads, kv_heads, dim):
    c = make([200], heads, kv_heads, dim, dtype, seed=31)
    with torch.no_grad():
        c["positions"][100] += 300.0
        c["slopes"].fill_(1.0)
    check(c)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_no_queries_at_all(dtype):
    # keys that nobody asks: an empty output, and gradients of 0
    c = make([5, 40, 0], 4, 2, 16, dtype, queries=[0, 0, 0], seed=32)
    out = call(c)
    assert out.shape == (0, 4, 16)
    for t in torch.autograd.grad(out, [c[n] for n in LEAVES], c["upstream"]):
        assert bool((t == 0).all())


@pytest.mark.parametrize("ptr", [[0, 5, 3, 10], [1, 5, 7, 10], [0, 5, 7, 9], [0, 5, 7, 11],
                                 [0, -5, 1 << 40, 10]])
def test_graphs_of_wrong_pointers_are_nan(ptr):
    c = make([10], 2, 2, 16, torch.float32)
    c["batch_ptr"] = torch.tensor(ptr, dtype=torch.int64, device=DEV)
    leaves = [c[n] for n in LEAVES if c[n] is not None]
    grads = torch.autograd.grad(call(c), leaves, c["upstream"], create_graph=True)
    again = torch.autograd.grad(sum(t.sum() for t in grads), leaves)
    for t in (*grads, *again):
        assert bool(torch.isnan(t).all())


def test_graphs_without_pairs():
    for lengths, queries in (([], None), ([0, 0], None), ([0, 3], [2, 0]), ([3], [0])):
        c = make(lengths, 2, 1, 16, torch.float32, queries=queries, seed=33)
        leaves = [c[n] for n in LEAVES if c[n] is not None]
        for t in torch.autograd.grad(call(c), leaves, c["upstream"], create_graph=True):
            assert bool((t == 0).all())


def test_graph_of_a_row_without_weight():
    c = make([4], 2, 2, 16, torch.float32, queries=[2], grad=False)
    c["query_positions"][1] = float("inf")
    c["slopes"] = torch.ones(2, device=DEV)
    leaves = [c[n].requires_grad_() for n in ("q", "k", "v")]
    out = call(c)
    plain = torch.autograd.grad(out, leaves, c["upstream"], retain_graph=True)
    graph = torch.autograd.grad(out, leaves, c["upstream"], create_graph=True)
    for a, e in zip(graph, plain):
        assert_near(a, e)
    for t in torch.autograd.grad(sum((t * t).sum() for t in graph), leaves):
        assert bool(torch.isfinite(t).all())


def test_graph_beyond_the_memory():
    c = make([1500], 8, 8, 64, torch.float32, seed=34)
    out = call(c)
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    torch.cuda.set_per_process_memory_fraction(2.0 * 2**30 / total)
    try:
        with pytest.raises(torch.OutOfMemoryError, match="create_graph holds .* fewer structures"):
            torch.autograd.grad(out, c["positions"], c["upstream"], create_graph=True)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert bool(torch.isfinite(torch.autograd.grad(out, c["positions"], c["upstream"])[0]).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("softcap", [None, 4.0])
@pytest.mark.parametrize("queries", [None, [3] * 50])
def test_one_key_is_its_value(dtype, softcap, queries):
    # the weight is 1 whatever the score, and nothing moves it: exact, to the bit
    c = make([1] * 50, 4, 2, 24, dtype, queries=queries, seed=35)
    out = call(c, softcap)
    of = torch.arange(50, device=DEV) if queries is None else torch.arange(50, device=DEV).repeat_interleave(3)
    assert torch.equal(out, c["v"][of].repeat_interleave(2, 1))
    names = [n for n in LEAVES if c[n] is not None and n != "v"]
    for n, t in zip(names, torch.autograd.grad(out, [c[n] for n in names], c["upstream"])):
        assert bool((t == 0).all()), n
