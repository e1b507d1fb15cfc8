"""Cases of the operators that an atomistic transformer runs next to a neighbor list.

``species_embedding``   rows of a table by the atoms' species, and the table's gradient
``structure_attention`` atoms attend to all atoms of their own structure (batch_ptr), with a bias
                        that falls with distance and an optional tanh cap of the scores
``neighbor_attention``  the same along the pairs (i, j, d) of a neighbor list

``run`` computes them in their plain form (elementary torch operations in 32 bits, rounded once at
the end) or, where ``own`` is true, through this repository's operators.  Sizes are those of the
repository's workloads (512-atom box, 256 crystals of 2 to 64 atoms, 1024 molecules of 20 to 120
atoms, the 100,000-atom box, 64 slabs of 2,000 to 20,000 atoms) with generic widths.

With x = scale q.k and c the cap (u = x without one), a query's score of a key is
u - slope r, u = c tanh(x / c); its output is the softmax-weighted sum of the values.
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
CUTOFF = 6.0


# ------------------------------------------------------------------ the cases


def _embedding(name, direction, dtype, atoms, species, channels):
    return {"name": name, "operator": "embedding", "direction": direction, "dtype": dtype,
            "atoms": atoms, "species": species, "channels": channels}


def _structure(name, direction, dtype, structures, shortest, longest, heads, kv_heads, dim, cap,
               queries=0):
    """queries: that many query atoms for each structure, 0 for all of its own atoms."""
    return {"name": name, "operator": "structure", "direction": direction, "dtype": dtype,
            "structures": structures, "shortest": shortest, "longest": longest, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "cap": cap, "queries": queries}


def _neighbor(name, direction, dtype, structures, shortest, longest, neighbors, heads, kv_heads,
              dim, cap):
    """neighbors: mean pairs of an atom within CUTOFF, which sets the density."""
    return {"name": name, "operator": "neighbor", "direction": direction, "dtype": dtype,
            "structures": structures, "shortest": shortest, "longest": longest,
            "neighbors": neighbors, "heads": heads, "kv_heads": kv_heads, "dim": dim, "cap": cap}


def listed():
    return [
        # one small box of a running simulation: latency counts
        _embedding("embed_box", "forward", "float32", 512, 119, 64),
        # the species of a training batch of molecules
        _embedding("embed_batch", "training", "bfloat16", 71_681, 119, 256),
        # a large training batch, packed from many structures
        _embedding("embed_packed", "training", "float32", 1_048_576, 95, 128),
        # inference over a batch of molecules
        _structure("molecules", "forward", "bfloat16", 1024, 20, 120, 8, 8, 32, 0.0),
        # a training step over a smaller batch, scores capped
        _structure("molecules_step", "training", "float16", 256, 20, 120, 8, 8, 32, 30.0),
        # one large cluster, shared key and value heads, capped
        _structure("cluster_step", "training", "bfloat16", 1, 4001, 4001, 8, 2, 64, 30.0),
        # ragged clusters in single precision, a head width that fills no tile
        _structure("ragged_step", "training", "float32", 48, 1, 509, 4, 4, 48, 0.0),
        # one moved or inserted atom in each of 64 slabs asks all of its slab's atoms
        _structure("one_atom", "forward", "bfloat16", 64, 2000, 20_000, 8, 2, 64, 0.0, 1),
        # one small box of a running simulation: latency counts
        _neighbor("list_box", "forward", "float32", 1, 512, 512, 33, 4, 4, 16, 0.0),
        # a training step over a batch of crystals, capped
        _neighbor("list_crystals_step", "training", "float32", 256, 2, 64, 150, 8, 8, 16, 30.0),
        # inference over the 100,000-atom box
        _neighbor("list_large", "forward", "bfloat16", 1, 100_000, 100_000, 90, 8, 8, 16, 0.0),
        # a training step over a large box, shared key and value heads
        _neighbor("list_step", "training", "bfloat16", 1, 32_768, 32_768, 90, 8, 2, 32, 0.0),
    ]


def _spread(rng, low, high):
    """A whole number whose logarithm is uniform over [low, high]."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    operator = rng.choice(["embedding", "structure", "structure", "neighbor", "neighbor"])
    direction = rng.choice(["forward", "training"])
    dtype = rng.choice(sorted(DTYPES))
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    cap = rng.choice([0.0, 20.0, 30.0])
    largest = [work(c) for c in listed() if c["operator"] == operator]
    most = {k: max(w[k] for w in largest) for k in ("bytes", "flops")}
    while True:
        if operator == "embedding":
            case = _embedding("", direction, dtype, _spread(rng, 512, 1_048_576),
                              _spread(rng, 4, 2000), 4 * _spread(rng, 8, 96))
        elif operator == "structure":
            dim = 8 * rng.randint(2, 12)
            longest = _spread(rng, 20, 20_000)
            case = _structure("", direction, dtype, _spread(rng, 1, 1024),
                              max(1, int(longest * rng.random())), longest, heads, kv_heads, dim,
                              cap, rng.choice([0, 0, 1, 3]))
        else:
            dim = 8 * rng.randint(1, 8)
            longest = _spread(rng, 8, 100_000)
            structures = _spread(rng, 1, 256) if longest <= 512 else 1
            shortest = max(1, int(longest * rng.random())) if structures > 1 else longest
            case = _neighbor("", direction, dtype, structures, shortest, longest,
                             _spread(rng, 10, 150), heads, kv_heads, dim, cap)
        del case["name"]
        w = work(case)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"]:
            return case


def _lengths(case):
    """Atoms of each structure: from the shortest to the longest, in a scattered order."""
    B, low, high = case["structures"], case["shortest"], case["longest"]
    golden = 0.5 * (math.sqrt(5.0) - 1.0)
    spread = [low + int((high - low + 1) * ((b * golden + 0.5) % 1.0)) for b in range(B)]
    return [min(high, n) for n in spread]


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    training = case["direction"] == "training"
    if case["operator"] == "embedding":
        rows, table = case["atoms"] * case["channels"], case["species"] * case["channels"]
        b = 8 * case["atoms"] + size * (rows + table)
        if training:
            b += 8 * case["atoms"] + size * (rows + table)
        return {"bytes": b, "flops": rows * (2 if training else 1)}
    lengths = _lengths(case)
    atoms = sum(lengths)
    wide, narrow = case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
    if case["operator"] == "structure":
        queries = case["structures"] * case["queries"] if case["queries"] else atoms
        pairs = sum(n * (case["queries"] or n) for n in lengths)
        geometry = 12 * (atoms + (queries if case["queries"] else 0)) + 8 * len(lengths)
    else:
        queries, pairs = atoms, atoms * case["neighbors"]
        geometry = 20 * pairs  # i, j and d
    tensors = size * (2 * queries * wide + 2 * atoms * narrow)  # q, output, k, v
    b = tensors + geometry
    if training:  # all of it again and the output's gradient in; three gradients and the geometry's out
        b += size * 3 * queries * wide + size * 4 * atoms * narrow + geometry
        b += 4 * pairs if case["operator"] == "neighbor" else 12 * atoms
    return {"bytes": b, "flops": (14 if training else 4) * pairs * wide}


# ----------------------------------------------------------------- the inputs


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _pointer(lengths):
    total, ptr = 0, [0]
    for n in lengths:
        total += n
        ptr.append(total)
    return torch.tensor(ptr, dtype=torch.int64, device=DEVICE)


def _nearest(i, j, d, count):
    """The `count` nearest of the pairs, in their order: a list whose length the case fixes."""
    keep = torch.sort(torch.argsort(d, stable=True)[:count]).values
    return i[keep], j[keep], d[keep]


def _box_list(n, edge, reach, g):
    """Pairs within `reach`, at most half the edge, of one periodic cubic box, sorted by source."""
    x = torch.rand(n, 3, generator=g, device=DEVICE) * edge
    rows = max(1, 1 << 27 >> (n - 1).bit_length())
    parts = []
    for low in range(0, n, rows):
        r2 = None
        for c in range(3):
            t = x[low:low + rows, c, None] - x[None, :, c]
            t -= edge * torch.round(t / edge)
            r2 = t * t if r2 is None else r2.addcmul_(t, t)
        pair = torch.nonzero(r2 < reach * reach)
        pair = pair[pair[:, 0] + low != pair[:, 1]]
        d = torch.sqrt(r2[pair[:, 0], pair[:, 1]])
        parts.append((pair[:, 0] + low, pair[:, 1], d))
    return tuple(torch.cat([p[k] for p in parts]) for k in range(3))


def _crystal_lists(lengths, neighbors, reach, g):
    """Pairs of a batch of cubic crystals with all their images within `reach`, sorted by source."""
    sphere = 4.0 / 3.0 * math.pi * CUTOFF**3
    parts, first = [], 0
    for n in lengths:
        edge = (n * sphere / neighbors) ** (1.0 / 3.0)
        x = torch.rand(n, 3, generator=g, device=DEVICE) * edge
        images = math.ceil(reach / edge)
        span = torch.arange(-images, images + 1, dtype=torch.float32, device=DEVICE)
        image = torch.cartesian_prod(span, span, span) * edge
        t = (x[None, :, None, :] - x[:, None, None, :]) + image
        r2 = (t * t).sum(-1)
        pair = torch.nonzero((r2 < reach * reach) & (r2 > 0))
        parts.append((pair[:, 0] + first, pair[:, 1] + first,
                      torch.sqrt(r2[pair[:, 0], pair[:, 1], pair[:, 2]])))
        first += n
    return tuple(torch.cat([p[k] for p in parts]) for k in range(3))


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    training = case["direction"] == "training"
    s = {"operator": case["operator"], "training": training}
    if case["operator"] == "embedding":
        # a few species make most of the atoms, as carbon and hydrogen do
        u = torch.rand(case["atoms"], generator=g, device=DEVICE)
        s["species"] = (u**3 * case["species"]).long().clamp_(max=case["species"] - 1)
        s["weight"] = torch.randn(case["species"], case["channels"], generator=g,
                                  device=DEVICE).to(dtype)
        s["scale"] = math.sqrt(case["channels"])
        shape = (case["atoms"], case["channels"])
        s["leaves"] = ["weight"]
    else:
        lengths = _lengths(case)
        atoms, H, K, D = sum(lengths), case["heads"], case["kv_heads"], case["dim"]
        queries = case.get("queries", 0)
        n_q = queries * len(lengths) if queries else atoms
        for name, shape in (("q", (n_q, H, D)), ("k", (atoms, K, D)), ("v", (atoms, K, D))):
            s[name] = torch.randn(*shape, generator=g, device=DEVICE).to(dtype)
        s["slopes"] = torch.rand(H, generator=g, device=DEVICE) * 0.5 + 0.05
        s["cap"] = case["cap"] or None
        s["scale"] = 1.0 / math.sqrt(D)
        shape = (n_q, H, D)
        if case["operator"] == "structure":
            ptr = s["batch_ptr"] = _pointer(lengths)
            s["lengths"], s["longest"] = torch.diff(ptr), max(lengths)
            # about the density of a molecule or a solid, 0.1 atoms in each cubic Angstrom
            edge = torch.repeat_interleave((s["lengths"].float() * 10.0) ** (1.0 / 3.0), s["lengths"])
            s["positions"] = torch.rand(atoms, 3, generator=g, device=DEVICE) * edge[:, None]
            s["query_ptr"] = s["query_positions"] = None
            s["query_lengths"], s["query_longest"] = s["lengths"], s["longest"]
            if queries:
                counts = [queries] * len(lengths)
                s["query_ptr"] = _pointer(counts)
                s["query_lengths"], s["query_longest"] = torch.diff(s["query_ptr"]), queries
                side = torch.repeat_interleave((s["lengths"].float() * 10.0) ** (1.0 / 3.0),
                                               s["query_lengths"])
                s["query_positions"] = torch.rand(n_q, 3, generator=g, device=DEVICE) * side[:, None]
            s["leaves"] = ["q", "k", "v", "positions", "slopes"]
            if queries:
                s["leaves"].append("query_positions")
        else:
            sphere = 4.0 / 3.0 * math.pi * CUTOFF**3
            edge = (lengths[0] * sphere / case["neighbors"]) ** (1.0 / 3.0)
            # searched a little further, the nearest kept
            if len(lengths) == 1 and edge >= 2.3 * CUTOFF:
                found = _box_list(atoms, edge, 1.15 * CUTOFF, g)
            else:
                found = _crystal_lists(lengths, case["neighbors"], 1.5 * CUTOFF, g)
            s["i"], s["j"], s["d"] = _nearest(*found, atoms * case["neighbors"])
            s["leaves"] = ["q", "k", "v", "d", "slopes"]
    if training:
        s["grad"] = torch.randn(*shape, generator=g, device=DEVICE).to(dtype)
        for name in s["leaves"]:
            s[name].requires_grad_()
    return s


# ------------------------------------------------------------- the plain form


def _scores(x, cap, bias):
    return (x if cap is None else cap * torch.tanh(x / cap)) - bias


def _plain_embedding(s):
    return (s["weight"].float().index_select(0, s["species"]) * s["scale"]).to(s["weight"].dtype)


def _places(ptr, lengths, longest):
    """Each atom's row where structures take `longest` rows each, and which (structures, longest) are atoms."""
    here = torch.arange(longest, device=ptr.device) < lengths[:, None]
    return torch.nonzero(here.view(-1)).squeeze(1), here


def _padded(t, places, structures, longest):
    flat = torch.zeros(structures * longest, *t.shape[1:], device=t.device)
    return flat.index_copy(0, places, t).view(structures, longest, *t.shape[1:])


def _plain_structure(s):
    H, D, K = s["q"].shape[1], s["q"].shape[2], s["k"].shape[1]
    B, n_k, n_q = s["batch_ptr"].shape[0] - 1, s["longest"], s["query_longest"]
    at_k, is_k = _places(s["batch_ptr"], s["lengths"], n_k)
    k, v, x_k = (_padded(s[n].float(), at_k, B, n_k) for n in ("k", "v", "positions"))
    at_q, x_q = at_k, x_k
    if s["query_ptr"] is not None:
        at_q, _ = _places(s["query_ptr"], s["query_lengths"], n_q)
        x_q = _padded(s["query_positions"], at_q, B, n_q)
    # (B, K, H / K * n_q, D) queries against (B, K, n_k, D) keys and values
    q = _padded(s["q"].float(), at_q, B, n_q).view(B, n_q, K, H // K, D).permute(0, 2, 3, 1, 4)
    x = torch.matmul(q.reshape(B, K, -1, D), k.permute(0, 2, 3, 1).contiguous()) * s["scale"]
    t = x_q[:, :, None, :] - x_k[:, None, :, :]
    r2 = (t * t).sum(-1)
    apart = r2 > 0
    r = torch.where(apart, torch.sqrt(torch.where(apart, r2, 1.0)), 0.0)
    bias = s["slopes"].view(1, K, H // K, 1, 1) * r[:, None, None]
    score = _scores(x.view(B, K, H // K, n_q, n_k), s["cap"], bias)
    score = score.masked_fill(~is_k[:, None, None, None, :], -math.inf)
    weight = torch.exp(score - score.detach().amax(-1, keepdim=True))
    weight = weight / weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(B, K, -1, n_k), v.permute(0, 2, 1, 3).contiguous())
    out = out.view(B, K, H // K, n_q, D).permute(0, 3, 1, 2, 4).reshape(B * n_q, H, D)
    return out.index_select(0, at_q).to(s["q"].dtype)


def _plain_neighbor(s):
    q, k, v, i, j = s["q"].float(), s["k"].float(), s["v"].float(), s["i"], s["j"]
    N, H, D = q.shape
    K, E = k.shape[1], i.shape[0]
    qi, kj, vj = q.index_select(0, i), k.index_select(0, j), v.index_select(0, j)
    x = (qi.view(E, K, H // K, D) * kj.unsqueeze(2)).sum(-1).view(E, H) * s["scale"]
    score = _scores(x, s["cap"], s["slopes"] * s["d"][:, None])
    top = torch.full((N, H), -math.inf, device=q.device)
    top = top.scatter_reduce(0, i[:, None].expand(E, H), score.detach(), "amax")
    weight = torch.exp(score - top.index_select(0, i))
    total = torch.zeros(N, H, device=q.device).index_add(0, i, weight)
    weight = weight / total.index_select(0, i)
    out = (weight.view(E, K, H // K, 1) * vj.unsqueeze(2)).view(E, H, D)
    return torch.zeros(N, H, D, device=q.device).index_add(0, i, out).to(s["q"].dtype)


# ------------------------------------------------------ this repository's own


def _own_embedding(s):
    from tonari_amd.embedding import species_embedding

    return species_embedding(s["species"], s["weight"], scale=s["scale"])


def _own_structure(s):
    from tonari_amd.attention import structure_attention

    return structure_attention(s["q"], s["k"], s["v"], s["positions"], s["batch_ptr"], s["slopes"],
                               softcap=s["cap"], scale=s["scale"],
                               query_positions=s["query_positions"], query_ptr=s["query_ptr"])


def _own_neighbor(s):
    from tonari_amd.attention import neighbor_attention, neighbor_rows

    # the list is new in every step: its rows are laid out within the pass
    rows = neighbor_rows(s["i"], s["j"], s["q"].shape[0], s["k"].shape[0], transpose=s["training"])
    return neighbor_attention(s["q"], s["k"], s["v"], s["d"], rows, s["slopes"], softcap=s["cap"],
                              scale=s["scale"])


PLAIN = {"embedding": _plain_embedding, "structure": _plain_structure, "neighbor": _plain_neighbor}
OWN = {"embedding": _own_embedding, "structure": _own_structure, "neighbor": _own_neighbor}


def run(state):
    out = (OWN if own else PLAIN)[state["operator"]](state)
    if not state["training"]:
        return {"out": out}
    leaves = [state[name] for name in state["leaves"]]
    grads = torch.autograd.grad(out, leaves, state["grad"])
    return {"out": out.detach(), **{"grad_" + n: t for n, t in zip(state["leaves"], grads)}}


# ------------------------------------------------------------ in 64 bits, apart


def _exact_rows(q, k, v, r, slope, cap, scale, grad):
    """One head's queries (n, D) against keys (m, D) at distances r (n, m), by the formulas.

    Returns the output, and with the output's gradient also those of q, k, v, r and the slope.
    """
    x = scale * (q @ k.t())
    t = torch.tanh(x / cap) if cap is not None else None
    s = (cap * t if cap is not None else x) - slope * r
    p = torch.softmax(s, dim=1)
    out = p @ v
    if grad is None:
        return (out,)
    dp = grad @ v.t()
    ds = p * (dp - (grad * out).sum(1, keepdim=True))
    dx = scale * (ds * (1.0 - t * t) if cap is not None else ds)
    return out, dx @ k, dx.t() @ q, p.t() @ grad, -slope * ds, -(ds * r).sum()


def _exact_embedding(case, s):
    w, at = s["weight"].detach().double(), s["species"]
    found = {"out": s["scale"] * w.index_select(0, at)}
    if s["training"]:
        hot = torch.zeros_like(w)
        for low in range(0, at.shape[0], 1 << 17):
            hot.index_add_(0, at[low:low + (1 << 17)], s["grad"][low:low + (1 << 17)].double())
        found["grad_weight"] = s["scale"] * hot
    return found


def _exact_structure(case, s):
    q, k, v, x = (s[n].detach().double() for n in ("q", "k", "v", "positions"))
    H, K = q.shape[1], k.shape[1]
    apart = s["query_ptr"] is not None
    y = s["query_positions"].detach().double() if apart else x
    ptr = s["batch_ptr"].tolist()
    ptr_q = s["query_ptr"].tolist() if apart else ptr
    slopes = s["slopes"].detach().double()
    found = {"out": torch.zeros_like(q)}
    if s["training"]:
        g = s["grad"].double()
        for name in s["leaves"]:
            found["grad_" + name] = torch.zeros_like(s[name], dtype=torch.float64)
        of_y = found["grad_query_positions" if apart else "grad_positions"]
    for b in range(len(ptr) - 1):
        of_k, of_q = slice(ptr[b], ptr[b + 1]), slice(ptr_q[b], ptr_q[b + 1])
        t = y[of_q, None, :] - x[None, of_k, :]
        r = torch.linalg.vector_norm(t, dim=2)
        unit = t / torch.where(r > 0, r, 1.0)[:, :, None]
        for h in range(H):
            c = h * K // H
            got = _exact_rows(q[of_q, h], k[of_k, c], v[of_k, c], r, slopes[h], s["cap"], s["scale"],
                              g[of_q, h] if s["training"] else None)
            found["out"][of_q, h] = got[0]
            if s["training"]:
                found["grad_q"][of_q, h] = got[1]
                found["grad_k"][of_k, c] += got[2]
                found["grad_v"][of_k, c] += got[3]
                push = got[4][:, :, None] * unit
                of_y[of_q] += push.sum(1)
                found["grad_positions"][of_k] -= push.sum(0)
                found["grad_slopes"][h] += got[5]
    return found


def _exact_neighbor(case, s):
    q, k, v, d = (s[n].detach().double() for n in ("q", "k", "v", "d"))
    i, j, slopes, cap = s["i"], s["j"], s["slopes"].detach().double(), s["cap"]
    N, H, D = q.shape
    K = k.shape[1]
    found = {"out": torch.zeros_like(q)}
    if s["training"]:
        g = s["grad"].double()
        for name in s["leaves"]:
            found["grad_" + name] = torch.zeros_like(s[name], dtype=torch.float64)

    def summed(rows, of, n):
        return torch.zeros(n, *rows.shape[1:], dtype=torch.float64, device=DEVICE).index_add_(
            0, of, rows)

    for h in range(H):  # head by head, so that the pairs' rows stay small
        c = h * K // H
        kj, vj, qi = k[j, c], v[j, c], q[i, h]
        x = s["scale"] * (qi * kj).sum(1)
        t = torch.tanh(x / cap) if cap is not None else None
        e = torch.exp((cap * t if cap is not None else x) - slopes[h] * d)  # scores are far from overflow
        p = e / summed(e, i, N)[i]
        out = found["out"][:, h] = summed(p[:, None] * vj, i, N)
        if s["training"]:
            gi = g[i, h]
            ds = p * ((gi * vj).sum(1) - (g[:, h] * out).sum(1)[i])
            dx = s["scale"] * (ds * (1.0 - t * t) if cap is not None else ds)
            found["grad_q"][:, h] = summed(dx[:, None] * kj, i, N)
            found["grad_k"][:, c] += summed(dx[:, None] * qi, j, k.shape[0])
            found["grad_v"][:, c] += summed(p[:, None] * gi, j, k.shape[0])
            found["grad_d"] -= slopes[h] * ds
            found["grad_slopes"][h] = -(ds * d).sum()
    return found


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"embedding": _exact_embedding, "structure": _exact_structure,
                "neighbor": _exact_neighbor}[case["operator"]](case, s)
