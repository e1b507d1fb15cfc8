// The operators of include/tonari_operators.h for torch tensors: allocation of
// outputs and workspaces, the calls on torch's current stream, and autograd.
// Arguments come checked from tonari_amd/embedding.py and attention.py.
//
// A gradient's own graph (create_graph, for training on forces) comes, for the
// attentions, from the operator's expression in torch operations, as for the
// list's d and D; the embedding's is the embedding again.

#include "../../../include/tonari_operators.h"

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <algorithm>
#include <limits>
#include <optional>
#include <vector>

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr size_t kErrLen = 256;

void* stream_of(const Tensor& t) {
    return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

int32_t code_of(const Tensor& t) {
    return t.scalar_type() == at::kFloat      ? TNR_FLOAT32
           : t.scalar_type() == at::kBFloat16 ? TNR_BFLOAT16
                                              : TNR_FLOAT16;
}

void require(int code, const char* err) {
    TORCH_CHECK_VALUE(code != TNR_INPUT_ERROR, err);
    TORCH_CHECK(code == TNR_OK, err);
}

Tensor bytes_on(const Tensor& like, size_t n) {
    return at::empty({(int64_t)n}, like.options().dtype(at::kByte).requires_grad(false));
}

// (atoms, heads, dim) as the kernels read it: contiguous channels, and
// addresses and strides in multiples of 16 bytes; a copy where it is not.
Tensor laid(const Tensor& x) {
    const Tensor t = x.detach();
    const int64_t unit = 16 / t.element_size();
    if (t.numel() == 0) return t.contiguous();
    const auto fits = [&](int64_t s) { return s % unit == 0 && s <= (int64_t(1) << 24); };
    if (t.stride(2) == 1 && fits(t.stride(0)) && fits(t.stride(1)) &&
        (uintptr_t)t.data_ptr() % 16 == 0)
        return t;
    return t.clone(at::MemoryFormat::Contiguous);
}
// Contiguous, at a multiple of 16 bytes.
Tensor flat(const Tensor& x) {
    const Tensor t = x.detach().contiguous();
    return t.numel() == 0 || (uintptr_t)t.data_ptr() % 16 == 0
               ? t
               : t.clone(at::MemoryFormat::Contiguous);
}

// What these calls would lose without a word: tangents of forward-mode
// derivatives, and themselves in a trace (which would record outputs that nothing fills).
void refuse_untracked(std::initializer_list<Tensor> inputs) {
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing(),
                                "the operators cannot be traced (torch.jit.trace)");
    for (const Tensor& t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(),
                                    "the operators have no forward-mode derivatives");
}

bool wants(std::initializer_list<Tensor> inputs) {
    refuse_untracked(inputs);
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor& t : inputs)
        if (t.defined() && t.requires_grad()) return true;
    return false;
}

void set_strides(int64_t (&to)[2], const Tensor& t) {
    to[0] = t.stride(0);
    to[1] = t.stride(1);
}

// --------------------------------------------------------------- embedding

tnr_embedding embedding_request(const Tensor& species, const Tensor& like, int64_t n_species,
                                double scale) {
    tnr_embedding r{};
    r.dtype = code_of(like);
    r.index_bytes = (int32_t)species.element_size();
    r.n_atoms = species.numel();
    r.n_species = n_species;
    r.channels = like.size(-1);
    r.species = species.data_ptr();
    r.scale = (float)scale;
    return r;
}

Tensor embedding_forward(const Tensor& species, const Tensor& weight, double scale) {
    c10::DeviceGuard guard(weight.device());
    const Tensor z = species.contiguous(), w = flat(weight);
    std::vector<int64_t> shape = species.sizes().vec();
    shape.push_back(weight.size(1));
    const Tensor out = at::empty(shape, w.options());
    tnr_embedding r = embedding_request(z, w, w.size(0), scale);
    r.weight = w.data_ptr();
    r.out = out.data_ptr();
    char err[kErrLen] = {0};
    require(tnr_embedding_forward(&r, stream_of(w), err, kErrLen), err);
    return out;
}

Tensor embedding_gradient(const Tensor& grad_out, const Tensor& species, int64_t rows,
                          double scale) {
    c10::DeviceGuard guard(grad_out.device());
    const Tensor z = species.contiguous(), go = flat(grad_out);
    const Tensor grad = at::empty({rows, go.size(-1)}, go.options());
    tnr_embedding r = embedding_request(z, go, rows, scale);
    r.grad_out = go.data_ptr();
    r.grad_weight = grad.data_ptr();
    const Tensor space = bytes_on(go, tnr_embedding_workspace_size(&r));
    char err[kErrLen] = {0};
    require(tnr_embedding_backward(&r, space.data_ptr(), (size_t)space.numel(), stream_of(go), err,
                                   kErrLen),
            err);
    return grad;
}

Tensor species_embedding(const Tensor& species, const Tensor& weight, double scale);

// The table's gradient as a function of the output's: linear, and its own gradient
// is the embedding of the table's (0 for a species outside it).
struct EmbeddingGradient : torch::autograd::Function<EmbeddingGradient> {
    static Tensor forward(AutogradContext* ctx, const Tensor& grad_out, const Tensor& species,
                          int64_t rows, double scale) {
        ctx->save_for_backward({species});
        ctx->saved_data["scale"] = scale;
        return embedding_gradient(grad_out, species, rows, scale);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        variable_list all(4);
        const Tensor &g = grads[0], species = ctx->get_saved_variables()[0];
        if (!g.defined()) return all;
        const Tensor out = species_embedding(species, g, ctx->saved_data["scale"].toDouble());
        const Tensor in = species.ge(0).logical_and(species.lt(g.size(0))).unsqueeze(-1);
        all[0] = at::where(in, out, at::zeros({}, out.options()));
        return all;
    }
};

struct Embedding : torch::autograd::Function<Embedding> {
    static Tensor forward(AutogradContext* ctx, const Tensor& weight, const Tensor& species,
                          double scale) {
        ctx->save_for_backward({species});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["rows"] = weight.size(0);
        return embedding_forward(species, weight, scale);
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const Tensor species = ctx->get_saved_variables()[0];
        const double scale = ctx->saved_data["scale"].toDouble();
        const int64_t rows = ctx->saved_data["rows"].toInt();
        const Tensor& g = grads[0];
        if (!g.defined()) return {Tensor(), Tensor(), Tensor()};
        // (wants refuses a tangent of g)
        return {wants({g}) ? EmbeddingGradient::apply(g, species, rows, scale)
                           : embedding_gradient(g, species, rows, scale),
                Tensor(), Tensor()};
    }
};

Tensor species_embedding(const Tensor& species, const Tensor& weight, double scale) {
    return wants({weight}) ? Embedding::apply(weight, species, scale)
                           : embedding_forward(species, weight, scale);
}

// ------------------------------------------------- attention, as an expression

// Attention over pairs (source, target) at distances r, in 32-bit torch
// operations: what a graph of the gradient is built from.  It holds the rows of q, k and
// v of every pair and head.
Tensor pair_expression(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& r,
                      const Tensor& slopes, const Tensor& source, const Tensor& target,
                      double scale, double softcap) {
    const int64_t n = q.size(0), heads = q.size(1), dim = q.size(2), group = heads / k.size(1);
    const auto wide = [&](const Tensor& t) {
        return t.to(at::kFloat).index_select(0, target).repeat_interleave(group, 1);
    };
    const Tensor qs = q.to(at::kFloat).index_select(0, source);
    Tensor x = (qs * wide(k)).sum(-1) * scale;
    if (softcap > 0.0) x = at::tanh(x / softcap) * softcap;
    const Tensor score = x - slopes * r.unsqueeze(1);
    const Tensor at = source.unsqueeze(1).expand({source.numel(), heads});
    Tensor top = at::full({n, heads}, -std::numeric_limits<double>::infinity(), score.options());
    top = top.scatter_reduce(0, at, score.detach(), "amax");
    top = at::where(top.isinf(), at::zeros_like(top), top);
    const Tensor e = at::exp(score - top.index_select(0, source));
    const Tensor sum = at::zeros({n, heads}, e.options()).index_add(0, source, e);
    // (a row that no key weighs in on is 0)
    const Tensor p = e / at::where(sum.eq(0), at::ones_like(sum), sum).index_select(0, source);
    return at::zeros({n, heads, dim}, e.options())
        .index_add(0, source, p.unsqueeze(-1) * wide(v))
        .to(q.scalar_type());
}

Tensor pair_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& r,
                      const Tensor& slopes, const Tensor& source, const Tensor& target,
                      double scale, double softcap) {
    try {
        return pair_expression(q, k, v, r, slopes, source, target, scale, softcap);
    } catch (const c10::OutOfMemoryError& e) {
        const double gib = 4.0 * (double)source.numel() * q.size(1) * q.size(2) / (1 << 30);
        TORCH_CHECK_WITH(OutOfMemoryError, false,
                         "create_graph holds several tensors of pairs x heads x dim floats (",
                         source.numel(), " x ", q.size(1), " x ", q.size(2), ": ", gib,
                         " GiB each); take the gradient of fewer structures at a time.  ",
                         e.what_without_backtrace());
    }
}

// 1 or, where `ok` (a truth value on the device) does not hold, NaN: inputs are
// multiplied by it, so that all that follows from them is NaN, as in the kernels.
Tensor nan_unless(const Tensor& ok) {
    return at::where(ok, at::ones({}, ok.options().dtype(at::kFloat)),
                     at::full({}, std::numeric_limits<double>::quiet_NaN(),
                              ok.options().dtype(at::kFloat)));
}
variable_list times(const variable_list& nodes, const Tensor& factor) {
    variable_list all;
    for (const Tensor& t : nodes) all.push_back(t.defined() ? t * factor : t);
    return all;
}

// Whether pointers rise from 0 to n.
Tensor rising(const Tensor& ptr, int64_t n) {
    return (ptr.slice(0, 1) - ptr.slice(0, 0, -1))
        .ge(0)
        .all()
        .logical_and(ptr.select(0, 0).eq(0))
        .logical_and(ptr.select(0, -1).eq(n));
}

// Whether the rows are of a valid list of these sizes (their head says both).
Tensor rows_hold(const Tensor& rows, int64_t pairs, int64_t sources, int64_t targets) {
    const Tensor head = rows.slice(0, 0, 16).view(at::kInt);
    return head.select(0, 0)
        .eq(0)
        .logical_and(head.select(0, 1).eq(pairs))
        .logical_and(head.select(0, 2).eq(sources))
        .logical_and(head.select(0, 3).eq(targets));
}

// The inputs as nodes of their own: the gradient for one of them then takes no
// path through another (q may well depend on the positions).
variable_list own_nodes(const variable_list& saved, size_t n) {
    variable_list nodes;
    for (size_t i = 0; i < n; ++i)
        nodes.push_back(saved[i].defined() ? saved[i].view_as(saved[i]) : Tensor());
    return nodes;
}

// The gradients, with a graph, of `out` for the inputs that need one.
variable_list graph_of(const Tensor& out, const Tensor& upstream, const variable_list& inputs,
                       const std::vector<bool>& needed) {
    variable_list wrt;
    for (size_t i = 0; i < inputs.size(); ++i)
        if (needed[i]) wrt.push_back(inputs[i]);
    const variable_list found = torch::autograd::grad(
        {out}, wrt, {upstream}, std::nullopt, /*create_graph=*/true, /*allow_unused=*/true);
    variable_list all(inputs.size());
    for (size_t i = 0, k = 0; i < inputs.size(); ++i)
        if (needed[i]) all[i] = found[k++];
    return all;
}

// ------------------------------------------------------ structure attention

struct StructureCall {
    Tensor q, k, v, query_positions, positions, slopes, query_ptr, key_ptr, tiles;
    tnr_structure_attention r{};

    StructureCall(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& x,
                  const Tensor& slopes_, const Tensor& x_q, const Tensor& batch_ptr,
                  const Tensor& query_ptr_, double scale, double softcap,
                  const Tensor& tiles_ = Tensor())
        : q(laid(q_)), k(laid(k_)), v(laid(v_)), positions(x.detach().contiguous()),
          slopes(slopes_.detach().contiguous()), key_ptr(batch_ptr.contiguous()) {
        if (x_q.defined()) query_positions = x_q.detach().contiguous();
        query_ptr = query_ptr_.defined() ? query_ptr_.contiguous() : key_ptr;
        r.dtype = code_of(q);
        r.heads = (int32_t)q.size(1);
        r.kv_heads = (int32_t)k.size(1);
        r.dim = (int32_t)q.size(2);
        r.n_structures = key_ptr.numel() - 1;
        r.n_queries = q.size(0);
        r.n_keys = k.size(0);
        r.query_ptr = (const int64_t*)query_ptr.data_ptr();
        r.key_ptr = (const int64_t*)key_ptr.data_ptr();
        r.q = q.data_ptr();
        r.k = k.data_ptr();
        r.v = v.data_ptr();
        set_strides(r.q_stride, q);
        set_strides(r.k_stride, k);
        set_strides(r.v_stride, v);
        if (x_q.defined()) r.query_positions = (const float*)query_positions.data_ptr();
        r.positions = (const float*)positions.data_ptr();
        r.slopes = (const float*)slopes.data_ptr();
        r.scale = (float)scale;
        r.softcap = (float)softcap;
        tiles = tiles_.defined() ? tiles_ : bytes_on(q, tnr_structure_tiles_size(&r));
        r.tiles = tiles.data_ptr();
    }
};

// `lse` and `full`: what the backward reads, NULL where there is none.
Tensor structure_forward(StructureCall& c, Tensor* lse, Tensor* full) {
    const Tensor out = at::empty(c.q.sizes(), c.q.options());
    c.r.out = out.data_ptr();
    if (full && c.r.dtype != TNR_FLOAT32) {
        *full = at::empty(c.q.sizes(), c.slopes.options());
        c.r.out32 = (float*)full->data_ptr();
    }
    if (lse) {
        *lse = at::empty({c.q.size(1), c.q.size(0)}, c.slopes.options());
        c.r.lse = (float*)lse->data_ptr();
    }
    const Tensor space = bytes_on(c.q, tnr_structure_forward_workspace_size(&c.r));
    char err[kErrLen] = {0};
    require(tnr_structure_forward(&c.r, space.data_ptr(), (size_t)space.numel(), stream_of(c.q), err,
                                  kErrLen),
            err);
    return out;
}

struct StructureAttention : torch::autograd::Function<StructureAttention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                          const Tensor& x, const Tensor& slopes,
                          const std::optional<Tensor>& query_positions, const Tensor& batch_ptr,
                          const std::optional<Tensor>& query_ptr_, double scale, double softcap) {
        const Tensor x_q = query_positions.value_or(Tensor());
        const Tensor query_ptr = query_ptr_.value_or(Tensor());
        StructureCall c(q, k, v, x, slopes, x_q, batch_ptr, query_ptr, scale, softcap);
        Tensor lse, full;
        const Tensor out = structure_forward(c, &lse, &full);
        ctx->save_for_backward(
            {q, k, v, x, slopes, x_q, batch_ptr, query_ptr, out, lse, c.tiles, full});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["softcap"] = softcap;
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const double scale = ctx->saved_data["scale"].toDouble();
        const double softcap = ctx->saved_data["softcap"].toDouble();
        variable_list all(10);
        if (!grads[0].defined()) return all;
        refuse_untracked({grads[0]});
        c10::DeviceGuard guard(s[0].device());
        std::vector<bool> needed;
        for (size_t i = 0; i < 6; ++i) needed.push_back(s[i].defined() && ctx->needs_input_grad(i));
        if (at::GradMode::is_enabled()) {
            const variable_list nodes = own_nodes(s, 6);
            const Tensor &kp = s[6], &qp = s[7].defined() ? s[7] : s[6];
            const Tensor ok = rising(kp, s[1].size(0)).logical_and(rising(qp, s[0].size(0)));
            const variable_list n = times(nodes, nan_unless(ok));
            const Tensor &x = n[3], &x_q = n[5];
            // (pointers that are wrong make no pairs, so that nothing goes by them)
            const Tensor nq = (qp.slice(0, 1) - qp.slice(0, 0, -1)) * ok;
            const Tensor nk = (kp.slice(0, 1) - kp.slice(0, 0, -1)) * ok;
            const Tensor pairs = nq * nk;
            const Tensor b = at::repeat_interleave(pairs);
            const Tensor place = at::arange(b.numel(), b.options()) -
                                 (pairs.cumsum(0) - pairs).index_select(0, b);
            const Tensor width = nk.index_select(0, b);
            const Tensor source = qp.index_select(0, b) + place.div(width, "floor");
            const Tensor target = kp.index_select(0, b) + place.remainder(width);
            const Tensor t = (x_q.defined() ? x_q : x).index_select(0, source) -
                             x.index_select(0, target);
            const Tensor r2 = (t * t).sum(-1), one = at::ones({}, r2.options());
            const Tensor apart = r2.gt(0);
            const Tensor r = at::where(apart, at::where(apart, r2, one).sqrt(), one * 0);
            const Tensor out =
                pair_attention(n[0], n[1], n[2], r, n[4], source, target, scale, softcap);
            const variable_list found = graph_of(out, grads[0], nodes, needed);
            for (size_t i = 0; i < 6; ++i) all[i] = found[i];
            return all;
        }
        StructureCall c(s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], scale, softcap, s[10]);
        const Tensor &out = s[8], &lse = s[9], &full = s[11];
        const Tensor go = flat(grads[0]);
        c.r.out = out.data_ptr();
        c.r.out32 = full.defined() ? (float*)full.data_ptr() : nullptr;
        c.r.lse = (float*)lse.data_ptr();
        c.r.grad_out = go.data_ptr();
        all[0] = at::empty(c.q.sizes(), c.q.options());
        all[1] = at::empty(c.k.sizes(), c.k.options());
        all[2] = at::empty(c.v.sizes(), c.v.options());
        c.r.grad_q = all[0].data_ptr();
        c.r.grad_k = all[1].data_ptr();
        c.r.grad_v = all[2].data_ptr();
        if (needed[3]) {
            all[3] = at::empty(c.positions.sizes(), c.positions.options());
            c.r.grad_positions = (float*)all[3].data_ptr();
        }
        if (needed[4]) {
            all[4] = at::empty(c.slopes.sizes(), c.slopes.options());
            c.r.grad_slopes = (float*)all[4].data_ptr();
        }
        if (needed[5]) {
            all[5] = at::empty(c.query_positions.sizes(), c.query_positions.options());
            c.r.grad_query_positions = (float*)all[5].data_ptr();
        }
        const Tensor space = bytes_on(go, tnr_structure_backward_workspace_size(&c.r));
        char err[kErrLen] = {0};
        require(tnr_structure_backward(&c.r, space.data_ptr(), (size_t)space.numel(), stream_of(go),
                                       err, kErrLen),
                err);
        return all;
    }
};

Tensor structure_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& x,
                           const Tensor& batch_ptr, const Tensor& slopes,
                           const std::optional<Tensor>& query_positions,
                           const std::optional<Tensor>& query_ptr, double scale, double softcap) {
    c10::DeviceGuard guard(q.device());  // (for both paths: launches go to the current device)
    const Tensor x_q = query_positions.value_or(Tensor()), q_ptr = query_ptr.value_or(Tensor());
    if (wants({q, k, v, x, slopes, x_q}))
        return StructureAttention::apply(q, k, v, x, slopes, query_positions, batch_ptr, query_ptr,
                                         scale, softcap);
    StructureCall c(q, k, v, x, slopes, x_q, batch_ptr, q_ptr, scale, softcap);
    return structure_forward(c, nullptr, nullptr);
}

// ------------------------------------------------------- neighbor attention

tnr_neighbor_list list_of(int64_t pairs, int64_t sources, int64_t targets, bool transpose) {
    tnr_neighbor_list l{};
    l.n_pairs = pairs;
    l.n_sources = sources;
    l.n_targets = targets;
    l.transpose = transpose;
    return l;
}

Tensor neighbor_rows(const Tensor& i, const Tensor& j, int64_t n_sources, int64_t n_targets,
                     bool transpose) {
    refuse_untracked({});
    c10::DeviceGuard guard(i.device());
    const Tensor sources = i.contiguous(), targets = j.contiguous();
    tnr_neighbor_list l = list_of(i.numel(), n_sources, n_targets, transpose);
    const Tensor rows = bytes_on(sources, tnr_neighbor_rows_size(&l));
    const Tensor space = bytes_on(sources, tnr_neighbor_rows_workspace_size(&l));
    l.sources = (const int64_t*)sources.data_ptr();
    l.targets = (const int64_t*)targets.data_ptr();
    l.rows = rows.data_ptr();
    char err[kErrLen] = {0};
    require(tnr_neighbor_rows(&l, space.data_ptr(), (size_t)space.numel(), stream_of(sources), err,
                              kErrLen),
            err);
    return rows;
}

struct NeighborCall {
    Tensor q, k, v, d, slopes;
    tnr_neighbor_attention r{};

    NeighborCall(const Tensor& q_, const Tensor& k_, const Tensor& v_, const Tensor& d_,
                 const Tensor& slopes_, const Tensor& rows, bool transpose, double scale,
                 double softcap)
        : q(laid(q_)), k(laid(k_)), v(laid(v_)), d(d_.detach().contiguous()),
          slopes(slopes_.detach().contiguous()) {
        r.dtype = code_of(q);
        r.heads = (int32_t)q.size(1);
        r.kv_heads = (int32_t)k.size(1);
        r.dim = (int32_t)q.size(2);
        r.list = list_of(d.numel(), q.size(0), k.size(0), transpose);
        r.list.rows = rows.data_ptr();
        r.q = q.data_ptr();
        r.k = k.data_ptr();
        r.v = v.data_ptr();
        set_strides(r.q_stride, q);
        set_strides(r.k_stride, k);
        set_strides(r.v_stride, v);
        r.distances = (const float*)d.data_ptr();
        r.slopes = (const float*)slopes.data_ptr();
        r.scale = (float)scale;
        r.softcap = (float)softcap;
    }
};

struct NeighborAttention : torch::autograd::Function<NeighborAttention> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                          const Tensor& d, const Tensor& slopes, const Tensor& rows,
                          const Tensor& i, const Tensor& j, bool transpose, double scale,
                          double softcap) {
        NeighborCall c(q, k, v, d, slopes, rows, transpose, scale, softcap);
        const Tensor out = at::empty(c.q.sizes(), c.q.options());
        const Tensor lse = at::empty({c.q.size(0), c.q.size(1)}, c.slopes.options());
        Tensor full;  // unrounded: the gradients of d and of the slopes have 32 bits
        if (c.r.dtype != TNR_FLOAT32) {
            full = at::empty(c.q.sizes(), c.slopes.options());
            c.r.out32 = (float*)full.data_ptr();
        }
        c.r.out = out.data_ptr();
        c.r.lse = (float*)lse.data_ptr();
        char err[kErrLen] = {0};
        require(tnr_neighbor_forward(&c.r, stream_of(c.q), err, kErrLen), err);
        ctx->save_for_backward({q, k, v, d, slopes, rows, i, j, out, lse, full});
        ctx->saved_data["transpose"] = transpose;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["softcap"] = softcap;
        return out;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto s = ctx->get_saved_variables();
        const double scale = ctx->saved_data["scale"].toDouble();
        const double softcap = ctx->saved_data["softcap"].toDouble();
        variable_list all(11);
        if (!grads[0].defined()) return all;
        refuse_untracked({grads[0]});
        c10::DeviceGuard guard(s[0].device());
        if (at::GradMode::is_enabled()) {
            std::vector<bool> needed;
            for (size_t i = 0; i < 5; ++i) needed.push_back(ctx->needs_input_grad(i));
            const variable_list nodes = own_nodes(s, 5);
            const int64_t sources = s[0].size(0), targets = s[1].size(0);
            const variable_list n =
                times(nodes, nan_unless(rows_hold(s[5], s[3].numel(), sources, targets)));
            // (a list may name atoms that do not exist)
            const Tensor out = pair_attention(n[0], n[1], n[2], n[3], n[4],
                                              s[6].clamp(0, std::max<int64_t>(sources - 1, 0)),
                                              s[7].clamp(0, std::max<int64_t>(targets - 1, 0)),
                                              scale, softcap);
            const variable_list found = graph_of(out, grads[0], nodes, needed);
            for (size_t i = 0; i < 5; ++i) all[i] = found[i];
            return all;
        }
        NeighborCall c(s[0], s[1], s[2], s[3], s[4], s[5], ctx->saved_data["transpose"].toBool(),
                       scale, softcap);
        const Tensor &out = s[8], &lse = s[9], &full = s[10];
        const Tensor go = flat(grads[0]);
        c.r.out = out.data_ptr();
        c.r.out32 = full.defined() ? (float*)full.data_ptr() : nullptr;
        c.r.lse = (float*)lse.data_ptr();
        c.r.grad_out = go.data_ptr();
        all[0] = at::empty(c.q.sizes(), c.q.options());
        all[1] = at::empty(c.k.sizes(), c.k.options());
        all[2] = at::empty(c.v.sizes(), c.v.options());
        all[3] = at::empty(c.d.sizes(), c.d.options());
        all[4] = at::empty(c.slopes.sizes(), c.slopes.options());
        c.r.grad_q = all[0].data_ptr();
        c.r.grad_k = all[1].data_ptr();
        c.r.grad_v = all[2].data_ptr();
        c.r.grad_distances = (float*)all[3].data_ptr();
        c.r.grad_slopes = (float*)all[4].data_ptr();
        const Tensor space = bytes_on(go, tnr_neighbor_backward_workspace_size(&c.r));
        char err[kErrLen] = {0};
        require(tnr_neighbor_backward(&c.r, space.data_ptr(), (size_t)space.numel(), stream_of(go),
                                      err, kErrLen),
                err);
        return all;
    }
};

Tensor neighbor_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& d,
                          const Tensor& slopes, const Tensor& rows, const Tensor& i,
                          const Tensor& j, bool transpose, double scale, double softcap) {
    c10::DeviceGuard guard(q.device());
    const tnr_neighbor_list l = list_of(d.numel(), q.size(0), k.size(0), transpose);
    TORCH_CHECK_VALUE(rows.scalar_type() == at::kByte && rows.dim() == 1 && rows.is_contiguous() &&
                          rows.numel() == (int64_t)tnr_neighbor_rows_size(&l),
                      "rows are not those of this list");
    if (wants({q, k, v, d, slopes}))
        return NeighborAttention::apply(q, k, v, d, slopes, rows, i, j, transpose, scale, softcap);
    NeighborCall c(q, k, v, d, slopes, rows, transpose, scale, softcap);
    const Tensor out = at::empty(c.q.sizes(), c.q.options());
    c.r.out = out.data_ptr();
    char err[kErrLen] = {0};
    require(tnr_neighbor_forward(&c.r, stream_of(c.q), err, kErrLen), err);
    return out;
}

// Runs without the GIL (see frontend.cpp).
template <typename R, typename... A>
auto free_of_gil(R (*f)(A...)) {
    return [f](A... a) -> R {
        HANDLE_TH_ERRORS
        pybind11::gil_scoped_release no_gil;
        return f(std::forward<A>(a)...);
        END_HANDLE_TH_ERRORS_PYBIND
    };
}

}  // namespace

void bind_operators(pybind11::module& m) {
    m.attr("operators_version") = TNR_OPERATORS_VERSION;
    m.def("species_embedding", free_of_gil(species_embedding));
    m.def("structure_attention", free_of_gil(structure_attention));
    m.def("neighbor_rows", free_of_gil(neighbor_rows));
    m.def("neighbor_attention", free_of_gil(neighbor_attention));
}
