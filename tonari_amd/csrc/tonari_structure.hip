// C ABI of structure attention (include/tonari_operators.h): checks of requests,
// workspaces and launches.  Every call returns a code; no exception crosses it.
#include "op_host.h"
#include "op_structure_backward.h"

using namespace tnr::op;

namespace {

// ------------------------------------------------------- structure attention

// Waves of 32 rows in a workgroup, which share the staged keys, by the batch's mean
// structure.  Four for long ones; for short ones two, of which fewer lie beyond a
// structure's end: 1,024 molecules of 20 to 120 atoms take 70 us at two and 73 at
// four (a training step over 256 of them 122 and 127), a cluster of 4,001 atoms 222
// us at four and 235 at two by queries, 247 and 254 by keys.
int waves_for(int64_t rows, int64_t structures) {
    const int64_t mean = structures > 0 ? rows / structures : 0;
    return mean <= 512 ? 2 : 4;
}

struct StructurePlan {
    int group, q_waves, k_waves;
    int f_splits, splits, k_splits;  // of the forward, the queries' pass back, the keys'
    int64_t q_tiles, k_tiles;
};

constexpr int64_t kMostAtoms = int64_t(1) << 30;
constexpr int64_t kSimds = 1024;

StructurePlan structure_plan(const tnr_structure_attention& r) {
    StructurePlan p{};
    p.group = r.heads / r.kv_heads;
    p.q_waves = waves_for(r.n_queries * p.group, r.n_structures);
    p.k_waves = waves_for(r.n_keys, r.n_structures);
    p.q_tiles = tile_start(r.n_queries, p.group, p.q_waves * kTile, r.n_structures);
    p.k_tiles = tile_start(r.n_keys, 1, p.k_waves * kTile, r.n_structures);
    // Few rows: the keys (or, for the keys' gradients, the rows) are split over
    // workgroups, at least 8 tiles each of the batch's mean structure, into as many
    // waves as the device holds of the kernel at once (`held` to a SIMD): a cluster of
    // 4,001 atoms split for three waves in all kernels takes 231 + 16 and 263 + 11 us
    // back, queries and keys with their joins, in place of 222 + 13 and 247 + 9.
    const auto split = [&](int64_t rows, int64_t others, int held) {
        const int64_t waves = (rows / kTile + r.n_structures) * r.kv_heads;
        const int64_t most = r.n_structures > 0 ? others / r.n_structures / (8 * kTile) : 0;
        int64_t n = waves > 0 ? kSimds * held / waves : 1;
        if (n > most) n = most;
        if (n > 64) n = 64;
        return n < 2 ? 1 : (int)n;
    };
    const bool wide = r.dtype == TNR_FLOAT32;
    p.f_splits = split(r.n_queries * p.group, r.n_keys, r.dim <= 64 ? 3 : 2);
    p.splits = split(r.n_queries * p.group, r.n_keys, wide && r.dim > 96 ? 1 : 2);
    p.k_splits = split(r.n_keys, r.n_queries * p.group, r.dim > 64 ? 1 : 2);
    return p;
}

int check_structure(const tnr_structure_attention* r, bool backward, char* err, size_t len) {
    if (!r) return refuse(err, len, "request is null");
    const int code = check_heads(r->dtype, r->heads, r->kv_heads, r->dim, r->scale, r->softcap, err,
                                 len);
    if (code != TNR_OK) return code;
    if (r->n_structures < 0 || r->n_queries < 0 || r->n_keys < 0 ||
        (r->n_structures == 0 && (r->n_queries > 0 || r->n_keys > 0)))
        return refuse(err, len, "invalid sizes");
    if (!r->query_positions && r->n_queries > 0 && r->n_queries != r->n_keys)
        return refuse(err, len, "queries of their own need positions of their own");
    if (r->n_queries >= INT32_MAX / r->heads || r->n_keys >= INT32_MAX / r->kv_heads ||
        r->n_queries >= kMostAtoms || r->n_keys >= kMostAtoms || r->n_structures >= kMostAtoms)
        return refuse(err, len, "too many atoms");
    const StructurePlan p = structure_plan(*r);
    // (the last kernel back: a thread for each coordinate, a workgroup for each slope)
    const int64_t coordinates = 3 * (r->n_queries + r->n_keys) + 1024 * (int64_t)(r->heads + 1);
    if ((backward && coordinates > kMostThreads) ||
        p.q_tiles * r->kv_heads * p.q_waves * kWave > kMostThreads ||
        p.k_tiles * r->kv_heads * p.k_waves * kWave > kMostThreads)
        return refuse(err, len, "too many atoms");
    if (r->n_structures > 0 && (!r->query_ptr || !r->key_ptr))
        return refuse(err, len, "required pointers are null");
    if (r->n_structures > 0 && (!r->tiles || (uintptr_t)r->tiles % 256 != 0))
        return refuse(err, len, "tiles must be given and aligned to 256 bytes");
    if (!r->slopes || (r->n_queries > 0 && (!r->q || !r->out)) ||
        (r->n_keys > 0 && (!r->k || !r->v || !r->positions)))
        return refuse(err, len, "required pointers are null");
    if (!aligned(r->q, r->q_stride, r->dtype) || !aligned(r->k, r->k_stride, r->dtype) ||
        !aligned(r->v, r->v_stride, r->dtype) || (uintptr_t)r->out % 16 != 0 ||
        (uintptr_t)r->out32 % 16 != 0)
        return refuse(err, len, "q, k, v and out must be aligned to 16 bytes, with strides up to 2^24");
    if (backward) {
        if ((r->n_queries > 0 && (!r->grad_out || !r->grad_q || !r->lse)) ||
            (r->n_keys > 0 && (!r->grad_k || !r->grad_v)))
            return refuse(err, len, "required pointers are null");
        if ((uintptr_t)r->grad_out % 16 != 0 || (uintptr_t)r->grad_q % 16 != 0 ||
            (uintptr_t)r->grad_k % 16 != 0 || (uintptr_t)r->grad_v % 16 != 0)
            return refuse(err, len, "gradients must be aligned to 16 bytes");
        if (r->grad_query_positions && !r->query_positions)
            return refuse(err, len, "the queries' positions are the keys'");
    }
    return TNR_OK;
}

// The batch's tiles: the queries', and the keys' for the backward.
size_t q_tile_bytes(const StructurePlan& p) {
    return padded((size_t)p.q_tiles * sizeof(StructureTile));
}
size_t k_tile_bytes(const StructurePlan& p) {
    return padded((size_t)p.k_tiles * sizeof(StructureTile));
}

StructureArgs structure_args(const tnr_structure_attention& r, const StructurePlan& p) {
    StructureArgs a{};
    a.q_tiles = (StructureTile*)r.tiles;
    a.k_tiles = (StructureTile*)((char*)r.tiles + q_tile_bytes(p));
    a.q = r.q;
    a.k = r.k;
    a.v = r.v;
    for (int i = 0; i < 2; ++i) {
        a.q_stride[i] = r.q_stride[i];
        a.k_stride[i] = r.k_stride[i];
        a.v_stride[i] = r.v_stride[i];
    }
    a.x_q = r.query_positions ? r.query_positions : r.positions;
    a.x_k = r.positions;
    a.slopes = r.slopes;
    a.rule = ScoreRule::of(r.scale, r.softcap);
    a.heads = r.heads;
    a.kv_heads = r.kv_heads;
    a.group = p.group;
    a.dim = r.dim;
    a.n_queries = (int)r.n_queries;
    a.n_keys = (int)r.n_keys;
    a.splits = p.splits;
    a.k_splits = p.k_splits;
    a.out = r.out;
    a.out32 = r.out32;
    a.lse = r.lse;
    a.grad_out = r.grad_out;
    a.grad_q = r.grad_q;
    a.grad_k = r.grad_k;
    a.grad_v = r.grad_v;
    return a;
}

struct StructureSpace {
    float *part, *part_k, *row, *push_q, *push_k, *turn;
    size_t bytes;
};
StructureSpace structure_space(const tnr_structure_attention& r, const StructurePlan& p,
                               bool backward, void* base) {
    size_t at = 0;
    const auto part = [&](size_t bytes) {
        char* q = (char*)base + at;
        at += padded(bytes);
        return q;
    };
    const size_t rows = (size_t)r.heads * r.n_queries;
    StructureSpace s{};
    const int splits = backward ? p.splits : p.f_splits;
    if (splits > 1)
        s.part = (float*)part(rows * splits * (r.dim + (backward ? kRowSums : 2)) * 4);
    if (backward) {
        if (p.k_splits > 1)
            s.part_k = (float*)part((size_t)r.kv_heads * r.n_keys * p.k_splits *
                                    (2 * r.dim + 3) * 4);
        s.row = (float*)part(rows * 4);
        if (r.grad_positions || r.grad_query_positions) {
            s.push_q = (float*)part(rows * 12);
            s.push_k = (float*)part((size_t)r.kv_heads * r.n_keys * 12);
        }
        if (r.grad_slopes) s.turn = (float*)part(rows * 4);
    }
    s.bytes = at;
    return s;
}

void lay_tiles(const tnr_structure_attention& r, const StructurePlan& p, const StructureArgs& a,
               bool keys, hipStream_t stream) {
    const int64_t blocks = (r.n_structures + 3) / 4;
    k_structure_tiles<<<(unsigned)(blocks < 64 ? blocks : 64), 256, 0, stream>>>(
        r.query_ptr, r.key_ptr, r.n_structures, r.n_queries, r.n_keys, p.group, p.q_waves * kTile,
        p.k_waves * kTile, a.q_tiles, keys ? a.k_tiles : nullptr);
}

template <typename F>
void with_dim(int32_t dim, F&& f) {
    if (dim <= 32)
        f(Int<32>{});
    else if (dim <= 64)
        f(Int<64>{});
    else if (dim <= 96)
        f(Int<96>{});
    else
        f(Int<128>{});
}
template <typename F>
void with_waves(int waves, bool cap, F&& f) {
    const auto capped = [&](auto w) {
        if (cap)
            f(w, std::true_type{});
        else
            f(w, std::false_type{});
    };
    if (waves == 2)
        capped(Int<2>{});
    else
        capped(Int<4>{});
}

}  // namespace

extern "C" {

size_t tnr_structure_tiles_size(const tnr_structure_attention* req) {
    if (!req || req->n_structures < 0 || req->n_queries < 0 || req->n_keys < 0 || req->heads < 1 ||
        req->kv_heads < 1 || req->heads % req->kv_heads != 0)
        return 0;
    const StructurePlan p = structure_plan(*req);
    return q_tile_bytes(p) + k_tile_bytes(p);
}

size_t tnr_structure_forward_workspace_size(const tnr_structure_attention* req) {
    if (tnr_structure_tiles_size(req) == 0) return 0;
    return structure_space(*req, structure_plan(*req), false, nullptr).bytes;
}

int tnr_structure_forward(const tnr_structure_attention* req, void* workspace,
                          size_t workspace_bytes, void* stream, char* err, size_t err_len) {
    const int code = check_structure(req, false, err, err_len);
    if (code != TNR_OK) return code;
    const tnr_structure_attention& r = *req;
    if (r.n_structures == 0) return TNR_OK;
    const StructurePlan p = structure_plan(r);
    const StructureSpace s = structure_space(r, p, false, workspace);
    if (s.bytes > 0 && (!workspace || (uintptr_t)workspace % 256 != 0 || workspace_bytes < s.bytes))
        return refuse(err, err_len, "workspace is too small or not aligned to 256 bytes");
    const hipStream_t st = (hipStream_t)stream;
    StructureArgs a = structure_args(r, p);
    a.part = s.part;
    a.splits = p.f_splits;
    // (no queries have no log-sums, and their backward reads the keys' tiles all the same)
    lay_tiles(r, p, a, r.lse != nullptr || r.n_queries == 0, st);
    if (r.n_queries == 0) return launched(err, err_len);
    with_type(r.dtype, [&](auto t) {
        using T = decltype(t);
        with_dim(r.dim, [&](auto d) {
            constexpr int DP = decltype(d)::value;
            with_waves(p.q_waves, r.softcap > 0.f, [&](auto w, auto c) {
                constexpr int NW = decltype(w)::value;
                constexpr bool CAP = decltype(c)::value;
                const dim3 grid((unsigned)(p.q_tiles * r.kv_heads), p.f_splits);
                k_structure_forward<T, DP, NW, CAP><<<grid, NW * kWave, 0, st>>>(a);
            });
        });
        if (p.f_splits > 1)
            k_structure_join<T>
                <<<(unsigned)((r.n_queries * r.heads + 3) / 4), 256, 0, st>>>(a);
    });
    return launched(err, err_len);
}

size_t tnr_structure_backward_workspace_size(const tnr_structure_attention* req) {
    if (tnr_structure_tiles_size(req) == 0) return 0;
    return structure_space(*req, structure_plan(*req), true, nullptr).bytes;
}

int tnr_structure_backward(const tnr_structure_attention* req, void* workspace,
                           size_t workspace_bytes, void* stream, char* err, size_t err_len) {
    const int code = check_structure(req, true, err, err_len);
    if (code != TNR_OK) return code;
    const tnr_structure_attention& r = *req;
    const StructurePlan p = structure_plan(r);
    const StructureSpace s = structure_space(r, p, true, workspace);
    if (s.bytes > 0 && (!workspace || (uintptr_t)workspace % 256 != 0 || workspace_bytes < s.bytes))
        return refuse(err, err_len, "workspace is too small or not aligned to 256 bytes");
    if (r.dtype != TNR_FLOAT32 && r.n_queries > 0 && !r.out32)
        return refuse(err, err_len, "required pointers are null");
    const hipStream_t st = (hipStream_t)stream;
    StructureArgs a = structure_args(r, p);
    a.part = s.part;
    a.part_k = s.part_k;
    a.row = s.row;
    a.push_q = s.push_q;
    a.push_k = s.push_k;
    a.turn = s.turn;
    with_type(r.dtype, [&](auto t) {
        using T = decltype(t);
        with_dim(r.dim, [&](auto d) {
            constexpr int DP = decltype(d)::value;
            if (r.n_queries > 0)
                with_waves(p.q_waves, r.softcap > 0.f, [&](auto w, auto c) {
                    constexpr int NW = decltype(w)::value;
                constexpr bool CAP = decltype(c)::value;
                    k_structure_dq<T, DP, NW, CAP>
                        <<<dim3((unsigned)(p.q_tiles * r.kv_heads), p.splits), NW * kWave, 0, st>>>(
                            a);
                });
            if (r.n_queries > 0 && p.splits > 1)
                k_structure_join_dq<T>
                    <<<(unsigned)((r.n_queries * r.heads + 3) / 4), 256, 0, st>>>(a);
            if (r.n_keys > 0)
                with_waves(p.k_waves, r.softcap > 0.f, [&](auto w, auto c) {
                    constexpr int NW = decltype(w)::value;
                constexpr bool CAP = decltype(c)::value;
                    k_structure_dkv<T, DP, NW, CAP>
                        <<<dim3((unsigned)(p.k_tiles * r.kv_heads), p.k_splits), NW * kWave, 0,
                           st>>>(a);
                });
            if (r.n_keys > 0 && p.k_splits > 1)
                k_structure_join_dkv<T>
                    <<<(unsigned)((r.kv_heads * r.n_keys * (2 * r.dim + 3) + 255) / 256), 256, 0,
                       st>>>(a);
        });
    });
    const int shared = !r.query_positions && r.n_queries > 0;
    const int64_t items = (r.grad_positions ? 3 * r.n_keys : 0) +
                          (r.grad_query_positions ? 3 * r.n_queries : 0);
    const int64_t blocks = (items + 1023) / 1024 + (r.grad_slopes ? r.heads : 0);
    if (blocks > 0)
        k_structure_finish<<<(unsigned)blocks, 1024, 0, st>>>(a, r.grad_query_positions,
                                                              r.grad_positions, r.grad_slopes, shared);
    return launched(err, err_len);
}

}  // extern "C"
