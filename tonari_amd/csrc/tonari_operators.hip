// C ABI of the species embedding and of neighbor attention
// (include/tonari_operators.h): checks of requests, workspaces and launches.
// Every call returns a code; no exception crosses it.
#include "op_embedding.h"
#include "op_host.h"
#include "op_neighbor.h"

using namespace tnr::op;

namespace {

void zero(void* p, size_t bytes, hipStream_t stream) {
    const int64_t words = (int64_t)(bytes / 4);
    if (words == 0) return;
    const int64_t blocks = (words + 1023) / 1024;
    k_op_zero<<<(unsigned)(blocks < 1024 ? blocks : 1024), 256, 0, stream>>>((int32_t*)p, words);
}

// ------------------------------------------------------------------ embedding

int check_embedding(const tnr_embedding* r, bool backward, char* err, size_t len) {
    if (!r) return refuse(err, len, "request is null");
    if (!is_type(r->dtype)) return refuse(err, len, "dtype must be float32, bfloat16 or float16");
    if (r->index_bytes != 4 && r->index_bytes != 8)
        return refuse(err, len, "species must be int32 or int64");
    if (r->n_atoms < 0 || r->n_species < 0 || r->channels < 1)
        return refuse(err, len, "invalid sizes");
    // a workgroup for each species, and at most 65,535 side by side for its channels
    if (r->n_atoms >= INT32_MAX || r->n_species > kMostThreads / 256 || r->channels > (1 << 18))
        return refuse(err, len, "too many atoms, species or channels");
    const bool rows = r->n_atoms > 0, table = r->n_species > 0;
    if ((rows && (!r->species || !(backward ? r->grad_out : r->out))) ||
        (table && !(backward ? r->grad_weight : r->weight)))
        return refuse(err, len, "required pointers are null");
    return TNR_OK;
}

// Channels that one thread takes: the most, up to 16 bytes, that divide a row
// and keep every row's address a multiple of them.
int vector_of(const tnr_embedding& r, const void* a, const void* b) {
    const int64_t size = (int64_t)size_of(r.dtype);
    for (int64_t n = 16 / size; n > 1; n /= 2)
        if (r.channels % n == 0 && (uintptr_t)a % (n * size) == 0 && (uintptr_t)b % (n * size) == 0)
            return (int)n;
    return 1;
}

template <typename F>
void with_vector(int vec, F&& f) {
    if (vec == 8)
        f(Int<8>{});
    else if (vec == 4)
        f(Int<4>{});
    else if (vec == 2)
        f(Int<2>{});
    else
        f(Int<1>{});
}

EmbeddingArgs embedding_args(const tnr_embedding& r) {
    return {r.species, r.weight, r.grad_out, r.out,  r.grad_weight,
            r.n_atoms, r.n_species, r.channels, r.scale};
}

// Sorted atoms of a group: enough groups for the device, and no more than 256
// atoms, whose partial rows are few beside them.  1,048,576 rows of 128 floats
// took 223 us at 256 atoms, which leaves two waves to a SIMD, and 171 at 64.
int64_t embedding_each(int64_t n) {
    const int64_t e = n / 16384;
    return e < 16 ? 16 : e > 256 ? 256 : e;
}

struct EmbeddingSpace {
    int32_t *counts, *totals, *key[2], *atom[2];
    int2* runs;
    float* partial;
    size_t bytes;
};
EmbeddingSpace embedding_space(const tnr_embedding& r, void* base) {
    size_t at = 0;
    const auto part = [&](size_t bytes) {
        char* p = (char*)base + at;
        at += padded(bytes);
        return p;
    };
    const int64_t each = embedding_each(r.n_atoms);
    EmbeddingSpace s{};
    s.counts = (int32_t*)part(sort_count_bytes(r.n_atoms));
    s.totals = (int32_t*)part((size_t)kSortRadix * 4);
    for (int i = 0; i < 2; ++i) {
        s.key[i] = (int32_t*)part((size_t)r.n_atoms * 4);
        s.atom[i] = (int32_t*)part((size_t)r.n_atoms * 4);
    }
    s.runs = (int2*)part((size_t)r.n_species * 8);
    s.partial = (float*)part((size_t)((r.n_atoms + each - 1) / each) * 2 * r.channels * 4);
    s.bytes = at;
    return s;
}

// A pass over `keys`, whose items `put` writes.
template <typename Keys, typename Put>
void sort_pass(Keys keys, int64_t n, SortPass pass, int32_t* counts, int32_t* totals, Put put,
               hipStream_t stream, int32_t* clear = nullptr, int64_t clear_words = 0) {
    const unsigned tiles = (unsigned)sort_tiles(n);
    const int radix = 1 << pass.bits;
    if (tiles == 1) {
        k_sort_move<<<1, kSortThreads, 0, stream>>>(keys, n, pass, (const int32_t*)nullptr,
                                                    (const int32_t*)nullptr, put, clear,
                                                    clear_words);
        return;
    }
    k_sort_count<<<tiles, kSortThreads, 0, stream>>>(keys, n, pass, counts, clear, clear_words);
    k_sort_scan<<<(radix + kSortWaves - 1) / kSortWaves, kSortThreads, 0, stream>>>(
        counts, tiles, radix, totals);
    k_sort_move<<<tiles, kSortThreads, 0, stream>>>(keys, n, pass, counts, totals, put, nullptr, 0);
}

template <typename I>
void sort_species(const tnr_embedding& r, const EmbeddingSpace& s, RunArgs& runs,
                  hipStream_t stream) {
    const SortPlan plan = sort_plan(r.n_species + 1);
    int from = 0;
    for (int p = 0; p < plan.passes; ++p) {
        if (p == 0)
            sort_pass(SpeciesOf<I>{(const I*)r.species, r.n_species}, r.n_atoms, plan.pass[p],
                      s.counts, s.totals, PutAtom{s.key[0], s.atom[0]}, stream, (int32_t*)s.runs,
                      2 * r.n_species);
        else {
            sort_pass(SortKeys{s.key[from]}, r.n_atoms, plan.pass[p], s.counts, s.totals,
                      MoveAtom{s.atom[from], s.key[1 - from], s.atom[1 - from]}, stream);
            from = 1 - from;
        }
    }
    runs.key = s.key[from];
    runs.atom = s.atom[from];
}

// -------------------------------------------------------- neighbor attention

constexpr int64_t kMostAtoms = kMostThreads / 256 * 4 + 1;  // a wave each, four to a workgroup

int check_list(const tnr_neighbor_list* l, char* err, size_t len) {
    if (!l) return refuse(err, len, "list is null");
    if (l->n_pairs < 0 || l->n_sources < 0 || l->n_targets < 0)
        return refuse(err, len, "invalid sizes");
    // (kernels look 64 pairs ahead with 32-bit numbers)
    if (l->n_pairs > INT32_MAX - 4096 || l->n_sources >= kMostAtoms || l->n_targets >= kMostAtoms)
        return refuse(err, len, "too many pairs or atoms");
    if (l->n_pairs > 0 && (l->n_sources == 0 || l->n_targets == 0))
        return refuse(err, len, "a list with pairs needs sources and targets");
    if (!l->rows || (uintptr_t)l->rows % 256 != 0)
        return refuse(err, len, "rows must be given and aligned to 256 bytes");
    return TNR_OK;
}

struct RowsSpace {
    int32_t *counts, *totals, *key[2];
    int2* order;
    size_t bytes;
};
RowsSpace rows_space(const tnr_neighbor_list& l, void* base) {
    size_t at = 0;
    const auto part = [&](size_t bytes) {
        char* q = (char*)base + at;
        at += padded(bytes);
        return q;
    };
    RowsSpace s{};
    if (!l.transpose || l.n_pairs == 0) return s;
    s.counts = (int32_t*)part(sort_count_bytes(l.n_pairs));
    s.totals = (int32_t*)part((size_t)kSortRadix * 4);
    s.key[0] = (int32_t*)part((size_t)l.n_pairs * 4);
    if (sort_plan(l.n_targets).passes > 1) {
        s.key[1] = (int32_t*)part((size_t)l.n_pairs * 4);
        s.order = (int2*)part((size_t)l.n_pairs * 8);
    }
    s.bytes = at;
    return s;
}

NeighborRows rows_of(const tnr_neighbor_list& l) {
    return neighbor_rows(l.rows, l.n_pairs, l.n_sources, l.n_targets, l.transpose != 0);
}

RowsHead head_of(const tnr_neighbor_list& l) {
    return {0, (int32_t)l.n_pairs, (int32_t)l.n_sources, (int32_t)l.n_targets};
}

int check_neighbor(const tnr_neighbor_attention* r, bool backward, char* err, size_t len) {
    if (!r) return refuse(err, len, "request is null");
    int code = check_heads(r->dtype, r->heads, r->kv_heads, r->dim, r->scale, r->softcap, err, len);
    if (code == TNR_OK) code = check_list(&r->list, err, len);
    if (code != TNR_OK) return code;
    if (r->list.n_sources >= INT32_MAX / r->heads || r->list.n_targets >= INT32_MAX / r->kv_heads)
        return refuse(err, len, "too many pairs or atoms");
    if (!r->slopes || (r->list.n_sources > 0 && (!r->q || !r->out)) ||
        (r->list.n_targets > 0 && (!r->k || !r->v)) || (r->list.n_pairs > 0 && !r->distances))
        return refuse(err, len, "required pointers are null");
    if (!aligned(r->q, r->q_stride, r->dtype) || !aligned(r->k, r->k_stride, r->dtype) ||
        !aligned(r->v, r->v_stride, r->dtype) || (uintptr_t)r->out % 16 != 0)
        return refuse(err, len, "q, k, v and out must be aligned to 16 bytes, with strides up to 2^24");
    if (backward) {
        if (!r->list.transpose) return refuse(err, len, "the backward needs the rows by target too");
        if ((r->list.n_sources > 0 && (!r->grad_out || !r->grad_q || !r->lse ||
                                       (r->dtype != TNR_FLOAT32 && !r->out32))) ||
            (r->list.n_targets > 0 && (!r->grad_k || !r->grad_v)) || !r->grad_slopes ||
            (r->list.n_pairs > 0 && !r->grad_distances))
            return refuse(err, len, "required pointers are null");
        if ((uintptr_t)r->grad_out % 16 != 0 || (uintptr_t)r->grad_q % 16 != 0 ||
            (uintptr_t)r->grad_k % 16 != 0 || (uintptr_t)r->grad_v % 16 != 0)
            return refuse(err, len, "gradients must be aligned to 16 bytes");
    }
    return TNR_OK;
}

NeighborArgs neighbor_args(const tnr_neighbor_attention& r) {
    NeighborArgs a{};
    a.rows = rows_of(r.list);
    a.head = head_of(r.list);
    a.n_pairs = (int)r.list.n_pairs;
    a.n_sources = (int)r.list.n_sources;
    a.n_targets = (int)r.list.n_targets;
    a.q = r.q;
    a.k = r.k;
    a.v = r.v;
    for (int i = 0; i < 2; ++i) {
        a.q_stride[i] = r.q_stride[i];
        a.k_stride[i] = r.k_stride[i];
        a.v_stride[i] = r.v_stride[i];
    }
    a.distances = r.distances;
    a.slopes = r.slopes;
    a.rule = ScoreRule::of(r.scale, r.softcap);
    a.heads = r.heads;
    a.kv_heads = r.kv_heads;
    a.group = r.heads / r.kv_heads;
    a.dim = r.dim;
    a.out = r.out;
    a.out32 = r.out32;
    a.lse = r.lse;
    a.grad_out = r.grad_out;
    a.out_full = r.dtype == TNR_FLOAT32 ? (const float*)r.out : r.out32;
    a.grad_q = r.grad_q;
    a.grad_k = r.grad_k;
    a.grad_v = r.grad_v;
    a.grad_distances = r.grad_distances;
    return a;
}

// How heads lie on lanes: R times 16 bytes to a lane, as many lanes as make a
// head's channels (a power of two), GH query heads to a lane where they share a
// key head.  What is done once for each score is done by every lane of a head,
// so one query head takes two pieces where the channels allow: 256 crystals (1.3 M
// pairs) of 8 capped heads of 16 floats take 48 + 70 + 63 us, forward and both
// passes back, and 51 + 89 + 75 at one piece.
template <typename T, typename F>
void with_lanes(int32_t dim, int group, bool cap, F&& f) {
    const auto capped = [&](auto lanes, auto of, auto pieces) {
        if (cap)
            f(lanes, of, pieces, std::true_type{});
        else
            f(lanes, of, pieces, std::false_type{});
    };
    const int units = (int)(dim * sizeof(T) / 16);
    const auto lanes_of = [&](int n, auto of, auto pieces) {
        constexpr int kMost = (int)(128 * sizeof(T) / 16) / decltype(pieces)::value;
        if (n <= 1)
            capped(Int<1>{}, of, pieces);
        else if (n <= 2)
            capped(Int<2>{}, of, pieces);
        else if (n <= 4)
            capped(Int<4>{}, of, pieces);
        else if (n <= 8)
            capped(Int<8>{}, of, pieces);
        else if constexpr (kMost >= 16) {
            if (n <= 16)
                capped(Int<16>{}, of, pieces);
            else if constexpr (kMost >= 32)
                capped(Int<32>{}, of, pieces);
        }
    };
    if (group % 4 == 0)
        lanes_of(units, Int<4>{}, Int<1>{});
    else if (group % 2 == 0)
        lanes_of(units, Int<2>{}, Int<1>{});
    else if (units % 2 == 0)
        lanes_of(units / 2, Int<1>{}, Int<2>{});
    else
        lanes_of(units, Int<1>{}, Int<1>{});
}

// Lanes of a slot: those of its units, a power of two, at most a wave.
int slot_of(int lanes, int units) {
    int slot = lanes;
    while (slot < kWave && slot < lanes * units) slot *= 2;
    return slot;
}

}  // namespace

extern "C" {

int tnr_operators_version(void) { return TNR_OPERATORS_VERSION; }

int tnr_embedding_forward(const tnr_embedding* req, void* stream, char* err, size_t err_len) {
    const int code = check_embedding(req, false, err, err_len);
    if (code != TNR_OK) return code;
    const tnr_embedding& r = *req;
    if (r.n_atoms == 0) return TNR_OK;
    const EmbeddingArgs a = embedding_args(r);
    with_type(r.dtype, [&](auto t) {
        using T = decltype(t);
        with_vector(vector_of(r, r.weight, r.out), [&](auto v) {
            constexpr int VEC = decltype(v)::value;
            if constexpr (VEC * sizeof(T) <= 16) {
                const int64_t blocks = (r.n_atoms * (r.channels / VEC) + 255) / 256;
                const unsigned grid = (unsigned)(blocks < 16384 ? blocks : 16384);
                if (r.index_bytes == 4)
                    k_embedding_forward<T, int32_t, VEC><<<grid, 256, 0, (hipStream_t)stream>>>(a);
                else
                    k_embedding_forward<T, int64_t, VEC><<<grid, 256, 0, (hipStream_t)stream>>>(a);
            }
        });
    });
    return launched(err, err_len);
}

size_t tnr_embedding_workspace_size(const tnr_embedding* req) {
    if (!req || req->n_atoms < 0 || req->n_species < 0 || req->channels < 1) return 0;
    return embedding_space(*req, nullptr).bytes;
}

int tnr_embedding_backward(const tnr_embedding* req, void* workspace, size_t workspace_bytes,
                           void* stream, char* err, size_t err_len) {
    const int code = check_embedding(req, true, err, err_len);
    if (code != TNR_OK) return code;
    const tnr_embedding& r = *req;
    if (r.n_species == 0) return TNR_OK;
    const EmbeddingSpace s = embedding_space(r, workspace);
    if (!workspace || (uintptr_t)workspace % 256 != 0 || workspace_bytes < s.bytes)
        return refuse(err, err_len, "workspace is too small or not aligned to 256 bytes");
    const hipStream_t st = (hipStream_t)stream;
    const EmbeddingArgs a = embedding_args(r);
    RunArgs runs{};
    runs.runs = s.runs;
    runs.partial = s.partial;
    runs.each = embedding_each(r.n_atoms);
    if (r.n_atoms == 0) {
        zero(s.runs, (size_t)r.n_species * 8, st);
    } else {
        if (r.index_bytes == 4)
            sort_species<int32_t>(r, s, runs, st);
        else
            sort_species<int64_t>(r, s, runs, st);
    }
    with_type(r.dtype, [&](auto t) {
        using T = decltype(t);
        with_vector(vector_of(r, r.grad_out, r.grad_weight), [&](auto v) {
            constexpr int VEC = decltype(v)::value;
            if constexpr (VEC * sizeof(T) <= 16) {
                int lanes = 1;
                while (lanes < 64 && lanes * VEC < r.channels) lanes *= 2;
                const unsigned y = (unsigned)((r.channels + lanes * VEC - 1) / (lanes * VEC));
                const int64_t groups = (r.n_atoms + runs.each - 1) / runs.each;
                const int64_t in_block = 256 / lanes;
                if (groups > 0)
                    k_embedding_runs<T, VEC>
                        <<<dim3((unsigned)((groups + in_block - 1) / in_block), y), 256, 0, st>>>(
                            a, runs, lanes);
                // few lanes a row: a frequent species has thousands of partial rows
                const int few = lanes < 8 ? lanes : 8;
                k_embedding_join<T, VEC>
                    <<<dim3((unsigned)r.n_species,
                            (unsigned)((r.channels + few * VEC - 1) / (few * VEC))),
                       256, 0, st>>>(a, runs, few);
            }
        });
    });
    return launched(err, err_len);
}

size_t tnr_neighbor_rows_size(const tnr_neighbor_list* list) {
    if (!list || list->n_pairs < 0 || list->n_sources < 0 || list->n_targets < 0) return 0;
    return neighbor_rows(nullptr, list->n_pairs, list->n_sources, list->n_targets,
                         list->transpose != 0)
        .bytes;
}

size_t tnr_neighbor_rows_workspace_size(const tnr_neighbor_list* list) {
    if (!list || list->n_pairs < 0 || list->n_sources < 0 || list->n_targets < 0) return 0;
    return rows_space(*list, nullptr).bytes;
}

int tnr_neighbor_rows(const tnr_neighbor_list* list, void* workspace, size_t workspace_bytes,
                      void* stream, char* err, size_t err_len) {
    const int code = check_list(list, err, err_len);
    if (code != TNR_OK) return code;
    const tnr_neighbor_list& l = *list;
    if (l.n_pairs > 0 && (!l.sources || !l.targets))
        return refuse(err, err_len, "required pointers are null");
    const RowsSpace s = rows_space(l, workspace);
    if (s.bytes > 0 && (!workspace || (uintptr_t)workspace % 256 != 0 || workspace_bytes < s.bytes))
        return refuse(err, err_len, "workspace is too small or not aligned to 256 bytes");
    const hipStream_t st = (hipStream_t)stream;
    const NeighborRows rows = rows_of(l);
    // the head and the runs, which lie at the front
    const int64_t words = ((char*)rows.target - (char*)rows.head) / 4;
    const int64_t blocks = (words + 1023) / 1024;
    k_neighbor_clear<<<(unsigned)(blocks < 1024 ? blocks : 1024), 256, 0, st>>>(rows.head,
                                                                                head_of(l), words);
    if (l.n_pairs > 0) {
        k_neighbor_rows<<<(unsigned)((l.n_pairs + kRowsBlock - 1) / kRowsBlock), 256, 0, st>>>(
            l.sources, l.targets, l.n_pairs, l.n_sources, l.n_targets, rows);
        if (l.transpose) {
            const SortPlan plan = sort_plan(l.n_targets);
            const int32_t* key = nullptr;
            for (int p = 0; p < plan.passes; ++p) {
                // the last pass writes the rows' own order
                const bool own = (plan.passes - 1 - p) % 2 == 0;
                int32_t* to = s.key[own ? 0 : 1];
                int2* order = own ? rows.order : s.order;
                if (p == 0)
                    sort_pass(PairKeys{rows.target}, l.n_pairs, plan.pass[p], s.counts, s.totals,
                              PutPair{l.sources, to, order}, st);
                else
                    sort_pass(SortKeys{key}, l.n_pairs, plan.pass[p], s.counts, s.totals,
                              MovePair{own ? s.order : rows.order, to, order}, st);
                key = to;
            }
            k_neighbor_targets<<<(unsigned)((l.n_pairs + 255) / 256), 256, 0, st>>>(
                key, l.n_pairs, rows.targets);
        }
    }
    return launched(err, err_len);
}

int tnr_neighbor_forward(const tnr_neighbor_attention* req, void* stream, char* err,
                         size_t err_len) {
    const int code = check_neighbor(req, false, err, err_len);
    if (code != TNR_OK) return code;
    const tnr_neighbor_attention& r = *req;
    if (r.list.n_sources == 0) return TNR_OK;
    NeighborArgs a = neighbor_args(r);
    with_type(r.dtype, [&](auto t) {
        using T = decltype(t);
        with_lanes<T>(r.dim, a.group, r.softcap > 0.f, [&](auto l, auto g, auto p, auto c) {
            constexpr int LPH = decltype(l)::value, GH = decltype(g)::value,
                          R = decltype(p)::value;
            constexpr bool CAP = decltype(c)::value;
            const int units = r.heads / GH;
            a.slot = slot_of(LPH, units);
            const int block = a.slot / LPH;
            k_neighbor_forward<T, LPH, GH, R, CAP>
                <<<dim3((unsigned)((r.list.n_sources + 3) / 4), (units + block - 1) / block), 256, 0,
                   (hipStream_t)stream>>>(a);
        });
    });
    return launched(err, err_len);
}

size_t tnr_neighbor_backward_workspace_size(const tnr_neighbor_attention* req) {
    if (!req || req->heads < 1 || req->list.n_sources < 0) return 0;
    const size_t rows = (size_t)req->list.n_sources * req->heads;
    return padded(rows * sizeof(float2)) + padded(rows * sizeof(float));
}

int tnr_neighbor_backward(const tnr_neighbor_attention* req, void* workspace,
                          size_t workspace_bytes, void* stream, char* err, size_t err_len) {
    const int code = check_neighbor(req, true, err, err_len);
    if (code != TNR_OK) return code;
    const tnr_neighbor_attention& r = *req;
    const size_t need = tnr_neighbor_backward_workspace_size(req);
    if (need > 0 && (!workspace || (uintptr_t)workspace % 256 != 0 || workspace_bytes < need))
        return refuse(err, err_len, "workspace is too small or not aligned to 256 bytes");
    const hipStream_t st = (hipStream_t)stream;
    NeighborArgs a = neighbor_args(r);
    a.stat = (float2*)workspace;
    a.turn = (float*)((char*)workspace +
                      padded((size_t)r.list.n_sources * r.heads * sizeof(float2)));
    with_type(r.dtype, [&](auto t) {
        using T = decltype(t);
        with_lanes<T>(r.dim, a.group, r.softcap > 0.f, [&](auto l, auto g, auto p, auto c) {
            constexpr int LPH = decltype(l)::value, GH = decltype(g)::value,
                          R = decltype(p)::value;
            constexpr bool CAP = decltype(c)::value;
            a.slot = slot_of(LPH, r.heads / GH);
            if (r.list.n_sources > 0)
                k_neighbor_dq<T, LPH, GH, R, CAP>
                    <<<(unsigned)((r.list.n_sources + 3) / 4), 256, 0, st>>>(a);
            a.slot = slot_of(LPH, r.kv_heads);
            const int block = a.slot / LPH;
            if (r.list.n_targets > 0)
                k_neighbor_dkv<T, LPH, GH, R, CAP><<<dim3((unsigned)((r.list.n_targets + 3) / 4),
                                                  (r.kv_heads + block - 1) / block),
                                             256, 0, st>>>(a);
        });
    });
    k_slopes<<<r.heads, 1024, 0, st>>>(a.turn, r.list.n_sources, r.grad_slopes);
    return launched(err, err_len);
}

}  // extern "C"
