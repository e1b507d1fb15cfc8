// Attention along the pairs of a neighbor list: each source atom i over its
// pairs (i, j) at distance d, scores and gradients as in op_structure.h with
// the pair's d for r (its gradient is an output: the list's own backward takes
// it on to positions and cell).
//
// A source's keys lie anywhere, so the work is a gather of k and v rows (512
// bytes a pair for 128 channels of 16 bits) and a few operations on each value
// read.  One wave takes a source: lanes of 16 or 32 bytes make a head, heads make
// a slot, and the wave's slots take pairs side by side, each with its own running
// maximum and sum; the slots are joined at the source's end.  Query heads that
// share a key head are taken by the same lanes, so that its rows are read once.
//
// What bounds it: where the rows of all atoms outgrow the 4 MB L2 of an XCD and
// the list is not in spatial order, the rate behind the L2 (100,000 atoms, 9 M
// pairs, 8 heads of 16 bfloat16: 4.6 GB in 593 us, 7.8 TB/s); else what is done
// for each score (256 crystals, 1.3 M pairs, 8 capped heads of 16 floats: 48 us
// forward, 70 and 63 back, vector instructions in 74 to 80 % of the busy cycles).
// Fewer registers and more waves lose: 32,768 atoms with 4 query heads to a key head
// take 179 us at five waves to a SIMD and 131 at four.
//
// Backward: by sources (grad_q, and grad_d, which needs the sum over heads of
// one pair), then by targets in the list's transposed order (grad_k, grad_v),
// both recomputing the weights from the forward's row statistics: no atomics,
// so the sums' order is the list's.
#pragma once

#include "op_sort.h"

namespace tnr {
namespace op {

// What the rows are of.  Rows whose head does not say what a call says are not read
// further, so that no call goes by the runs of another list.
struct RowsHead {
    int32_t status;  // not 0: the list is not valid (every result is NaN)
    int32_t pairs, sources, targets;
    __host__ __device__ bool holds(const RowsHead& o) const {
        return status == 0 && pairs == o.pairs && sources == o.sources && targets == o.targets;
    }
};
constexpr int kHeadWords = sizeof(RowsHead) / 4;

// What tnr_neighbor_rows writes, in this order (each part 256-byte aligned).
struct NeighborRows {
    RowsHead* head;
    int2* sources;     // [n_sources]: pairs [x, y)
    int32_t* target;   // [n_pairs]
    int2* targets;     // [n_targets]: places [x, y) of `order`
    int2* order;       // [n_pairs]: (pair, source) by target, in list order
    size_t bytes;
};
inline NeighborRows neighbor_rows(void* base, int64_t pairs, int64_t sources, int64_t targets,
                                  bool transpose) {
    size_t at = 0;
    char* p = (char*)base;
    const auto part = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return p + here;
    };
    NeighborRows r{};
    r.head = (RowsHead*)part(sizeof(RowsHead));
    r.sources = (int2*)part((size_t)sources * 8);
    if (transpose) r.targets = (int2*)part((size_t)targets * 8);
    r.target = (int32_t*)part((size_t)pairs * 4);
    if (transpose) r.order = (int2*)part((size_t)pairs * 8);
    r.bytes = at;
    return r;
}

// Clears `words` from the head on: the runs, but for what the head says.
__global__ __launch_bounds__(256) void k_neighbor_clear(RowsHead* at, RowsHead head, int64_t words) {
    const int32_t says[kHeadWords] = {head.status, head.pairs, head.sources, head.targets};
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words;
         i += (int64_t)gridDim.x * 256) {
        int32_t x = 0;
#pragma unroll
        for (int w = 0; w < kHeadWords; ++w)
            if (i == w) x = says[w];
        ((int32_t*)at)[i] = x;
    }
}

// The runs are cleared before.  A source whose pairs do not lie
// together finds its run taken.
constexpr int kRowsEach = 4, kRowsBlock = 256 * kRowsEach;
__global__ __launch_bounds__(256) void k_neighbor_rows(const int64_t* sources,
                                                       const int64_t* targets, int64_t n_pairs,
                                                       int64_t n_sources, int64_t n_targets,
                                                       NeighborRows r) {
    // a wave takes kRowsEach x 64 pairs that lie together, a lane one of each 64
    const int lane = lane_of();
    const int64_t base =
        (int64_t)blockIdx.x * kRowsBlock + (threadIdx.x / kWave) * (kWave * kRowsEach) + lane;
    int64_t i[kRowsEach], j[kRowsEach], edge = -1;
#pragma unroll
    for (int u = 0; u < kRowsEach; ++u) {
        const int64_t e = base + u * kWave;
        i[u] = e < n_pairs ? sources[e] : -1;
        j[u] = e < n_pairs ? targets[e] : -1;
    }
    // the sources before the wave's first pair and after its last
    const int64_t out = lane == 0 ? base - 1 : base + (kRowsEach - 1) * kWave + 1;
    if ((lane == 0 || lane == kWave - 1) && out >= 0 && out < n_pairs) edge = sources[out];
    int bad = 0;
#pragma unroll
    for (int u = 0; u < kRowsEach; ++u) {
        const int64_t e = base + u * kWave;
        int64_t before = __shfl_up((long long)i[u], 1), after = __shfl_down((long long)i[u], 1);
        const int64_t last = u > 0 ? __shfl((long long)i[u > 0 ? u - 1 : 0], kWave - 1) : edge;
        const int64_t next = u + 1 < kRowsEach
                                 ? __shfl((long long)i[u + 1 < kRowsEach ? u + 1 : u], 0)
                                 : edge;
        if (lane == 0) before = last;
        if (lane == kWave - 1) after = next;
        if (e >= n_pairs) continue;
        const bool in = i[u] >= 0 && i[u] < n_sources && j[u] >= 0 && j[u] < n_targets;
        bad |= !in;
        r.target[e] = in ? (int32_t)j[u] : 0;
        if (!in) continue;
        if (e == 0 || before != i[u])
            bad |= atomicExch(&r.sources[i[u]].x, (int)e + 1) != 0;  // 0: none yet
        if (e + 1 == n_pairs || after != i[u]) r.sources[i[u]].y = (int)e + 1;
    }
    if (__builtin_amdgcn_ballot_w64(bad != 0) != 0 && lane == 0) atomicOr(&r.head->status, 1);
}

struct PairKeys {
    const int32_t* target;
    __device__ __forceinline__ int operator()(int64_t i) const { return target[i]; }
};
struct PutPair {
    const int64_t* sources;
    int32_t* key;
    int2* order;
    __device__ __forceinline__ void operator()(int64_t place, int64_t i, int k) const {
        key[place] = k;
        order[place] = int2{(int)i, (int)sources[i]};
    }
};
struct MovePair {
    const int2* from;
    int32_t* key;
    int2* order;
    __device__ __forceinline__ void operator()(int64_t place, int64_t i, int k) const {
        key[place] = k;
        order[place] = from[i];
    }
};
__global__ __launch_bounds__(256) void k_neighbor_targets(const int32_t* key, int64_t n_pairs,
                                                          int2* targets) {
    const int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (p >= n_pairs) return;
    const int k = key[p];
    if (p == 0 || key[p - 1] != k) targets[k].x = (int)p + 1;
    if (p + 1 == n_pairs || key[p + 1] != k) targets[k].y = (int)p + 1;
}

// Runs hold begin + 1 and end: an atom without pairs has (0, 0).
__device__ __forceinline__ int2 run_of(const int2* runs, int64_t i) {
    const int2 r = runs[i];
    return int2{r.x > 0 ? r.x - 1 : 0, r.y};
}

struct NeighborArgs {
    NeighborRows rows;
    RowsHead head;  // what the rows have to be of
    int n_pairs, n_sources, n_targets;
    const void *q, *k, *v;
    int64_t q_stride[2], k_stride[2], v_stride[2];
    const float *distances, *slopes;
    ScoreRule rule;
    int heads, kv_heads, group, dim;
    int slot;  // lanes of a slot
    void* out;
    float *out32, *lse;
    const void* grad_out;
    const float* out_full;  // the forward's output in 32 bits
    void *grad_q, *grad_k, *grad_v;
    float* grad_distances;
    float2* stat;  // [n_sources][heads]: log-sum (inf: no weight) and delta
    float* turn;   // [heads][n_sources]
};

// A lane's part of a row, as it is loaded: R times 16 bytes.  Products of 16-bit
// values go two at a time into a 32-bit sum.
template <typename T, int R>
struct Raw {
    static constexpr int kEach = 16 / sizeof(T), kVec = R * kEach;
    Vec<T, kEach> x[R];
    __device__ __forceinline__ static Raw at(const char* p) {
        Raw raw;
#pragma unroll
        for (int r = 0; r < R; ++r) raw.x[r] = ((const Vec<T, kEach>*)p)[r];
        return raw;
    }
    __device__ __forceinline__ float get(int i) const { return (float)x[i / kEach][i % kEach]; }
    __device__ __forceinline__ float dot(const Raw& o, float sum) const {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int i = 0; i < kEach; ++i) sum = fmaf(x[r][i], o.x[r][i], sum);
            } else {
#pragma unroll
                for (int i = 0; i < kEach; i += 2) {
                    const Vec<T, 2> a = {x[r][i], x[r][i + 1]}, b = {o.x[r][i], o.x[r][i + 1]};
                    if constexpr (std::is_same_v<T, bf16>)
                        sum = __builtin_amdgcn_fdot2_f32_bf16(a, b, sum, false);
                    else
                        sum = __builtin_amdgcn_fdot2(a, b, sum, false);
                }
            }
        }
        return sum;
    }
    // acc += p x
    __device__ __forceinline__ void add(float p, float (&acc)[kVec]) const {
#pragma unroll
        for (int i = 0; i < kVec; ++i) acc[i] = fmaf(p, get(i), acc[i]);
    }
};
// 16 bytes at a time.
template <typename T, int N>
__device__ __forceinline__ void store_wide(T* p, const float (&x)[N]) {
    constexpr int kEach = 16 / sizeof(T);
#pragma unroll
    for (int b = 0; b < N; b += kEach) {
        Vec<T, kEach> v;
#pragma unroll
        for (int i = 0; i < kEach; ++i) v[i] = rounded<T>(x[b + i]);
        *(Vec<T, kEach>*)(p + b) = v;
    }
}

// Sum over the LPH lanes of a head, in all of them.
template <int LPH>
__device__ __forceinline__ float head_sum(float x) {
    if constexpr (LPH >= 2) x += dpp_of<0xb1>(x);    // lane ^ 1
    if constexpr (LPH >= 4) x += dpp_of<0x4e>(x);    // lane ^ 2
    if constexpr (LPH >= 8) x += dpp_of<0x141>(x);   // mirrored in 8
    if constexpr (LPH >= 16) x += dpp_of<0x140>(x);  // mirrored in 16
    if constexpr (LPH >= 32) x += __shfl_xor(x, 16);
    return x;
}

// Sum over the heads of a slot of what all lanes of a head hold, in all of them.
template <int LPH>
__device__ __forceinline__ float slot_sum(float x, int slot) {
    if (LPH <= 1 && slot > 1) x += dpp_of<0xb1>(x);
    if (LPH <= 2 && slot > 2) x += dpp_of<0x4e>(x);
    if (LPH <= 4 && slot > 4) x += dpp_of<0x141>(x);
    if (LPH <= 8 && slot > 8) x += dpp_of<0x140>(x);
    if (LPH <= 16 && slot > 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x),
                                                        false, false);
        x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    if (slot > 32) x = sum_halves(x);
    return x;
}

// u log2(e) of N products, and what their gradients are multiplied by.  (As in
// structure attention nothing is subtracted before a score is whole.)
template <bool CAP, int N>
__device__ __forceinline__ void capped_few(float (&u)[N], const ScoreRule& rule,
                                           float (&bend)[N]) {
    if (!CAP) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            u[i] *= rule.scale2;
            bend[i] = 1.f;
        }
        return;
    }
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        u[i] *= rule.inv;
        top = fmaxf(top, fabsf(u[i]));
    }
    // (the empty asm keeps this a branch of the wave: one side only is computed)
    if (__builtin_amdgcn_ballot_w64(!(top <= kTanhNear)) == 0) {
        asm volatile("");
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = tanh_near(u[i]);
    } else {
        asm volatile("");
#pragma unroll
        for (int i = 0; i < N; ++i) u[i] = tanh_of(u[i]);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        bend[i] = fmaf(-u[i], u[i], 1.f);
        u[i] *= rule.cap2;
    }
}

template <typename T>
__device__ __forceinline__ void fill_nan(T* p, int64_t n, int64_t from, int64_t step) {
    for (int64_t i = from; i < n; i += step) p[i] = rounded<T>(nan_of());
}

// Floats of any count, 16 bytes at a time.
template <int N>
__device__ __forceinline__ void load_wide(const float* p, float (&x)[N]) {
#pragma unroll
    for (int b = 0; b < N; b += 4) {
        const Vec<float, 4> t = *(const Vec<float, 4>*)(p + b);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[b + i] = t[i];
    }
}

// What a lane of a wave takes: R times 16 bytes of a key head's channels, for GH
// query heads that share it (`head` is the first).  A slot holds `block` such units.
// Lanes whose head or channels do not exist read those of others, which may be
// infinite, and add nothing: their products are left out, not multiplied by 0.
template <typename T, int LPH, int GH, int R>
struct Lane {
    static constexpr int VEC = Raw<T, R>::kVec;
    int lane, slot, in_slot, slots, head, kv, c;
    bool there, mine;  // the head exists; the channels too
    __device__ __forceinline__ Lane(const NeighborArgs& a, int first) {
        lane = lane_of();
        slot = lane / a.slot;
        in_slot = lane % a.slot;
        slots = kWave / a.slot;
        head = (first + in_slot / LPH) * GH;
        there = head < a.heads;
        c = (in_slot % LPH) * VEC;
        mine = there && c < a.dim;
        if (!there) head = 0;
        kv = head / a.group;
        if (!mine) c = 0;
    }
};
template <typename T>
__device__ __forceinline__ const char* row_at(const char* base, int row, uint32_t bytes) {
    return base + (uint64_t)(uint32_t)row * bytes;
}

// Waves that a SIMD is to hold: the gather lives by what is in flight.
constexpr int kHeld = 4, kHeldBack = 3;

// 64 pairs of a source, one to a lane, and the next 64 on their way.  A lane
// beyond the run holds its last pair.
struct PairChunk {
    int first, left;  // of the run's pairs; those from `first` on
    int target, next_target;
    float distance, next_distance;
    __device__ __forceinline__ PairChunk(const NeighborArgs& a, int2 run)
        : first(run.x - kWave), left(run.y - run.x + kWave), target(0), next_target(0),
          distance(0.f), next_distance(0.f) {
        fetch(a, run, run.x);
        next(a, run);
    }
    __device__ __forceinline__ void fetch(const NeighborArgs& a, int2 run, int from) {
        if (from >= run.y) return;
        const int e = min(from + lane_of(), run.y - 1);
        next_target = a.rows.target[e];
        next_distance = a.distances[e];
    }
    __device__ __forceinline__ void next(const NeighborArgs& a, int2 run) {
        first += kWave;
        left -= kWave;
        target = next_target;
        distance = next_distance;
        fetch(a, run, first + kWave);
    }
};

// grid: (sources / 4, blocks of units).
template <typename T, int LPH, int GH, int R, bool CAP>
__global__ __launch_bounds__(256, kHeld) void k_neighbor_forward(const NeighborArgs a) {
    constexpr int VEC = Raw<T, R>::kVec, kAhead = GH == 1 && R == 1 ? 4 : 2;
    const int64_t i = (int64_t)xcd_order(blockIdx.x, gridDim.x) * 4 + threadIdx.x / kWave;
    if (i >= a.n_sources) return;
    const Lane<T, LPH, GH, R> l(a, blockIdx.y * (a.slot / LPH));
    const int64_t row = i * a.heads + l.head;
    float acc[GH][VEC], top[GH], sum[GH];
#pragma unroll
    for (int g = 0; g < GH; ++g) {
        top[g] = -inf_of();
        sum[g] = 0.f;
#pragma unroll
        for (int x = 0; x < VEC; ++x) acc[g][x] = 0.f;
    }
    const bool valid = a.rows.head->holds(a.head);
    if (valid) {
        Raw<T, R> q[GH];
        float slope2[GH];
#pragma unroll
        for (int g = 0; g < GH; ++g) {
            q[g] = Raw<T, R>{};
            if (l.mine)
                q[g] = Raw<T, R>::at((const char*)((const T*)a.q + i * a.q_stride[0] +
                                                (l.head + g) * a.q_stride[1] + l.c));
            slope2[g] = a.slopes[l.head + g] * kLog2e;
        }
        const char* k = (const char*)((const T*)a.k + l.kv * a.k_stride[1] + l.c);
        const char* v = (const char*)((const T*)a.v + l.kv * a.v_stride[1] + l.c);
        const uint32_t k_row = (uint32_t)(a.k_stride[0] * sizeof(T));
        const uint32_t v_row = (uint32_t)(a.v_stride[0] * sizeof(T));
        const int2 run = run_of(a.rows.sources, i);
        // The targets and distances of 64 pairs are loaded together, one to a lane,
        // 64 pairs ahead.  A pair beyond the run's end repeats its last one, with
        // weight 0.
        PairChunk chunk(a, run);
        // `n` of the chunk's 64 places hold pairs; a step reaches beyond them, and
        // beyond 64 where a slot is a lane or two
        const auto step = [&](int p0, int n, auto whole) {
            Raw<T, R> kx[kAhead], vx[kAhead];
            float d[kAhead];
            bool in[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int p = p0 + u * l.slots + l.slot;
                in[u] = whole || p < n;
                const int j = __shfl(chunk.target, p);
                d[u] = __shfl(chunk.distance, p);
                kx[u] = Raw<T, R>::at(row_at<T>(k, j, k_row));
                vx[u] = Raw<T, R>::at(row_at<T>(v, j, v_row));
            }
            if (!whole)
#pragma unroll
                for (int u = 0; u < kAhead; ++u)
                    if (!in[u]) vx[u] = Raw<T, R>{};
            // weights relative to the slot's maximum when it was last set, which
            // is set anew where a score passes it by more than 2^8
            float s[GH][kAhead], high[GH], unused[kAhead];
            bool anew = false;
#pragma unroll
            for (int g = 0; g < GH; ++g) {
#pragma unroll
                for (int u = 0; u < kAhead; ++u)
                    s[g][u] = head_sum<LPH>(l.mine ? q[g].dot(kx[u], 0.f) : 0.f);
                const float ref = top[g] == -inf_of() ? 0.f : top[g];
                capped_few<CAP>(s[g], a.rule, unused);
                high[g] = -inf_of();
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    s[g][u] = fmaf(-slope2[g], d[u], s[g][u]) - ref;
                    if (!whole && !in[u]) s[g][u] = -inf_of();
                    high[g] = fmaxf(high[g], s[g][u]);
                }
                anew |= high[g] > 8.f || (top[g] == -inf_of() && high[g] > -inf_of());
            }
            if (__builtin_amdgcn_ballot_w64(anew) != 0) {
                asm volatile("");
#pragma unroll
                for (int g = 0; g < GH; ++g) {
                    const bool first = top[g] == -inf_of();
                    const bool move = first ? high[g] > -inf_of() : high[g] > 0.f;
                    // (the first maximum has no sums to fade, and may lie far below 0)
                    const float up = move ? high[g] : 0.f, fade = exp2_of(fminf(-up, 0.f));
                    if (move) top[g] = (first ? 0.f : top[g]) + high[g];
                    sum[g] *= fade;
#pragma unroll
                    for (int x = 0; x < VEC; ++x) acc[g][x] *= fade;
#pragma unroll
                    for (int u = 0; u < kAhead; ++u) s[g][u] -= up;
                }
            }
#pragma unroll
            for (int g = 0; g < GH; ++g)
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    const float p = exp2_of(s[g][u]);
                    sum[g] += p;
                    vx[u].add(p, acc[g]);
                }
        };
        for (; chunk.left > 0; chunk.next(a, run)) {
            const int n = min(chunk.left, kWave), stride = l.slots * kAhead;
            int p0 = 0;
            for (; p0 + stride <= n; p0 += stride) step(p0, n, std::true_type{});
            if (p0 < n) step(p0, n, std::false_type{});
        }
        // the slots' sums, in the largest maximum's terms
#pragma unroll
        for (int g = 0; g < GH; ++g) {
            const float high = join_lanes<max_of>(top[g], a.slot);
            const float w = exp2_of(top[g] - (high == -inf_of() ? 0.f : high));
            top[g] = high;
            sum[g] = join_lanes<sum_of>(sum[g] * w, a.slot);
#pragma unroll
            for (int x = 0; x < VEC; ++x) acc[g][x] = join_lanes<sum_of>(acc[g][x] * w, a.slot);
        }
    }
    if (!l.mine || l.slot != 0) return;
#pragma unroll
    for (int g = 0; g < GH; ++g) {
        const float by = sum[g] == 0.f ? 0.f : 1.f / sum[g];
        const int64_t at = (row + g) * a.dim + l.c;
#pragma unroll
        for (int x = 0; x < VEC; ++x) acc[g][x] = valid ? acc[g][x] * by : nan_of();
        store_wide<T, VEC>((T*)a.out + at, acc[g]);
        if (a.out32) store_wide<float, VEC>(a.out32 + at, acc[g]);
        if (a.lse && l.c == 0)
            a.lse[row + g] = !valid        ? nan_of()
                             : sum[g] == 0.f ? -inf_of()
                                             : top[g] + __builtin_amdgcn_logf(sum[g]);
    }
}

// By sources: grad_q, grad_d, delta and the slopes' gradient by rows.  Blocks of
// units that do not fit a wave follow one another in it, so that a pair's
// grad_d is summed by one lane.
template <typename T, int LPH, int GH, int R, bool CAP>
__global__ __launch_bounds__(256, kHeldBack) void k_neighbor_dq(const NeighborArgs a) {
    constexpr int VEC = Raw<T, R>::kVec, kAhead = GH == 4 ? 1 : GH == 2 || R == 2 ? 2 : 4;
    const int64_t i = (int64_t)xcd_order(blockIdx.x, gridDim.x) * 4 + threadIdx.x / kWave;
    if (i >= a.n_sources) return;
    if (!a.rows.head->holds(a.head)) {
        const int lane = lane_of();
        fill_nan((T*)a.grad_q + i * a.heads * a.dim, (int64_t)a.heads * a.dim, lane, kWave);
        fill_nan(a.grad_distances, a.n_pairs, i * kWave + lane, (int64_t)a.n_sources * kWave);
        for (int h = lane; h < a.heads; h += kWave) a.turn[(int64_t)h * a.n_sources + i] = nan_of();
        return;
    }
    const int2 run = run_of(a.rows.sources, i);
    const uint32_t k_row = (uint32_t)(a.k_stride[0] * sizeof(T));
    const uint32_t v_row = (uint32_t)(a.v_stride[0] * sizeof(T));
    for (int first = 0; first * GH < a.heads; first += a.slot / LPH) {
        const Lane<T, LPH, GH, R> l(a, first);
        const int64_t row = i * a.heads + l.head;
        Raw<T, R> q[GH], go[GH];
        float acc[GH][VEC], delta[GH], turn[GH], over[GH], mean[GH], lse[GH], slope[GH];
#pragma unroll
        for (int g = 0; g < GH; ++g) {
            q[g] = go[g] = Raw<T, R>{};
            delta[g] = turn[g] = over[g] = mean[g] = slope[g] = 0.f;
            lse[g] = inf_of();
            if (l.mine) {
                const int64_t at = (row + g) * a.dim + l.c;
                float o[VEC];
                q[g] = Raw<T, R>::at((const char*)((const T*)a.q + i * a.q_stride[0] +
                                                (l.head + g) * a.q_stride[1] + l.c));
                go[g] = Raw<T, R>::at((const char*)((const T*)a.grad_out + at));
                load_wide<VEC>(a.out_full + at, o);
#pragma unroll
                for (int x = 0; x < VEC; ++x) delta[g] = fmaf(go[g].get(x), o[x], delta[g]);
            }
            if (l.there) {  // in every lane of the head: slot_sum takes any of them
                lse[g] = a.lse[row + g];
                if (lse[g] == -inf_of()) lse[g] = inf_of();
                slope[g] = a.slopes[l.head + g];
            }
            delta[g] = head_sum<LPH>(delta[g]);
            if (l.mine && l.c == 0 && l.slot == 0) a.stat[row + g] = float2{lse[g], delta[g]};
#pragma unroll
            for (int x = 0; x < VEC; ++x) acc[g][x] = 0.f;
        }
        const char* k = (const char*)((const T*)a.k + l.kv * a.k_stride[1] + l.c);
        const char* v = (const char*)((const T*)a.v + l.kv * a.v_stride[1] + l.c);
        PairChunk chunk(a, run);
        // The slope's gradient is sum ds d, where ds sums to 0: what rounding leaves of
        // that sum, `over`, is taken out times the mean distance.
        const auto step = [&](int p0, int n, auto whole) {
            Raw<T, R> kx[kAhead], vx[kAhead];
            float d[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int p = p0 + u * l.slots + l.slot;
                const int j = __shfl(chunk.target, p);
                d[u] = __shfl(chunk.distance, p);
                kx[u] = Raw<T, R>::at(row_at<T>(k, j, k_row));
                vx[u] = Raw<T, R>::at(row_at<T>(v, j, v_row));
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int p = p0 + u * l.slots + l.slot;
                const bool in = whole || p < n;
                const int e = chunk.first + p;
                if (!whole && !in) kx[u] = Raw<T, R>{};
                float push = 0.f, s[GH], dp[GH], bend[GH];
#pragma unroll
                for (int g = 0; g < GH; ++g) {
                    s[g] = head_sum<LPH>(l.mine ? q[g].dot(kx[u], 0.f) : 0.f);
                    dp[g] = head_sum<LPH>(l.mine ? go[g].dot(vx[u], 0.f) : 0.f);
                }
                capped_few<CAP>(s, a.rule, bend);
#pragma unroll
                for (int g = 0; g < GH; ++g) {
                    s[g] = fmaf(-slope[g] * kLog2e, d[u], s[g]);
                    float w = exp2_of(s[g] - lse[g]), ds = w * (dp[g] - delta[g]);
                    if (!l.there || (!whole && !in)) w = ds = 0.f;
                    kx[u].add(CAP ? ds * bend[g] : ds, acc[g]);
                    turn[g] = fmaf(-ds, d[u], turn[g]);
                    over[g] += ds;
                    mean[g] = fmaf(w, d[u], mean[g]);
                    push = fmaf(-slope[g], ds, push);
                }
                push = slot_sum<LPH>(push, a.slot);
                if (in && l.in_slot == 0)
                    a.grad_distances[e] = first == 0 ? push : a.grad_distances[e] + push;
            }
        };
        for (; chunk.left > 0; chunk.next(a, run)) {
            const int n = min(chunk.left, kWave), stride = l.slots * kAhead;
            int p0 = 0;
            for (; p0 + stride <= n; p0 += stride) step(p0, n, std::true_type{});
            if (p0 < n) step(p0, n, std::false_type{});
        }
#pragma unroll
        for (int g = 0; g < GH; ++g) {
            turn[g] = join_lanes<sum_of>(turn[g], a.slot);
            over[g] = join_lanes<sum_of>(over[g], a.slot);
            mean[g] = join_lanes<sum_of>(mean[g], a.slot);
#pragma unroll
            for (int x = 0; x < VEC; ++x)
                acc[g][x] = join_lanes<sum_of>(acc[g][x], a.slot) * a.rule.scale;
            if (l.mine && l.slot == 0) {
                store_wide<T, VEC>((T*)a.grad_q + (row + g) * a.dim + l.c, acc[g]);
                if (l.c == 0)
                    a.turn[(int64_t)(l.head + g) * a.n_sources + i] =
                        fmaf(over[g], mean[g], turn[g]);
            }
        }
    }
}

// By targets: grad_k and grad_v.  grid: (targets / 4, blocks of key heads).  A
// unit here is a key head; its query heads are taken GH at a time.
template <typename T, int LPH, int GH, int R, bool CAP>
__global__ __launch_bounds__(256, kHeldBack) void k_neighbor_dkv(const NeighborArgs a) {
    constexpr int VEC = Raw<T, R>::kVec, kAhead = GH == 4 ? 1 : GH == 2 || R == 2 ? 2 : 4;
    const int64_t j = (int64_t)xcd_order(blockIdx.x, gridDim.x) * 4 + threadIdx.x / kWave;
    if (j >= a.n_targets) return;
    const int lane = lane_of(), slot = lane / a.slot, in_slot = lane % a.slot;
    const int slots = kWave / a.slot;
    int kv = blockIdx.y * (a.slot / LPH) + in_slot / LPH, c = (in_slot % LPH) * VEC;
    const bool mine = kv < a.kv_heads && c < a.dim;
    if (kv >= a.kv_heads) kv = 0;
    if (!mine) c = 0;
    const int64_t flat = (j * a.kv_heads + kv) * a.dim + c;
    float dk[VEC], dv[VEC];
    const bool valid = a.rows.head->holds(a.head);
#pragma unroll
    for (int x = 0; x < VEC; ++x) dk[x] = dv[x] = valid ? 0.f : nan_of();
    if (valid) {
        Raw<T, R> k{}, v{};
        if (mine) {
            k = Raw<T, R>::at((const char*)((const T*)a.k + j * a.k_stride[0] + kv * a.k_stride[1] + c));
            v = Raw<T, R>::at((const char*)((const T*)a.v + j * a.v_stride[0] + kv * a.v_stride[1] + c));
        }
        const int2 run = run_of(a.rows.targets, j);
        const uint32_t q_row = (uint32_t)(a.q_stride[0] * sizeof(T));
        const uint32_t q_head = (uint32_t)(a.q_stride[1] * sizeof(T));
        const uint32_t o_head = (uint32_t)(a.dim * sizeof(T)), o_row = a.heads * o_head;
        for (int g0 = 0; g0 < a.group; g0 += GH) {
            const int head = kv * a.group + g0;
            float slope2[GH];
#pragma unroll
            for (int g = 0; g < GH; ++g) slope2[g] = a.slopes[head + g] * kLog2e;
            const char* q = (const char*)((const T*)a.q + head * a.q_stride[1] + c);
            const char* go = (const char*)((const T*)a.grad_out + (int64_t)head * a.dim + c);
            const char* stat = (const char*)(a.stat + head);
            const uint32_t stat_row = a.heads * sizeof(float2);
            // 64 pairs of the target, one to a lane, and the next 64 on their way
            int2 pair{}, next_pair{};
            float distance = 0.f, next_distance = 0.f;
            const auto fetch = [&](int from) {
                if (from >= run.y) return;
                next_pair = a.rows.order[min(from + lane, run.y - 1)];
                next_distance = a.distances[next_pair.x];
            };
            fetch(run.x);
            for (int from = run.x; from < run.y; from += kWave) {
                pair = next_pair;
                distance = next_distance;
                fetch(from + kWave);
                const int n = min(run.y - from, kWave);
                const auto step = [&](int p0, auto whole) {
                    Raw<T, R> qx[kAhead][GH], ox[kAhead][GH];
                    float d[kAhead];
                    float2 st[kAhead][GH];
#pragma unroll
                    for (int u = 0; u < kAhead; ++u) {
                        const int p = p0 + u * slots + slot;
                        const int i = __shfl(pair.y, p);
                        d[u] = __shfl(distance, p);
                        const char* qi = row_at<T>(q, i, q_row);
                        const char* oi = row_at<T>(go, i, o_row);
                        const float2* si = (const float2*)row_at<T>(stat, i, stat_row);
#pragma unroll
                        for (int g = 0; g < GH; ++g) {
                            qx[u][g] = Raw<T, R>::at(qi + g * q_head);
                            ox[u][g] = Raw<T, R>::at(oi + g * o_head);
                            st[u][g] = si[g];
                        }
                    }
#pragma unroll
                    for (int u = 0; u < kAhead; ++u) {
                        const bool in = whole || p0 + u * slots + slot < n;
                        float s[GH], dp[GH], bend[GH];
#pragma unroll
                        for (int g = 0; g < GH; ++g) {
                            if (!whole && !in) qx[u][g] = ox[u][g] = Raw<T, R>{};
                            s[g] = head_sum<LPH>(mine ? qx[u][g].dot(k, 0.f) : 0.f);
                            dp[g] = head_sum<LPH>(mine ? ox[u][g].dot(v, 0.f) : 0.f);
                        }
                        capped_few<CAP>(s, a.rule, bend);
#pragma unroll
                        for (int g = 0; g < GH; ++g) {
                            float p = exp2_of(fmaf(-slope2[g], d[u], s[g]) - st[u][g].x);
                            if (!whole && !in) p = 0.f;
                            float dx = p * (dp[g] - st[u][g].y);
                            if (CAP) dx *= bend[g];
                            qx[u][g].add(dx, dk);
                            ox[u][g].add(p, dv);
                        }
                    }
                };
                const int stride = slots * kAhead;
                int p0 = 0;
                for (; p0 + stride <= n; p0 += stride) step(p0, std::true_type{});
                if (p0 < n) step(p0, std::false_type{});
            }
        }
#pragma unroll
        for (int x = 0; x < VEC; ++x) {
            dk[x] = join_lanes<sum_of>(dk[x], a.slot);
            dv[x] = join_lanes<sum_of>(dv[x], a.slot);
        }
    }
    if (!mine || slot != 0) return;
#pragma unroll
    for (int x = 0; x < VEC; ++x) dk[x] *= a.rule.scale;
    store_wide<T, VEC>((T*)a.grad_k + flat, dk);
    store_wide<T, VEC>((T*)a.grad_v + flat, dv);
}

}  // namespace op
}  // namespace tnr
