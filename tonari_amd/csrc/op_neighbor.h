// Attention along the pairs of a neighbor list: each source atom i over its
// pairs (i, j) at distance d, scores and gradients as in op_structure.h with
// the pair's d for r (its gradient is an output: the list's own backward takes
// it on to positions and cell).
//
// A source's keys lie anywhere, so the work is a gather of k and v rows (512
// bytes a pair for 128 channels of 16 bits) and a few operations on each value
// read: what bounds it is the rate at which the L2 and the memory behind it
// serve such rows.  One wave takes a source: lanes of 16 bytes make a head,
// heads make a slot, and the wave's slots take pairs side by side, each with
// its own running maximum and sum; the slots are joined at the source's end.
//
// Backward: by sources (grad_q, and grad_d, which needs the sum over heads of
// one pair), then by targets in the list's transposed order (grad_k, grad_v),
// both recomputing the weights from the forward's row statistics: no atomics,
// so the sums' order is the list's.
#pragma once

#include "op_sort.h"

namespace tnr {
namespace op {

// What tnr_neighbor_rows writes, in this order (each part 256-byte aligned).
struct NeighborRows {
    int32_t* status;   // not 0: the list is not valid (every result is NaN)
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
    r.status = (int32_t*)part(4);
    r.sources = (int2*)part((size_t)sources * 8);
    if (transpose) r.targets = (int2*)part((size_t)targets * 8);
    r.target = (int32_t*)part((size_t)pairs * 4);
    if (transpose) r.order = (int2*)part((size_t)pairs * 8);
    r.bytes = at;
    return r;
}

// status and the runs are cleared before.  A source whose pairs do not lie
// together finds its run taken.
__global__ __launch_bounds__(256) void k_neighbor_rows(const int64_t* sources,
                                                       const int64_t* targets, int64_t n_pairs,
                                                       int64_t n_sources, int64_t n_targets,
                                                       NeighborRows r) {
    int bad = 0;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n_pairs;
         e += (int64_t)gridDim.x * 256) {
        const int64_t i = sources[e], j = targets[e];
        const bool in = i >= 0 && i < n_sources && j >= 0 && j < n_targets;
        bad |= !in;
        r.target[e] = in ? (int32_t)j : 0;
        if (!in) continue;
        if (e == 0 || sources[e - 1] != i)
            bad |= atomicExch(&r.sources[i].x, (int)e + 1) != 0;  // 0: none yet
        if (e + 1 == n_pairs || sources[e + 1] != i) r.sources[i].y = (int)e + 1;
    }
    if (__builtin_amdgcn_ballot_w64(bad != 0) != 0 && lane_of() == 0) atomicOr(r.status, 1);
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
    float* delta;  // [n_sources][heads]
    float* turn;   // [heads][n_sources]
};

template <typename T>
constexpr int kVec = 16 / sizeof(T);

template <int CTRL>
__device__ __forceinline__ float dpp_of(float x) {
    return __int_as_float(
        __builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, false));
}

// Sum over the LPH lanes of a head, in all of them.
template <int LPH>
__device__ __forceinline__ float head_sum(float x) {
    if constexpr (LPH >= 2) x += dpp_of<0xb1>(x);   // lane ^ 1
    if constexpr (LPH >= 4) x += dpp_of<0x4e>(x);   // lane ^ 2
    if constexpr (LPH >= 8) x += dpp_of<0x141>(x);  // mirrored in 8
    if constexpr (LPH >= 16) x += dpp_of<0x140>(x); // mirrored in 16
    if constexpr (LPH >= 32) x += __shfl_xor(x, 16);
    return x;
}

// u log2(e) of one product, and tanh where there is a cap.
__device__ __forceinline__ float capped_one(float dot, const ScoreRule& rule, float& t) {
    t = 0.f;
    if (rule.cap > 0.f) {
        t = tanh_of(dot * rule.inv);
        return t * rule.cap2;
    }
    return dot * rule.scale2;
}

template <typename T>
__device__ __forceinline__ void fill_nan(T* p, int64_t n, int64_t from, int64_t step) {
    for (int64_t i = from; i < n; i += step) p[i] = rounded<T>(nan_of());
}

// grid: (sources / 4, head blocks).
template <typename T, int LPH>
__global__ __launch_bounds__(256) void k_neighbor_forward(const NeighborArgs a) {
    constexpr int VEC = kVec<T>, kAhead = 4;
    const int64_t i = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
    if (i >= a.n_sources) return;
    const int lane = lane_of(), slot = lane / a.slot, in_slot = lane % a.slot;
    const int head = blockIdx.y * (a.slot / LPH) + in_slot / LPH;
    const int c = (in_slot % LPH) * VEC;
    const bool mine = head < a.heads && c < a.dim;
    const int slots = kWave / a.slot;
    T* out = (T*)a.out + (i * a.heads + head) * a.dim + c;
    const int64_t row = i * a.heads + head;
    float acc[VEC];
#pragma unroll
    for (int x = 0; x < VEC; ++x) acc[x] = 0.f;
    float top = -inf_of(), sum = 0.f;
    const bool valid = *a.rows.status == 0;
    if (valid) {
        float q[VEC] = {};
        if (mine)
            load_floats<T, VEC>((const T*)a.q + i * a.q_stride[0] + head * a.q_stride[1] + c, q);
        const float slope2 = mine ? a.slopes[head] * kLog2e : 0.f;
        const int kv = mine ? head / a.group : 0;
        const T* k = (const T*)a.k + kv * a.k_stride[1] + (mine ? c : 0);
        const T* v = (const T*)a.v + kv * a.v_stride[1] + (mine ? c : 0);
        const int2 run = run_of(a.rows.sources, i);
        for (int e0 = run.x; e0 < run.y; e0 += slots * kAhead) {
            float kx[kAhead][VEC], vx[kAhead][VEC], d[kAhead], s[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int e = min(e0 + u * slots + slot, run.y - 1);
                const int64_t j = a.rows.target[e];
                d[u] = a.distances[e];
                load_floats<T, VEC>(k + j * a.k_stride[0], kx[u]);
                load_floats<T, VEC>(v + j * a.v_stride[0], vx[u]);
            }
            float high = top;
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                float dot = 0.f, t;
#pragma unroll
                for (int x = 0; x < VEC; ++x) dot = fmaf(q[x], kx[u][x], dot);
                dot = head_sum<LPH>(mine ? dot : 0.f);
                s[u] = fmaf(-slope2, d[u], capped_one(dot, a.rule, t));
                if (e0 + u * slots + slot >= run.y) s[u] = -inf_of();
                high = fmaxf(high, s[u]);
            }
            const float ref = high == -inf_of() ? 0.f : high;
            const float fade = exp2_of(top - ref);
            top = high;
            sum *= fade;
#pragma unroll
            for (int x = 0; x < VEC; ++x) acc[x] *= fade;
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                // a pair beyond the run's end repeats its last one, with weight 0
                const bool in = e0 + u * slots + slot < run.y;
                const float p = in ? exp2_of(s[u] - ref) : 0.f;
                sum += p;
#pragma unroll
                for (int x = 0; x < VEC; ++x) acc[x] = fmaf(p, in ? vx[u][x] : 0.f, acc[x]);
            }
        }
        for (int d = a.slot; d < kWave; d <<= 1) {
            const float other = __shfl_xor(top, d), high = fmaxf(top, other);
            const float ref = high == -inf_of() ? 0.f : high;
            const float w = exp2_of(top - ref), z = exp2_of(other - ref);
            sum = sum * w + __shfl_xor(sum, d) * z;
#pragma unroll
            for (int x = 0; x < VEC; ++x) acc[x] = acc[x] * w + __shfl_xor(acc[x], d) * z;
            top = high;
        }
    }
    if (!mine || slot != 0) return;
    const float by = !valid ? nan_of() : sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int x = 0; x < VEC; ++x) acc[x] = valid ? acc[x] * by : nan_of();
    store_floats<T, VEC>(out, acc);
    if (a.out32) store_floats<float, VEC>(a.out32 + row * a.dim + c, acc);
    if (a.lse && c == 0)
        a.lse[row] = !valid ? nan_of() : sum == 0.f ? -inf_of() : top + __builtin_amdgcn_logf(sum);
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

// By sources: grad_q, grad_d, delta and the slopes' gradient by rows.  Blocks of
// heads that do not fit a wave follow one another in it, so that a pair's
// grad_d is summed by one lane.
template <typename T, int LPH>
__global__ __launch_bounds__(256) void k_neighbor_dq(const NeighborArgs a) {
    constexpr int VEC = kVec<T>, kAhead = 4;
    const int64_t i = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
    if (i >= a.n_sources) return;
    const int lane = lane_of(), slot = lane / a.slot, in_slot = lane % a.slot;
    const int slots = kWave / a.slot, block = a.slot / LPH;
    const int c = (in_slot % LPH) * VEC;
    if (*a.rows.status != 0) {
        fill_nan((T*)a.grad_q + i * a.heads * a.dim, (int64_t)a.heads * a.dim, lane, kWave);
        fill_nan(a.grad_distances, a.n_pairs, i * kWave + lane, (int64_t)a.n_sources * kWave);
        for (int h = lane; h < a.heads; h += kWave) a.turn[(int64_t)h * a.n_sources + i] = nan_of();
        return;
    }
    const int2 run = run_of(a.rows.sources, i);
    for (int h0 = 0; h0 < a.heads; h0 += block) {
        const int head = h0 + in_slot / LPH;
        const bool mine = head < a.heads && c < a.dim;
        const int64_t row = i * a.heads + head;
        float q[VEC] = {}, go[VEC] = {}, acc[VEC];
        float delta = 0.f, turn = 0.f, lse = inf_of(), slope = 0.f;
        if (mine) {
            float o[VEC];
            load_floats<T, VEC>((const T*)a.q + i * a.q_stride[0] + head * a.q_stride[1] + c, q);
            load_floats<T, VEC>((const T*)a.grad_out + row * a.dim + c, go);
            load_wide<VEC>(a.out_full + row * a.dim + c, o);
#pragma unroll
            for (int x = 0; x < VEC; ++x) delta = fmaf(go[x], o[x], delta);
            lse = a.lse[row];
            if (lse == -inf_of()) lse = inf_of();
            slope = a.slopes[head];
        }
        delta = head_sum<LPH>(delta);
        // every lane of a head that is there holds its lse and slope
        const float slope2 = slope * kLog2e;
        if (mine && c == 0 && slot == 0) a.delta[row] = delta;
#pragma unroll
        for (int x = 0; x < VEC; ++x) acc[x] = 0.f;
        const int kv = mine ? head / a.group : 0;
        const T* k = (const T*)a.k + kv * a.k_stride[1] + (mine ? c : 0);
        const T* v = (const T*)a.v + kv * a.v_stride[1] + (mine ? c : 0);
        for (int e0 = run.x; e0 < run.y; e0 += slots * kAhead) {
            float kx[kAhead][VEC], vx[kAhead][VEC], d[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int e = min(e0 + u * slots + slot, run.y - 1);
                const int64_t j = a.rows.target[e];
                d[u] = a.distances[e];
                load_floats<T, VEC>(k + j * a.k_stride[0], kx[u]);
                load_floats<T, VEC>(v + j * a.v_stride[0], vx[u]);
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int e = e0 + u * slots + slot;
                const bool in = e < run.y;
                float dot = 0.f, dp = 0.f, t;
#pragma unroll
                for (int x = 0; x < VEC; ++x) {
                    dot = fmaf(q[x], kx[u][x], dot);
                    dp = fmaf(go[x], vx[u][x], dp);
                }
                dot = head_sum<LPH>(mine ? dot : 0.f);
                dp = head_sum<LPH>(mine ? dp : 0.f);
                const float s = fmaf(-slope2, d[u], capped_one(dot, a.rule, t));
                // (only lanes of the head's channels know its lse)
                const float ds = in && mine ? exp2_of(s - lse) * (dp - delta) : 0.f;
                const float dx = ds * fmaf(-t, t, 1.f);
#pragma unroll
                for (int x = 0; x < VEC; ++x) acc[x] = fmaf(dx, in ? kx[u][x] : 0.f, acc[x]);
                turn = fmaf(-ds, in ? d[u] : 0.f, turn);
                float push = -slope * ds;
                for (int w = LPH; w < a.slot; w <<= 1) push += __shfl_xor(push, w);
                if (in && in_slot == 0)
                    a.grad_distances[e] = h0 == 0 ? push : a.grad_distances[e] + push;
            }
        }
        for (int d = a.slot; d < kWave; d <<= 1) {
            turn += __shfl_xor(turn, d);
#pragma unroll
            for (int x = 0; x < VEC; ++x) acc[x] += __shfl_xor(acc[x], d);
        }
        if (mine && slot == 0) {
#pragma unroll
            for (int x = 0; x < VEC; ++x) acc[x] *= a.rule.scale;
            store_floats<T, VEC>((T*)a.grad_q + row * a.dim + c, acc);
            if (c == 0) a.turn[(int64_t)head * a.n_sources + i] = turn;
        }
    }
}

// By targets: grad_k and grad_v.  grid: (targets / 4, blocks of key heads).
template <typename T, int LPH>
__global__ __launch_bounds__(256) void k_neighbor_dkv(const NeighborArgs a) {
    constexpr int VEC = kVec<T>, kAhead = 2;
    const int64_t j = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
    if (j >= a.n_targets) return;
    const int lane = lane_of(), slot = lane / a.slot, in_slot = lane % a.slot;
    const int kv = blockIdx.y * (a.slot / LPH) + in_slot / LPH;
    const int c = (in_slot % LPH) * VEC;
    const bool mine = kv < a.kv_heads && c < a.dim;
    const int slots = kWave / a.slot;
    const int64_t flat = (j * a.kv_heads + kv) * a.dim + c;
    float dk[VEC], dv[VEC];
    const bool valid = *a.rows.status == 0;
#pragma unroll
    for (int x = 0; x < VEC; ++x) dk[x] = dv[x] = valid ? 0.f : nan_of();
    if (valid) {
        float k[VEC] = {}, v[VEC] = {};
        if (mine) {
            load_floats<T, VEC>((const T*)a.k + j * a.k_stride[0] + kv * a.k_stride[1] + c, k);
            load_floats<T, VEC>((const T*)a.v + j * a.v_stride[0] + kv * a.v_stride[1] + c, v);
        }
        const int2 run = run_of(a.rows.targets, j);
        for (int g = 0; g < a.group; ++g) {
            const int head = mine ? kv * a.group + g : 0;
            const float slope2 = a.slopes[head] * kLog2e;
            const T* q = (const T*)a.q + head * a.q_stride[1] + (mine ? c : 0);
            const T* go = (const T*)a.grad_out + (int64_t)head * a.dim + (mine ? c : 0);
            for (int p0 = run.x; p0 < run.y; p0 += slots * kAhead) {
                float qx[kAhead][VEC], ox[kAhead][VEC], d[kAhead], lse[kAhead], delta[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    const int2 at = a.rows.order[min(p0 + u * slots + slot, run.y - 1)];
                    const int64_t i = at.y;
                    d[u] = a.distances[at.x];
                    load_floats<T, VEC>(q + i * a.q_stride[0], qx[u]);
                    load_floats<T, VEC>(go + i * a.heads * a.dim, ox[u]);
                    lse[u] = a.lse[i * a.heads + head];
                    delta[u] = a.delta[i * a.heads + head];
                }
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    const bool in = p0 + u * slots + slot < run.y;
                    float dot = 0.f, dp = 0.f, t;
#pragma unroll
                    for (int x = 0; x < VEC; ++x) {
                        dot = fmaf(qx[u][x], k[x], dot);
                        dp = fmaf(ox[u][x], v[x], dp);
                    }
                    dot = head_sum<LPH>(mine ? dot : 0.f);
                    dp = head_sum<LPH>(mine ? dp : 0.f);
                    const float s = fmaf(-slope2, d[u], capped_one(dot, a.rule, t));
                    const bool any = in && lse[u] != -inf_of();
                    const float p = any ? exp2_of(s - lse[u]) : 0.f;
                    const float dx = any ? p * (dp - delta[u]) * fmaf(-t, t, 1.f) : 0.f;
#pragma unroll
                    for (int x = 0; x < VEC; ++x) {
                        dk[x] = fmaf(dx, in ? qx[u][x] : 0.f, dk[x]);
                        dv[x] = fmaf(p, in ? ox[u][x] : 0.f, dv[x]);
                    }
                }
            }
        }
        for (int d = a.slot; d < kWave; d <<= 1)
#pragma unroll
            for (int x = 0; x < VEC; ++x) {
                dk[x] += __shfl_xor(dk[x], d);
                dv[x] += __shfl_xor(dv[x], d);
            }
    }
    if (!mine || slot != 0) return;
#pragma unroll
    for (int x = 0; x < VEC; ++x) dk[x] *= a.rule.scale;
    store_floats<T, VEC>((T*)a.grad_k + flat, dk);
    store_floats<T, VEC>((T*)a.grad_v + flat, dv);
}

// A head's slope: the sum of its rows, one workgroup each.
__global__ __launch_bounds__(256) void k_neighbor_slopes(const float* turn, int64_t rows,
                                                         float* grad_slopes) {
    __shared__ float waves[4];
    const float* from = turn + (int64_t)blockIdx.x * rows;
    float sum = 0.f;
    for (int64_t i = threadIdx.x; i < rows; i += 256) sum += from[i];
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    if (lane_of() == 0) waves[threadIdx.x / kWave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) grad_slopes[blockIdx.x] = waves[0] + waves[1] + waves[2] + waves[3];
}

}  // namespace op
}  // namespace tnr
