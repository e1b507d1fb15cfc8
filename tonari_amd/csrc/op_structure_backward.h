// The gradients of structure attention (op_structure.h has the formulas), in
// two passes that both recompute a tile's weights from the forward's row
// statistics: by queries (grad_q, and for every row delta, its own share of
// the positions' gradient and the slope's) and by keys (grad_k, grad_v and the
// keys' share of the positions' gradient).  Neither needs an atomic, so the
// sums' order is fixed by the sizes.
//
// delta = do.o is taken from the forward's output in 32 bits.  The rounding of a
// 16-bit output, times sum p k, would show in grad_q where keys have a component
// in common: 200 keys of mean 3, bfloat16, 32 channels, a tenth of it.  What is
// left, e = sum p (dp - do.o) of the weights' own rounding, is summed by the
// queries' pass and taken out of the gradients of positions and slopes, which are
// 32-bit: sum p (dp - delta) f = sum p (dp - do.o) f - e sum p f.
//
// Both recompute a tile's scores, which costs seven products of matrices in place
// of five but needs no sums across workgroups.  As the forward they are bound by
// vector instructions: 4,001 atoms, 8 capped heads of 64 on 2, bfloat16: 222 us by
// queries (751 instructions a tile, 16 of them matrix products) and 247 by keys (701,
// 24), at two waves to a SIMD, whose accumulators and rows fill its registers.
//
// 16-bit types: dx and p go through two products, rounded and rest, so that each
// gradient is rounded once, at the end.
//
// float16: dx is scaled by a power of two that follows the largest |dx| that a
// row (or, in the keys' pass, a key) has met so far, to below 2^14, and p by 2^12, so
// that neither large values nor small upstream gradients nor the small weights
// of long rows fall out of the type's range.  bfloat16 has the range of 32 bits.
#pragma once

#include "op_structure.h"

namespace tnr {
namespace op {

// Sums of a query row besides grad_q: e, sum (ds u, p u) for the unit vectors
// u, sum (ds r, p r).
constexpr int kRowSums = 9;

__device__ __forceinline__ float power_of(int e) { return __builtin_amdgcn_ldexpf(1.f, e); }

// The scale of a lane's dx: 2^kMost / 2^e, where 2^e is above all of them so far.
struct Unit {
    static constexpr int kMost = 14;
    int e = -100;
    __device__ __forceinline__ float by() const { return power_of(kMost - e); }
    __device__ __forceinline__ float back() const { return power_of(e - kMost); }
    // Takes the 16 of a tile; sums of earlier ones change their unit with it.
    template <int N>
    __device__ __forceinline__ void meet(const f32x16& dx, f32x16 (&sums)[N]) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(dx[i]));
        top = max_halves(top);
        const int next = top > 0.f && top < inf_of() ? __builtin_amdgcn_frexp_expf(top) : e;
        if (next <= e) return;
        const float fade = power_of(e - next);
#pragma unroll
        for (int d = 0; d < N; ++d) sums[d] *= fade;
        e = next;
    }
};

// What a row's sums make, for its own lane.
__device__ __forceinline__ void finish_row(const StructureArgs& a, int head, int query,
                                           float delta, float slope,
                                           const float (&w)[kRowSums]) {
    const int64_t at = (int64_t)head * a.n_queries + query;
    a.row[at] = delta + w[0];
    if (a.push_q)
        for (int c = 0; c < 3; ++c) a.push_q[3 * at + c] = -slope * (w[1 + c] - w[0] * w[4 + c]);
    if (a.turn) a.turn[at] = -(w[7] - w[0] * w[8]);
}

// grid: (query tiles * kv_heads, splits).
template <typename T, int DP, int NW, bool CAP>
__global__ __launch_bounds__(NW* kWave, waves_held<T>(DP <= 32 ? 64 : 2 * DP)) void k_structure_dq(
    const StructureArgs a) {
    using M = Mat<T>;
    using Row = typename M::template Row<DP>;
    using Pair = StagePair<T, DP, NW>;
    constexpr int kTiles = Pair::kTiles, kKeys = kTiles * kTile;
    __shared__ alignas(16) T k_rows[kTiles * Pair::kRows];
    __shared__ alignas(16) T k_cols[M::kSeparateCols ? kTiles * Pair::kCols : 8];
    __shared__ alignas(16) T v_rows[kTiles * Pair::kRows];
    __shared__ TilePositions<kTiles> x_k;

    const uint32_t order = xcd_order(blockIdx.x, gridDim.x), block = order / (uint32_t)a.kv_heads;
    const StructureTile t = a.q_tiles[block];
    const int lane = lane_of(), half = lane / 32, wave = threadIdx.x / kWave;
    const int kv = (int)(order - block * a.kv_heads), split = blockIdx.y;
    const int g = a.group;
    if (t.n_q < 0) {
        const int64_t row = (int64_t)block * (NW * kTile) + wave * kTile + lane % 32;
        if (row >= (int64_t)a.n_queries * g || half) return;
        const int query = (int)(row / g), head = kv * g + (int)(row % g);
        const int64_t at = (int64_t)head * a.n_queries + query;
        if (a.splits > 1) {
            float* part = a.part + ((int64_t)split * a.heads * a.n_queries + at) * (a.dim + kRowSums);
            for (int c = 0; c < a.dim + kRowSums; ++c) part[c] = nan_of();
            if (split == 0) a.row[at] = nan_of();
            return;
        }
        T* dq = (T*)a.grad_q + ((int64_t)query * a.heads + head) * a.dim;
        for (int c = 0; c < a.dim; ++c) dq[c] = rounded<T>(nan_of());
        const float w[kRowSums] = {nan_of()};
        finish_row(a, head, query, 0.f, 1.f, w);
        return;
    }
    const int rows = t.n_q * g;
    if (t.first >= rows) return;

    const int row = t.first + wave * kTile + lane % 32;
    const bool valid = row < rows;
    const bool busy = t.first + wave * kTile < rows;  // a wave without rows only helps to stage
    // (a division costs as much as a short row's tile does)
    const int nth = !valid ? 0 : g == 1 ? row : (int)((uint32_t)row / (uint32_t)g);
    const int query = t.q_lo + nth, head = kv * g + (valid ? row - nth * g : 0);
    const int64_t at = (int64_t)head * a.n_queries + query;
    const int64_t flat = ((int64_t)query * a.heads + head) * a.dim;
    Row qr, dor;
    qr.load(valid ? (const T*)a.q + (int64_t)query * a.q_stride[0] + head * a.q_stride[1] : nullptr,
            a.dim);
    dor.load(valid ? (const T*)a.grad_out + flat : nullptr, a.dim);
    const float* full = sizeof(T) == 4 ? (const float*)a.out : a.out32;
    const float delta = dor.dot32(valid ? full + flat : nullptr, a.dim);
    Unit unit;
    float xq = 0.f, yq = 0.f, zq = 0.f, slope = 0.f, lse = inf_of();
    if (valid) {
        xq = a.x_q[3 * (int64_t)query];
        yq = a.x_q[3 * (int64_t)query + 1];
        zq = a.x_q[3 * (int64_t)query + 2];
        slope = a.slopes[head];
        lse = a.lse[at];
        if (lse == -inf_of()) lse = inf_of();  // no weight anywhere
    }
    const float slope2 = slope * kLog2e;
    const bool geometry = a.push_q != nullptr || a.push_k != nullptr || a.turn != nullptr;
    const T* kb = (const T*)a.k + (int64_t)t.k_lo * a.k_stride[0] + kv * a.k_stride[1];
    const T* vb = (const T*)a.v + (int64_t)t.k_lo * a.v_stride[0] + kv * a.v_stride[1];
    const float* xb = a.x_k + 3 * (int64_t)t.k_lo;

    const int tiles = (t.n_k + kTile - 1) / kTile;
    const int each = (tiles + a.splits - 1) / a.splits;
    const int from = min(tiles, split * each), to = min(tiles, from + each);

    f32x16 acc[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) acc[d] = f32x16{};
    float w[kRowSums];
#pragma unroll
    for (int i = 0; i < kRowSums; ++i) w[i] = 0.f;

    Pair stage;
    float xs[3];
    const auto fetch = [&](int tile) {
        const int k0 = tile * kTile, n = min(t.n_k, to * kTile) - k0;
        stage.fetch(kb + (int64_t)k0 * a.k_stride[0], (int)a.k_stride[0],
                   vb + (int64_t)k0 * a.v_stride[0], (int)a.v_stride[0], n, a.dim);
        if (threadIdx.x < kKeys) {
            const float* p = xb + 3 * (int64_t)(k0 + min((int)threadIdx.x, n - 1));
#pragma unroll
            for (int c = 0; c < 3; ++c) xs[c] = p[c];
        }
    };
    const auto place = [&] {
        __syncthreads();
        stage.place(k_rows, M::kSeparateCols ? k_cols : nullptr, v_rows, nullptr);
        if (threadIdx.x < kKeys)
#pragma unroll
            for (int c = 0; c < 3; ++c) x_k.x[c][threadIdx.x] = xs[c];
        __syncthreads();
    };
    const auto push = [&](int sub, int left) {
        f32x16 dot{}, dp{};
        M::template rows<DP>(dot, k_rows + sub * Pair::kRows, qr, a.dim);
        M::template rows<DP>(dp, v_rows + sub * Pair::kRows, dor, a.dim);
        typename M::Weights p, rest;
        const bool near = all_near<CAP>(dot, a.rule);
        // the tile's own sums: a long row's are then sums of few terms each
        float tw[kRowSums] = {};
#pragma unroll
        for (int run = 0; run < 4; ++run) {
            const int first = sub * kTile;
            const Vec<float, 4> x = four_of(x_k.x[0] + first, run, half),
                                y = four_of(x_k.x[1] + first, run, half),
                                z = four_of(x_k.x[2] + first, run, half);
            float dx[4], dy[4], dz[4], r[4], s[4], u[4], bend[4];
            capped<CAP>(dot, run, a.rule, near, u, bend);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                dx[e] = xq - x[e];
                dy[e] = yq - y[e];
                dz[e] = zq - z[e];
                r[e] = __builtin_amdgcn_sqrtf(
                    fmaf(dx[e], dx[e], fmaf(dy[e], dy[e], dz[e] * dz[e])));
                s[e] = exp2_of(fmaf(-slope2, r[e], u[e]) - lse);
            }
            if (left < kTile) {
                asm volatile("");  // a branch: only a structure's last tile pays for the selects
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (8 * run + e >= left - 4 * half) s[e] = 0.f;
            }
            float ds[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 4 * run + e;
                ds[e] = s[e] * (dp[i] - delta);
                tw[0] += ds[e];
                const float dx_i = CAP ? ds[e] * bend[e] : ds[e];
                if constexpr (kNarrow<T>) {
                    dot[i] = dx_i;  // (its product is done with)
                } else {
                    p.set(i, dx_i);
                    if (sizeof(T) == 2) rest.set(i, dx_i - p.get(i));
                }
            }
            if (geometry) {
                asm volatile("");  // one branch for the run
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float over = r[e] > 0.f ? __builtin_amdgcn_rcpf(r[e]) : 0.f;
                    const float wd = ds[e] * over, wp = s[e] * over;
                    tw[1] = fmaf(wd, dx[e], tw[1]);
                    tw[2] = fmaf(wd, dy[e], tw[2]);
                    tw[3] = fmaf(wd, dz[e], tw[3]);
                    tw[4] = fmaf(wp, dx[e], tw[4]);
                    tw[5] = fmaf(wp, dy[e], tw[5]);
                    tw[6] = fmaf(wp, dz[e], tw[6]);
                    tw[7] = fmaf(ds[e], r[e], tw[7]);
                    tw[8] = fmaf(s[e], r[e], tw[8]);
                }
            }
            __builtin_amdgcn_sched_barrier(kLoadsPass);
        }
#pragma unroll
        for (int i = 0; i < kRowSums; ++i) w[i] += tw[i];
        if constexpr (kNarrow<T>) {
            unit.meet(dot, acc);
            const float by = unit.by();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                p.set(i, dot[i] * by);
                rest.set(i, dot[i] * by - p.get(i));
            }
        }
        // Their sum over a row is 0, so grad_q is a difference: what the rounding of
        // dx leaves out goes through a second product.
        const T* cols = M::kSeparateCols ? k_cols + sub * Pair::kCols : k_rows + sub * Pair::kRows;
        M::template cols<DP>(acc, cols, p);
        if constexpr (sizeof(T) == 2) M::template cols<DP>(acc, cols, rest);
    };
    if (from < to) fetch(from);
    for (int tile = from; tile < to; tile += kTiles) {
        place();
        if (tile + kTiles < to) fetch(tile + kTiles);
        if (busy)
            for (int sub = 0; sub < min(kTiles, to - tile); ++sub)
                push(sub, t.n_k - (tile + sub) * kTile);
    }
#pragma unroll
    for (int i = 0; i < kRowSums; ++i) w[i] = sum_halves(w[i]);
    if (!valid) return;
    if (a.splits > 1) {
        float* part = a.part + ((int64_t)split * a.heads * a.n_queries + at) * (a.dim + kRowSums);
        const float by = kNarrow<T> ? unit.back() : 1.f;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int c = 32 * d + row_of(i, half);
                if (c < a.dim) part[c] = acc[d][i] * by;
            }
        if (half == 0) {
#pragma unroll
            for (int i = 0; i < kRowSums; ++i) part[a.dim + i] = w[i];
            if (split == 0) a.row[at] = delta;
        }
        return;
    }
    store_channels<T, DP>((T*)a.grad_q + flat, a.dim, acc,
                          kNarrow<T> ? a.rule.scale * unit.back() : a.rule.scale);
    if (half == 0) finish_row(a, head, query, delta, slope, w);
}

// Joins the splits of a row of the queries' pass: one wave each.  (The first
// split has put the row's delta down.)
template <typename T>
__global__ __launch_bounds__(256) void k_structure_join_dq(const StructureArgs a) {
    const int64_t at = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
    const int64_t rows = (int64_t)a.heads * a.n_queries;
    if (at >= rows) return;
    const int lane = lane_of();
    const int head = (int)(at / a.n_queries), query = (int)(at % a.n_queries);
    const int64_t flat = ((int64_t)query * a.heads + head) * a.dim;
    const int64_t step = rows * (a.dim + kRowSums);
    const float* part = a.part + at * (a.dim + kRowSums);
    float x0 = 0.f, x1 = 0.f, w[kRowSums] = {};
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
        const float* p = part + s * step;
        if (lane < a.dim) x0 += p[lane];
        if (lane + kWave < a.dim) x1 += p[lane + kWave];
        for (int i = 0; i < kRowSums; ++i) w[i] += p[a.dim + i];
    }
    T* dq = (T*)a.grad_q + flat;
    if (lane < a.dim) dq[lane] = rounded<T>(x0 * a.rule.scale);
    if (lane + kWave < a.dim) dq[lane + kWave] = rounded<T>(x1 * a.rule.scale);
    if (lane == 0) finish_row(a, head, query, a.row[at], a.slopes[head], w);
}

// grid: (key tiles * kv_heads, k_splits); NW waves of 32 keys each.
template <typename T, int DP, int NW, bool CAP>
__global__ __launch_bounds__(NW* kWave, DP > 64 ? 1 : DP > 32 || CAP || sizeof(T) == 4 ? 2 : 3) void
k_structure_dkv(const StructureArgs a) {
    using M = Mat<T>;
    using Row = typename M::template Row<DP>;
    constexpr float kLift = kNarrow<T> ? 12.f : 0.f;
    constexpr float kLower = kNarrow<T> ? 1.f / 4096.f : 1.f;
    using Pair = StagePair<T, DP, NW>;
    constexpr int kTiles = Pair::kTiles, kQueries = kTiles * kTile;
    __shared__ alignas(16) T q_rows[kTiles * Pair::kRows];
    __shared__ alignas(16) T o_rows[kTiles * Pair::kRows];
    __shared__ alignas(16) T q_cols[M::kSeparateCols ? kTiles * Pair::kCols : 8];
    __shared__ alignas(16) T o_cols[M::kSeparateCols ? kTiles * Pair::kCols : 8];
    __shared__ TilePositions<kTiles> x_q;
    __shared__ alignas(16) float stat[2][kQueries];  // log-sum, delta

    const uint32_t order = xcd_order(blockIdx.x, gridDim.x), block = order / (uint32_t)a.kv_heads;
    const StructureTile t = a.k_tiles[block];
    const int lane = lane_of(), half = lane / 32, wave = threadIdx.x / kWave;
    const int kv = (int)(order - block * a.kv_heads), split = blockIdx.y;
    if (t.n_q < 0) {
        const int64_t key = (int64_t)block * (NW * kTile) + wave * kTile + lane % 32;
        if (key >= a.n_keys || half) return;
        if (a.k_splits > 1) {
            float* part = a.part_k + (((int64_t)split * a.kv_heads + kv) * a.n_keys + key) *
                                         (2 * a.dim + 3);
            for (int c = 0; c < 2 * a.dim + 3; ++c) part[c] = nan_of();
            return;
        }
        for (int c = 0; c < a.dim; ++c) {
            ((T*)a.grad_k)[(key * a.kv_heads + kv) * a.dim + c] = rounded<T>(nan_of());
            ((T*)a.grad_v)[(key * a.kv_heads + kv) * a.dim + c] = rounded<T>(nan_of());
        }
        if (a.push_k)
            for (int c = 0; c < 3; ++c)
                a.push_k[3 * ((int64_t)kv * a.n_keys + key) + c] = nan_of();
        return;
    }
    if (t.first >= t.n_k) return;
    const int place = t.first + wave * kTile + lane % 32;
    const bool valid = place < t.n_k;
    const int64_t key = t.k_lo + (valid ? place : 0);
    Row kr, vr;
    kr.load(valid ? (const T*)a.k + key * a.k_stride[0] + kv * a.k_stride[1] : nullptr, a.dim);
    vr.load(valid ? (const T*)a.v + key * a.v_stride[0] + kv * a.v_stride[1] : nullptr, a.dim);
    const float xk = valid ? a.x_k[3 * key] : 0.f, yk = valid ? a.x_k[3 * key + 1] : 0.f,
                zk = valid ? a.x_k[3 * key + 2] : 0.f;

    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) dk[d] = dv[d] = f32x16{};
    float px = 0.f, py = 0.f, pz = 0.f;
    Unit unit;  // what dk is held in

    // stages of kTiles tiles, of one head after the other
    const int per_head = (t.n_q + kQueries - 1) / kQueries, stages = per_head * a.group;
    Pair stage;
    float xs[3], ss[2];
    const auto fetch = [&](int at_stage) {
        const int head = kv * a.group + at_stage / per_head;
        const int q0 = (at_stage % per_head) * kQueries, n = t.n_q - q0;
        const int64_t first = t.q_lo + q0;
        stage.fetch((const T*)a.q + first * a.q_stride[0] + head * a.q_stride[1], (int)a.q_stride[0],
                    (const T*)a.grad_out + (first * a.heads + head) * a.dim, a.heads * a.dim, n,
                    a.dim);
        if (threadIdx.x < kQueries) {
            const bool in = (int)threadIdx.x < n;
            const int64_t query = first + (in ? threadIdx.x : 0);
            const int64_t at = (int64_t)head * a.n_queries + query;
#pragma unroll
            for (int c = 0; c < 3; ++c) xs[c] = a.x_q[3 * query + c];
            ss[0] = in ? a.lse[at] : inf_of();  // no weight beyond the rows
            if (ss[0] == -inf_of()) ss[0] = inf_of();
            ss[0] -= kLift;
            ss[1] = a.row[at];
        }
    };
    const auto pull = [&](int sub, float slope) {
        const float slope2 = slope * kLog2e;
        f32x16 dot{}, dp{};
        M::template rows<DP>(dot, q_rows + sub * Pair::kRows, kr, a.dim);
        M::template rows<DP>(dp, o_rows + sub * Pair::kRows, vr, a.dim);
        typename M::Weights p, p_rest, dx, dx_rest;
        const bool near = all_near<CAP>(dot, a.rule);
        float ux = 0.f, uy = 0.f, uz = 0.f;
#pragma unroll
        for (int run = 0; run < 4; ++run) {
            const int first = sub * kTile;
            const Vec<float, 4> x = four_of(x_q.x[0] + first, run, half),
                                y = four_of(x_q.x[1] + first, run, half),
                                z = four_of(x_q.x[2] + first, run, half),
                                lse = four_of(stat[0] + first, run, half),
                                delta = four_of(stat[1] + first, run, half);
            float u[4], bend[4];
            capped<CAP>(dot, run, a.rule, near, u, bend);
            float ex[4], ey[4], ez[4], r[4], ds[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = 4 * run + e;
                ex[e] = x[e] - xk;
                ey[e] = y[e] - yk;
                ez[e] = z[e] - zk;
                r[e] = __builtin_amdgcn_sqrtf(
                    fmaf(ex[e], ex[e], fmaf(ey[e], ey[e], ez[e] * ez[e])));
                const float w = exp2_of(fmaf(-slope2, r[e], u[e]) - lse[e]);
                ds[e] = (kNarrow<T> ? w * kLower : w) * (dp[i] - delta[e]);
                p.set(i, w);
                // (the rests are what the rounding leaves out)
                if constexpr (sizeof(T) == 2) p_rest.set(i, w - p.get(i));
                const float dx_i = CAP ? ds[e] * bend[e] : ds[e];
                if constexpr (kNarrow<T>) {
                    dot[i] = dx_i;  // (its product is done with)
                } else {
                    dx.set(i, dx_i);
                    if constexpr (sizeof(T) == 2) dx_rest.set(i, dx_i - dx.get(i));
                }
            }
            if (a.push_k) {
                asm volatile("");  // one branch for the run
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float wd = ds[e] * (r[e] > 0.f ? __builtin_amdgcn_rcpf(r[e]) : 0.f);
                    ux = fmaf(wd, ex[e], ux);
                    uy = fmaf(wd, ey[e], uy);
                    uz = fmaf(wd, ez[e], uz);
                }
            }
            __builtin_amdgcn_sched_barrier(kLoadsPass);
        }
        px = fmaf(slope, ux, px);
        py = fmaf(slope, uy, py);
        pz = fmaf(slope, uz, pz);
        const T* oc = M::kSeparateCols ? o_cols + sub * Pair::kCols : o_rows + sub * Pair::kRows;
        const T* qc = M::kSeparateCols ? q_cols + sub * Pair::kCols : q_rows + sub * Pair::kRows;
        M::template cols<DP>(dv, oc, p);
        if constexpr (sizeof(T) == 2) M::template cols<DP>(dv, oc, p_rest);
        if constexpr (kNarrow<T>) {
            unit.meet(dot, dk);
            const float by = unit.by();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                dx.set(i, dot[i] * by);
                dx_rest.set(i, dot[i] * by - dx.get(i));
            }
        }
        M::template cols<DP>(dk, qc, dx);
        if constexpr (sizeof(T) == 2) M::template cols<DP>(dk, qc, dx_rest);
    };
    const bool busy = t.first + wave * kTile < t.n_k;  // a wave without keys only helps to stage
    const int each = (stages + a.k_splits - 1) / a.k_splits;
    const int from = min(stages, split * each), to = min(stages, from + each);
    if (from < to) fetch(from);
    for (int i = from; i < to; ++i) {
        __syncthreads();
        stage.place(q_rows, M::kSeparateCols ? q_cols : nullptr, o_rows,
                    M::kSeparateCols ? o_cols : nullptr);
        if (threadIdx.x < kQueries)
#pragma unroll
            for (int c = 0; c < 3; ++c) {
                x_q.x[c][threadIdx.x] = xs[c];
                if (c < 2) stat[c][threadIdx.x] = ss[c];
            }
        __syncthreads();
        if (i + 1 < to) fetch(i + 1);
        const int n = t.n_q - (i % per_head) * kQueries;
        if (busy)
            for (int sub = 0; sub < kTiles && sub * kTile < n; ++sub)
                pull(sub, a.slopes[kv * a.group + i / per_head]);
    }
    px = sum_halves(px);
    py = sum_halves(py);
    pz = sum_halves(pz);
    if (!valid) return;
    const int64_t flat = (key * a.kv_heads + kv) * a.dim;
    const float back = kNarrow<T> ? unit.back() : 1.f;
    if (a.k_splits > 1) {
        float* part =
            a.part_k + (((int64_t)split * a.kv_heads + kv) * a.n_keys + key) * (2 * a.dim + 3);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int c = 32 * d + row_of(i, half);
                if (c >= a.dim) continue;
                part[c] = dk[d][i] * back;
                part[a.dim + c] = dv[d][i] * kLower;
            }
        if (half == 0) {
            part[2 * a.dim] = px;
            part[2 * a.dim + 1] = py;
            part[2 * a.dim + 2] = pz;
        }
        return;
    }
    store_channels<T, DP>((T*)a.grad_k + flat, a.dim, dk, a.rule.scale * back);
    store_channels<T, DP>((T*)a.grad_v + flat, a.dim, dv, kLower);
    if (a.push_k && half == 0) {
        float* push = a.push_k + 3 * ((int64_t)kv * a.n_keys + key);
        push[0] = px;
        push[1] = py;
        push[2] = pz;
    }
}

// Joins the splits of a key: threads over its 2 dim + 3 sums.
template <typename T>
__global__ __launch_bounds__(256) void k_structure_join_dkv(const StructureArgs a) {
    const int64_t width = 2 * a.dim + 3, keys = (int64_t)a.kv_heads * a.n_keys;
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (u >= keys * width) return;
    const int64_t at = u / width;
    const int c = (int)(u - at * width);
    float sum = 0.f;
#pragma unroll 4
    for (int s = 0; s < a.k_splits; ++s) sum += a.part_k[s * keys * width + u];
    const int64_t kv = at / a.n_keys, key = at - kv * a.n_keys;
    const int64_t flat = (key * a.kv_heads + kv) * a.dim;
    if (c < a.dim)
        ((T*)a.grad_k)[flat + c] = rounded<T>(sum * a.rule.scale);
    else if (c < 2 * a.dim)
        ((T*)a.grad_v)[flat + c - a.dim] = rounded<T>(sum);
    else if (a.push_k)
        a.push_k[3 * at + c - 2 * a.dim] = sum;
}

// Sums over the heads of the positions' gradients, threads over atoms and axes;
// where slopes are wanted, the first `heads` workgroups sum their rows.
__global__ __launch_bounds__(1024) void k_structure_finish(const StructureArgs a, float* grad_x_q,
                                                           float* grad_x_k, float* grad_slopes,
                                                           int shared) {
    int64_t block = blockIdx.x;
    if (grad_slopes) {
        if (block < a.heads) {
            const float sum = block_sum(a.turn + block * a.n_queries, a.n_queries);
            if (threadIdx.x == 0) grad_slopes[block] = sum;
            return;
        }
        block -= a.heads;
    }
    const int64_t nk = 3 * (int64_t)a.n_keys, nq = 3 * (int64_t)a.n_queries;
    int64_t i = block * 1024 + threadIdx.x;
    if (grad_x_k) {
        if (i < nk) {
            float sum = 0.f;
            for (int h = 0; h < a.kv_heads; ++h) sum += a.push_k[h * nk + i];
            if (shared)
                for (int h = 0; h < a.heads; ++h) sum += a.push_q[h * nq + i];
            grad_x_k[i] = sum;
            return;
        }
        i -= nk;
    }
    if (grad_x_q && i < nq) {
        float sum = 0.f;
        for (int h = 0; h < a.heads; ++h) sum += a.push_q[h * nq + i];
        grad_x_q[i] = sum;
    }
}

}  // namespace op
}  // namespace tnr
