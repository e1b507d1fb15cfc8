// Attention within the structures of a batch.  For a query i and a key j of
// one structure at distance r, with x = scale q.k, u = c tanh(x / c) (u = x
// without a cap) and a slope m of the head:
//   s = u - m r,  p = softmax_j(s),  o = sum_j p v_j
// and back, with dp = do.v_j and delta = sum_j p dp:
//   ds = p (dp - delta),  dx = scale ds (1 - (u / c)^2),
//   dq = sum_j dx k_j,  dk_j = sum_i dx q_i,  dv_j = sum_i p do_i,
//   dr = -m ds (to both atoms along their line),  dm = -sum ds r.
//
// One pass over the keys with the running maximum and sum of the softmax
// (scores never leave the registers), in tiles of 32 x 32 on the matrix
// cores.  The forward and the queries' gradients hold the tile transposed,
// keys x queries: a lane then has 16 keys of ONE query, so that the row's
// maximum, sum and rescaling are the lane's own but for one exchange with the
// lane 32 away, and the weights of the tile are, as they stand in the
// registers, the right operand of the next product (out^T = v^T p^T); the
// rows of v^T are read in the order that the weights happen to have.  The
// keys' gradients hold queries x keys for the same reason.
//
// The query heads that share a key head are rows of one tile (row = query *
// group + head in the group): keys and values are read once for all of them,
// and one moved atom with 4 query heads to a key head fills 4 rows.
//
// The distance is computed in the tile from the positions, 32 bits.  Scores,
// statistics and sums are 32 bits.  The matrix products with 16-bit values take
// 16-bit weights: these go in two pieces, rounded and rest, which hold 16 bits of a
// bfloat16 weight and 22 of a float16 one.  Against the output's own rounding at the
// end that is nothing (2 values in 1,000 round to their neighbour); one piece alone
// adds as much error as it.  float16 weights are lifted by 2^7, so that those of keys far below
// the largest keep digits down to 2^-31 of it.
//
// What bounds it: vector instructions, not the matrix cores.  A tile of 32 x 32
// and one head takes about 29 instructions for each of a lane's 16 products
// (distance 7, cap 10, the weights' two pieces 4, the rest softmax) besides three
// that run at a quarter of the rate, and 12 matrix products of 32 cycles for 64
// channels.  Measured: 4,001 atoms, 8 capped heads of 64 on 2 key heads, bfloat16,
// 145 us (0.23 PFLOP/s, vector instructions in 79 % of the busy cycles, matrix
// products in 15 %); 1,024 molecules of 20 to 120 atoms, 8 heads of 32, 71 us
// (vector instructions in 94 %); one query in each of 64 structures of 2,000 to 20,000
// atoms, 8 heads of 64 on 2, 123 us (the keys' and values' rows); float32 is bound by
// its matrix products, a sixteenth of the rate (48 structures of 1 to 509 atoms, 4
// heads of 48: 85 us).
#pragma once

#include "op_common.h"

namespace tnr {
namespace op {

constexpr int kTile = 32;  // keys (or query rows) staged at a time, and rows of a wave

// A workgroup's part of a structure: its rows (or keys) from `first` on.
// n_q < 0: the batch's pointers are not valid (every result is NaN).
struct StructureTile {
    int q_lo, n_q, k_lo, n_k;
    int first, pad0, pad1, pad2;
};

struct StructureArgs {
    StructureTile *q_tiles, *k_tiles;
    const void *q, *k, *v;
    int64_t q_stride[2], k_stride[2], v_stride[2];
    const float *x_q, *x_k, *slopes;
    ScoreRule rule;
    int heads, kv_heads, group, dim;
    int n_queries, n_keys;
    int splits, k_splits;
    void* out;
    float* out32;  // out before its rounding to 16 bits, NULL: not wanted
    float* lse;   // [heads][n_queries], base 2
    float* part;    // splits of a row: [split][heads][n_queries][dim + 2], or dim + kRowSums
    float* part_k;  // splits of a key: [split][kv_heads][n_keys][2 dim + 3]
    const void* grad_out;
    void *grad_q, *grad_k, *grad_v;
    float* row;     // [heads][n_queries]: delta
    float* push_q;  // [heads][n_queries][3], NULL: not wanted
    float* push_k;  // [kv_heads][n_keys][3]
    float* turn;    // [heads][n_queries]: the slope's gradient by rows, NULL: not wanted
};

// ------------------------------------------------------------ the batch's tiles

// Structure b's tiles start at floor(ptr[b] * mult / rows) + b: room for all of
// them, at a place that no other structure's count is needed for.
__host__ __device__ inline int64_t tile_start(int64_t at, int64_t mult, int64_t rows, int64_t b) {
    return at * mult / rows + b;
}

// Tiles of `q_rows` query rows and of `k_rows` keys.  Every workgroup looks
// at all pointers, so that no tile of a batch whose pointers are wrong is left
// valid.
__global__ __launch_bounds__(256) void k_structure_tiles(const int64_t* q_ptr, const int64_t* k_ptr,
                                                         int64_t n_structures, int64_t n_queries,
                                                         int64_t n_keys, int group, int q_rows,
                                                         int k_rows, StructureTile* q_tiles,
                                                         StructureTile* k_tiles) {
    int bad = 0;
    for (int64_t b = threadIdx.x; b < n_structures; b += 256)
        bad |= q_ptr[b + 1] < q_ptr[b] || k_ptr[b + 1] < k_ptr[b];
    if (threadIdx.x == 0)
        bad |= q_ptr[0] != 0 || k_ptr[0] != 0 || q_ptr[n_structures] != n_queries ||
               k_ptr[n_structures] != n_keys;
    bad = __syncthreads_or(bad);
    const int lane = lane_of();
    const int64_t waves = (int64_t)gridDim.x * 4;
    if (bad) {
        const int64_t nq = tile_start(n_queries, group, q_rows, n_structures);
        const int64_t nk = tile_start(n_keys, 1, k_rows, n_structures);
        const StructureTile none{0, -1, 0, -1, 0, 0, 0, 0};
        for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < nq; i += waves * kWave)
            q_tiles[i] = none;
        if (k_tiles)
            for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < nk; i += waves * kWave)
                k_tiles[i] = none;
        return;
    }
    for (int64_t b = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave; b < n_structures; b += waves) {
        const int64_t q0 = q_ptr[b], q1 = q_ptr[b + 1], k0 = k_ptr[b], k1 = k_ptr[b + 1];
        StructureTile t{(int)q0, (int)(q1 - q0), (int)k0, (int)(k1 - k0), 0, 0, 0, 0};
        const int64_t from = tile_start(q0, group, q_rows, b);
        const int64_t to = tile_start(q1, group, q_rows, b + 1);
        for (int64_t i = from + lane; i < to; i += kWave) {
            t.first = (int)((i - from) * q_rows);
            q_tiles[i] = t;
        }
        if (!k_tiles) continue;
        const int64_t kfrom = tile_start(k0, 1, k_rows, b);
        const int64_t kto = tile_start(k1, 1, k_rows, b + 1);
        for (int64_t i = kfrom + lane; i < kto; i += kWave) {
            t.first = (int)((i - kfrom) * k_rows);
            k_tiles[i] = t;
        }
    }
}

// ---------------------------------------------------------- matrix products

// One staged tile of 32 rows of DP channels in LDS, and the two products with
// it.  `row` operands contract over channels, `col` operands over the tile's
// rows, whose order is that in which a lane's 16 results of a product lie:
// row_of(i, half).
__device__ __forceinline__ int row_of(int i, int half) { return 8 * (i / 4) + 4 * half + i % 4; }

// The value at a lane's own row and column of a 32 x 32 result.
__device__ __forceinline__ float diagonal(const f32x16& all) {
    const int lane = lane_of();
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (row_of(i, lane / 32) == lane % 32) x = all[i];
    return sum_halves(x);  // the other half's lane has none
}

template <typename T>
struct Mat;

// The scheduler keeps the work on four products together, which bounds the
// registers, but may read the next four's rows from LDS meanwhile.
constexpr int kLoadsPass = 0x100;

template <typename T, typename F>
struct Mat16 {
    using Frag = Vec<T, 8>;
    // Rows are 16 bytes longer than their channels, columns 8 bytes longer
    // than their rows: both then spread over the LDS banks.
    static constexpr int kRows(int dp) { return kTile * (dp + 8); }
    static constexpr int kCols(int dp) { return dp * (kTile + 4); }

    // A lane's own row: channels 16 s + 8 half + 0..7.
    template <int DP>
    struct Row {
        Frag x[DP / 16];
        __device__ __forceinline__ void load(const T* p, int dim) {
            const int half = lane_of() / 32;
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) {
                const int c = 16 * s + 8 * half;
                x[s] = Frag{};
                if (p && c < dim) x[s] = *(const Frag*)(p + c);
            }
        }
        // With a row of 32 bits, in three pieces of T (float16's are lifted by
        // 2^11 each, which its range would else cut off), by the matrix product
        // that also makes a query's product with a value: a row that T holds gives
        // the same bits as that product.
        __device__ __forceinline__ float dot32(const float* p, int dim) const {
            constexpr float kLift = std::is_same_v<T, f16> ? 2048.f : 1.f;
            const int half = lane_of() / 32;
            float rest[DP / 16][8], sum = 0.f, by = 1.f;
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) {
                const int c = 16 * s + 8 * half;
                Vec<float, 4> lo{}, hi{};
                if (p && c < dim) {
                    lo = *(const Vec<float, 4>*)(p + c);
                    hi = *(const Vec<float, 4>*)(p + c + 4);
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) rest[s][e] = e < 4 ? lo[e % 4] : hi[e % 4];
            }
#pragma unroll
            for (int piece = 0; piece < 3; ++piece) {
                f32x16 all{};
#pragma unroll
                for (int s = 0; s < DP / 16; ++s) {
                    Frag o;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        o[e] = rounded<T>(rest[s][e]);
                        rest[s][e] = (rest[s][e] - (float)o[e]) * kLift;
                    }
                    all = F::mma(o, x[s], all);
                }
                sum = fmaf(diagonal(all), by, sum);
                by *= 1.f / kLift;
            }
            return sum;
        }
    };

    // acc += tile . row^T over the first `dim` channels
    template <int DP>
    static __device__ __forceinline__ void rows(f32x16& acc, const T* tile, const Row<DP>& b,
                                                int dim) {
        const int lane = lane_of();
        const T* p = tile + (lane % 32) * (DP + 8) + 8 * (lane / 32);
#pragma unroll
        for (int s = 0; s < DP / 16; ++s) {
            if (16 * s > DP - 32 && 16 * s >= dim) break;
            acc = F::mma(*(const Frag*)(p + 16 * s), b.x[s], acc);
        }
    }

    // A lane's 16 weights of a tile, rounded for the second product.
    struct Weights {
        Frag b[2];
        __device__ __forceinline__ void set(int i, float x) { b[i / 8][i % 8] = rounded<T>(x); }
        __device__ __forceinline__ float get(int i) const { return (float)b[i / 8][i % 8]; }
    };
    // acc[channel block] += tile^T . p
    template <int DP>
    static __device__ __forceinline__ void cols(f32x16 (&acc)[DP / 32], const T* tile,
                                                const Weights& p) {
        const int lane = lane_of();
        const T* at = tile + (lane % 32) * (kTile + 4) + 4 * (lane / 32);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const T* c = at + d * 32 * (kTile + 4) + 16 * s;
                const Vec<T, 4> lo = *(const Vec<T, 4>*)c, hi = *(const Vec<T, 4>*)(c + 8);
                const Frag a = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                acc[d] = F::mma(a, p.b[s], acc[d]);
            }
    }

    // Threads stage units of 4 rows x 8 channels.
    template <int DP>
    struct Stage {
        static constexpr int kUnits = (kTile / 4) * (DP / 8);
        Frag x[4];
        __device__ __forceinline__ void load(int unit, const T* base, int stride, int rows,
                                             int dim) {
            const int r = 4 * (unit % (kTile / 4)), c = 8 * (unit / (kTile / 4));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = Frag{};
                if (r + i < rows && c < dim)
                    x[i] = *(const Frag*)(base + (uint32_t)((r + i) * stride + c));
            }
        }
        __device__ __forceinline__ void store(int unit, T* row, T* col) const {
            const int r = 4 * (unit % (kTile / 4)), c = 8 * (unit / (kTile / 4));
            if (row)
#pragma unroll
                for (int i = 0; i < 4; ++i) *(Frag*)(row + (r + i) * (DP + 8) + c) = x[i];
            if (col)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const Vec<T, 4> t = {x[0][e], x[1][e], x[2][e], x[3][e]};
                    *(Vec<T, 4>*)(col + (c + e) * (kTile + 4) + r) = t;
                }
        }
    };
    static constexpr bool kSeparateCols = true;
};

struct MmaBf16 {
    static __device__ __forceinline__ f32x16 mma(Vec<bf16, 8> a, Vec<bf16, 8> b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
struct MmaF16 {
    static __device__ __forceinline__ f32x16 mma(Vec<f16, 8> a, Vec<f16, 8> b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Mat<bf16> : Mat16<bf16, MmaBf16> {};
template <>
struct Mat<f16> : Mat16<f16, MmaF16> {};

// 32-bit products: two channels to an instruction, of which the lower lanes
// take those of the row's first half and the upper lanes the second's, so that
// a lane reads neighbouring floats.  They run at a sixteenth of the 16-bit rate
// and bound the 32-bit kernels, so channels beyond `dim` are left out.
template <>
struct Mat<float> {
    static constexpr int kRows(int dp) { return kTile * (dp + 4); }
    static constexpr int kCols(int) { return 0; }

    template <int DP>
    struct Row {
        Vec<float, 4> x[DP / 8];
        __device__ __forceinline__ void load(const float* p, int dim) {
            const int half = lane_of() / 32;
#pragma unroll
            for (int s = 0; s < DP / 8; ++s) {
                x[s] = Vec<float, 4>{};
                if (p && 8 * s < dim)
                    x[s] = *(const Vec<float, 4>*)(p + half * (dim / 2) + 4 * s);
            }
        }
        __device__ __forceinline__ float dot32(const float* p, int dim) const {
            Row o;
            o.load(p, dim);
            f32x16 all{};
#pragma unroll
            for (int s = 0; s < DP / 8; ++s)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    all = __builtin_amdgcn_mfma_f32_32x32x2f32(o.x[s][e], x[s][e], all, 0, 0, 0);
            return diagonal(all);
        }
    };

    template <int DP>
    static __device__ __forceinline__ void rows(f32x16& acc, const float* tile, const Row<DP>& b,
                                                int dim) {
        const int lane = lane_of();
        const float* p = tile + (lane % 32) * (DP + 4) + (lane / 32) * (dim / 2);
#pragma unroll
        for (int s = 0; s < DP / 8; ++s) {
            if (8 * s > DP - 32 && 8 * s >= dim) break;
            const Vec<float, 4> a = *(const Vec<float, 4>*)(p + 4 * s);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                acc = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b.x[s][e], acc, 0, 0, 0);
        }
    }

    struct Weights {
        float b[16];
        __device__ __forceinline__ void set(int i, float x) { b[i] = x; }
        __device__ __forceinline__ float get(int i) const { return b[i]; }
    };
    template <int DP>
    static __device__ __forceinline__ void cols(f32x16 (&acc)[DP / 32], const float* tile,
                                                const Weights& p) {
        const int lane = lane_of();
        const float* at = tile + lane % 32;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                acc[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(
                    at[row_of(i, lane / 32) * (DP + 4) + 32 * d], p.b[i], acc[d], 0, 0, 0);
    }

    // Threads stage units of 4 rows x 4 channels.
    template <int DP>
    struct Stage {
        static constexpr int kUnits = (kTile / 4) * (DP / 4);
        Vec<float, 4> x[4];
        __device__ __forceinline__ void load(int unit, const float* base, int stride, int rows,
                                             int dim) {
            const int r = unit / (DP / 4), c = 4 * (unit % (DP / 4));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = Vec<float, 4>{};
                if (r + 8 * i < rows && c < dim)
                    x[i] = *(const Vec<float, 4>*)(base + (uint32_t)((r + 8 * i) * stride + c));
            }
        }
        __device__ __forceinline__ void store(int unit, float* row, float*) const {
            const int r = unit / (DP / 4), c = 4 * (unit % (DP / 4));
#pragma unroll
            for (int i = 0; i < 4; ++i) *(Vec<float, 4>*)(row + (r + 8 * i) * (DP + 4) + c) = x[i];
        }
    };
    static constexpr bool kSeparateCols = false;
};

// Two staged tensors, kTiles tiles of 32 rows each: as many as give the
// workgroup's threads a unit each.  With one unit they are loaded a stage ahead,
// with more (few waves, wide heads) when their stage is placed: their registers
// are worth more than the wait.
template <typename T, int DP, int NW>
struct StagePair {
    using S = typename Mat<T>::template Stage<DP>;
    static constexpr int kOne = S::kUnits, kThreads = NW * kWave;
    static constexpr int kTiles = kThreads >= 8 * kOne ? 4 : kThreads >= 4 * kOne ? 2 : 1;
    static constexpr int kAll = 2 * kOne * kTiles;
    static constexpr int kEach = (kAll + kThreads - 1) / kThreads;
    static constexpr bool kAhead = kEach == 1;
    static constexpr int kRows = Mat<T>::kRows(DP);  // elements of a tile, as rows and as columns
    static constexpr int kCols = Mat<T>::kSeparateCols ? Mat<T>::kCols(DP) : 0;
    const T *a, *b;
    int a_stride, b_stride, rows, dim;
    S ahead;

    // unit u: of tile u / (2 kOne), and there of one tensor, then of the other
    __device__ __forceinline__ void load(S& s, int u) const {
        const int tile = u / (2 * kOne), v = u % (2 * kOne);
        const bool first = v < kOne;
        if (u < kAll)
            s.load(first ? v : v - kOne, (first ? a : b) + (int64_t)tile * kTile * (first ? a_stride : b_stride),
                   first ? a_stride : b_stride, rows - tile * kTile, dim);
    }
    // (null: that form of the tensor is not wanted)
    static __device__ __forceinline__ void put(const S& s, int u, T* a_row, T* a_col, T* b_row,
                                               T* b_col) {
        const int tile = u / (2 * kOne), v = u % (2 * kOne);
        const bool first = v < kOne;
        if (u >= kAll) return;
        if (first)
            s.store(v, a_row ? a_row + tile * kRows : nullptr, a_col ? a_col + tile * kCols : nullptr);
        else
            s.store(v - kOne, b_row ? b_row + tile * kRows : nullptr,
                    b_col ? b_col + tile * kCols : nullptr);
    }
    __device__ __forceinline__ void fetch(const T* a_, int a_stride_, const T* b_, int b_stride_,
                                          int rows_, int dim_) {
        a = a_;
        b = b_;
        a_stride = a_stride_;
        b_stride = b_stride_;
        rows = rows_;
        dim = dim_;
        if (kAhead) load(ahead, threadIdx.x);
    }
    __device__ __forceinline__ void place(T* a_row, T* a_col, T* b_row, T* b_col) const {
        if (kAhead) {
            put(ahead, threadIdx.x, a_row, a_col, b_row, b_col);
            return;
        }
#pragma unroll 2
        for (int i = 0; i < kEach; ++i) {
            S s;
            load(s, threadIdx.x + i * kThreads);
            put(s, threadIdx.x + i * kThreads, a_row, a_col, b_row, b_col);
        }
    }
};

// ------------------------------------------------------------------ forward

// Channels 8 (i / 4) + 4 half + i % 4 of block d: groups of four, written whole.
template <typename T, int DP>
__device__ __forceinline__ void store_channels(T* row, int dim, const f32x16 (&acc)[DP / 32],
                                               float by) {
    const int half = lane_of() / 32;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = 32 * d + 8 * g + 4 * half;
            if (c >= dim) continue;
            const float x[4] = {acc[d][4 * g] * by, acc[d][4 * g + 1] * by, acc[d][4 * g + 2] * by,
                                acc[d][4 * g + 3] * by};
            store_floats<T, 4>(row + c, x);
        }
}

// Whether the tile's 16 products all lie where tanh needs no exp.
template <bool CAP>
__device__ __forceinline__ bool all_near(const f32x16& dot, const ScoreRule& rule) {
    if (!CAP) return true;
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, fabsf(dot[i]));
    return __builtin_amdgcn_ballot_w64(!(top * fabsf(rule.inv) <= kTanhNear)) == 0;
}
// u log2(e) of the products of run `run`, and what their gradients are multiplied
// by.  (What is subtracted from a score comes after the score is whole, in every pass:
// its rounding is then the same bits in all of them, and delta is the mean of dp
// under the weights that the backward finds.)
template <bool CAP>
__device__ __forceinline__ void capped(const f32x16& dot, int run, const ScoreRule& rule, bool near,
                                       float (&u)[4], float (&bend)[4]) {
    if (!CAP) {
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = dot[4 * run + e] * rule.scale2;
        return;
    }
    // (the empty asm keeps this a branch of the wave: one side only is computed)
    if (near) {
        asm volatile("");
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = tanh_near(dot[4 * run + e] * rule.inv);
    } else {
        asm volatile("");
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = tanh_of(dot[4 * run + e] * rule.inv);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        bend[e] = fmaf(-u[e], u[e], 1.f);
        u[e] *= rule.cap2;
    }
}

// Positions of a staged tile, by axes: a lane's 16 rows are 4 runs of 4.
template <int TILES>
struct TilePositions {
    alignas(16) float x[3][TILES * kTile];
};
__device__ __forceinline__ Vec<float, 4> four_of(const float* x, int run, int half) {
    return *(const Vec<float, 4>*)(x + 8 * run + 4 * half);
}

// Waves that a SIMD is to hold, of 512 registers: the accumulators and rows of
// one wave grow with the head dimension.
template <typename T>
constexpr int waves_held(int dp) {
    return sizeof(T) == 4 ? (dp <= 32 ? 3 : dp <= 64 ? 2 : 1) : (dp <= 32 ? 4 : dp <= 64 ? 3 : 2);
}

// float16 has small values down to 2^-24 and large ones below 2^16.
template <typename T>
constexpr bool kNarrow = std::is_same_v<T, f16>;
// The exponent that a row's largest weight has in the forward: reached exactly, so that
// a row of one key is that key's value to the bit.
template <typename T>
constexpr float kWeightLift = kNarrow<T> ? 7.f : 0.f;

// grid: (tiles * kv_heads, splits); NW waves of 32 query rows each.
template <typename T, int DP, int NW, bool CAP>
__global__ __launch_bounds__(NW* kWave, waves_held<T>(DP)) void k_structure_forward(
    const StructureArgs a) {
    using M = Mat<T>;
    using Row = typename M::template Row<DP>;
    using Pair = StagePair<T, DP, NW>;
    constexpr int kTiles = Pair::kTiles, kKeys = kTiles * kTile;
    constexpr int kValues = M::kSeparateCols ? Pair::kCols : Pair::kRows;
    __shared__ alignas(16) T k_rows[kTiles * Pair::kRows];
    __shared__ alignas(16) T v_tile[kTiles * kValues];
    __shared__ TilePositions<kTiles> x_k;

    // a tile's key heads lie next to each other in memory: they follow one another
    const uint32_t order = xcd_order(blockIdx.x, gridDim.x), block = order / (uint32_t)a.kv_heads;
    const StructureTile t = a.q_tiles[block];
    const int lane = lane_of(), half = lane / 32, wave = threadIdx.x / kWave;
    const int kv = (int)(order - block * a.kv_heads), split = blockIdx.y;
    const int g = a.group;
    if (t.n_q < 0) {  // NaN for the rows that lie here in the batch
        const int64_t all = (int64_t)a.n_queries * g;
        const int64_t row = (int64_t)block * (NW * kTile) + wave * kTile + lane % 32;
        if (row >= all || split > 0 || half) return;
        const int query = (int)(row / g), head = kv * g + (int)(row % g);
        T* out = (T*)a.out + ((int64_t)query * a.heads + head) * a.dim;
        for (int c = 0; c < a.dim; ++c) out[c] = rounded<T>(nan_of());
        if (a.out32)
            for (int c = 0; c < a.dim; ++c)
                a.out32[((int64_t)query * a.heads + head) * a.dim + c] = nan_of();
        if (a.lse) a.lse[(int64_t)head * a.n_queries + query] = nan_of();
        if (a.splits > 1)
            for (int s = 0; s < a.splits; ++s) {
                float* part = a.part + (((int64_t)s * a.heads + head) * a.n_queries + query) *
                                           (a.dim + 2);
                for (int c = 0; c < a.dim; ++c) part[c] = nan_of();
                part[a.dim] = 0.f;
                part[a.dim + 1] = 1.f;
            }
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
    Row qr;
    qr.load(valid ? (const T*)a.q + (int64_t)query * a.q_stride[0] + head * a.q_stride[1] : nullptr,
            a.dim);
    float xq = 0.f, yq = 0.f, zq = 0.f, slope2 = 0.f;
    if (valid) {
        xq = a.x_q[3 * (int64_t)query];
        yq = a.x_q[3 * (int64_t)query + 1];
        zq = a.x_q[3 * (int64_t)query + 2];
        slope2 = a.slopes[head] * kLog2e;
    }
    const T* kb = (const T*)a.k + (int64_t)t.k_lo * a.k_stride[0] + kv * a.k_stride[1];
    const T* vb = (const T*)a.v + (int64_t)t.k_lo * a.v_stride[0] + kv * a.v_stride[1];
    const float* xb = a.x_k + 3 * (int64_t)t.k_lo;

    const int tiles = (t.n_k + kTile - 1) / kTile;
    const int each = (tiles + a.splits - 1) / a.splits;
    const int from = min(tiles, split * each), to = min(tiles, from + each);

    f32x16 acc[DP / 32];
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) acc[d] = f32x16{};
    float top = -inf_of(), sum = 0.f;

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
        if constexpr (M::kSeparateCols)
            stage.place(k_rows, nullptr, nullptr, v_tile);
        else
            stage.place(k_rows, nullptr, v_tile, nullptr);
        if (threadIdx.x < kKeys)
#pragma unroll
            for (int c = 0; c < 3; ++c) x_k.x[c][threadIdx.x] = xs[c];
        __syncthreads();
    };
    // Weights are taken relative to `top`, the maximum when it was last set: it
    // is set anew only where a score passes it by more than 2^8 (the row's sums
    // then change their unit), so that most tiles neither subtract nor rescale.
    constexpr float kLift = kWeightLift<T>;
    const auto weigh = [&](int sub, int left) {
        f32x16 dot{};
        M::template rows<DP>(dot, k_rows + sub * Pair::kRows, qr, a.dim);
        float s[16], unused[4];
        const float ref = top == -inf_of() ? 0.f : top - kLift;
        const bool near = all_near<CAP>(dot, a.rule);
        float high = -inf_of();
#pragma unroll
        for (int run = 0; run < 4; ++run) {
            const int first = sub * kTile;
            const Vec<float, 4> x = four_of(x_k.x[0] + first, run, half),
                                y = four_of(x_k.x[1] + first, run, half),
                                z = four_of(x_k.x[2] + first, run, half);
            float u[4];
            capped<CAP>(dot, run, a.rule, near, u, unused);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float dx = xq - x[e], dy = yq - y[e], dz = zq - z[e];
                const float r = __builtin_amdgcn_sqrtf(fmaf(dx, dx, fmaf(dy, dy, dz * dz)));
                s[4 * run + e] = fmaf(-slope2, r, u[e]) - ref;
            }
            if (left < kTile) {
                asm volatile("");  // a branch: only a structure's last tile pays for the selects
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (8 * run + e >= left - 4 * half) s[4 * run + e] = -inf_of();
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) high = fmaxf(high, s[4 * run + e]);
            __builtin_amdgcn_sched_barrier(kLoadsPass);
        }
        high = max_halves(high);
        const bool anew = high > 8.f + kLift || (top == -inf_of() && high > -inf_of());
        if (__builtin_amdgcn_ballot_w64(anew) != 0) {
            const float up = anew ? high : 0.f, lift = anew ? kLift : 0.f;
            // (the first maximum has no sums to fade, and may lie far below 0)
            const float fade = exp2_of(fminf(lift - up, 0.f));
            top = anew ? ref + high : top;
            sum *= fade;
#pragma unroll
            for (int d = 0; d < DP / 32; ++d) acc[d] *= fade;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = kNarrow<T> ? (s[i] - up) + lift : s[i] - up;
        }
        float part[4] = {};
        typename M::Weights p, rest;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float w = exp2_of(s[i]);
            part[i % 4] += w;
            p.set(i, w);
            if constexpr (sizeof(T) == 2) rest.set(i, w - p.get(i));
        }
        sum += (part[0] + part[1]) + (part[2] + part[3]);
        M::template cols<DP>(acc, v_tile + sub * kValues, p);
        if constexpr (sizeof(T) == 2) M::template cols<DP>(acc, v_tile + sub * kValues, rest);
    };
    if (from < to) fetch(from);
    for (int tile = from; tile < to; tile += kTiles) {
        place();
        if (tile + kTiles < to) fetch(tile + kTiles);
        if (busy)
            for (int sub = 0; sub < min(kTiles, to - tile); ++sub)
                weigh(sub, t.n_k - (tile + sub) * kTile);
    }
    sum = sum_halves(sum);
    if (!valid) return;
    if (a.splits > 1) {
        float* part =
            a.part + (((int64_t)split * a.heads + head) * a.n_queries + query) * (a.dim + 2);
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int c = 32 * d + row_of(i, half);
                if (c < a.dim) part[c] = acc[d][i];
            }
        if (half == 0) {
            part[a.dim] = top;
            part[a.dim + 1] = sum;
        }
        return;
    }
    const float by = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t flat = ((int64_t)query * a.heads + head) * a.dim;
    store_channels<T, DP>((T*)a.out + flat, a.dim, acc, by);
    if (a.out32) store_channels<float, DP>(a.out32 + flat, a.dim, acc, by);
    if (a.lse && half == 0)
        a.lse[(int64_t)head * a.n_queries + query] =
            sum == 0.f ? -inf_of() : top + (__builtin_amdgcn_logf(sum) - kLift);
}

// Joins the splits of a row: one wave each, lanes over channels.
template <typename T>
__global__ __launch_bounds__(256) void k_structure_join(const StructureArgs a) {
    const int64_t at = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
    const int64_t rows = (int64_t)a.heads * a.n_queries;
    if (at >= rows) return;
    const int lane = lane_of();
    const int64_t step = rows * (a.dim + 2);
    const float* part = a.part + at * (a.dim + 2);
    // a lane for each split: its maximum and sum
    const bool there = lane < a.splits;
    const float high = there ? part[lane * step + a.dim] : -inf_of();
    float sum = there ? part[lane * step + a.dim + 1] : 0.f;
    const float top = join_lanes<max_of>(high, 1);
    const float w = exp2_of(high - (top == -inf_of() ? 0.f : top));
    sum = join_lanes<sum_of>(there ? sum * w : 0.f, 1);
    float x0 = 0.f, x1 = 0.f;
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) {
        const float* p = part + s * step;
        const float ws = __shfl(w, s);
        if (lane < a.dim) x0 = fmaf(ws, p[lane], x0);
        if (lane + kWave < a.dim) x1 = fmaf(ws, p[lane + kWave], x1);
    }
    const int head = (int)(at / a.n_queries), query = (int)(at % a.n_queries);
    const float by = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t flat = ((int64_t)query * a.heads + head) * a.dim;
    T* out = (T*)a.out + flat;
    if (lane < a.dim) out[lane] = rounded<T>(x0 * by);
    if (lane + kWave < a.dim) out[lane + kWave] = rounded<T>(x1 * by);
    if (a.out32) {
        if (lane < a.dim) a.out32[flat + lane] = x0 * by;
        if (lane + kWave < a.dim) a.out32[flat + lane + kWave] = x1 * by;
    }
    if (a.lse && lane == 0)
        a.lse[at] = sum == 0.f ? -inf_of()
                               : top + (__builtin_amdgcn_logf(sum) - kWeightLift<T>);
}

}  // namespace op
}  // namespace tnr
