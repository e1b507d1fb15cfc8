// Stable sort of small whole keys with a payload, by the digits of the key from
// the lowest on.  Each pass counts the digits of every tile of kSortTile items
// (one workgroup), scans the counts digit by digit, and moves the items: a
// wave ranks 64 items of equal digits among themselves by ballots, in the
// order that they have, so the result depends on the input alone.
//
// A digit has up to 10 bits (1,024 counters for each of a workgroup's 4 waves
// in LDS), so that keys below 1,024 take one pass and below 2^20 two.
//
// A pass over 2.9 M pairs (8-byte payloads) takes 6 + 5 + 41 us: the move writes
// runs of a few items, and what lies next to them comes from the next tiles.  With
// tiles dealt to the XCDs in turn it took 64, since each wrote parts of all lines.
#pragma once

#include "op_common.h"

namespace tnr {
namespace op {

constexpr int kSortThreads = 256;
constexpr int kSortWaves = kSortThreads / kWave;
constexpr int kSortRounds = 8;                            // items of a lane
constexpr int kSortTile = kSortThreads * kSortRounds;     // items of a workgroup
constexpr int kSortBits = 10;
constexpr int kSortRadix = 1 << kSortBits;

struct SortPass {
    int shift, bits;
};
// The passes for keys in [0, n_keys).
struct SortPlan {
    int passes;
    SortPass pass[4];
};
inline SortPlan sort_plan(int64_t n_keys) {
    int bits = 1;
    while (bits < 31 && (int64_t(1) << bits) < n_keys) ++bits;
    SortPlan p;
    p.passes = (bits + kSortBits - 1) / kSortBits;
    for (int i = 0, shift = 0; i < p.passes; ++i) {
        const int width = (bits - shift + p.passes - i - 1) / (p.passes - i);
        p.pass[i] = {shift, width};
        shift += width;
    }
    return p;
}
inline int64_t sort_tiles(int64_t n) { return (n + kSortTile - 1) / kSortTile; }
__host__ __device__ inline int64_t sort_stride(int64_t tiles) { return (tiles + 3) / 4 * 4; }  // of a digit's counts
inline size_t sort_count_bytes(int64_t n) {
    return (size_t)kSortRadix * sort_stride(sort_tiles(n)) * sizeof(int32_t);
}

// Keys and payloads of the first pass; later passes read what the one before
// wrote.
struct SortKeys {
    const int32_t* key;
    __device__ __forceinline__ int operator()(int64_t i) const { return key[i]; }
};

// Clears `words` that a later kernel wants zero.
__device__ __forceinline__ void sort_clear(int32_t* clear, int64_t words) {
    for (int64_t w = (int64_t)blockIdx.x * kSortThreads + threadIdx.x; w < words;
         w += (int64_t)gridDim.x * kSortThreads)
        clear[w] = 0;
}

// counts[digit * stride + tile]; and `clear`, which a later kernel wants zero.
template <typename Keys>
__global__ __launch_bounds__(kSortThreads) void k_sort_count(Keys keys, int64_t n, SortPass pass,
                                                             int32_t* counts, int32_t* clear,
                                                             int64_t clear_words) {
    __shared__ int32_t hist[kSortRadix];
    const int radix = 1 << pass.bits;
    sort_clear(clear, clear_words);
    for (int d = threadIdx.x; d < radix; d += kSortThreads) hist[d] = 0;
    __syncthreads();
    const int64_t tile = xcd_order(blockIdx.x, gridDim.x), base = tile * kSortTile;
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        const int64_t i = base + r * kSortThreads + threadIdx.x;
        if (i < n) atomicAdd(&hist[(keys(i) >> pass.shift) & (radix - 1)], 1);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < radix; d += kSortThreads)
        counts[(int64_t)d * sort_stride(gridDim.x) + tile] = hist[d];
}

__device__ __forceinline__ int sort_wave_scan(int x) {  // inclusive
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const int y = __shfl_up(x, d);
        if (lane_of() >= d) x += y;
    }
    return x;
}

// One wave a digit: its tiles' counts become their exclusive sums, its total
// goes to totals[digit].
__global__ __launch_bounds__(kSortThreads) void k_sort_scan(int32_t* counts, int64_t tiles,
                                                            int radix, int32_t* totals) {
    const int digit = blockIdx.x * kSortWaves + threadIdx.x / kWave;
    if (digit >= radix) return;
    int32_t* at = counts + (int64_t)digit * sort_stride(tiles);
    int before = 0;
    for (int64_t t = 0; t < tiles; t += 4 * kWave) {
        const int64_t i = t + 4 * lane_of();
        int4 x = i < tiles ? *(const int4*)(at + i) : int4{};  // (the counts end at a multiple of 4)
        if (i + 1 >= tiles) x.y = 0;
        if (i + 2 >= tiles) x.z = 0;
        if (i + 3 >= tiles) x.w = 0;
        const int sum = x.x + x.y + x.z + x.w, up = sort_wave_scan(sum);
        int4 y;
        y.x = before + up - sum;
        y.y = y.x + x.x;
        y.z = y.y + x.y;
        y.w = y.z + x.z;
        if (i < tiles) *(int4*)(at + i) = y;
        before += __shfl(up, kWave - 1);
    }
    if (lane_of() == 0) totals[digit] = before;
}

// Moves the items of a tile.  `put(place, index, key)` writes an item.  Where there
// is one tile it counts for itself (counts null), and clears what the counting
// kernel else does.
template <typename Keys, typename Put>
__global__ __launch_bounds__(kSortThreads) void k_sort_move(Keys keys, int64_t n, SortPass pass,
                                                            const int32_t* counts,
                                                            const int32_t* totals, Put put,
                                                            int32_t* clear, int64_t clear_words) {
    __shared__ int32_t seen[kSortWaves][kSortRadix];
    __shared__ int32_t wave_sum[kSortWaves];
    const int radix = 1 << pass.bits, lane = lane_of(), wave = threadIdx.x / kWave;
    if (!counts) sort_clear(clear, clear_words);
    for (int d = threadIdx.x; d < radix; d += kSortThreads)
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) seen[w][d] = 0;
    __syncthreads();
    // a wave's items are consecutive, in rounds of 64
    const int64_t tile = xcd_order(blockIdx.x, gridDim.x);
    const int64_t base = tile * kSortTile + wave * (kWave * kSortRounds);
    int key[kSortRounds], rank[kSortRounds];
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        const int64_t i = base + r * kWave + lane;
        key[r] = i < n ? keys(i) : -1;
    }
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        const bool in = base + r * kWave + lane < n;
        const int digit = (key[r] >> pass.shift) & (radix - 1);
        unsigned long long same = __builtin_amdgcn_ballot_w64(in);
        for (int b = 0; b < pass.bits; ++b) {
            const unsigned long long ones = __builtin_amdgcn_ballot_w64((digit >> b) & 1);
            same &= (digit >> b) & 1 ? ones : ~ones;
        }
        const int below = __popcll(same & ((1ull << lane) - 1));
        if (in) {
            const int before = seen[wave][digit];
            rank[r] = before + below;
            // the last of its kind counts them all, after every lane has read
            __builtin_amdgcn_wave_barrier();
            if ((same >> lane) == 1) seen[wave][digit] = before + below + 1;
        }
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    // a digit's place in the whole output, and in it those of this tile's waves
    int carry = 0;
    for (int d0 = 0; d0 < radix; d0 += kSortThreads) {
        const int d = d0 + threadIdx.x;
        int x = 0;
        if (d < radix) {
            if (counts)
                x = totals[d];
            else
#pragma unroll
                for (int w = 0; w < kSortWaves; ++w) x += seen[w][d];
        }
        const int up = sort_wave_scan(x);
        if (lane == kWave - 1) wave_sum[wave] = up;
        __syncthreads();
        int before = carry, all = 0;
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) {
            if (w < wave) before += wave_sum[w];
            all += wave_sum[w];
        }
        if (d < radix) {
            int at = before + up - x;
            if (counts) at += counts[(int64_t)d * sort_stride(gridDim.x) + tile];
#pragma unroll
            for (int w = 0; w < kSortWaves; ++w) {
                const int c = seen[w][d];
                seen[w][d] = at;
                at += c;
            }
        }
        carry += all;
        __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
        const int64_t i = base + r * kWave + lane;
        if (i < n) {
            const int digit = (key[r] >> pass.shift) & (radix - 1);
            put((int64_t)seen[wave][digit] + rank[r], i, key[r]);
        }
    }
}

}  // namespace op
}  // namespace tnr
