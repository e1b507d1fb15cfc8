// Rows of a table by species, out[n] = scale weight[z_n], and the table's
// gradient, grad_weight[z] = scale sum_{n: z_n = z} grad_out[n].
//
// Both are bound by the rows: the forward writes them once (the table stays in
// the L2), the backward reads them once.  The backward sorts the atoms by
// species (op_sort.h) and sums runs: each group of threads takes as many
// sorted atoms as fill the device, adds their rows in registers, 32 bits, and
// writes a species' sum where its run lies within them; runs that reach over
// their ends go to partial rows, which a second kernel adds in the order of the
// atoms.  No atomics, so the sums' order is fixed by the inputs.
//
// Measured: 1,048,576 rows of 128 floats, forward 122 us (537 MB written, 4.4
// TB/s); backward the sort 26, the runs 157 (3.4 TB/s: rows of 512 bytes come in
// sorted, not in memory order), the join 21.
#pragma once

#include "op_sort.h"

namespace tnr {
namespace op {

struct EmbeddingArgs {
    const void *species, *weight, *grad_out;
    void *out, *grad_weight;
    int64_t n_atoms, n_species, channels;
    float scale;
};

template <typename I>
struct SpeciesOf {
    const I* species;
    int64_t n_species;
    // species outside the table sort behind it
    __device__ __forceinline__ int operator()(int64_t i) const {
        const int64_t z = (int64_t)species[i];
        return (int)(z < 0 || z >= n_species ? n_species : z);
    }
};

// One thread for VEC channels of an atom.
template <typename T, typename I, int VEC>
__global__ __launch_bounds__(256) void k_embedding_forward(const EmbeddingArgs a) {
    const int64_t units = a.channels / VEC, all = a.n_atoms * units;
    const SpeciesOf<I> of{(const I*)a.species, a.n_species};
    for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < all;
         u += (int64_t)gridDim.x * 256) {
        const int64_t n = all < INT32_MAX ? (int64_t)((uint32_t)u / (uint32_t)units) : u / units;
        const int64_t c = (u - n * units) * VEC;
        const int64_t z = of(n);
        float x[VEC];
        if (z < a.n_species) {
            load_floats<T, VEC>((const T*)a.weight + z * a.channels + c, x);
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[i] *= a.scale;
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[i] = nan_of();
        }
        store_floats<T, VEC>((T*)a.out + n * a.channels + c, x);
    }
}

// After the last pass: the atom at a place, and where species' runs begin and
// end (found from the sorted keys by k_embedding_runs).
struct PutAtom {
    int32_t *key, *atom;
    __device__ __forceinline__ void operator()(int64_t place, int64_t i, int k) const {
        key[place] = k;
        atom[place] = (int32_t)i;
    }
};
struct MoveAtom {
    const int32_t* from;
    int32_t *key, *atom;
    __device__ __forceinline__ void operator()(int64_t place, int64_t i, int k) const {
        key[place] = k;
        atom[place] = from[i];
    }
};

struct RunArgs {
    const int32_t *key, *atom;  // sorted
    int2* runs;                 // [n_species]: places [x, y), zeros before
    float* partial;             // [groups][2][channels]
    int64_t each;               // sorted atoms of a group
};

// `lanes` threads (a power of two) take VEC channels each of a group's rows,
// blockIdx.y tiles the channels.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void k_embedding_runs(const EmbeddingArgs a, const RunArgs r,
                                                        int lanes) {
    const int64_t group = (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
    const int64_t c = ((int64_t)blockIdx.y * lanes + threadIdx.x % lanes) * VEC;
    const int64_t from = group * r.each, to = min(a.n_atoms, from + r.each);
    if (from >= to) return;
    const bool mine = c < a.channels, first = blockIdx.y == 0 && threadIdx.x % lanes == 0;
    float sum[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[i] = 0.f;
    int run = r.key[from];
    // the group's first run may have begun before it
    bool head = from > 0 && r.key[from - 1] == run;
    if (first && !head && run < a.n_species) r.runs[run].x = (int)from;
    const auto flush = [&](bool open) {
        if (run >= a.n_species || !mine) return;
        if (head || open) {
            float* p = r.partial + (group * 2 + (head ? 0 : 1)) * a.channels + c;
            store_floats<float, VEC>(p, sum);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum[i] *= a.scale;
            store_floats<T, VEC>((T*)a.grad_weight + (int64_t)run * a.channels + c, sum);
        }
    };
    constexpr int kAhead = 8;
    int next_key[kAhead], next_atom[kAhead];
    const auto look = [&](int64_t p0) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int64_t p = min(p0 + j, to - 1);
            next_key[j] = r.key[p];
            next_atom[j] = r.atom[p];
        }
    };
    look(from);
    for (int64_t p0 = from; p0 < to; p0 += kAhead) {
        float x[kAhead][VEC];
        int key[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            key[j] = next_key[j];
            if (mine)
                load_floats<T, VEC>((const T*)a.grad_out + (int64_t)next_atom[j] * a.channels + c,
                                    x[j]);
        }
        look(p0 + kAhead);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (p0 + j >= to) break;
            if (key[j] != run) {
                flush(false);
                if (first) {
                    if (run < a.n_species) r.runs[run].y = (int)(p0 + j);
                    if (key[j] < a.n_species) r.runs[key[j]].x = (int)(p0 + j);
                }
                run = key[j];
                head = false;
#pragma unroll
                for (int i = 0; i < VEC; ++i) sum[i] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum[i] += x[j][i];
        }
    }
    const bool open = to < a.n_atoms && r.key[to] == run;
    if (first && !open && run < a.n_species) r.runs[run].y = (int)to;
    flush(open);
}

// Zeros for species without atoms, and the sums of those whose run spans
// several groups: one workgroup a species and tile of channels.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void k_embedding_join(const EmbeddingArgs a, const RunArgs r,
                                                        int lanes) {
    __shared__ float part[256 * VEC];
    const int64_t z = blockIdx.x;
    const int2 run = r.runs[z];
    const int64_t c = ((int64_t)blockIdx.y * lanes + threadIdx.x % lanes) * VEC;
    const bool mine = c < a.channels;
    T* out = (T*)a.grad_weight + z * a.channels + c;
    float sum[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[i] = 0.f;
    if (run.y <= run.x) {
        if (mine && (int)threadIdx.x < lanes) store_floats<T, VEC>(out, sum);
        return;
    }
    const int64_t g0 = run.x / r.each, g1 = (run.y - 1) / r.each;
    // (a run that neither began before its group nor goes on after it is whole)
    if (g0 == g1) return;
    const int64_t team = threadIdx.x / lanes, teams = 256 / lanes;
    if (mine)
#pragma unroll 4
        for (int64_t g = g0 + team; g <= g1; g += teams) {
            // it began within its first group, and before the others
            float x[VEC];
            load_floats<float, VEC>(r.partial + (g * 2 + (g > g0 ? 0 : 1)) * a.channels + c, x);
#pragma unroll
            for (int i = 0; i < VEC; ++i) sum[i] += x[i];
        }
#pragma unroll
    for (int i = 0; i < VEC; ++i) part[threadIdx.x * VEC + i] = sum[i];
    __syncthreads();
    if (!mine || (int)threadIdx.x >= lanes) return;
    for (int64_t t = 1; t < teams; ++t)
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] += part[(t * lanes + threadIdx.x) * VEC + i];
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[i] *= a.scale;
    store_floats<T, VEC>(out, sum);
}

// Sets `n` words to zero.
__global__ __launch_bounds__(256) void k_op_zero(int32_t* p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
        p[i] = 0;
}

}  // namespace op
}  // namespace tnr
