// row_norm.cuh — what the fused norms share: teams of threads that hold a row in registers, sums over a team, and the
// column sums of a backward pass.
//
// Every element is read once and written once, so the norms are bound by memory: a team loads all its operands of a
// row before it adds anything up, 16 bytes at a time where the rows allow it, and blocks stay to take more rows.
#pragma once

#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace bcm {
namespace row_norm {

// T threads hold a row of up to 8 T elements, 8 each: few registers, so that many rows are in flight (8 or 32 elements
// a thread in smaller teams spilled in the backward passes).  VEC: eight neighbouring elements at a time (rows on 16
// bytes, a width that is a multiple of 8); else neighbouring threads hold neighbouring elements.
template <int T, bool VEC>
struct Team {
    static constexpr int n = 8, threads = T > 256 ? T : 256, teams = threads / T;
    // a backward pass with 64 registers a thread has none to hold the next row
    static constexpr bool ahead_back = T < 1024;

    __device__ __forceinline__ static int lane() { return threadIdx.x % T; }
    __device__ __forceinline__ static int id() { return threadIdx.x / T; }
    __device__ __forceinline__ static int col(int j) { return VEC ? lane() * 8 + j : j * T + lane(); }

    // a thread's elements of a row as they lie in memory, 0 behind `width`; values() makes numbers of them
    template <typename E>
    struct Raw {
        typename std::conditional<VEC, uint4[sizeof(E) / 2], E[8]>::type v;
    };
    template <typename E>
    __device__ __forceinline__ static void fetch(const E* row, int width, Raw<E>& raw) {
        if constexpr (VEC) {
            const int c = lane() * 8;
#pragma unroll
            for (int q = 0; q < (int)sizeof(E) / 2; ++q) raw.v[q] = c < width ? ((const uint4*)(row + c))[q] : make_uint4(0, 0, 0, 0);
        } else {
#pragma unroll
            for (int j = 0; j < n; ++j) raw.v[j] = j * T + lane() < width ? row[j * T + lane()] : from_f32<E>(0.0f);
        }
    }
    template <typename E>
    __device__ __forceinline__ static void values(const Raw<E>& raw, float (&x)[n]) {
#pragma unroll
        for (int e = 0; e < n; ++e) x[e] = to_f32(((const E*)raw.v)[e]);
    }
    template <typename E>
    __device__ __forceinline__ static void load(const E* row, int width, float (&x)[n]) {
        Raw<E> raw;
        fetch(row, width, raw);
        values(raw, x);
    }
    template <typename E>
    __device__ __forceinline__ static void store(E* row, int width, const float (&x)[n]) {
        if (VEC) {
            const int c = lane() * 8;
            if (c < width) {
                struct alignas(16) Eight { E v[8]; } raw;
#pragma unroll
                for (int e = 0; e < 8; ++e) raw.v[e] = from_f32<E>(x[e]);
#pragma unroll
                for (int q = 0; q < (int)sizeof(E) / 2; ++q) ((uint4*)(row + c))[q] = ((uint4*)&raw)[q];
            }
        } else {
#pragma unroll
            for (int j = 0; j < n; ++j) {
                const int c = j * T + lane();
                if (c < width) row[c] = from_f32<E>(x[j]);
            }
        }
    }
    // both sums over the team; `room` for teams of several warps, `turn` alternates between calls
    __device__ __forceinline__ static void sum(float& a, float& b, float (*room)[32][2], int turn) {
#pragma unroll
        for (int o = (T < 32 ? T : 32) / 2; o; o >>= 1) {
            a += __shfl_xor_sync(kFull, a, o);
            b += __shfl_xor_sync(kFull, b, o);
        }
        if (T > 32) {
            if (lane_id() == 0) {
                room[turn][threadIdx.x >> 5][0] = a;
                room[turn][threadIdx.x >> 5][1] = b;
            }
            __syncthreads();
            a = b = 0.0f;
#pragma unroll
            for (int w = 0; w < T / 32; ++w) {
                a += room[turn][id() * (T / 32) + w][0];
                b += room[turn][id() * (T / 32) + w][1];
            }
        }
    }
    // column sums of the block's teams, in their order, to out[width]; `room` [teams][width] shared
    __device__ __forceinline__ static void columns(const float (&x)[n], int width, float* room, float* out) {
        if (teams == 1) {
#pragma unroll
            for (int j = 0; j < n; ++j)
                if (col(j) < width) out[col(j)] = x[j];
            return;
        }
#pragma unroll
        for (int j = 0; j < n; ++j)
            if (col(j) < width) room[id() * width + col(j)] = x[j];
        __syncthreads();
        for (int c = threadIdx.x; c < width; c += threads) {
            float s = 0.0f;
            for (int t = 0; t < teams; ++t) s += room[t * width + c];
            out[c] = s;
        }
        __syncthreads();
    }
};

// calls f(Team) for rows of `width`
template <bool VEC, typename F>
bcm_status by_width(int64_t width, F&& f) {
    if (width <= 64) return f(Team<8, VEC>());
    if (width <= 256) return f(Team<32, VEC>());
    if (width <= 1024) return f(Team<128, VEC>());
    if (width <= 2048) return f(Team<256, VEC>());
    if (width <= 4096) return f(Team<512, VEC>());
    return f(Team<1024, VEC>());
}
constexpr int64_t kMostWidth = 8192;

// Blocks for rows of `groups` norms each (a block keeps to one group of columns): as many as are resident at once with
// `per_sm` threads on an SM, which the kernels' launch bounds hold to.  More blocks than that ran as one and a half waves
// (the gated norm of 512000 x 256 bf16 took 237 us forward).
constexpr int resident(int threads, int per_sm) { return per_sm > threads ? per_sm / threads : 1; }
inline int64_t most_row_blocks(int64_t groups, int threads, int per_sm) {
    return std::max<int64_t>(1, (int64_t)sm_count() * resident(threads, per_sm) / groups);
}
inline int64_t row_blocks(int64_t rows, int64_t groups, int teams, int threads, int per_sm) {
    return std::max<int64_t>(1, std::min((rows + teams - 1) / teams, most_row_blocks(groups, threads, per_sm)));
}

// out[c] = sum of part[b][c] over the blocks in an order that only their number sets: 32 columns a block, 32 rows of
// threads, so that a thread waits for few loads in turn.  A second block row does the same for the parts behind, to `more`.
static __global__ void __launch_bounds__(1024) add_blocks_kernel(const float* part, int blocks, int64_t cols, float* out, float* more) {
    __shared__ float room[32][33];
    const int64_t c = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
    const int w = threadIdx.x >> 5;
    if (blockIdx.y) {
        part += (int64_t)blocks * cols;
        out = more;
    }
    float s = 0.0f;
    if (c < cols) {
#pragma unroll 8
        for (int b = w; b < blocks; b += 32) s += part[b * cols + c];
    }
    room[w][threadIdx.x & 31] = s;
    __syncthreads();
    if (w == 0 && c < cols) {
        for (int k = 1; k < 32; ++k) s += room[k][threadIdx.x & 31];
        out[c] = s;
    }
}

inline bool on_16(const void* p, int64_t stride_bytes) { return (((uintptr_t)p | (uintptr_t)stride_bytes) & 15) == 0; }

}  // namespace row_norm
}  // namespace bcm
