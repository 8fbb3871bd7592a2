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

    __device__ __forceinline__ static int lane() { return threadIdx.x % T; }
    __device__ __forceinline__ static int id() { return threadIdx.x / T; }
    __device__ __forceinline__ static int col(int j) { return VEC ? lane() * 8 + j : j * T + lane(); }

    template <typename E>
    __device__ __forceinline__ static void load(const E* row, int width, float (&x)[n]) {
        if (VEC) {
            struct alignas(16) Eight { E v[8]; } raw;
            const int c = lane() * 8;
            if (c < width) {
#pragma unroll
                for (int q = 0; q < (int)sizeof(E) / 2; ++q) ((uint4*)&raw)[q] = ((const uint4*)(row + c))[q];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = c < width ? to_f32(raw.v[e]) : 0.0f;
        } else {
#pragma unroll
            for (int j = 0; j < n; ++j) {
                const int c = j * T + lane();
                x[j] = c < width ? to_f32(row[c]) : 0.0f;
            }
        }
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

// Blocks for rows of `groups` norms each (a block keeps to one group of columns): about as many as stay resident.
constexpr int kThreadsPerSm = 1536;
inline int64_t most_row_blocks(int64_t groups, int threads) {
    return std::max<int64_t>(1, (int64_t)sm_count() * std::max(1, kThreadsPerSm / threads) / groups);
}
inline int64_t row_blocks(int64_t rows, int64_t groups, int teams, int threads) {
    return std::max<int64_t>(1, std::min((rows + teams - 1) / teams, most_row_blocks(groups, threads)));
}

// out[c] = sum of part[b][c] over the blocks in their order: 32 columns a block, 8 rows of threads
static __global__ void __launch_bounds__(256) add_blocks_kernel(const float* part, int blocks, int64_t cols, float* out) {
    __shared__ float room[8][33];
    const int64_t c = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31);
    const int w = threadIdx.x >> 5;
    float s = 0.0f;
    if (c < cols) {
#pragma unroll 4
        for (int b = w; b < blocks; b += 8) s += part[b * cols + c];
    }
    room[w][threadIdx.x & 31] = s;
    __syncthreads();
    if (w == 0 && c < cols) {
        for (int k = 1; k < 8; ++k) s += room[k][threadIdx.x & 31];
        out[c] = s;
    }
}

inline bool on_16(const void* p, int64_t stride_bytes) { return (((uintptr_t)p | (uintptr_t)stride_bytes) & 15) == 0; }

}  // namespace row_norm
}  // namespace bcm
