// tensor5.cuh — the fifth-generation tensor cores (tcgen05) for tiles of 64 rows in bf16 with fp32 sums: operands in
// shared memory (or, for A, in tensor memory), accumulators in tensor memory.
//
// A tile in shared memory has 64 rows of 16, 32 or 64 bf16 in blocks of 8 rows, its 16-byte units swizzled by the row's
// number in its block (a swizzle of the row's own width); wider rows continue in a further tile.  A tile serves as an
// operand in both senses: with its columns along the sum ("K-major") or with its rows along it ("MN-major").
// Accumulators of 64 rows lie in the first 16 lanes of each warp's 32 (row 16 w + i in lane 32 w + i).
#pragma once

#include "common.cuh"

namespace bcm {
namespace t5 {

using bf16 = __nv_bfloat16;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

template <int W>
struct Tile {
    static constexpr int elements = 64 * W, bytes = 2 * elements;
    static constexpr int step_k = 32, step_mn = 32 * W;      // bytes to the next 16 of the sum, K-major (in a row) and MN-major

    // element (row, col); units of 8 columns stay together
    __device__ __forceinline__ static int at(int row, int col) {
        constexpr int units = W / 8;
        return row * W + (((col >> 3) ^ (row / (8 / units) & (units - 1))) << 3) + (col & 7);
    }
    // the lower half of the descriptor of a tile's start, `far` bytes to the tile that continues the rows (MN-major operands
    // that are wider than a tile), and the upper half, the same for all; tiles are aligned to 1024 bytes
    __device__ __forceinline__ static uint32_t low(uint32_t addr, uint32_t far) { return (addr & 0x3ffff) >> 4 | (far >> 4) << 16; }
    static constexpr uint32_t high = (16 * W >> 4) | 1u << 14 | (W == 64 ? 2u : W == 32 ? 4u : 6u) << 29;
};

// bf16 x bf16 -> fp32, 64 rows, n columns; a_mn, b_mn: MN-major operands
__host__ __device__ constexpr uint32_t instr(int n, bool a_mn, bool b_mn) {
    return 1u << 4 | 1u << 7 | 1u << 10 | (a_mn ? 1u << 15 : 0) | (b_mn ? 1u << 16 : 0) | (uint32_t)(n >> 3) << 17 | (uint32_t)(64 >> 4) << 24;
}

// an operand in shared memory: the two halves of its descriptor
struct Desc {
    uint32_t low, high;
};

__device__ __forceinline__ void mma(uint32_t d, Desc a, Desc b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %4};\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %5, p;\n\t}" ::"r"(d), "r"(a.low), "r"(a.high), "r"(b.low), "r"(b.high), "r"(idesc),
        "r"((uint32_t)add)
        : "memory");
}
// A at an address of tensor memory
__device__ __forceinline__ void mma(uint32_t d, uint32_t a, Desc b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d), "r"(a), "r"(b.low), "r"(b.high), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}

// arrives at the barrier once all products issued before by this thread are done
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void bar_init(uint64_t* bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
// Waits for the phase, a warp as one (its threads leave together: what follows moves all their registers to or from tensor
// memory).  After 2^31 cycles (about a second; products of a tile take microseconds) it gives up and sets *failed to the bits
// of a NaN, and where that is set it does not wait.
__device__ __forceinline__ void bar_wait(uint64_t* bar, uint32_t phase, int* failed) {
    __syncwarp();
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        ".reg .b32 f;\n\t"
        ".reg .b64 t, s;\n\t"
        "ld.volatile.shared.b32 f, [%2];\n\t"
        "setp.ne.b32 p, f, 0;\n\t"
        "vote.sync.any.pred p, p, 0xffffffff;\n\t"
        "@p bra.uni DONE;\n\t"
        "mov.u64 s, %%clock64;\n"
        "AGAIN:\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%0], %1;\n\t"
        "vote.sync.all.pred p, p, 0xffffffff;\n\t"
        "@p bra.uni DONE;\n\t"
        "mov.u64 t, %%clock64;\n\t"
        "sub.u64 t, t, s;\n\t"
        "setp.lt.u64 p, t, 0x80000000;\n\t"
        "vote.sync.any.pred p, p, 0xffffffff;\n\t"
        "@p bra.uni AGAIN;\n\t"
        "st.volatile.shared.b32 [%2], 0x7fc00000;\n"
        "DONE:\n\t"
        "}" ::"r"(smem_u32(bar)), "r"(phase), "r"(smem_u32(failed))
        : "memory");
    __syncwarp();
}

// a warp lets 2^31 cycles pass where *failed is set (without a branch that the compiler sees: one behind a kernel's walk made
// it hold more registers in the walk)
__device__ __forceinline__ void rest_if(const int* failed) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        ".reg .b32 f;\n\t"
        ".reg .b64 t, s;\n\t"
        "ld.volatile.shared.b32 f, [%0];\n\t"
        "setp.eq.b32 p, f, 0;\n\t"
        "@p bra DONE;\n\t"
        "mov.u64 s, %%clock64;\n"
        "AGAIN:\n\t"
        "mov.u64 t, %%clock64;\n\t"
        "sub.u64 t, t, s;\n\t"
        "setp.lt.u64 p, t, 0x80000000;\n\t"
        "@p bra AGAIN;\n"
        "DONE:\n\t"
        "}" ::"r"(smem_u32(failed))
        : "memory");
    __syncwarp();
}

// one thread of a warp (all of it, together), known to the compiler to be one: what it computes alike for the whole warp
// (descriptors) stays in uniform registers, from which products are issued
__device__ __forceinline__ bool elect() {
    uint32_t is;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(is));
    return is != 0;
}
__device__ __forceinline__ int warp_id() { return __shfl_sync(kFull, (int)(threadIdx.x >> 5), 0); }

// writes to shared memory become visible to the tensor cores' reads
__device__ __forceinline__ void fence_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// one warp; columns a power of two of at least 32
__device__ __forceinline__ void alloc(uint32_t* addr, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(addr)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void dealloc(uint32_t addr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}

// All threads of a warp take part in what follows, together: callers bring the warp together before (a wait or a store
// under a condition may have left its threads apart).  A load's registers hold nothing before its wait, so both are one
// statement.

// 16 rows x 16 columns of an accumulator: row l / 4, columns 2 (l % 4) and the next (+ 8: second half), then row l / 4 + 8
__device__ __forceinline__ void ld16(float (&r)[2][4], uint32_t addr) {
    uint32_t x[8];
    __syncwarp();
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=&r"(x[0]), "=&r"(x[1]), "=&r"(x[2]), "=&r"(x[3]), "=&r"(x[4]), "=&r"(x[5]), "=&r"(x[6]), "=&r"(x[7])
                 : "r"(addr)
                 : "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i >> 2][i & 3] = __uint_as_float(x[i]);
}
// 16 rows x 8 columns
__device__ __forceinline__ void ld8(float (&r)[4], uint32_t addr) {
    uint32_t x[4];
    __syncwarp();
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x1.b32 {%0,%1,%2,%3}, [%4];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=&r"(x[0]), "=&r"(x[1]), "=&r"(x[2]), "=&r"(x[3])
                 : "r"(addr)
                 : "memory");
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = __uint_as_float(x[i]);
}
// 32 columns
__device__ __forceinline__ void ld32(float (&r)[4][4], uint32_t addr) {
    uint32_t x[16];
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=&r"(x[0]), "=&r"(x[1]), "=&r"(x[2]), "=&r"(x[3]), "=&r"(x[4]), "=&r"(x[5]), "=&r"(x[6]), "=&r"(x[7]), "=&r"(x[8]), "=&r"(x[9]), "=&r"(x[10]),
          "=&r"(x[11]), "=&r"(x[12]), "=&r"(x[13]), "=&r"(x[14]), "=&r"(x[15])
        : "r"(addr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i >> 2][i & 3] = __uint_as_float(x[i]);
}
// 16 columns at each of two addresses
__device__ __forceinline__ void ld16x2(float (&r)[2][4], uint32_t addr, float (&r2)[2][4], uint32_t addr2) {
    uint32_t x[16];
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%16];\n\t"
        "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%8,%9,%10,%11,%12,%13,%14,%15}, [%17];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=&r"(x[0]), "=&r"(x[1]), "=&r"(x[2]), "=&r"(x[3]), "=&r"(x[4]), "=&r"(x[5]), "=&r"(x[6]), "=&r"(x[7]), "=&r"(x[8]), "=&r"(x[9]), "=&r"(x[10]),
          "=&r"(x[11]), "=&r"(x[12]), "=&r"(x[13]), "=&r"(x[14]), "=&r"(x[15])
        : "r"(addr), "r"(addr2)
        : "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        r[i >> 2][i & 3] = __uint_as_float(x[i]);
        r2[i >> 2][i & 3] = __uint_as_float(x[8 + i]);
    }
}
// 16 rows x 16 bf16 columns of an A operand (8 columns of 32 bits), in the accumulators' layout: r[2 q + half] the pair
// of columns 8 q + 2 (l % 4), half: row l / 4 + 8
__device__ __forceinline__ void st16(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
    __syncwarp();
    asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r0), "r"(r1), "r"(r2), "r"(r3) : "memory");
}
// 16 rows x 16 columns of an accumulator
__device__ __forceinline__ void st_acc16(uint32_t addr, const float (&r)[2][4]) {
    __syncwarp();
    asm volatile("tcgen05.st.sync.aligned.16x256b.x2.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(__float_as_uint(r[0][0])),
                 "r"(__float_as_uint(r[0][1])), "r"(__float_as_uint(r[0][2])), "r"(__float_as_uint(r[0][3])), "r"(__float_as_uint(r[1][0])),
                 "r"(__float_as_uint(r[1][1])), "r"(__float_as_uint(r[1][2])), "r"(__float_as_uint(r[1][3]))
                 : "memory");
}
__device__ __forceinline__ void wait_st() {
    __syncwarp();
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

}  // namespace t5
}  // namespace bcm
