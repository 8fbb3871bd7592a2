// decay_attn.cuh — what the kernels of the linear attention with a decay for each head share: tiles and their products,
// the decays' running sums, the state, and the work items that sequences are cut into.
//
// Per head, a_t = exp(g_t):  S_t = a_t S_(t-1) + k_t v_t^T (N x P),  y_t = S_t^T q_t.
// In chunks of 64 tokens with G the running sum of g inside the chunk, D_ij = exp(G_i - G_j) for j <= i, 0 elsewhere:
//   Y = ((Q K^T) o D) V + diag(exp G) Q S_in,    S_out = exp(G_64) S_in + sum_j exp(G_64 - G_j) k_j v_j^T.
// All products are of 64 rows and run on the tensor cores; a block walks the chunks of its item, 64 columns of the
// values wide.
//
// Numbers.  The products are of bf16 with fp32 sums.  An operand of more bits is a sum of bf16 pieces, each the rounding
// of what the pieces before it left: float32 is three pieces (exact), float16 two (exact), and what a kernel computes
// itself (masked scores, states, values times decays) has as many as its products need: two (relative 2^-18) where
// they end in 16 bits, three where they end in float32.  Of the pieces' products those whose weight lies below that are
// left out, and the small ones are added up first: the tensor cores cut sums off instead of rounding them, so that few
// additions may be made at the full sum.  States are float32 between chunks.  G is summed in float64 and kept as two
// floats, so that a difference of two of its values keeps full precision after a decay of any size.
#pragma once

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "tensor5.cuh"

namespace bcm {
namespace decay_attn {

using bf16 = __nv_bfloat16;

constexpr int kChunk = 64;
constexpr int kP = 64;        // columns of the values that a block takes

// pieces of an input, and of what is computed for products that end in T; for those that end in float32 there are three
template <typename T> struct Pieces;
template <> struct Pieces<float> { static constexpr int in = 3, out = 3; };
template <> struct Pieces<__half> { static constexpr int in = 2, out = 2; };
template <> struct Pieces<bf16> { static constexpr int in = 1, out = 2; };
constexpr int kFull3 = 3;

// Tiles of 64 rows and NT columns (of queries, keys, states): one of up to 64 columns, or two of 64
template <int NT>
struct Wide {
    static constexpr int W = NT < 64 ? NT : 64;
    using Tile = t5::Tile<W>;
    static constexpr int elements = 64 * NT, bytes = 2 * elements;     // of a piece
    __device__ __forceinline__ static int at(int row, int col) { return col / W * Tile::elements + Tile::at(row, col % W); }
};

__device__ __forceinline__ float low_f(uint32_t r) { return __uint_as_float(r << 16); }
__device__ __forceinline__ float high_f(uint32_t r) { return __uint_as_float(r & 0xffff0000u); }

__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// two values as M pieces each
template <int M>
__device__ __forceinline__ void split(float x, float y, uint32_t (&r)[M]) {
#pragma unroll
    for (int m = 0; m < M; ++m) {
        r[m] = pack(x, y);
        if (m + 1 < M) {
            x -= low_f(r[m]);
            y -= high_f(r[m]);
        }
    }
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// --------------------------------------------------------------------- products ----
// An operand of NT columns at a shared address, its pieces one behind the other; K: columns along the sum, else rows.
template <int NT, bool K>
struct Operand {
    using X = Wide<NT>;
    uint32_t addr;
    __device__ __forceinline__ uint64_t desc(int piece, int step) const {
        constexpr int in_tile = X::W / 16;
        const uint32_t off = piece * X::bytes + (K ? step / in_tile * X::Tile::bytes + step % in_tile * X::Tile::step_k : step * X::Tile::step_mn);
        return X::Tile::desc(addr + off, X::Tile::bytes);
    }
};

// d (+)= A B over `steps` of 16, products (s, u) of A's NA and B's NB pieces with s + u < D, small ones first; one thread.
// a(s, step), b(u, step): descriptors (or A's address in tensor memory)
template <int NA, int NB, int D, typename FA, typename FB>
__device__ __forceinline__ void products(uint32_t d, FA&& a, FB&& b, int steps, uint32_t idesc, bool add) {
#pragma unroll
    for (int order = (NA + NB - 2 < D - 1 ? NA + NB - 2 : D - 1); order >= 0; --order)
#pragma unroll
        for (int s = 0; s < NA; ++s) {
            const int u = order - s;
            if (u < 0 || u >= NB) continue;
#pragma unroll 1
            for (int k = 0; k < steps; ++k) {
                const auto x = a(s, k);
                if constexpr (sizeof(x) == 4) t5::mma_ts(d, x, b(u, k), idesc, add);
                else t5::mma_ss(d, x, b(u, k), idesc, add);
                add = true;
            }
        }
}

__device__ __forceinline__ void named_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// ------------------------------------------------------------------- decays ----
// Of one chunk: the running sums of g log2(e) as two floats, what has decayed since the chunk's start and what will
// until its end, and the decay of the whole chunk.
struct alignas(16) Decays {
    float hi[kChunk], lo[kChunk], since[kChunk], until[kChunk];
    float whole, pad[3];
};

// D_ij, i >= j
__device__ __forceinline__ float between(float hi_i, float lo_i, float hi_j, float lo_j) {
    return ex2((hi_i - hi_j) + (lo_i - lo_j));
}

constexpr double kLog2e = 1.4426950408889634;

// One warp; g0, g1 the logarithms of token 2 lane and 2 lane + 1 (0 behind the last).  A decay below 2^-256 is 0
// in float32 next to anything, and bounded so it leaves the sums their precision.  The coarse part is a multiple of
// 2^-9 below 2^15: differences of it are exact.  Returns the chunk's sum.
__device__ __forceinline__ double decays_of(Decays& d, float g0, float g1) {
    const int l = lane_id();
    const double x0 = g0 < -177.0f ? -256.0 : (double)g0 * kLog2e, x1 = g1 < -177.0f ? -256.0 : (double)g1 * kLog2e;
    double s = x0 + x1;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const double o = __shfl_up_sync(kFull, s, off);
        if (l >= off) s += o;
    }
    const double all = __shfl_sync(kFull, s, 31);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const double v = q ? s : s - x1;
        const float h = rintf((float)v * 512.0f) * (1.0f / 512.0f);
        const int at = 2 * l + q;
        d.hi[at] = h;
        d.lo[at] = (float)(v - (double)h);
        d.since[at] = exp2f((float)v);
        d.until[at] = exp2f((float)(all - v));
    }
    if (l == 0) d.whole = exp2f((float)all);
    return all;
}

// ---------------------------------------------------------------- work items ----
// A sequence is cut into items of `span` tokens (a multiple of the chunk); a packed batch has them in a table.
struct Item {
    int seq, t0, t1;          // sequence and tokens (of the packed rows, or of the sequence's own), seq < 0: none
    int chunk;                // number of its first chunk among all the kept states
    int first, last;          // whether it begins and whether it ends its sequence
};

struct Tables {               // of a packed batch, in the workspace
    Item* items;
    int* seq_item;            // [batch + 1]: each sequence's first item
};

struct Sizes {
    int batch, heads, qk_heads, n, p, seqlen;
    int span, items, per_seq; // items in all (packed: at most), per sequence (dense)
    int chunks;               // kept states of a head in all (packed: at most)
    int slices;               // of kP columns of the values
    const int32_t* cu;
    Tables tables;
};

__device__ __forceinline__ Item item_of(const Sizes& z, int i) {
    if (z.cu) return z.tables.items[i];
    Item it;
    it.seq = i / z.per_seq;
    const int s = i - it.seq * z.per_seq;
    it.t0 = s * z.span;
    it.t1 = min(z.seqlen, it.t0 + z.span);
    it.chunk = it.seq * ((z.seqlen + kChunk - 1) / kChunk) + it.t0 / kChunk;
    it.first = s == 0;
    it.last = s == z.per_seq - 1;
    return it;
}

// rows of a tensor (batch, tokens, heads, width); packed: b is 0
struct Rows {
    const void* p;
    int64_t sb, st, sh;
};

template <typename T>
__device__ __forceinline__ const T* row_ptr(const Rows& r, const Sizes& z, int seq, int64_t t, int h) {
    return (const T*)r.p + (z.cu ? 0 : (int64_t)seq * r.sb) + t * r.st + (int64_t)h * r.sh;
}

// ---------------------------------------------------------------------- tiles ----
// whether v's pieces are not finite
__device__ __forceinline__ bool not_finite(float v) { return !(fabsf(v) <= 3.38e38f); }

template <typename T> struct alignas(16) Eight { T v[8]; };

// 64 rows x W columns on their way to shared memory: each of TH threads has groups of eight columns.  Rows and columns
// behind the last are 0.
template <typename T, int W, int TH>
struct Pending {
    static constexpr int all = 64 * W / 8, n = (all + TH - 1) / TH;
    Eight<T> g[n];

    __device__ __forceinline__ static int row(int i) { return (threadIdx.x + i * TH) / (W / 8); }
    __device__ __forceinline__ static int col(int i) { return (threadIdx.x + i * TH) % (W / 8) * 8; }

    // how: elements at a time that the rows' alignment allows (8, 2 or 1)
    __device__ __forceinline__ void fetch(const T* src, int64_t stride, int rows, int cols, int how) {
        if (how == 8) {
#pragma unroll
            for (int i = 0; i < n; ++i) {
                const T* p = src + row(i) * stride + col(i);
                if (row(i) < rows && col(i) + 8 <= cols) {
#pragma unroll
                    for (int u = 0; u < (int)sizeof(T) / 2; ++u) ((uint4*)&g[i])[u] = ((const uint4*)p)[u];
                } else {
#pragma unroll
                    for (int u = 0; u < 8; ++u) g[i].v[u] = row(i) < rows && col(i) + u < cols ? p[u] : from_f32<T>(0.0f);
                }
            }
            return;
        }
        using Two = typename std::conditional<sizeof(T) == 4, uint2, uint32_t>::type;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const T* p = src + row(i) * stride + col(i);
            const int in = row(i) < rows ? cols - col(i) : 0;
            if (how == 2) {
#pragma unroll
                for (int u = 0; u < 8; u += 2) {
                    if (u + 2 <= in) {
                        *(Two*)&g[i].v[u] = *(const Two*)(p + u);
                    } else {
                        g[i].v[u] = u < in ? p[u] : from_f32<T>(0.0f);
                        g[i].v[u + 1] = from_f32<T>(0.0f);
                    }
                }
            } else {
#pragma unroll
                for (int u = 0; u < 8; ++u) g[i].v[u] = u < in ? p[u] : from_f32<T>(0.0f);
            }
        }
    }
    __device__ __forceinline__ bool bad() const {
        bool b = false;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            if (all % TH != 0 && threadIdx.x + i * TH >= all) continue;
            if constexpr (std::is_same<T, bf16>::value) {
                const uint4 q = *(const uint4*)&g[i];
                const uint32_t e = 0x7f807f80u;                        // exponents of all ones
                b |= (__vcmpeq2(q.x & e, e) | __vcmpeq2(q.y & e, e) | __vcmpeq2(q.z & e, e) | __vcmpeq2(q.w & e, e)) != 0;
            } else {
#pragma unroll
                for (int u = 0; u < 8; ++u) b |= not_finite(to_f32(g[i].v[u]));
            }
        }
        return b;
    }
    // the values' pieces
    __device__ __forceinline__ void put(bf16* dst) const {
        constexpr int NS = Pieces<T>::in;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            if (all % TH != 0 && threadIdx.x + i * TH >= all) continue;
            bf16* to = dst + Wide<W>::at(row(i), col(i));
            if constexpr (NS == 1) {
                *(uint4*)to = *(const uint4*)&g[i];
            } else {
                uint32_t r[4][NS];
#pragma unroll
                for (int u = 0; u < 4; ++u) split<NS>(to_f32(g[i].v[2 * u]), to_f32(g[i].v[2 * u + 1]), r[u]);
#pragma unroll
                for (int s = 0; s < NS; ++s) *(uint4*)(to + s * Wide<W>::elements) = make_uint4(r[0][s], r[1][s], r[2][s], r[3][s]);
            }
        }
    }
    // three pieces of the values times their row's weight
    __device__ __forceinline__ void put_weighted(bf16* dst, const float* weight) const {
#pragma unroll
        for (int i = 0; i < n; ++i) {
            if (all % TH != 0 && threadIdx.x + i * TH >= all) continue;
            bf16* to = dst + Wide<W>::at(row(i), col(i));
            const float w = weight[row(i)];
            uint32_t r[4][kFull3];
#pragma unroll
            for (int u = 0; u < 4; ++u) split<kFull3>(to_f32(g[i].v[2 * u]) * w, to_f32(g[i].v[2 * u + 1]) * w, r[u]);
#pragma unroll
            for (int s = 0; s < kFull3; ++s) *(uint4*)(to + s * Wide<W>::elements) = make_uint4(r[0][s], r[1][s], r[2][s], r[3][s]);
        }
    }
};

// elements at a time for rows that start at p and lie `stride` apart
template <typename T>
__device__ __forceinline__ int alignment(const T* p, int64_t stride) {
    const uint64_t x = (uint64_t)(uintptr_t)p | (uint64_t)(stride * (int64_t)sizeof(T));
    return (x & 15) == 0 ? 8 : (x & (2 * sizeof(T) - 1)) == 0 ? 2 : 1;
}

// two neighbouring values from their pieces
template <int NS>
__device__ __forceinline__ float2 from_pieces(const bf16* m, int piece) {
    float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int s = NS - 1; s >= 0; --s) {
        const uint32_t r = *(const uint32_t*)(m + s * piece);
        v.x += low_f(r);
        v.y += high_f(r);
    }
    return v;
}

// Writes a warp's 16 x 16 fragment (rows r0 and r0 + 8 of this lane) to rows of `st` elements; `how` as in alignment().
// 16-bit values of four lanes are brought together, so that a lane stores 16 bytes.
template <typename T>
__device__ __forceinline__ void store_rows(T* out, int64_t st, int rows, int cols, int r0, int c0, const float (&x)[2][4], int how) {
    const int lq = lane_id() & 3;
    if (sizeof(T) == 2 && how == 8 && c0 + 16 <= cols) {
        // two tiles of 8 columns, rows r0 and r0 + 8: lane lq gathers tile lq & 1 of row r0 + 8 (lq >> 1)
        uint32_t v[4];                                                 // [tile + 2 half]
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                struct alignas(4) Two { T a, b; } t{from_f32<T>(x[q][2 * h]), from_f32<T>(x[q][2 * h + 1])};
                v[q + 2 * h] = *(uint32_t*)&t;
            }
        uint32_t a = lq & 1 ? v[0] : v[1], b = lq & 1 ? v[2] : v[3];
        a = __shfl_xor_sync(kFull, a, 1);
        b = __shfl_xor_sync(kFull, b, 1);
        // now this lane and its neighbour hold tile lq & 1 of both rows: (mine, the neighbour's) words
        uint32_t m0 = lq & 1 ? v[1] : v[0], m1 = lq & 1 ? v[3] : v[2];
        uint32_t lo0 = lq & 1 ? a : m0, hi0 = lq & 1 ? m0 : a, lo1 = lq & 1 ? b : m1, hi1 = lq & 1 ? m1 : b;
        const bool up = lq >> 1;
        uint32_t s0 = up ? lo0 : lo1, s1 = up ? hi0 : hi1;
        s0 = __shfl_xor_sync(kFull, s0, 2);
        s1 = __shfl_xor_sync(kFull, s1, 2);
        const uint32_t k0 = up ? lo1 : lo0, k1 = up ? hi1 : hi0;
        const uint4 all = up ? make_uint4(s0, s1, k0, k1) : make_uint4(k0, k1, s0, s1);
        const int r = r0 + 8 * (lq >> 1);
        if (r < rows) *(uint4*)(out + r * st + c0 + 8 * (lq & 1)) = all;
        return;
    }
    struct alignas(2 * sizeof(T)) Two { T a, b; };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int r = r0 + 8 * h;
        if (r < rows)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int c = c0 + 8 * q + 2 * lq;
                const T a = from_f32<T>(x[q][2 * h]), b = from_f32<T>(x[q][2 * h + 1]);
                T* to = out + r * st + c;
                if (how > 1 && c + 1 < cols) {
                    *(Two*)to = Two{a, b};
                } else {
                    if (c < cols) to[0] = a;
                    if (c + 1 < cols) to[1] = b;
                }
            }
    }
}

// ---------------------------------------------------------------------- state ----
// The transposed state (64 columns of the values by NT of the keys) in the registers of four warps (which begin at a
// multiple of four), in the accumulators' layout.
template <int NT>
struct State {
    float s[NT / 8][4];

    __device__ __forceinline__ static int p(int half) { return ((threadIdx.x >> 5) & 3) * 16 + (lane_id() >> 2) + 8 * half; }
    __device__ __forceinline__ static int n(int c) { return 8 * c + 2 * (lane_id() & 3); }

    // calls f(value, value, p, n) for pairs of neighbouring n
    template <typename F>
    __device__ __forceinline__ void pairs(F&& f) {
#pragma unroll
        for (int c = 0; c < NT / 8; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) f(s[c][2 * h], s[c][2 * h + 1], p(h), n(c));
    }
    __device__ __forceinline__ void zero() {
        pairs([](float& x, float& y, int, int) { x = y = 0.0f; });
    }
    // from (n, p) of rows of `stride` floats
    __device__ __forceinline__ void load(const float* src, int rows, int cols, int stride) {
        pairs([&](float& x, float& y, int p, int n) {
            x = p < cols && n < rows ? src[(int64_t)n * stride + p] : 0.0f;
            y = p < cols && n + 1 < rows ? src[(int64_t)(n + 1) * stride + p] : 0.0f;
        });
    }
    __device__ __forceinline__ void store(float* dst, int rows, int cols, int stride) {
        pairs([&](float& x, float& y, int p, int n) {
            if (p < cols && n < rows) dst[(int64_t)n * stride + p] = x;
            if (p < cols && n + 1 < rows) dst[(int64_t)(n + 1) * stride + p] = y;
        });
    }
    // its pieces to shared memory; whether a value was not finite
    template <int MS>
    __device__ __forceinline__ bool put(bf16* dst) {
        bool bad = false;
        pairs([&](float& x, float& y, int p, int n) {
            uint32_t q[MS];
            split<MS>(x, y, q);
            bad |= not_finite(x) | not_finite(y);
            bf16* to = dst + Wide<NT>::at(p, n);
#pragma unroll
            for (int k = 0; k < MS; ++k) *(uint32_t*)(to + k * Wide<NT>::elements) = q[k];
        });
        return bad;
    }
    // s = whole s + the accumulator at addr (this warp's lanes)
    __device__ __forceinline__ void advance(uint32_t addr, float whole) {
#pragma unroll
        for (int c = 0; c < NT / 16; ++c) {
            float x[2][4];
            t5::ld16(x, addr + 16 * c);
            t5::wait_ld();
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[2 * c + q][e] = fmaf(whole, s[2 * c + q][e], x[q][e]);
        }
    }
};

// What has to be initialised and awaited: barriers of the tensor cores' work, the tensor memory's address, and whether
// a wait has run out of time, after which no wait is made any more and results are NaN.
template <int BARS>
struct Sync {
    uint64_t bars[BARS];
    uint32_t tmem;
    int failed;

    __device__ __forceinline__ void init(uint32_t cols) {
        if (threadIdx.x < 32) t5::alloc(&tmem, cols);
        if (threadIdx.x == 0) {
            failed = 0;
            for (int i = 0; i < BARS; ++i) t5::bar_init(&bars[i], 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        t5::fence_before();
        __syncthreads();
        t5::fence_after();
    }
    __device__ __forceinline__ void wait(int bar, uint32_t phase) {
        if (!*(volatile int*)&failed && !t5::bar_wait(&bars[bar], phase)) *(volatile int*)&failed = 1;
        t5::fence_after();
    }
    // the whole block, all products awaited
    __device__ __forceinline__ void end(uint32_t cols) {
        t5::fence_before();
        __syncthreads();
        t5::fence_after();
        if (threadIdx.x < 32) t5::dealloc(tmem, cols);
    }
};

// dynamic shared memory from the next multiple of 1024 bytes (tiles want it)
__device__ __forceinline__ unsigned char* tiles_base(unsigned char* raw) { return raw + ((1024 - (t5::smem_u32(raw) & 1023)) & 1023); }

// The rows of a packed batch behind its last sequence are written as zeros: each block has its share of them.
template <typename T>
__device__ __forceinline__ void zero_rows(T* out, int64_t from, int64_t rows, int64_t row_stride, int cols, int part, int parts) {
    for (int64_t t = from + part; t < rows; t += parts)
        for (int c = threadIdx.x; c < cols; c += blockDim.x) out[t * row_stride + c] = from_f32<T>(0.0f);
}

}  // namespace decay_attn
}  // namespace bcm

// ------------------------------------------------------------------ host side ----
namespace bcm {
namespace decay_attn {

// The state that every item but a sequence's first (backwards: last) enters with, in two steps: each item's own part
// (`part`, from a zero state) and decay, then sums along the sequence.
struct Parts {
    float* state;             // [items][heads][n][p]: the item's part, then the state that it enters with
    float* whole;             // [items][heads]: its decay
};

// Sizes and tables of a call; what it takes of the workspace (offsets from its start, 0 bytes where there is none)
struct Plan {
    Sizes z;
    size_t items_at, seq_at, state_at, whole_at, bytes;
    bool cut;                 // some sequence may have more than one item
};

bcm_status check(const bcm_decay_attn_args* a, const char* what);
Plan plan_of(const bcm_decay_attn_args* a, bool backward);
bcm_status fill_tables(Plan& plan, void* workspace, cudaStream_t stream);
Parts parts_of(const Plan& plan, void* workspace);
// entering states along each sequence, from `end` (nullptr: zeros) at its first (backwards: last) item
bcm_status join(const Plan& plan, const Parts& parts, const float* end, bool backward, cudaStream_t stream);

inline Rows rows_of(const void* p, int64_t sb, int64_t st, int64_t sh) { return Rows{p, sb, st, sh}; }

// calls f(T, NT as an integral constant)
template <typename F>
bcm_status dispatch(bcm_dtype t, int64_t n, F&& f) {
    return dispatch_dtype(t, [&](auto type) -> bcm_status {
        if (n <= 16) return f(type, std::integral_constant<int, 16>());
        if (n <= 32) return f(type, std::integral_constant<int, 32>());
        if (n <= 64) return f(type, std::integral_constant<int, 64>());
        return f(type, std::integral_constant<int, 128>());
    });
}

// a kernel's dynamic shared memory, allowed once per device; the opt-in is per kernel
template <typename K>
bcm_status allow_smem(K kernel, size_t bytes) {
    BCM_CUDA_TRY(cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    return BCM_OK;
}

// ------------------------------------------------------------- an item's part ----
// Forward: sum_j exp(G_end - G_j) k_j v_j^T.  Backward (of the state's gradient, towards the item's start):
// sum_i exp(G_i) q_i dy_i^T.  a holds k or q, b v or dy.
struct PartArgs {
    Sizes z;
    Rows a, b;                // b.p NULL: zeros
    const float* g;
    int64_t g_sb, g_st, g_sh;
    Parts parts;
};

template <typename T, int NT>
struct PartSmem {
    bf16 a[Pieces<T>::in][Wide<NT>::elements];
    bf16 bw[kFull3][Wide<kP>::elements];
    Decays d[2];
    Sync<1> sync;
};

constexpr int kPartThreads = 128;

template <typename T, int NT, bool BACK>
__global__ void __launch_bounds__(kPartThreads) part_kernel(const __grid_constant__ PartArgs p) {
    extern __shared__ unsigned char smem_raw[];
    PartSmem<T, NT>& sm = *(PartSmem<T, NT>*)tiles_base(smem_raw);
    constexpr int NS = Pieces<T>::in;
    constexpr uint32_t kCols = NT < 32 ? 32 : NT;
    const Sizes& z = p.z;
    const int across = z.heads * z.slices;
    const int item = blockIdx.x / across, hs = blockIdx.x % across, h = hs / z.slices, col = hs % z.slices * kP;
    const Item it = item_of(z, item);
    if (it.seq < 0 || (BACK ? it.first : it.last)) return;
    const int cols = min(kP, z.p - col), ha = h / (z.heads / z.qk_heads);
    const T* a = row_ptr<T>(p.a, z, it.seq, it.t0, ha);
    const T* b = row_ptr<T>(p.b, z, it.seq, it.t0, h) + col;
    const float* g = p.g + (z.cu ? 0 : it.seq * p.g_sb) + it.t0 * p.g_st + h * p.g_sh;
    const int va = alignment(a, p.a.st), vb = alignment(b, p.b.st);
    const int len = it.t1 - it.t0, nc = (len + kChunk - 1) / kChunk, l = lane_id();
    State<NT> st;
    st.zero();
    double all = 0.0;
    Pending<T, NT, kPartThreads> pa;
    Pending<T, kP, kPartThreads> pb;
    float g0 = 0.0f, g1 = 0.0f;
    auto fetch = [&](int i) {                             // the i-th chunk of the walk
        const int t = (BACK ? nc - 1 - i : i) * kChunk, rows = min(kChunk, len - t);
        pa.fetch(a + t * p.a.st, p.a.st, rows, z.n, va);
        pb.fetch(b + t * p.b.st, p.b.st, p.b.p ? rows : 0, cols, vb);
        if (threadIdx.x < 32) {
            g0 = 2 * l < rows ? g[(int64_t)(t + 2 * l) * p.g_st] : 0.0f;
            g1 = 2 * l + 1 < rows ? g[(int64_t)(t + 2 * l + 1) * p.g_st] : 0.0f;
        }
    };
    if (nc > 0) fetch(0);
    sm.sync.init(kCols);
    if (threadIdx.x < 32) all += decays_of(sm.d[0], g0, g1);
    const uint32_t acc = sm.sync.tmem;
    for (int i = 0; i < nc; ++i) {
        __syncthreads();
        // (what is not finite stays so in the sums, and the walk takes such chunks token by token)
        const Decays& d = sm.d[i & 1];
        pa.put(sm.a[0]);
        pb.put_weighted(sm.bw[0], BACK ? d.since : d.until);
        t5::fence_smem();
        t5::fence_before();
        __syncthreads();
        if (threadIdx.x == 0) {
            t5::fence_after();
            const Operand<kP, false> A{t5::smem_u32(sm.bw)};
            const Operand<NT, false> B{t5::smem_u32(sm.a)};
            products<kFull3, NS, kFull3>(acc, [&](int s, int k) { return A.desc(s, k); }, [&](int u, int k) { return B.desc(u, k); },
                                         kChunk / 16, t5::instr(NT, true, true), false);
            t5::commit(&sm.sync.bars[0]);
        }
        __syncwarp();
        if (i + 1 < nc) {
            fetch(i + 1);
            if (threadIdx.x < 32) all += decays_of(sm.d[(i + 1) & 1], g0, g1);
        }
        sm.sync.wait(0, i & 1);
        st.advance(acc + ((threadIdx.x >> 5) << 21), d.whole);
        t5::fence_before();
    }
    if (sm.sync.failed) st.pairs([](float& x, float& y, int, int) { x = y = __int_as_float(0x7fc00000); });
    const int64_t at = (int64_t)item * z.heads + h;
    st.store(p.parts.state + at * z.n * z.p + col, z.n, cols, z.p);
    if (threadIdx.x == 0 && col == 0) p.parts.whole[at] = exp2f((float)all);
    sm.sync.end(kCols);
}

template <typename T, int NT, bool BACK>
bcm_status launch_part(const PartArgs& p, cudaStream_t stream) {
    constexpr size_t smem = sizeof(PartSmem<T, NT>) + 1024;
    auto kernel = part_kernel<T, NT, BACK>;
    bcm_status st = allow_smem(kernel, smem);
    if (st != BCM_OK) return st;
    kernel<<<(unsigned)(p.z.items * p.z.heads * p.z.slices), kPartThreads, smem, stream>>>(p);
    BCM_LAUNCH_CHECK();
    return BCM_OK;
}

}  // namespace decay_attn
}  // namespace bcm
