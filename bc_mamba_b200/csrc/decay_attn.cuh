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
// itself (masked scores, states, values times decays) has as many as its products need: two (within 2^-17, 2.5e-6 in the
// root mean square) where they end in 16 bits, three where they end in float32.  Of the pieces' products those that lie
// below that are left out: under 2^-24 of the whole product where results are float32 (a third piece times all but the
// first), under 2^-16 where they are 16 bits wide (the two second pieces of float16 operands, or of a computed one and an
// input).  The small ones are added up first: the tensor cores cut sums off instead of rounding them, so that few
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

// as pack(), but what rounds beyond bf16's largest number becomes that number
__device__ __forceinline__ uint32_t pack_within(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Two values as M pieces each.  A float32 within 2^-9 of the largest would round up to an infinite first piece: it gets
// bf16's largest number instead, and the next piece the rest.  An infinity stays one, in the last piece.
template <int M>
__device__ __forceinline__ void split(float x, float y, uint32_t (&r)[M]) {
#pragma unroll
    for (int m = 0; m < M; ++m) {
        r[m] = m + 1 < M ? pack_within(x, y) : pack(x, y);
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
// An operand of NT columns, its pieces one behind the other; K: columns along the sum, else rows.
template <int NT, bool K>
struct Operand {
    using X = Wide<NT>;
    uint32_t base;
    __device__ __forceinline__ explicit Operand(const void* m) {
        base = X::Tile::low(t5::smem_u32(m), X::Tile::bytes);
    }
    // of a piece's step of 16 along the sum (constants once loops are unrolled; shared addresses do not leave the field)
    __device__ __forceinline__ t5::Desc operator()(int piece, int step) const {
        constexpr int in_tile = X::W / 16;
        const int off = piece * X::bytes + (K ? step / in_tile * X::Tile::bytes + step % in_tile * X::Tile::step_k : step * X::Tile::step_mn);
        return t5::Desc{base + (uint32_t)(off >> 4), X::Tile::high};
    }
};

// d (+)= A B over STEPS of 16, products (s, u) of A's NA and B's NB pieces with s + u < D, small ones first; one thread.
// a(s, step), b(u, step): descriptors (or A's address in tensor memory)
template <int NA, int NB, int D, int STEPS, typename FA, typename FB>
__device__ __forceinline__ void products(uint32_t d, FA&& a, FB&& b, uint32_t idesc, bool add) {
#pragma unroll
    for (int order = (NA + NB - 2 < D - 1 ? NA + NB - 2 : D - 1); order >= 0; --order)
#pragma unroll
        for (int s = 0; s < NA; ++s) {
            const int u = order - s;
            if (u < 0 || u >= NB) continue;
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
                t5::mma(d, a(s, k), b(u, k), idesc, add);
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
    it.t1 = it.t0 + min(z.span, z.seqlen - it.t0);            // (t0 + span may pass 2^31)
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
// 0 as long as every value seen is finite (or within 2^-8 of float32's largest: such a value is taken token by token too,
// where it enters no product of scores)
__device__ __forceinline__ float seen(float v, float so_far) { return fmaf(v * 1.00390625f, 0.0f, so_far); }

// 64 rows x W columns on their way to shared memory: each of TH threads has groups of eight columns.  Rows and columns
// behind the last are 0.  VEC: rows on 16 bytes, a multiple of 8 columns.  What is loaded is not touched before put(), so
// that nothing waits for it earlier.
template <typename T, int W, int TH, bool VEC>
struct Pending {
    static constexpr int all = 64 * W / 8, n = (all + TH - 1) / TH, step = TH / (W / 8);    // rows between a thread's groups
    static_assert(TH % (W / 8) == 0 && step % 8 == 0, "a thread's groups lie in one column, alike in the swizzle");
    using Word = typename std::conditional<sizeof(T) == 4, float, typename std::conditional<VEC, uint32_t, unsigned short>::type>::type;
    static constexpr int words = VEC ? 2 * (int)sizeof(T) : 8;
    Word g[n][words];

    __device__ __forceinline__ static bool mine(int i) { return all % TH == 0 || threadIdx.x + i * TH < all; }

    __device__ __forceinline__ void fetch(const T* src, int64_t stride, int rows, int cols) {
        const int tid = threadIdx.x, row0 = tid / (W / 8), col = tid % (W / 8) * 8, in = cols - col;
        const T* p = src + row0 * stride + col;
#pragma unroll
        for (int i = 0; i < n; ++i, p += step * stride) {
            const bool here = row0 + i * step < rows;
            if (VEC) {
#pragma unroll
                for (int u = 0; u < (int)sizeof(T) / 2; ++u) {
                    uint4 q = make_uint4(0, 0, 0, 0);
                    if (here && in > 0) q = ((const uint4*)p)[u];
                    ((uint32_t*)g[i])[4 * u] = q.x;
                    ((uint32_t*)g[i])[4 * u + 1] = q.y;
                    ((uint32_t*)g[i])[4 * u + 2] = q.z;
                    ((uint32_t*)g[i])[4 * u + 3] = q.w;
                }
            } else {
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    Word x = 0;
                    if (here && u < in) x = ((const Word*)p)[u];
                    g[i][u] = x;
                }
            }
        }
    }
    // two of a group's values, as loaded (16-bit types)
    __device__ __forceinline__ uint32_t pair(int i, int u) const {
        if constexpr (sizeof(T) == 4) return 0;
        else return VEC ? (uint32_t)g[i][u] : (uint32_t)g[i][2 * u] | (uint32_t)g[i][2 * u + 1] << 16;
    }
    __device__ __forceinline__ float2 two(int i, int u) const {
        if constexpr (sizeof(T) == 4) {
            return make_float2(g[i][2 * u], g[i][2 * u + 1]);
        } else {
            const uint32_t r = pair(i, u);
            if constexpr (std::is_same<T, bf16>::value) return make_float2(low_f(r), high_f(r));
            else return __half22float2(*(const __half2*)&r);
        }
    }
    // whether a value is not finite
    __device__ __forceinline__ bool bad() const {
        if constexpr (std::is_same<T, bf16>::value) {
            __nv_bfloat162 sum = __float2bfloat162_rn(0.0f);
#pragma unroll
            for (int i = 0; i < n; ++i)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const uint32_t r = pair(i, u);
                    sum = __hfma2(*(const __nv_bfloat162*)&r, __float2bfloat162_rn(0.0f), sum);
                }
            return (*(const uint32_t*)&sum & 0x7fff7fffu) != 0;        // (0 times what is not finite is NaN)
        } else {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < n; ++i)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float2 v = two(i, u);
                    sum = seen(v.x, seen(v.y, sum));
                }
            return sum != 0.0f;
        }
    }
    // M pieces of the values, or of the values times their row's weight
    template <int M, bool WEIGHTED>
    __device__ __forceinline__ void put(bf16* dst, const float* weight) const {
        const int tid = threadIdx.x, row0 = tid / (W / 8);
        bf16* to = dst + Wide<W>::at(row0, tid % (W / 8) * 8);
#pragma unroll
        for (int i = 0; i < n; ++i, to += step * Wide<W>::W) {
            if (!mine(i)) continue;
            const float w = WEIGHTED ? weight[row0 + i * step] : 1.0f;
            uint32_t r[4][M];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if constexpr (std::is_same<T, bf16>::value && M == 1) {
                    r[u][0] = pair(i, u);
                } else {
                    const float2 v = two(i, u);
                    split<M>(WEIGHTED ? v.x * w : v.x, WEIGHTED ? v.y * w : v.y, r[u]);
                }
            }
#pragma unroll
            for (int s = 0; s < M; ++s) *(uint4*)(to + s * Wide<W>::elements) = make_uint4(r[0][s], r[1][s], r[2][s], r[3][s]);
        }
    }
    __device__ __forceinline__ void put(bf16* dst) const { put<Pieces<T>::in, false>(dst, nullptr); }
    __device__ __forceinline__ void put_weighted(bf16* dst, const float* weight) const { put<kFull3, true>(dst, weight); }
};

// whether rows that start at p and lie `stride` apart are on 16 bytes
inline bool on_16(const void* p, int64_t stride_bytes) { return (((uintptr_t)p | (uintptr_t)stride_bytes) & 15) == 0; }

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

// Writes a warp's 16 x 16 fragment (rows r0 and r0 + 8 of this lane) to rows of `st` elements.  VEC: rows on 16 bytes, a
// multiple of 8 columns; 16-bit values of four lanes are brought together, so that a lane stores 16 bytes.
template <bool VEC, typename T>
__device__ __forceinline__ void store_rows(T* out, int64_t st, int rows, int cols, int r0, int c0, const float (&x0)[4], const float (&x1)[4]) {
    const int lq = lane_id() & 3;
    if constexpr (VEC && sizeof(T) == 2) {
        // two tiles of 8 columns, rows r0 and r0 + 8: lane lq gathers tile lq & 1 of row r0 + 8 (lq >> 1)
        uint32_t v[4];                                                 // [tile + 2 half]
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            struct alignas(4) Two { T a, b; } t{from_f32<T>(x0[2 * h]), from_f32<T>(x0[2 * h + 1])}, t2{from_f32<T>(x1[2 * h]), from_f32<T>(x1[2 * h + 1])};
            v[2 * h] = *(uint32_t*)&t;
            v[1 + 2 * h] = *(uint32_t*)&t2;
        }
        const uint32_t a = __shfl_xor_sync(kFull, lq & 1 ? v[0] : v[1], 1), b = __shfl_xor_sync(kFull, lq & 1 ? v[2] : v[3], 1);
        // this lane and its neighbour now hold tile lq & 1 of both rows
        const uint32_t m0 = lq & 1 ? v[1] : v[0], m1 = lq & 1 ? v[3] : v[2];
        const uint32_t lo0 = lq & 1 ? a : m0, hi0 = lq & 1 ? m0 : a, lo1 = lq & 1 ? b : m1, hi1 = lq & 1 ? m1 : b;
        const bool up = lq >> 1;
        const uint32_t s0 = __shfl_xor_sync(kFull, up ? lo0 : lo1, 2), s1 = __shfl_xor_sync(kFull, up ? hi0 : hi1, 2);
        const uint32_t k0 = up ? lo1 : lo0, k1 = up ? hi1 : hi0;
        const int r = r0 + 8 * (lq >> 1), c = c0 + 8 * (lq & 1);
        if (r < rows && c < cols) *(uint4*)(out + r * st + c) = up ? make_uint4(s0, s1, k0, k1) : make_uint4(k0, k1, s0, s1);
    } else {
        struct alignas(2 * sizeof(T)) Two { T a, b; };
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            T* to = out + (r0 + 8 * h) * st + c0 + 2 * lq;
            const int in = r0 + 8 * h < rows ? cols - c0 - 2 * lq : 0;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const T a = from_f32<T>(q ? x1[2 * h] : x0[2 * h]), b = from_f32<T>(q ? x1[2 * h + 1] : x0[2 * h + 1]);
                if (VEC) {
                    if (8 * q < in) *(Two*)(to + 8 * q) = Two{a, b};
                } else {
                    if (8 * q < in) to[8 * q] = a;
                    if (8 * q + 1 < in) to[8 * q + 1] = b;
                }
            }
        }
    }
}

// ---------------------------------------------------------------------- state ----
// The transposed state (64 columns of the values by NT of the keys) in the registers of PARTS groups of four warps (which
// begin at multiples of four; each has NT / PARTS of the keys' columns), in the accumulators' layout.
template <int NT, int PARTS>
struct State {
    static constexpr int C = NT / PARTS;
    float s[C / 8][4];
    int first;                   // of the group's columns
    __device__ __forceinline__ explicit State(int part) : first(part * C) {}

    // calls f(value, value, p, n) for pairs of neighbouring n
    template <typename F>
    __device__ __forceinline__ void pairs(F&& f) {
        const int tid = threadIdx.x, p = (tid >> 5 & 3) * 16 + (tid >> 2 & 7), n = first + 2 * (tid & 3);
#pragma unroll
        for (int c = 0; c < C / 8; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) f(s[c][2 * h], s[c][2 * h + 1], p + 8 * h, n + 8 * c);
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
    // Its pieces to shared memory.  What is not finite becomes NaN there, in every piece: no product with a state is masked, so
    // that it reaches what it reaches by the formulas, without a walk token by token.  LATER: in a second pass where there is
    // any, so that a finite state costs only the question; else on the way.  Which is faster goes by the registers that the
    // walk around it has left (16 x 4096 tokens of 8 heads of 64 x 64 bf16, both ways, 540 us and 562 on the way; packed 30011
    // of 12 heads of 128 x 64 float16 1450 and 1420).
    template <int MS, bool LATER>
    __device__ __forceinline__ void put(bf16* dst) {
        float bad = 0.0f;
        pairs([&](float& x, float& y, int p, int n) {
            uint32_t q[MS];
            if (LATER) {
                split<MS>(x, y, q);
                bad = fmaf(x, 0.0f, fmaf(y, 0.0f, bad));
            } else {
                split<MS>(fmaf(x, 0.0f, x), fmaf(y, 0.0f, y), q);
            }
            bf16* to = dst + Wide<NT>::at(p, n);
#pragma unroll
            for (int k = 0; k < MS; ++k) *(uint32_t*)(to + k * Wide<NT>::elements) = q[k];
        });
        if (LATER && bad != 0.0f)
            pairs([&](float& x, float& y, int p, int n) {
                unsigned short* to = (unsigned short*)(dst + Wide<NT>::at(p, n));
                for (int k = 0; k < MS; ++k, to += Wide<NT>::elements) {
                    if (!isfinite(x)) to[0] = 0x7fff;
                    if (!isfinite(y)) to[1] = 0x7fff;
                }
            });
    }
    // s = whole s + the accumulator at addr (this warp's lanes)
    __device__ __forceinline__ void advance(uint32_t addr, float whole) {
        constexpr int many = C >= 32 ? 4 : C / 8;              // 8-column tiles a load
#pragma unroll
        for (int c = 0; c < C / 8; c += many) {
            float x[many][4];
            if constexpr (many == 4) t5::ld32(x, addr + first + 8 * c);
            else if constexpr (many == 2) t5::ld16(x, addr + first + 8 * c);
            else t5::ld8(x[0], addr + first + 8 * c);
#pragma unroll
            for (int q = 0; q < many; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[c + q][e] = fmaf(whole, s[c + q][e], x[q][e]);
        }
    }
};

// The logarithms of a chunk's decays on their way (one warp), two chunks ahead of the walk.
struct Logs {
    const float* g;
    int64_t st;
    float a, b;                  // of token 2 lane and 2 lane + 1
    __device__ __forceinline__ void fetch(int t, int len) {
        const int l = lane_id();
        a = t + 2 * l < len && t >= 0 ? g[(int64_t)(t + 2 * l) * st] : 0.0f;
        b = t + 2 * l + 1 < len && t >= 0 ? g[(int64_t)(t + 2 * l + 1) * st] : 0.0f;
    }
    __device__ __forceinline__ bool bad() const { return !(a <= 3.38e38f && b <= 3.38e38f); }
};

// What has to be initialised and awaited: barriers of the tensor cores' work, the tensor memory's address, and whether
// a wait has run out of time (t5::bar_wait).  After that no wait is made any more: the walk goes to its end with whatever
// its sums hold, the products still under way are awaited, and all that the block writes from then on, or in the end all
// that it has written, is NaN.
template <int BARS>
struct Sync {
    uint64_t bars[BARS];
    uint32_t tmem;
    int failed;

    // the first barrier awaits `first` arrivals, the others one
    __device__ __forceinline__ void init(uint32_t cols, int first = 1) {
        if (threadIdx.x < 32) t5::alloc(&tmem, cols);
        if (threadIdx.x == 0) {
            failed = 0;
            for (int i = 0; i < BARS; ++i) t5::bar_init(&bars[i], i == 0 ? first : 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        t5::fence_before();
        __syncthreads();
        t5::fence_after();
    }
    __device__ __forceinline__ void wait(int bar, uint32_t phase) {
        t5::bar_wait(&bars[bar], phase, &failed);
        t5::fence_after();
    }
    // 0, or NaN once a wait has run out
    __device__ __forceinline__ float poison() const { return __int_as_float(*(const volatile int*)&failed); }
    // the whole block, its walk over: whether a wait ran out
    __device__ __forceinline__ bool lost() {
        __syncthreads();
        return failed != 0;
    }
    // The whole block, all products awaited.  Where a wait ran out, products may be under way that use this block's memory:
    // they have as long again to end.
    __device__ __forceinline__ void end(uint32_t cols) {
        t5::fence_before();
        __syncthreads();
        t5::fence_after();
        if (threadIdx.x < 32) {
            t5::rest_if(&failed);
            t5::dealloc(tmem, cols);
        }
    }
};

// the rows of a block that lost a wait; all its threads
template <typename T>
__device__ __noinline__ void nan_rows(T* out, int64_t stride, int rows, int cols) {
    for (int64_t e = threadIdx.x; e < (int64_t)rows * cols; e += blockDim.x) out[e / cols * stride + e % cols] = from_f32<T>(__int_as_float(0x7fc00000));
}

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

// whether all rows of a call are on 16 bytes (NULL pointers count)
bool aligned(const bcm_decay_attn_args* a, bool backward);

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

// allows a kernel its dynamic shared memory, on the current device (with every launch: the attribute is the device's)
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

constexpr int kPartThreads = 256;
// Blocks on an SM: four hide one another's barriers (1 x 65536 tokens of 32 heads of 64 x 64 bf16 240 us with two, 185 with
// four); float32 and 128 features need the registers of two.
template <typename T, int NT>
constexpr int kPartResident = sizeof(T) == 2 && NT <= 64 ? 4 : 2;

template <typename T, int NT, bool BACK, bool VEC>
__global__ void __launch_bounds__(kPartThreads, kPartResident<T, NT>) part_kernel(const __grid_constant__ PartArgs p) {
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
    const int len = it.t1 - it.t0, nc = (len + kChunk - 1) / kChunk, l = lane_id();
    State<NT, 2> st(threadIdx.x >> 7);
    st.zero();
    double all = 0.0;
    Pending<T, NT, kPartThreads, VEC> pa;
    Pending<T, kP, kPartThreads, VEC> pb;
    Logs logs{g, p.g_st};
    const bool decay_warp = threadIdx.x >= 128 && threadIdx.x < 160;
    auto start = [&](int i) { return (BACK ? nc - 1 - i : i) * kChunk; };      // of the i-th chunk of the walk
    auto fetch = [&](int i) {
        const int t = start(i), rows = p.b.p ? min(kChunk, len - t) : 0;       // (no gradient: nothing, whatever q holds)
        pa.fetch(a + t * p.a.st, p.a.st, rows, z.n);
        pb.fetch(b + t * p.b.st, p.b.st, rows, cols);
    };
    sm.sync.init(kCols);
    if (decay_warp) {
        logs.fetch(start(0), len);
        all += decays_of(sm.d[0], logs.a, logs.b);
        logs.fetch(nc > 1 ? start(1) : -1, len);
    }
    const uint32_t acc = __shfl_sync(kFull, sm.sync.tmem, 0);
    const int warp = t5::warp_id();
    for (int i = -1; i < nc; ++i) {
        if (i >= 0) {
            __syncthreads();
            // (what is not finite stays so in the sums, and the walk takes such chunks token by token)
            pa.put(sm.a[0]);
            pb.put_weighted(sm.bw[0], BACK ? sm.d[i & 1].since : sm.d[i & 1].until);
            t5::fence_smem();
            t5::fence_before();
            __syncthreads();
            if (warp == 0 && t5::elect()) {
                t5::fence_after();
                const Operand<kP, false> A(sm.bw);
                const Operand<NT, false> B(sm.a);
                products<kFull3, NS, kFull3, kChunk / 16>(acc, A, B, t5::instr(NT, true, true), false);
                t5::commit(&sm.sync.bars[0]);
            }
            __syncwarp();
        }
        if (i + 1 < nc) fetch(i + 1);
        if (i < 0) continue;
        if (decay_warp && i + 1 < nc) {
            all += decays_of(sm.d[(i + 1) & 1], logs.a, logs.b);
            logs.fetch(i + 2 < nc ? start(i + 2) : -1, len);
        }
        sm.sync.wait(0, i & 1);
        st.advance(acc + ((warp & 3) << 21), sm.d[i & 1].whole);
        t5::fence_before();
    }
    const int64_t at = (int64_t)item * z.heads + h;
    st.store(p.parts.state + at * z.n * z.p + col, z.n, cols, z.p);
    if (threadIdx.x == 128 && col == 0) p.parts.whole[at] = exp2f((float)all);
    // (the items behind begin with it)
    if (sm.sync.lost()) nan_rows(p.parts.state + at * z.n * z.p + col, z.p, z.n, cols);
    sm.sync.end(kCols);
}

template <typename T, int NT, bool BACK>
bcm_status launch_part(const PartArgs& p, bool vec, cudaStream_t stream) {
    constexpr size_t smem = sizeof(PartSmem<T, NT>) + 1024;
    auto kernel = vec ? part_kernel<T, NT, BACK, true> : part_kernel<T, NT, BACK, false>;
    bcm_status st = allow_smem(kernel, smem);
    if (st != BCM_OK) return st;
    kernel<<<(unsigned)(p.z.items * p.z.heads * p.z.slices), kPartThreads, smem, stream>>>(p);
    BCM_LAUNCH_CHECK();
    return BCM_OK;
}

}  // namespace decay_attn
}  // namespace bcm
