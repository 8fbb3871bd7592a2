// decay_attn.cuh — what the kernels of the linear attention with a decay for each head share: tiles in shared memory,
// their matrix products, the decays' running sums, and the work items that sequences are cut into.
//
// Per head, a_t = exp(g_t):  S_t = a_t S_(t-1) + k_t v_t^T (N x P),  y_t = S_t^T q_t.
// In chunks of 64 tokens with G the running sum of g inside the chunk, D_ij = exp(G_i - G_j) for j <= i, 0 elsewhere:
//   Y = ((Q K^T) o D) V + diag(exp G) Q S_in,    S_out = exp(G_64) S_in + sum_j exp(G_64 - G_j) k_j v_j^T.
//
// Numbers.  The products run on the tensor cores in bf16 with fp32 sums.  An operand of more bits is a sum of bf16
// pieces, each the rounding of what the pieces before it left: float32 is three pieces (exact), float16 two (exact),
// and what a kernel computes itself (masked scores, states, keys times decays) has as many as its products need: two
// (relative 2^-18) where they end in 16 bits, three where they end in float32.  Of the pieces' products those whose
// weight lies below that are left out, and the small ones are added up first: the tensor cores cut sums off instead of
// rounding them, so that only few additions may be made at the full sum.  States are float32 between chunks.  G is
// summed in float64 and kept as two floats, so that a difference of two of its values keeps full precision after a
// decay of any size.
#pragma once

#include <algorithm>
#include <type_traits>

#include "common.cuh"

namespace bcm {
namespace decay_attn {

using bf16 = __nv_bfloat16;

constexpr int kChunk = 64;

// pieces of an input, and of what is computed for products that end in T; for those that end in float32 there are three
template <typename T> struct Pieces;
template <> struct Pieces<float> { static constexpr int in = 3, out = 3; };
template <> struct Pieces<__half> { static constexpr int in = 2, out = 2; };
template <> struct Pieces<bf16> { static constexpr int in = 1, out = 2; };
constexpr int kFull3 = 3;

// ------------------------------------------------------------ matrix products ----
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const bf16* p) {
    const uint32_t s = (uint32_t)__cvta_generic_to_shared(p);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s) : "memory");
}

__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], const bf16* p) {
    const uint32_t s = (uint32_t)__cvta_generic_to_shared(p);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s) : "memory");
}

// A of 16 rows x 16: stored by rows
__device__ __forceinline__ void load_a(uint32_t (&r)[4], const bf16* m, int ld, int row, int col) {
    const int l = lane_id();
    ldsm4(r, m + (row + (l & 15)) * ld + col + 8 * (l >> 4));
}
// A of 16 rows x 16, stored transposed (m[k][row])
__device__ __forceinline__ void load_at(uint32_t (&r)[4], const bf16* m, int ld, int row, int k) {
    const int l = lane_id();
    ldsm4t(r, m + (k + (l & 7) + 8 * (l >> 4)) * ld + row + 8 * ((l >> 3) & 1));
}
// B of 16 (k) x 16 (n), stored m[n][k]: r[0], r[1] the first eight n, r[2], r[3] the others
__device__ __forceinline__ void load_bn(uint32_t (&r)[4], const bf16* m, int ld, int n, int k) {
    const int l = lane_id();
    ldsm4(r, m + (n + (l & 7) + 8 * (l >> 4)) * ld + k + 8 * ((l >> 3) & 1));
}
// B of 16 (k) x 16 (n), stored m[k][n]
__device__ __forceinline__ void load_bk(uint32_t (&r)[4], const bf16* m, int ld, int k, int n) {
    const int l = lane_id();
    ldsm4t(r, m + (k + (l & 15)) * ld + n + 8 * (l >> 4));
}
// B of 32 (k) x 8 (n), stored m[k][n]: r[0], r[1] the first sixteen k, r[2], r[3] the others
__device__ __forceinline__ void load_bk32(uint32_t (&r)[4], const bf16* m, int ld, int k, int n) {
    ldsm4t(r, m + (k + lane_id()) * ld + n);
}

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
        x -= low_f(r[m]);
        y -= high_f(r[m]);
    }
}

// the four registers of an A operand as M pieces, from the two accumulator tiles that cover its 16 columns
template <int M>
__device__ __forceinline__ void split_a(const float (&c0)[4], const float (&c1)[4], uint32_t (&a)[M][4]) {
    uint32_t r[M];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const float(&c)[4] = q < 2 ? c0 : c1;
        split<M>(c[2 * (q & 1)], c[2 * (q & 1) + 1], r);
#pragma unroll
        for (int m = 0; m < M; ++m) a[m][q] = r[m];
    }
}

// acc[2 i], acc[2 i + 1] += A B over K16 steps of 16 and the N16 blocks of 16 columns.  la(regs, piece, step) loads A's
// NA pieces; B's NB pieces lie `piece` elements apart, stored m[k][n] (BK) or m[n][k].  Products (s, u) of pieces with
// s + u < D.  With many products to a step all but the largest go in a pass of their own.
template <int NA, int NB, int D, int K16, int N16, bool BK, typename LA>
__device__ __forceinline__ void gemm(float (&acc)[2 * N16][4], LA&& la, const bf16* b, int ldb, int piece, int k0, int n0) {
    constexpr bool two = NA * NB > 4;
#pragma unroll
    for (int pass = two ? 0 : 1; pass < 2; ++pass) {
#pragma unroll
        for (int kk = 0; kk < K16; ++kk) {
            uint32_t a[NA][4];
#pragma unroll
            for (int s = 0; s < NA; ++s)
                if (!(two && pass == 1 && s > 0)) la(a[s], s, kk);
#pragma unroll
            for (int nb = 0; nb < N16; ++nb)
#pragma unroll
                for (int u = NB - 1; u >= 0; --u) {
                    if (two && pass == 1 && u > 0) continue;
                    if (u >= D) continue;
                    uint32_t r[4];
                    if (BK) load_bk(r, b + u * piece, ldb, k0 + kk * 16, n0 + nb * 16);
                    else load_bn(r, b + u * piece, ldb, n0 + nb * 16, k0 + kk * 16);
#pragma unroll
                    for (int s = NA - 1; s >= 0; --s) {
                        if (s + u >= D) continue;
                        if (two && (pass == 1) != (s + u == 0)) continue;
                        mma(acc[2 * nb], a[s], r[0], r[1]);
                        mma(acc[2 * nb + 1], a[s], r[2], r[3]);
                    }
                }
        }
    }
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

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
    int chunks;               // kept states in all (packed: at most)
    int slices;               // of PT columns of the values
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

// A tile of R rows x W columns on its way to shared memory: each of TH threads has groups of eight columns.  Rows and
// columns behind the last are 0.
template <typename T, int R, int W, int TH>
struct Pending {
    static constexpr int all = R * W / 8, n = (all + TH - 1) / TH;
    Eight<T> g[n];

    __device__ __forceinline__ void fetch(const T* src, int64_t stride, int rows, int cols, bool vec) {
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const int at = threadIdx.x + i * TH, row = at / (W / 8), col = at % (W / 8) * 8;
            const T* p = src + row * stride + col;
            if (row < rows && vec && col + 8 <= cols) {
                const uint4* q = (const uint4*)p;
#pragma unroll
                for (int u = 0; u < (int)sizeof(T) / 2; ++u) ((uint4*)&g[i])[u] = q[u];
            } else {
#pragma unroll
                for (int u = 0; u < 8; ++u) g[i].v[u] = row < rows && col + u < cols ? p[u] : from_f32<T>(0.0f);
            }
        }
    }
    // writes the pieces, R rows of ld each; whether a value was not finite
    __device__ __forceinline__ bool put(bf16* dst, int ld) const {
        constexpr int NS = Pieces<T>::in;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const int at = threadIdx.x + i * TH, row = at / (W / 8), col = at % (W / 8) * 8;
            if (all % TH != 0 && at >= all) continue;
            if constexpr (std::is_same<T, bf16>::value) {
                const uint4 q = *(const uint4*)&g[i];
                const uint32_t e = 0x7f807f80u;
                // exponents of all ones
                bad |= (__vcmpeq2(q.x & e, e) | __vcmpeq2(q.y & e, e) | __vcmpeq2(q.z & e, e) | __vcmpeq2(q.w & e, e)) != 0;
                *(uint4*)(dst + row * ld + col) = q;
            } else {
                uint32_t r[4][NS];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float x = to_f32(g[i].v[2 * u]), y = to_f32(g[i].v[2 * u + 1]);
                    split<NS>(x, y, r[u]);
                    bad |= not_finite(x) | not_finite(y);
                }
#pragma unroll
                for (int s = 0; s < NS; ++s) *(uint4*)(dst + (s * R + row) * ld + col) = make_uint4(r[0][s], r[1][s], r[2][s], r[3][s]);
            }
        }
        return bad;
    }
};

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

template <typename T>
__device__ __forceinline__ bool on_16(const T* p, int64_t stride) {
    return (((uintptr_t)p | (uintptr_t)(stride * (int64_t)sizeof(T))) & 15) == 0;
}

// ---------------------------------------------------------------------- state ----
// An NT x PT state in the registers of four warps (which begin at a multiple of four), in the accumulators' layout.
template <int NT, int PT>
struct State {
    static constexpr int rows16 = NT / 16;
    static constexpr int M = rows16 >= 4 ? rows16 / 4 : 1;             // 16-row tiles of a warp
    static constexpr int across = rows16 >= 4 ? 1 : 4 / rows16;        // warps side by side over the columns
    static constexpr int C = PT / 8 / across;                          // 8-column tiles of a warp
    float s[M][C][4];

    __device__ __forceinline__ static int row(int m) {                 // first of the tile's rows
        const int w = (threadIdx.x >> 5) & 3;
        return rows16 >= 4 ? (w * M + m) * 16 : w / across * 16;
    }
    __device__ __forceinline__ static int col(int c) {
        const int w = (threadIdx.x >> 5) & 3;
        return ((rows16 >= 4 ? 0 : w % across * C) + c) * 8;
    }
    // calls f(value, row, column) for pairs of neighbouring columns
    template <typename F>
    __device__ __forceinline__ void pairs(F&& f) {
        const int l = lane_id();
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    f(s[m][c][2 * h], s[m][c][2 * h + 1], row(m) + (l >> 2) + 8 * h, col(c) + 2 * (l & 3));
    }
    __device__ __forceinline__ void zero() {
        pairs([](float& x, float& y, int, int) { x = y = 0.0f; });
    }
    // from rows of `stride` floats, n x p of them
    __device__ __forceinline__ void load(const float* src, int n, int p, int stride) {
        const bool even = ((stride & 1) | ((uintptr_t)src & 7)) == 0;
        pairs([&](float& x, float& y, int r, int c) {
            x = y = 0.0f;
            if (r < n && c < p) {
                const float* q = src + (int64_t)r * stride + c;
                if (even && c + 1 < p) {
                    const float2 v = *(const float2*)q;
                    x = v.x;
                    y = v.y;
                } else {
                    x = q[0];
                    if (c + 1 < p) y = q[1];
                }
            }
        });
    }
    __device__ __forceinline__ void store(float* dst, int n, int p, int stride) {
        const bool even = ((stride & 1) | ((uintptr_t)dst & 7)) == 0;
        pairs([&](float& x, float& y, int r, int c) {
            if (r < n && c < p) {
                float* q = dst + (int64_t)r * stride + c;
                if (even && c + 1 < p) {
                    *(float2*)q = make_float2(x, y);
                } else {
                    q[0] = x;
                    if (c + 1 < p) q[1] = y;
                }
            }
        });
    }
    // its pieces to shared memory [M][NT][PT + 8]; whether a value was not finite
    template <int MS>
    __device__ __forceinline__ bool put(bf16* dst) {
        bool bad = false;
        pairs([&](float& x, float& y, int r, int c) {
            uint32_t q[MS];
            split<MS>(x, y, q);
            bad |= not_finite(x) | not_finite(y);
#pragma unroll
            for (int k = 0; k < MS; ++k) *(uint32_t*)(dst + (k * NT + r) * (PT + 8) + c) = q[k];
        });
        return bad;
    }
    // s = whole s + sum over the 64 tokens of weight[t] a[t] b[t]^T; weighted a in three pieces.  Half of the tokens at
    // a time is added up from 0 and then to the state, whose own roundings stay those of float32.
    template <int NS>
    __device__ __forceinline__ void advance(const bf16* a, const bf16* b, const float* weight, float whole) {
        constexpr int lda = NT + 8, ldb = PT + 8, MS = kFull3;
        const int l = lane_id();
        pairs([&](float& x, float& y, int, int) {
            x *= whole;
            y *= whole;
        });
#pragma unroll
        for (int k = 0; k < kChunk; k += 32) {
            uint32_t f[M][2][MS][4];
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t raw[NS][4];
#pragma unroll
                    for (int q = 0; q < NS; ++q) load_at(raw[q], a + q * kChunk * lda, lda, row(m), k + 16 * h);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float2 w2 = *(const float2*)(weight + k + 16 * h + 2 * (l & 3) + 8 * (r >> 1));
                        float x = 0.0f, y = 0.0f;
#pragma unroll
                        for (int q = NS - 1; q >= 0; --q) {
                            x += low_f(raw[q][r]);
                            y += high_f(raw[q][r]);
                        }
                        uint32_t w[MS];
                        split<MS>(x * w2.x, y * w2.y, w);
#pragma unroll
                        for (int q = 0; q < MS; ++q) f[m][h][q][r] = w[q];
                    }
                }
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float sum[M][4] = {};
                uint32_t v[NS][4];
#pragma unroll
                for (int u = NS - 1; u >= 0; --u) load_bk32(v[u], b + u * kChunk * ldb, ldb, k, col(c));
                // pieces of small weight first
#pragma unroll
                for (int order = MS - 1; order >= 0; --order)
#pragma unroll
                    for (int u = 0; u < NS && u <= order; ++u)
#pragma unroll
                        for (int m = 0; m < M; ++m) {
                            mma(sum[m], f[m][0][order - u], v[u][0], v[u][1]);
                            mma(sum[m], f[m][1][order - u], v[u][2], v[u][3]);
                        }
#pragma unroll
                for (int m = 0; m < M; ++m)
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[m][c][r] += sum[m][r];
            }
        }
    }
};

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
    int pt;                   // columns of a block's tile
    size_t items_at, seq_at, state_at, whole_at, bytes;
    bool cut;                 // some sequence may have more than one item
};

int padded_n(int64_t n);
bcm_status check(const bcm_decay_attn_args* a, const char* what);
Plan plan_of(const bcm_decay_attn_args* a, bool backward);
bcm_status fill_tables(Plan& plan, void* workspace, cudaStream_t stream);
Parts parts_of(const Plan& plan, void* workspace);
// entering states along each sequence, from `end` (nullptr: zeros) at its first (backwards: last) item
bcm_status join(const Plan& plan, const Parts& parts, const float* end, bool backward, cudaStream_t stream);

inline Rows rows_of(const void* p, int64_t sb, int64_t st, int64_t sh) { return Rows{p, sb, st, sh}; }

// calls f(T, NT, PT as integral constants)
template <typename F>
bcm_status dispatch(bcm_dtype t, int nt, int pt, F&& f) {
    return dispatch_dtype(t, [&](auto type) -> bcm_status {
        auto by_pt = [&](auto n) -> bcm_status {
            if (pt == 32) return f(type, n, std::integral_constant<int, 32>());
            return f(type, n, std::integral_constant<int, 64>());
        };
        switch (nt) {
            case 16: return by_pt(std::integral_constant<int, 16>());
            case 32: return by_pt(std::integral_constant<int, 32>());
            case 64: return by_pt(std::integral_constant<int, 64>());
            default: return by_pt(std::integral_constant<int, 128>());
        }
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

template <typename T, int NT, int PT>
struct PartSmem {
    bf16 a[Pieces<T>::in][kChunk][NT + 8];
    bf16 b[Pieces<T>::in][kChunk][PT + 8];
    Decays d;
};

constexpr int kPartThreads = 128;

template <typename T, int NT, int PT, bool BACK>
__global__ void __launch_bounds__(kPartThreads) part_kernel(const __grid_constant__ PartArgs p) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    PartSmem<T, NT, PT>& sm = *(PartSmem<T, NT, PT>*)smem_raw;
    const Sizes& z = p.z;
    const int across = z.heads * z.slices;
    const int item = blockIdx.x / across, hs = blockIdx.x % across, h = hs / z.slices, col = hs % z.slices * PT;
    const Item it = item_of(z, item);
    if (it.seq < 0 || (BACK ? it.first : it.last)) return;
    const int cols = min(PT, z.p - col), ha = h / (z.heads / z.qk_heads);
    const T* a = row_ptr<T>(p.a, z, it.seq, it.t0, ha);
    const T* b = row_ptr<T>(p.b, z, it.seq, it.t0, h) + col;
    const float* g = p.g + (z.cu ? 0 : it.seq * p.g_sb) + it.t0 * p.g_st + h * p.g_sh;
    const bool va = on_16(a, p.a.st), vb = on_16(b, p.b.st);
    State<NT, PT> st;
    st.zero();
    double all = 0.0;
    const int len = it.t1 - it.t0, nc = (len + kChunk - 1) / kChunk, l = lane_id();
    Pending<T, kChunk, NT, kPartThreads> pa;
    Pending<T, kChunk, PT, kPartThreads> pb;
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
    for (int i = 0; i < nc; ++i) {
        __syncthreads();
        if (threadIdx.x < 32) all += decays_of(sm.d, g0, g1);
        // (what is not finite stays so in the sums, and the walk takes such chunks token by token)
        pa.put(&sm.a[0][0][0], NT + 8);
        pb.put(&sm.b[0][0][0], PT + 8);
        __syncthreads();
        if (i + 1 < nc) fetch(i + 1);
        st.template advance<Pieces<T>::in>(&sm.a[0][0][0], &sm.b[0][0][0], BACK ? sm.d.since : sm.d.until, sm.d.whole);
    }
    const int64_t at = (int64_t)item * z.heads + h;
    st.store(p.parts.state + at * z.n * z.p + col, z.n, z.p - col, z.p);
    if (threadIdx.x == 0 && col == 0) p.parts.whole[at] = exp2f((float)all);
}

template <typename T, int NT, int PT, bool BACK>
bcm_status launch_part(const PartArgs& p, cudaStream_t stream) {
    constexpr size_t smem = sizeof(PartSmem<T, NT, PT>);
    auto kernel = part_kernel<T, NT, PT, BACK>;
    bcm_status st = allow_smem(kernel, smem);
    if (st != BCM_OK) return st;
    kernel<<<(unsigned)(p.z.items * p.z.heads * p.z.slices), kPartThreads, smem, stream>>>(p);
    BCM_LAUNCH_CHECK();
    return BCM_OK;
}

}  // namespace decay_attn
}  // namespace bcm
