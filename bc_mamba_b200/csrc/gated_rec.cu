// gated_rec.cu — gated linear recurrence, forward, backward and one-token step.
//
// Per feature d with c the decay scale, s = softplus(lam[d]):
//   u_t = -c s sigmoid(r_t),  a_t = exp(u_t),  m_t = sqrt(1 - a_t^2),
//   h_t = a_t h_{t-1} + m_t sigmoid(i_t) x_t,  y_t = h_t.
// Backward, with G_t = dy_t + a_{t+1} G_{t+1} (dh_last enters at the last
// token, nothing passes over a sequence's end):
//   dx_t = G_t m_t sigmoid(i_t),       di_t = dx_t x_t (1 - sigmoid(i_t)),
//   du_t = G_t (a_t h_{t-1} - (a_t^2 / m_t) sigmoid(i_t) x_t),
//   dr_t = du_t u_t (1 - sigmoid(r_t)),
//   dlam = -c sigmoid(lam) sum_t du_t sigmoid(r_t),  dh0 = a_1 G_1.
// The second term of du is 0 where m_t = 0 (its limit after the factor u).
#include <algorithm>
#include <cstring>

#include "common.cuh"

namespace bcm {
namespace {

__device__ __forceinline__ float sigmoid_(float v) { return 1.0f / (1.0f + expf(-v)); }
__device__ __forceinline__ float softplus_(float v) { return v > 20.0f ? v : log1pf(expf(v)); }

// ---- two gates at a time ----------------------------------------------------
// The scan kernels' arithmetic works on pairs (packed fp32 instructions): two
// neighbouring features of a token, or two tokens of a feature.  What bounds it
// is the special-function unit (one result per lane every 8 cycles), so:
//  * a - 1 = expm1(u) is a polynomial for |u| <= kPolyEnd (degree 4 times u,
//    interpolated at Chebyshev nodes, relative error 1.4e-8): no cancellation in
//    1 - a^2 = (1 - a)(1 + a) and a correctly rounded a = 1 + (a - 1), so that a
//    memory of a thousand tokens does not add up a biased decay;
//  * FAST (every gate of the warp's batch above -40, every cs below kPolyEnd)
//    shares one reciprocal between the two sigmoids and needs no exponential for
//    a: 4 results per pair member instead of 6.
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPolyEnd = 0.35f;
constexpr float kGateLow = -40.0f;   // below: (1 + e^-r)(1 + e^-i) may overflow

__device__ __forceinline__ float ex2_(float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float rcp_(float v) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float rsqrt_(float v) { float r; asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float min_nan_(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }

struct Gates {
    float2 sr, si, w, rs;     // sigmoid(r), sigmoid(i), a - 1, 1 / m (0 where m = 0)
};

__device__ __forceinline__ float2 one_minus_a2(float2 w) { return __fmul2_rn(w, __ffma2_rn(w, f2(-1.0f), f2(-2.0f))); }

template <bool FAST>
__device__ __forceinline__ Gates gates(float2 r, float2 i, float2 ncs) {
    Gates g;
    const float2 tr = __fmul2_rn(r, f2(-kLog2e)), ti = __fmul2_rn(i, f2(-kLog2e));
    const float2 dr = __fadd2_rn(make_float2(ex2_(tr.x), ex2_(tr.y)), f2(1.0f));
    const float2 di = __fadd2_rn(make_float2(ex2_(ti.x), ex2_(ti.y)), f2(1.0f));
    if (FAST) {
        const float2 both = __fmul2_rn(dr, di);
        const float2 inv = make_float2(rcp_(both.x), rcp_(both.y));
        g.sr = __fmul2_rn(di, inv);
        g.si = __fmul2_rn(dr, inv);
    } else {
        g.sr = make_float2(rcp_(dr.x), rcp_(dr.y));
        g.si = make_float2(rcp_(di.x), rcp_(di.y));
    }
    const float2 u = __fmul2_rn(ncs, g.sr);
    float2 q = __ffma2_rn(u, f2(0.007211245596408844f), f2(0.04133187234401703f));
    q = __ffma2_rn(u, q, f2(0.16662530601024628f));
    q = __ffma2_rn(u, q, f2(0.49999821186065674f));
    q = __ffma2_rn(u, q, f2(1.0f));
    g.w = __fmul2_rn(u, q);
    if (!FAST) {
        const float2 t = __fmul2_rn(u, f2(kLog2e));
        if (!(u.x >= -kPolyEnd)) g.w.x = ex2_(t.x) - 1.0f;
        if (!(u.y >= -kPolyEnd)) g.w.y = ex2_(t.y) - 1.0f;
    }
    const float2 m2 = one_minus_a2(g.w);
    g.rs.x = m2.x > 1e-37f ? rsqrt_(m2.x) : 0.0f;
    g.rs.y = m2.y > 1e-37f ? rsqrt_(m2.y) : 0.0f;
    return g;
}

__device__ __forceinline__ float2 m_of(const Gates& g) { return __fmul2_rn(one_minus_a2(g.w), g.rs); }

struct RecPtr {
    const void* x; const void* r; const void* i; const void* dy;
    int64_t xb, xt, rb, rt, ib, it, gb, gt;
};

struct RecOut {
    const float* h0; void* y; float* h_last; float* ckpt;          // forward
    const float* dh_last; void* dx; void* dr; void* di; float* part; float* dh0;   // backward
};

// ---- layout of the scan kernels -----------------------------------------------
// A lane owns VEC neighbouring features, a warp a few consecutive tokens, a block
// kWarps times as many (a chunk) of a tile of 32 * VEC features.
// A block's chunks follow one another in a loop that carries the state; P blocks
// of a cluster take P consecutive chunks per turn, so that few tiles with long
// sequences still fill the GPU.  Every input is read once: the composition
// h -> A h + H of a warp's tokens goes to shared memory, the other warps' and
// blocks' compositions give the state that enters, and the tokens, still in
// registers, are replayed from it.
//
// Mode: kDense, one sequence per block; kGroup, a block takes `per` consecutive
// dense sequences as one run of tokens (short sequences would leave most of a
// chunk empty); kPacked, one run of tokens with the sequences' offsets in cu.
// Where a sequence starts inside a run, nothing passes and its own state enters.
constexpr int kWarps = 8;
constexpr int kChunkFwd = 64, kChunkBwd = 32;    // tokens of a block's turn: 8 and 4 a warp (the backward keeps 7 values a token)
constexpr int kCkpt = 32;                        // the forward keeps the state that enters every kCkpt tokens of a run
constexpr int kMaxCluster = 16;
constexpr float kCut = -1.0f;   // in place of a product of decays: nothing passes (a sequence starts inside)

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, bool ok, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = ok ? to_f32<T>(*p) : 0.0f;
    } else if constexpr (sizeof(T) == 4) {
        const float2 w = ok ? __ldg(reinterpret_cast<const float2*>(p)) : make_float2(0.0f, 0.0f);
        v[0] = w.x;
        v[1] = w.y;
    } else {
        const uint32_t w = ok ? __ldg(reinterpret_cast<const uint32_t*>(p)) : 0u;
        T e[2];
        memcpy(e, &w, 4);
        v[0] = to_f32<T>(e[0]);
        v[1] = to_f32<T>(e[1]);
    }
}

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        *p = from_f32<T>(v[0]);
    } else if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
    } else {
        const T e[2] = {from_f32<T>(v[0]), from_f32<T>(v[1])};
        uint32_t w;
        memcpy(&w, e, 4);
        *reinterpret_cast<uint32_t*>(p) = w;
    }
}

// Arrays of pairs hold S tokens of VEC features: pair j = token j's two features, or the tokens 2j, 2j + 1 of one.
template <int VEC, int N>
__device__ __forceinline__ float get(const float2 (&p)[N], int j, int v) {
    if (VEC == 2) return v ? p[j].y : p[j].x;
    return (j & 1) ? p[j >> 1].y : p[j >> 1].x;
}
template <int VEC, int N>
__device__ __forceinline__ void put(float2 (&p)[N], int j, int v, float e) {
    if (VEC == 2) {
        if (v) p[j].y = e;
        else p[j].x = e;
    } else {
        if (j & 1) p[j >> 1].y = e;
        else p[j >> 1].x = e;
    }
}
template <int VEC, int N>
__device__ __forceinline__ void put_row(float2 (&p)[N], int j, const float (&e)[VEC]) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) put<VEC>(p, j, v, e[v]);
}

// The sequence that holds token t: the last s with cu[s] <= t, in [0, n).  Called by whole warps; t is uniform.
__device__ __forceinline__ int seq_of(const int32_t* __restrict__ cu, int n, int t) {
    int lo = 0, hi = n - 1;                          // the answer lies in [lo, hi]
    const int lane = threadIdx.x & 31;
    while (hi > lo) {
        const int step = (hi - lo + 31) / 32;        // lanes look at lo + step, lo + 2 step, ...
        const int at = lo + (lane + 1) * step;
        const unsigned m = __ballot_sync(kFull, at <= hi && cu[at] <= t);
        const int c = __popc(m);
        lo += c * step;
        hi = min(hi, lo + step - 1);
    }
    return lo;
}

enum Mode { kDense, kGroup, kPacked };

// What the kernels know of the sizes: a run holds L tokens (kGroup: its last may hold fewer), a sequence Ls (kDense,
// kGroup), per sequences make a run (kGroup); n sequences, D features, P blocks in a cluster.
struct RecDim {
    const int32_t* cu;
    int64_t n;
    int L, Ls, per, D, P;
};

// The sequence around a token of the run, moved along by a warp: its index s, its first token and its end.
template <int MODE>
struct Seq {
    const int32_t* cu;
    int n, Ls;
    int64_t s0, s;
    int beg, end;
    __device__ __forceinline__ void at(int t) {
        if (MODE == kPacked) {
            const int k = seq_of(cu, n, t);
            s = k;
            beg = cu[k];
            end = cu[k + 1];
        } else if (MODE == kGroup) {
            const int k = t / Ls;
            s = s0 + k;
            beg = k * Ls;
            end = beg + Ls;
        }
    }
};

// (A1, H1) followed by (A2, H2)
template <bool CUTS>
__device__ __forceinline__ void then(float& A1, float& H1, float A2, float H2) {
    if (CUTS && A2 < 0.0f) {
        A1 = kCut;
        H1 = H2;
    } else {
        H1 = fmaf(A2, H1, H2);
        A1 = CUTS && A1 < 0.0f ? kCut : A1 * A2;
    }
}

template <bool CUTS>
__device__ __forceinline__ float apply(float A, float H, float h) {
    return CUTS && A < 0.0f ? H : fmaf(A, h, H);
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void st_cluster(uint32_t addr, int rank, float2 v) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(remote), "f"(v.x), "f"(v.y) : "memory");
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Whether a warp's batch of gates can take the shorter form (uniform over the warp; false where a gate is NaN).
template <int N>
__device__ __forceinline__ bool fast_batch(bool small, const float2 (&r)[N], const float2 (&i)[N]) {
    if (!small) return false;
    float low = 0.0f;
#pragma unroll
    for (int k = 0; k < N; ++k) low = min_nan_(min_nan_(low, min_nan_(r[k].x, r[k].y)), min_nan_(i[k].x, i[k].y));
    return __all_sync(kFull, low >= kGateLow);
}

template <typename T, int VEC, int MODE, bool CLUSTER>
__global__ void __launch_bounds__(kWarps * 32)
rec_fwd_kernel(RecPtr p, RecOut o, RecDim n, const float* __restrict__ lam, float c) {
    constexpr bool CUTS = MODE != kDense;
    constexpr int kChunk = kChunkFwd, S = kChunk / kWarps, NP = S * VEC / 2;
    __shared__ float2 ex[2][kWarps][VEC][32];
    __shared__ float2 pub[CLUSTER ? 2 : 1][CLUSTER ? kMaxCluster : 1][VEC][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int D = n.D, P = n.P, tiles = (D + 32 * VEC - 1) / (32 * VEC);
    const int rank = CLUSTER ? blockIdx.x % P : 0;
    const int64_t run_id = blockIdx.x / (CLUSTER ? P : 1) / tiles;
    const int tile = blockIdx.x / (CLUSTER ? P : 1) - (int)run_id * tiles;
    // the run's first sequence and its tokens
    const int64_t b = MODE == kGroup ? run_id * n.per : run_id;
    const int L = MODE == kGroup ? (int)min((int64_t)n.per, n.n - b) * n.Ls : n.L;
    const int d = (tile * 32 + lane) * VEC;
    const bool mine = d < D;
    const int dd = mine ? d : 0;
    const T* x = static_cast<const T*>(p.x) + (MODE == kPacked ? 0 : b * p.xb) + dd;
    const T* r = static_cast<const T*>(p.r) + (MODE == kPacked ? 0 : b * p.rb) + dd;
    const T* i = static_cast<const T*>(p.i) + (MODE == kPacked ? 0 : b * p.ib) + dd;
    T* y = static_cast<T*>(o.y) + (MODE == kPacked ? 0 : b * n.Ls * D) + dd;
    const int chunks = (n.L + kChunk - 1) / kChunk, turns = (chunks + P - 1) / P;   // (of a full run)
    float* ck = o.ckpt ? o.ckpt + run_id * ((n.L + kCkpt - 1) / kCkpt) * D + dd : nullptr;
    float run[VEC];
    const float2 ncs = make_float2(-c * softplus_(lam[dd]), -c * softplus_(lam[dd + VEC - 1]));
    const bool small = __all_sync(kFull, -ncs.x <= kPolyEnd && -ncs.y <= kPolyEnd);
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        run[v] = MODE == kDense && o.h0 ? o.h0[b * D + dd + v] : 0.0f;
    }
    Seq<MODE> seq{n.cu, (int)n.n, n.Ls, b, 0, 0, 0};
    if (CLUSTER) cluster_sync();       // every block of the cluster runs before its shared memory is written to
    for (int turn = 0; turn < turns; ++turn) {
        const int buf = turn & 1;
        const int chunk = turn * P + rank;
        const int t0 = chunk * kChunk + warp * S;
        float2 a[NP], e[NP];
        {
            float2 xv[NP], rv[NP], iv[NP];
            if (MODE == kGroup) seq.at(t0);
            int64_t sl = seq.s - b;
            int tl = t0 - seq.beg;
#pragma unroll
            for (int j = 0; j < S; ++j) {
                const bool ok = mine && t0 + j < L;
                const int64_t t = MODE == kGroup ? tl : t0 + j, q = MODE == kGroup ? sl : 0;
                float row[VEC];
                load_vec<T, VEC>(r + q * p.rb + t * p.rt, ok, row);
                put_row<VEC>(rv, j, row);
                load_vec<T, VEC>(i + q * p.ib + t * p.it, ok, row);
                put_row<VEC>(iv, j, row);
                load_vec<T, VEC>(x + q * p.xb + t * p.xt, ok, row);
                put_row<VEC>(xv, j, row);
                if (MODE == kGroup && ++tl == n.Ls) {
                    tl = 0;
                    ++sl;
                }
            }
            if (MODE == kPacked && t0 < L) seq.at(t0);
            if (fast_batch(small, rv, iv)) {
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    const Gates g = gates<true>(rv[k], iv[k], ncs);
                    a[k] = __fadd2_rn(g.w, f2(1.0f));
                    e[k] = __fmul2_rn(__fmul2_rn(m_of(g), g.si), xv[k]);
                }
            } else {
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    const Gates g = gates<false>(rv[k], iv[k], ncs);
                    a[k] = __fadd2_rn(g.w, f2(1.0f));
                    e[k] = __fmul2_rn(__fmul2_rn(m_of(g), g.si), xv[k]);
                }
            }
            if (t0 + S > L)               // tokens past the end change nothing
#pragma unroll
                for (int j = 0; j < S; ++j)
                    if (t0 + j >= L)
#pragma unroll
                        for (int v = 0; v < VEC; ++v) {
                            put<VEC>(a, j, v, 1.0f);
                            put<VEC>(e, j, v, 0.0f);
                        }
        }
        unsigned starts = 0;      // bit j: a sequence starts at token t0 + j (its entering state goes into e)
        if (CUTS && t0 < L && (seq.beg == t0 || seq.end < t0 + S)) {
            Seq<MODE> q = seq;
#pragma unroll
            for (int j = 0; j < S; ++j) {
                const int t = t0 + j;
                if (t < L && t == q.end) q.at(t);
                if (t < L && t == q.beg) {
                    starts |= 1u << j;
#pragma unroll
                    for (int v = 0; v < VEC; ++v)
                        put<VEC>(e, j, v, fmaf(get<VEC>(a, j, v), o.h0 ? o.h0[q.s * D + dd + v] : 0.0f, get<VEC>(e, j, v)));
                }
            }
        }
        float A[VEC], H[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            A[v] = 1.0f;
            H[v] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const bool cut = CUTS && (starts >> j & 1u);
#pragma unroll
            for (int v = 0; v < VEC; ++v) then<CUTS>(A[v], H[v], cut ? kCut : get<VEC>(a, j, v), get<VEC>(e, j, v));
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) ex[buf][warp][v][lane] = make_float2(A[v], H[v]);
        __syncthreads();
        float preA[VEC], preH[VEC], totA[VEC], totH[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            totA[v] = 1.0f;
            totH[v] = 0.0f;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) {
                if (k == warp) {
                    preA[v] = totA[v];
                    preH[v] = totH[v];
                }
                const float2 f = ex[buf][k][v][lane];
                then<CUTS>(totA[v], totH[v], f.x, f.y);
            }
        }
        float h[VEC];
        if (CLUSTER) {
            for (int k = warp; k < P; k += kWarps)
#pragma unroll
                for (int v = 0; v < VEC; ++v) st_cluster(smem_addr(&pub[buf][rank][v][lane]), k, make_float2(totA[v], totH[v]));
            cluster_sync();
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                for (int k = 0; k < P; ++k) {
                    if (k == rank) h[v] = run[v];
                    const float2 f = pub[buf][k][v][lane];
                    run[v] = apply<CUTS>(f.x, f.y, run[v]);
                }
            }
        } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                h[v] = run[v];
                run[v] = apply<CUTS>(totA[v], totH[v], run[v]);
            }
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) h[v] = apply<CUTS>(preA[v], preH[v], h[v]);
        if (ck && warp * S % kCkpt == 0 && mine && t0 < L)
#pragma unroll
            for (int v = 0; v < VEC; ++v) ck[(int64_t)(t0 / kCkpt) * D + v] = h[v];
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const int t = t0 + j;
            const bool cut = CUTS && (starts >> j & 1u);
#pragma unroll
            for (int v = 0; v < VEC; ++v) h[v] = cut ? get<VEC>(e, j, v) : fmaf(get<VEC>(a, j, v), h[v], get<VEC>(e, j, v));
            if (mine && t < L) store_vec<T, VEC>(y + (int64_t)t * D, h);
            if (CUTS && t < L) {
                if (t == seq.end) seq.at(t);
                if (t == seq.end - 1 && mine)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) o.h_last[seq.s * D + d + v] = h[v];
            }
        }
    }
    if (rank != 0 || !mine) return;
    if (MODE == kDense) {
        if (warp == 0)
#pragma unroll
            for (int v = 0; v < VEC; ++v) o.h_last[b * D + d + v] = run[v];
    } else if (MODE == kPacked) {
        for (int64_t s = warp; s < n.n; s += kWarps)       // empty sequences keep their state
            if (n.cu[s] >= n.cu[s + 1])
#pragma unroll
                for (int v = 0; v < VEC; ++v) o.h_last[s * D + d + v] = o.h0 ? o.h0[s * D + d + v] : 0.0f;
    }
}

// Chunks from the last to the first.  The states that enter a chunk come from
// the forward; back_t = a_t G_t passes from right to left by the same products
// of decays, back -> A back + K.
template <typename T, int VEC, int MODE, bool CLUSTER>
__global__ void __launch_bounds__(kWarps * 32)
rec_bwd_kernel(RecPtr p, RecOut o, RecDim n, const float* __restrict__ lam, float c) {
    constexpr bool CUTS = MODE != kDense;
    constexpr int kChunk = kChunkBwd, S = kChunk / kWarps, NP = S * VEC / 2;
    __shared__ float ex[2][kWarps][3][VEC][32];
    __shared__ float2 pub[CLUSTER ? 2 : 1][CLUSTER ? kMaxCluster : 1][VEC][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int D = n.D, P = n.P, tiles = (D + 32 * VEC - 1) / (32 * VEC);
    const int rank = CLUSTER ? blockIdx.x % P : 0;
    const int64_t run_id = blockIdx.x / (CLUSTER ? P : 1) / tiles;
    const int tile = blockIdx.x / (CLUSTER ? P : 1) - (int)run_id * tiles;
    // the run's first sequence and its tokens
    const int64_t b = MODE == kGroup ? run_id * n.per : run_id;
    const int L = MODE == kGroup ? (int)min((int64_t)n.per, n.n - b) * n.Ls : n.L;
    const int d = (tile * 32 + lane) * VEC;
    const bool mine = d < D;
    const int dd = mine ? d : 0;
    const T* x = static_cast<const T*>(p.x) + (MODE == kPacked ? 0 : b * p.xb) + dd;
    const T* r = static_cast<const T*>(p.r) + (MODE == kPacked ? 0 : b * p.rb) + dd;
    const T* i = static_cast<const T*>(p.i) + (MODE == kPacked ? 0 : b * p.ib) + dd;
    const T* dy = static_cast<const T*>(p.dy) + (MODE == kPacked ? 0 : b * p.gb) + dd;
    const bool has_dy = p.dy != nullptr;
    const int64_t base = (MODE == kPacked ? 0 : b * n.Ls * D) + dd;
    T* dx = static_cast<T*>(o.dx) + base;
    T* dr = static_cast<T*>(o.dr) + base;
    T* di = static_cast<T*>(o.di) + base;
    const int chunks = (n.L + kChunk - 1) / kChunk, turns = (chunks + P - 1) / P;   // (of a full run)
    const float* ck = o.ckpt + run_id * ((n.L + kCkpt - 1) / kCkpt) * D + dd;
    Seq<MODE> seq{n.cu, (int)n.n, n.Ls, b, 0, 0, 0};
    float run[VEC];
    float2 sum = f2(0.0f);
    const float2 ncs = make_float2(-c * softplus_(lam[dd]), -c * softplus_(lam[dd + VEC - 1]));
    const bool small = __all_sync(kFull, -ncs.x <= kPolyEnd && -ncs.y <= kPolyEnd);
    if (CUTS) seq.at(L - 1);
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        run[v] = o.dh_last ? o.dh_last[(CUTS ? seq.s : b) * D + dd + v] : 0.0f;
    }
    if (CLUSTER) cluster_sync();
    for (int turn = turns - 1; turn >= 0; --turn) {
        const int buf = turn & 1;
        const int chunk = turn * P + rank;
        const int t0 = chunk * kChunk + warp * S;
        float2 xv[NP], gv[NP], sr[NP], si[NP], w[NP], rs[NP];
        float enter[VEC];
        {
            float2 rv[NP], iv[NP];
            if (MODE == kGroup) seq.at(t0);
            int64_t sl = seq.s - b;
            int tl = t0 - seq.beg;
#pragma unroll
            for (int j = 0; j < S; ++j) {
                const bool ok = mine && t0 + j < L;
                const int64_t t = MODE == kGroup ? tl : t0 + j, q = MODE == kGroup ? sl : 0;
                float row[VEC];
                load_vec<T, VEC>(r + q * p.rb + t * p.rt, ok, row);
                put_row<VEC>(rv, j, row);
                load_vec<T, VEC>(i + q * p.ib + t * p.it, ok, row);
                put_row<VEC>(iv, j, row);
                load_vec<T, VEC>(x + q * p.xb + t * p.xt, ok, row);
                put_row<VEC>(xv, j, row);
                load_vec<T, VEC>(dy + q * p.gb + t * p.gt, ok && has_dy, row);
                put_row<VEC>(gv, j, row);
                if (MODE == kGroup && ++tl == n.Ls) {
                    tl = 0;
                    ++sl;
                }
            }
#pragma unroll
            for (int v = 0; v < VEC; ++v) enter[v] = chunk * kChunk < L ? ck[(int64_t)chunk * D + v] : 0.0f;
            if (MODE == kPacked && t0 < L) seq.at(t0);
            if (fast_batch(small, rv, iv)) {
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    const Gates g = gates<true>(rv[k], iv[k], ncs);
                    sr[k] = g.sr; si[k] = g.si; w[k] = g.w; rs[k] = g.rs;
                }
            } else {
#pragma unroll
                for (int k = 0; k < NP; ++k) {
                    const Gates g = gates<false>(rv[k], iv[k], ncs);
                    sr[k] = g.sr; si[k] = g.si; w[k] = g.w; rs[k] = g.rs;
                }
            }
            if (t0 + S > L)               // tokens past the end change nothing
#pragma unroll
                for (int j = 0; j < S; ++j)
                    if (t0 + j >= L)
#pragma unroll
                        for (int v = 0; v < VEC; ++v) {
                            put<VEC>(w, j, v, 0.0f);
                            put<VEC>(rs, j, v, 0.0f);
                            put<VEC>(sr, j, v, 0.0f);
                        }
        }
        float2 a[NP], msi[NP], prev[NP];
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            a[k] = __fadd2_rn(w[k], f2(1.0f));
            msi[k] = __fmul2_rn(__fmul2_rn(one_minus_a2(w[k]), rs[k]), si[k]);
            prev[k] = __fmul2_rn(msi[k], xv[k]);        // for now what enters at the token
        }
        // forward composition (A, H), backward composition (A, K) of the warp's tokens
        unsigned starts = 0;
        if (CUTS && t0 < L && (seq.beg == t0 || seq.end < t0 + S)) {
            Seq<MODE> q = seq;
#pragma unroll
            for (int j = 0; j < S; ++j) {
                const int t = t0 + j;
                if (t < L && t == q.end) q.at(t);
                if (t < L && t == q.beg) starts |= 1u << j;
            }
        }
        auto state0 = [&](int t, int v) -> float {          // the state entering the sequence that starts at t
            Seq<MODE> q = seq;
            q.at(t);
            return o.h0 ? o.h0[q.s * D + dd + v] : 0.0f;
        };
        auto back0 = [&](int t, int v) -> float {           // what enters, from the right, the sequence that ends at t
            if (t < 0) return 0.0f;
            Seq<MODE> q = seq;
            q.at(t);
            return o.dh_last ? o.dh_last[q.s * D + dd + v] : 0.0f;
        };
        float A[VEC], H[VEC], K[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            A[v] = 1.0f;
            H[v] = 0.0f;
            K[v] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const bool cut = CUTS && (starts >> j & 1u);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float e = get<VEC>(prev, j, v);
                if (cut) {
                    A[v] = kCut;
                    H[v] = fmaf(get<VEC>(a, j, v), state0(t0 + j, v), e);
                } else {
                    then<CUTS>(A[v], H[v], get<VEC>(a, j, v), e);
                }
            }
        }
#pragma unroll
        for (int j = S - 1; j >= 0; --j) {
            const bool cut = CUTS && (starts >> j & 1u);
#pragma unroll
            for (int v = 0; v < VEC; ++v) K[v] = cut ? back0(t0 + j - 1, v) : get<VEC>(a, j, v) * (get<VEC>(gv, j, v) + K[v]);
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            ex[buf][warp][0][v][lane] = A[v];
            ex[buf][warp][1][v][lane] = H[v];
            ex[buf][warp][2][v][lane] = K[v];
        }
        __syncthreads();
        float sufA[VEC], sufK[VEC], totA[VEC], totK[VEC], h[VEC], back[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            totA[v] = 1.0f;
            totK[v] = 0.0f;
#pragma unroll
            for (int k = kWarps - 1; k >= 0; --k) {
                if (k == warp) {
                    sufA[v] = totA[v];
                    sufK[v] = totK[v];
                }
                then<CUTS>(totA[v], totK[v], ex[buf][k][0][v][lane], ex[buf][k][2][v][lane]);
            }
            h[v] = enter[v];
            for (int k = 0; k < warp; ++k) h[v] = apply<CUTS>(ex[buf][k][0][v][lane], ex[buf][k][1][v][lane], h[v]);
        }
        if (CLUSTER) {
            for (int k = warp; k < P; k += kWarps)
#pragma unroll
                for (int v = 0; v < VEC; ++v) st_cluster(smem_addr(&pub[buf][rank][v][lane]), k, make_float2(totA[v], totK[v]));
            cluster_sync();
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                for (int k = P - 1; k >= 0; --k) {
                    if (k == rank) back[v] = run[v];
                    const float2 f = pub[buf][k][v][lane];
                    run[v] = apply<CUTS>(f.x, f.y, run[v]);
                }
        } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                back[v] = run[v];
                run[v] = apply<CUTS>(totA[v], totK[v], run[v]);
            }
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) back[v] = apply<CUTS>(sufA[v], sufK[v], back[v]);
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const bool cut = CUTS && (starts >> j & 1u);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                if (cut) h[v] = state0(t0 + j, v);
                const float e = get<VEC>(prev, j, v);
                put<VEC>(prev, j, v, h[v]);
                h[v] = fmaf(get<VEC>(a, j, v), h[v], e);
            }
        }
#pragma unroll
        for (int j = S - 1; j >= 0; --j) {              // gv becomes G
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float G = get<VEC>(gv, j, v) + back[v];
                put<VEC>(gv, j, v, G);
                back[v] = t0 + j < L ? get<VEC>(a, j, v) * G : back[v];
            }
            if (CUTS && (starts >> j & 1u)) {
                Seq<MODE> q = seq;
                q.at(t0 + j);
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    if (o.dh0 && mine) o.dh0[q.s * D + d + v] = back[v];
                    back[v] = back0(t0 + j - 1, v);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            const float2 G = gv[k];
            const float2 ox = __fmul2_rn(G, msi[k]);
            const float2 oi = __fmul2_rn(__fmul2_rn(ox, xv[k]), __ffma2_rn(si[k], f2(-1.0f), f2(1.0f)));
            // du = G a (prev - (a / m) sigmoid(i) x)
            const float2 slope = __fmul2_rn(__fmul2_rn(a[k], rs[k]), __fmul2_rn(si[k], xv[k]));
            const float2 du = __fmul2_rn(__fmul2_rn(G, a[k]), __ffma2_rn(slope, f2(-1.0f), prev[k]));
            const float2 ds = __fmul2_rn(du, sr[k]);
            sum = __fadd2_rn(sum, ds);
            const float2 orr = __fmul2_rn(__fmul2_rn(ds, ncs), __ffma2_rn(sr[k], f2(-1.0f), f2(1.0f)));
#pragma unroll
            for (int half = 0; half < 2 / VEC; ++half) {
                const int t = t0 + (VEC == 2 ? k : 2 * k + half);
                if (mine && t < L) {
                    float vx[VEC], vr[VEC], vi[VEC];
#pragma unroll
                    for (int v = 0; v < VEC; ++v) {
                        const bool y = VEC == 2 ? v : half;
                        vx[v] = y ? ox.y : ox.x;
                        vr[v] = y ? orr.y : orr.x;
                        vi[v] = y ? oi.y : oi.x;
                    }
                    store_vec<T, VEC>(dx + (int64_t)t * D, vx);
                    store_vec<T, VEC>(dr + (int64_t)t * D, vr);
                    store_vec<T, VEC>(di + (int64_t)t * D, vi);
                }
            }
        }
    }
    __syncthreads();
    float* red = &ex[0][0][0][0][0];
#pragma unroll
    for (int v = 0; v < VEC; ++v) red[(warp * VEC + v) * 32 + lane] = VEC == 2 ? (v ? sum.y : sum.x) : sum.x + sum.y;
    __syncthreads();
    if (warp == 0 && mine)
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            float s = 0.0f;
            for (int k = 0; k < kWarps; ++k) s += red[(k * VEC + v) * 32 + lane];
            o.part[(run_id * P + rank) * D + d + v] = s;
        }
    if (rank != 0 || !mine || !o.dh0) return;
    if (MODE == kDense) {
        if (warp == 0)
#pragma unroll
            for (int v = 0; v < VEC; ++v) o.dh0[b * D + d + v] = run[v];
    } else if (MODE == kPacked) {
        for (int64_t s = warp; s < n.n; s += kWarps)
            if (n.cu[s] >= n.cu[s + 1])
#pragma unroll
                for (int v = 0; v < VEC; ++v)
                    o.dh0[s * D + d + v] = o.dh_last ? o.dh_last[s * D + d + v] : 0.0f;
    }
}

// dlam[d] = -c sigmoid(lam[d]) * sum of the partials of feature d, in order.
__global__ void rec_dlam_kernel(const float* __restrict__ part, int64_t n, int64_t D, const float* __restrict__ lam, float c,
                                float* __restrict__ dlam) {
    const int64_t d = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (d >= D) return;
    float s = 0.0f;
    for (int64_t k = 0; k < n; ++k) s += part[k * D + d];
    dlam[d] = -c * sigmoid_(lam[d]) * s;
}

// One token of every sequence: reads 3 values and a state, writes a value and a state.
template <typename T>
__global__ void rec_step_kernel(RecPtr p, int64_t B, int64_t D, const float* __restrict__ lam, float c, float* __restrict__ h,
                                T* __restrict__ y) {
    const int64_t n = B * D, stride = (int64_t)gridDim.x * blockDim.x;
    for (int64_t k = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; k < n; k += stride) {
        const int64_t b = k / D, d = k - b * D;
        const Gates g = gates<false>(f2(to_f32<T>(static_cast<const T*>(p.r)[b * p.rb + d])),
                                     f2(to_f32<T>(static_cast<const T*>(p.i)[b * p.ib + d])), f2(-c * softplus_(lam[d])));
        const float v = fmaf(1.0f + g.w.x, h[k], m_of(g).x * g.si.x * to_f32<T>(static_cast<const T*>(p.x)[b * p.xb + d]));
        h[k] = v;
        y[k] = from_f32<T>(v);
    }
}

bcm_status rec_validate(const bcm_gated_rec_args* a, const char* what) {
    BCM_REQUIRE(a != nullptr, "%s: null arguments", what);
    BCM_REQUIRE(dtype_ok(a->dtype), "%s: unsupported dtype %d", what, (int)a->dtype);
    BCM_REQUIRE(a->batch >= 0 && a->seqlen >= 0 && a->dim >= 1, "%s: bad sizes", what);
    BCM_REQUIRE(a->batch < (1ll << 31) && a->seqlen < (1ll << 31) - 4096 && a->dim < (1ll << 30),
                "%s: batch must be below 2^31, seqlen below 2^31 - 4096, dim below 2^30", what);
    BCM_REQUIRE(a->decay_scale >= 0.0f, "%s: decay_scale must not be negative", what);
    return BCM_OK;
}

RecPtr rec_ptr(const bcm_gated_rec_args* a) {
    RecPtr p;
    p.x = a->x; p.r = a->r; p.i = a->i; p.dy = a->dy;
    p.xb = a->x_stride_b; p.xt = a->x_stride_t;
    p.rb = a->r_stride_b; p.rt = a->r_stride_t;
    p.ib = a->i_stride_b; p.it = a->i_stride_t;
    p.gb = a->dy_stride_b; p.gt = a->dy_stride_t;
    return p;
}

int64_t rec_rows(const bcm_gated_rec_args* a) { return a->cu_seqlens ? a->seqlen : a->batch * a->seqlen; }
int64_t rec_parts(int64_t L, int part) { return (L + part - 1) / part; }

// How the tokens are dealt out.  It goes by sizes alone: forward and backward have to agree on the runs.
struct Plan {
    int mode, per, L, vec, P;
    int64_t runs;
};

Plan rec_plan(const bcm_gated_rec_args* a, int vec) {
    Plan pl = {kDense, 1, (int)a->seqlen, vec, 1, a->batch};
    // in units of the widest tile, so that the runs do not depend on alignment
    const int64_t wide = (a->dim + 63) / 64, tiles = (a->dim + 32 * vec - 1) / (32 * vec);
    if (a->cu_seqlens) {
        pl.mode = kPacked;
        pl.runs = 1;
    } else if (a->seqlen < 4 * kChunkFwd && a->batch > 1) {
        // runs of about 8 chunks (an eighth of the last one empty at most), fewer where that leaves SMs without a block
        pl.mode = kGroup;
        int64_t per = (8 * kChunkFwd + a->seqlen - 1) / a->seqlen;
        while (per > 1 && per * a->seqlen > kChunkFwd && ((a->batch + per - 1) / per) * wide < 4 * (int64_t)sm_count()) per = (per + 1) / 2;
        pl.per = (int)std::min<int64_t>(per, a->batch);
        pl.L = (int)(pl.per * a->seqlen);
        pl.runs = (a->batch + pl.per - 1) / pl.per;
    }
    // blocks of a cluster: as many as the chunks allow until the GPU holds three blocks per SM
    while (pl.P < kMaxCluster && pl.runs * tiles * pl.P < 3 * (int64_t)sm_count() && 2 * pl.P <= rec_parts(pl.L, kChunkFwd)) pl.P *= 2;
    return pl;
}

// Two features a lane where rows are even and aligned for it.
int rec_vec(const bcm_gated_rec_args* a, bool bwd) {
    const size_t s = 2 * dtype_size(a->dtype);
    int64_t odd = a->dim;
    uintptr_t at = 0;
    auto see = [&](const void* p, int64_t sb, int64_t st) {
        at |= (uintptr_t)p;
        odd |= (a->cu_seqlens || a->batch == 1 ? 0 : sb) | (a->seqlen == 1 ? 0 : st);
    };
    see(a->x, a->x_stride_b, a->x_stride_t);
    see(a->r, a->r_stride_b, a->r_stride_t);
    see(a->i, a->i_stride_b, a->i_stride_t);
    if (bwd) {
        if (a->dy) see(a->dy, a->dy_stride_b, a->dy_stride_t);
        at |= (uintptr_t)a->dx | (uintptr_t)a->dr | (uintptr_t)a->di;
    } else {
        at |= (uintptr_t)a->y;
    }
    return (odd & 1) == 0 && at % s == 0 ? 2 : 1;
}

template <typename F>
bcm_status rec_launch_as(F* kernel, const bcm_gated_rec_args* a, const RecOut& o, const Plan& pl, cudaStream_t stream) {
    const int64_t blocks = ((a->dim + 32 * pl.vec - 1) / (32 * pl.vec)) * pl.runs * pl.P;
    BCM_REQUIRE(blocks < (1ll << 31), "gated_rec: batch x dim too large");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)pl.P;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pl.P > 1 ? 1 : 0;
    if (pl.P > 8) BCM_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    const RecDim n = {a->cu_seqlens, a->batch, pl.L, (int)a->seqlen, pl.per, (int)a->dim, pl.P};
    BCM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, rec_ptr(a), o, n, a->lam, a->decay_scale));
    return BCM_OK;
}

template <bool BWD, typename T, int VEC, int MODE>
bcm_status rec_launch_p(const bcm_gated_rec_args* a, const RecOut& o, const Plan& pl, cudaStream_t stream) {
    if constexpr (BWD) {
        return pl.P > 1 ? rec_launch_as(rec_bwd_kernel<T, VEC, MODE, true>, a, o, pl, stream)
                        : rec_launch_as(rec_bwd_kernel<T, VEC, MODE, false>, a, o, pl, stream);
    } else {
        return pl.P > 1 ? rec_launch_as(rec_fwd_kernel<T, VEC, MODE, true>, a, o, pl, stream)
                        : rec_launch_as(rec_fwd_kernel<T, VEC, MODE, false>, a, o, pl, stream);
    }
}

template <bool BWD, typename T, int VEC>
bcm_status rec_launch_v(const bcm_gated_rec_args* a, const RecOut& o, const Plan& pl, cudaStream_t stream) {
    if (pl.mode == kDense) return rec_launch_p<BWD, T, VEC, kDense>(a, o, pl, stream);
    if (pl.mode == kGroup) return rec_launch_p<BWD, T, VEC, kGroup>(a, o, pl, stream);
    return rec_launch_p<BWD, T, VEC, kPacked>(a, o, pl, stream);
}

template <bool BWD>
bcm_status rec_launch(const bcm_gated_rec_args* a, const RecOut& o, const Plan& pl, cudaStream_t stream) {
    return dispatch_dtype(a->dtype, [&](auto tag) -> bcm_status {
        using T = decltype(tag);
        return pl.vec == 2 ? rec_launch_v<BWD, T, 2>(a, o, pl, stream) : rec_launch_v<BWD, T, 1>(a, o, pl, stream);
    });
}

}  // namespace
}  // namespace bcm

using namespace bcm;

extern "C" size_t bcm_gated_rec_ckpt_bytes(const bcm_gated_rec_args* a) {
    if (!a || a->batch < 0 || a->seqlen < 0 || a->dim < 1) return 0;
    if (rec_rows(a) == 0) return 0;
    const Plan pl = rec_plan(a, 1);
    return align_up((size_t)pl.runs * (size_t)rec_parts(pl.L, kCkpt) * (size_t)a->dim * sizeof(float), 256);
}

extern "C" size_t bcm_gated_rec_bwd_workspace_bytes(const bcm_gated_rec_args* a) {
    if (!a || a->batch < 0 || a->seqlen < 0 || a->dim < 1) return 0;
    if (rec_rows(a) == 0) return 0;
    const Plan pl = rec_plan(a, 2);         // one lane a feature takes no more blocks to a cluster than two
    return align_up((size_t)pl.runs * (size_t)pl.P * (size_t)a->dim * sizeof(float), 256);
}

extern "C" bcm_status bcm_gated_rec_fwd(const bcm_gated_rec_args* a, cudaStream_t stream) {
    clear_error();
    if (bcm_status st = rec_validate(a, "gated_rec_fwd"); st != BCM_OK) return st;
    if (a->batch == 0) return BCM_OK;
    BCM_REQUIRE(a->lam && a->h_last && (rec_rows(a) == 0 || (a->x && a->r && a->i && a->y)), "gated_rec_fwd: null pointer");
    if (a->ckpt && a->ckpt_bytes < bcm_gated_rec_ckpt_bytes(a)) {
        set_error("gated_rec_fwd: ckpt of %zu bytes < required %zu", a->ckpt_bytes, bcm_gated_rec_ckpt_bytes(a));
        return BCM_ERR_WORKSPACE;
    }
    if (rec_rows(a) == 0) {                 // no token: the states stay
        const size_t bytes = sizeof(float) * (size_t)a->batch * (size_t)a->dim;
        if (a->h0) BCM_CUDA_TRY(cudaMemcpyAsync(a->h_last, a->h0, bytes, cudaMemcpyDeviceToDevice, stream));
        else BCM_CUDA_TRY(cudaMemsetAsync(a->h_last, 0, bytes, stream));
        return BCM_OK;
    }
    RecOut o = {};
    o.h0 = a->h0; o.y = a->y; o.h_last = a->h_last; o.ckpt = static_cast<float*>(a->ckpt);
    return rec_launch<false>(a, o, rec_plan(a, rec_vec(a, false)), stream);
}

extern "C" bcm_status bcm_gated_rec_bwd(const bcm_gated_rec_args* a, cudaStream_t stream) {
    clear_error();
    if (bcm_status st = rec_validate(a, "gated_rec_bwd"); st != BCM_OK) return st;
    BCM_REQUIRE(a->lam && a->dlam, "gated_rec_bwd: null pointer");
    if (rec_rows(a) == 0) {
        const size_t bytes = sizeof(float) * (size_t)a->batch * (size_t)a->dim;
        BCM_CUDA_TRY(cudaMemsetAsync(a->dlam, 0, sizeof(float) * a->dim, stream));
        if (a->dh0 && a->dh_last) BCM_CUDA_TRY(cudaMemcpyAsync(a->dh0, a->dh_last, bytes, cudaMemcpyDeviceToDevice, stream));
        else if (a->dh0) BCM_CUDA_TRY(cudaMemsetAsync(a->dh0, 0, bytes, stream));
        return BCM_OK;
    }
    BCM_REQUIRE(a->batch >= 1 && a->x && a->r && a->i && a->dx && a->dr && a->di && a->ckpt, "gated_rec_bwd: null pointer");
    const size_t need = bcm_gated_rec_bwd_workspace_bytes(a), ck = bcm_gated_rec_ckpt_bytes(a);
    if (!a->workspace || a->workspace_bytes < need || a->ckpt_bytes < ck) {
        set_error("gated_rec_bwd: workspace of %zu bytes or ckpt of %zu bytes < required %zu and %zu", a->workspace_bytes,
                  a->ckpt_bytes, need, ck);
        return BCM_ERR_WORKSPACE;
    }
    RecOut o = {};
    o.h0 = a->h0; o.ckpt = static_cast<float*>(a->ckpt);
    o.dh_last = a->dh_last; o.dx = a->dx; o.dr = a->dr; o.di = a->di;
    o.part = static_cast<float*>(a->workspace); o.dh0 = a->dh0;
    const Plan pl = rec_plan(a, rec_vec(a, true));
    if (bcm_status st = rec_launch<true>(a, o, pl, stream); st != BCM_OK) return st;
    rec_dlam_kernel<<<(unsigned)ceil_div(a->dim, 128), 128, 0, stream>>>(o.part, pl.runs * pl.P, a->dim, a->lam, a->decay_scale,
                                                                        a->dlam);
    BCM_LAUNCH_CHECK();
    return BCM_OK;
}

extern "C" bcm_status bcm_gated_rec_step(const void* x, int64_t x_stride_b, const void* r, int64_t r_stride_b, const void* i,
                                         int64_t i_stride_b, bcm_dtype dtype, int64_t batch, int64_t dim, const float* lam,
                                         float decay_scale, float* h, void* y, cudaStream_t stream) {
    clear_error();
    BCM_REQUIRE(dtype_ok(dtype), "gated_rec_step: unsupported dtype %d", (int)dtype);
    BCM_REQUIRE(batch >= 0 && dim >= 1 && batch < (1ll << 31) && dim < (1ll << 31), "gated_rec_step: bad sizes");
    BCM_REQUIRE(decay_scale >= 0.0f, "gated_rec_step: decay_scale must not be negative");
    if (batch == 0) return BCM_OK;
    BCM_REQUIRE(x && r && i && lam && h && y, "gated_rec_step: null pointer");
    RecPtr p = {};
    p.x = x; p.r = r; p.i = i;
    p.xb = x_stride_b; p.rb = r_stride_b; p.ib = i_stride_b;
    const int64_t want = (batch * dim + 255) / 256;
    const unsigned grid = (unsigned)std::min<int64_t>(want, (int64_t)sm_count() * 8);
    return dispatch_dtype(dtype, [&](auto tag) -> bcm_status {
        using T = decltype(tag);
        rec_step_kernel<T><<<grid, 256, 0, stream>>>(p, batch, dim, lam, decay_scale, h, static_cast<T*>(y));
        BCM_LAUNCH_CHECK();
        return BCM_OK;
    });
}
