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

// ---- the gates of two features at a time ------------------------------------
// A lane owns two neighbouring features; its arithmetic is packed fp32 (two
// results an instruction).  What bounds it then is the special-function unit
// (8 cycles a warp instruction), so:
//  * v = 1 - a = -expm1(u) is a polynomial for U = -u <= kPolyEnd (degree 4 times
//    U, interpolated at Chebyshev nodes, relative error 2.5e-8).  It also gives
//    1 - a^2 = v + v a without cancellation and a correctly rounded a = 1 - v, so
//    that a memory of a thousand tokens does not add up a biased decay.  Beyond, a
//    is the exponential itself and v = 1 - a: gradients are proportional to a, and
//    1 - v would leave it a multiple of 2^-24, 0 from U = 17 on;
//  * FAST shares one reciprocal between the four sigmoids of a pair and needs no
//    exponential for a: 7 special functions a pair instead of 12.  It holds where
//    every c s lies in [kCsLow, kPolyEnd] and the product of a pair's four
//    denominators (1 + e^-r)(1 + e^-i) stays below kProdEnd (U is a normal number
//    then); a warp that finds a larger one (gates below about -10, infinite, NaN)
//    computes its batch again in the long form.  One feature in 64 outside the range
//    (an open gate's decay below 0.705 a token) costs its warp as much as all of them:
//    128 x 4000 x 256 bf16 forward 261 -> 385 us, backward 540 -> 640 us, fp32 348 ->
//    410 and 620 -> 658 us.
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPolyEnd = 0.35f, kCsLow = 1e-18f;
constexpr float kProdEnd = 1e18f;

__device__ __forceinline__ float ex2_(float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float rcp_(float v) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float rsqrt_(float v) { float r; asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float max_nan_(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float2 f2(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 mul(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 fma(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }

// Constants as register pairs: packed instructions take no immediates, and left to itself the compiler sets each pair
// up again at every use (a quarter of the loop's instructions).
__device__ __forceinline__ float2 pinned(float v) {
    float2 r;
    asm volatile("mov.b32 %0, %2; mov.b32 %1, %2;" : "=f"(r.x), "=f"(r.y) : "f"(v));
    return r;
}
struct Consts {
    float2 nlog2e, one, c1, c2, c3, c4;
    __device__ __forceinline__ Consts()
        : nlog2e(pinned(-kLog2e)), one(pinned(1.0f)), c1(pinned(-0.49999821186065674f)), c2(pinned(0.16662530601024628f)),
          c3(pinned(-0.04133187234401703f)), c4(pinned(0.007211245596408844f)) {}
};

struct Gates {
    float2 sr, si, a, m, rs;     // sigmoid(r), sigmoid(i), a, m, 1 / m (0 where m = 0)
};

template <bool FAST>
__device__ __forceinline__ Gates gates(float2 r, float2 i, float2 cs, const Consts& k, float& prod) {
    Gates g;
    const float2 tr = mul(r, k.nlog2e), ti = mul(i, k.nlog2e);
    const float2 dr = add(make_float2(ex2_(tr.x), ex2_(tr.y)), k.one);
    const float2 di = add(make_float2(ex2_(ti.x), ex2_(ti.y)), k.one);
    if (FAST) {
        const float2 both = mul(dr, di);
        const float all = both.x * both.y;
        prod = max_nan_(prod, all);
        const float inv = rcp_(all);
        const float2 each = make_float2(both.y * inv, both.x * inv);
        g.sr = mul(di, each);
        g.si = mul(dr, each);
    } else {
        g.sr = make_float2(rcp_(dr.x), rcp_(dr.y));
        g.si = make_float2(rcp_(di.x), rcp_(di.y));
    }
    const float2 U = mul(cs, g.sr);
    float2 q = fma(U, k.c4, k.c3);
    q = fma(U, q, k.c2);
    q = fma(U, q, k.c1);
    float2 v = fma(mul(U, U), q, U);
    g.a = make_float2(1.0f - v.x, 1.0f - v.y);
    if (!FAST) {
        if (!(U.x <= kPolyEnd)) {
            g.a.x = ex2_(U.x * -kLog2e);
            v.x = 1.0f - g.a.x;
        }
        if (!(U.y <= kPolyEnd)) {
            g.a.y = ex2_(U.y * -kLog2e);
            v.y = 1.0f - g.a.y;
        }
    }
    const float2 m2 = fma(v, g.a, v);
    g.rs = make_float2(rsqrt_(m2.x), rsqrt_(m2.y));
    if (!FAST) {
        if (m2.x == 0.0f || g.rs.x == __int_as_float(0x7f800000)) g.rs.x = 0.0f;
        if (m2.y == 0.0f || g.rs.y == __int_as_float(0x7f800000)) g.rs.y = 0.0f;
    }
    g.m = mul(m2, g.rs);
    return g;
}

// ---- layout of the scan kernels -----------------------------------------------
// A warp owns a few consecutive tokens of 64 features, a block kWarps times as
// many (a chunk).  A block's chunks follow one another in a loop (turns) that
// carries the state; P blocks of a cluster take P consecutive chunks per turn, so
// that few features with long sequences still fill the GPU.  Every input is read
// once: the composition h -> A h + H of a warp's tokens goes to shared memory,
// the other warps' and blocks' compositions give the state that enters, and the
// tokens, still in registers, are replayed from it.  Rows arrive by 16-byte
// cp.async a few turns ahead; a warp copies its own rows only.  Two blocks share
// an SM: one computes while the other exchanges.  (Computing the next turn's gates
// before a turn is replayed, with a split cluster barrier, needs both turns in
// registers: it spilled and ran 20 to 30 % slower.)  128 x 4000 x 256: fp32 forward
// 336 us (6.2 TB/s), backward 618 us (5.9 TB/s), bound by memory; bf16 261 and 541 us,
// bound by instructions and their latency (42 and 89 instructions a value, issue slots
// 60 % busy with 3.5 warps a scheduler at 128 x 1000 x 256).
//
// Mode: kDense, one sequence per block; kGroup, a block takes `per` consecutive
// dense sequences as one run of tokens (short sequences would leave most of a
// chunk empty); kPacked, the sequences' offsets stand in cu, and run g of G takes
// the sequences that start in the g-th part of the tokens (found on the device).
// Where a sequence starts inside a run, nothing passes and its own state enters.
//
// Few features with long sequences: a sequence (kDense) or the whole packed run is
// cut into segments of fixed length.  A first launch (SUM) only composes every
// segment, a small kernel carries the state over them, and the second launch starts
// each segment from its own.
constexpr int kWarps = 8;
constexpr int kTile = 64;                        // features of a block
constexpr int kStepsFwd = 8, kStepsBwd = 4;      // tokens of a warp's turn (the backward keeps 7 values a token)
constexpr int kCkpt = kWarps * kStepsBwd;        // the forward keeps the state that enters every kCkpt tokens of a run
constexpr int kMaxCluster = 8;                   // (16 measured no faster: a turn's exchange grew with the blocks)
constexpr float kCut = -1.0f;                    // in place of a product of decays: nothing passes (a sequence starts inside)

enum Mode { kDense, kGroup, kPacked };

struct RecPtr {
    const void* x; const void* r; const void* i; const void* dy;
    int64_t xb, xt, rb, rt, ib, it, gb, gt;
};

struct RecOut {
    const float* h0; void* y; float* h_last; float* ckpt;                          // forward
    const float* dh_last; void* dx; void* dr; void* di; float* part; float* dh0;   // backward
    const float* seg; float* sum;                  // segments: what enters each of them; their compositions [2] (SUM)
};

// A run holds L tokens (kGroup: its last may hold fewer; kPacked: all runs together), a sequence Ls (kDense, kGroup),
// per sequences make a run (kGroup), runs of them (kPacked); n sequences, D features, P blocks in a cluster.
struct RecDim {
    const int32_t* cu;
    int64_t n;
    int L, Ls, per, runs, D, P;
    int segs, seg;            // segments of a sequence (1: none) and their length
};

// The sequence that holds token t: the last s with cu[s] <= t, in [0, n).  Called by whole warps; t is uniform.
__device__ __forceinline__ int seq_of(const int32_t* cu, int n, int t) {
    int lo = 0, hi = n - 1;                          // the answer lies in [lo, hi]
    const int lane = threadIdx.x & 31;
    while (hi > lo) {
        const int step = (hi - lo + 31) / 32;        // lanes look at lo + step, lo + 2 step, ...
        const int64_t at = lo + (int64_t)(lane + 1) * step;
        const int c = __popc(__ballot_sync(kFull, at <= hi && cu[at] <= t));
        lo += c * step;
        hi = min(hi, lo + step - 1);
    }
    return lo;
}

// The sequence around a token of the run, moved along by a warp: its index s, its first token and its end.
template <int MODE>
struct Seq {
    const int32_t* cu;
    int n, Ls, off;           // off: the run's first token (kPacked)
    int64_t s0, s;
    int beg, end;
    __device__ __forceinline__ void at(int t) {
        if (MODE == kDense || (beg <= t && t < end)) return;
        if (MODE == kPacked) {
            const int k = seq_of(cu, n, t + off);
            s = k;
            beg = cu[k] - off;
            end = cu[k + 1] - off;
        } else {
            const int k = t / Ls;
            s = s0 + k;
            beg = k * Ls;
            end = beg + Ls;
        }
    }
};

// (A1, H1) followed by (A2, H2)
template <bool CUTS>
__device__ __forceinline__ void then(float2& A1, float2& H1, float2 A2, float2 H2) {
    if (!CUTS) {
        H1 = fma(A2, H1, H2);
        A1 = mul(A1, A2);
    } else if (A2.x < 0.0f) {                        // (cuts lie between tokens: both features have them)
        A1 = f2(kCut);
        H1 = H2;
    } else {
        const bool cut = A1.x < 0.0f;
        H1 = fma(A2, H1, H2);
        A1 = cut ? f2(kCut) : mul(A1, A2);
    }
}
template <bool CUTS>
__device__ __forceinline__ float2 apply(float2 A, float2 H, float2 h) {
    return CUTS && A.x < 0.0f ? H : fma(A, h, H);
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void st_cluster(uint32_t addr, int rank, float4 v) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(remote), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Where a block works.
struct Place {
    int lane, warp, rank, tile, d, L;
    int off;                  // the run's first token (kPacked, segments)
    int64_t run, b;           // the run and its first sequence (kDense, kGroup)
    bool has0, has1;          // the lane's features exist
};
template <int MODE, bool CLUSTER>
__device__ __forceinline__ Place place(const RecDim& n, const int32_t* cu) {
    Place q;
    q.off = 0;
    q.lane = threadIdx.x & 31;
    q.warp = threadIdx.x >> 5;
    const int P = CLUSTER ? n.P : 1, tiles = (n.D + kTile - 1) / kTile;
    q.rank = CLUSTER ? blockIdx.x % P : 0;
    q.run = blockIdx.x / P / tiles;
    q.tile = (int)(blockIdx.x / P - q.run * tiles);
    q.b = MODE == kGroup ? q.run * n.per : q.run / n.segs;
    q.L = MODE == kGroup ? (int)min((int64_t)n.per, n.n - q.b) * n.Ls : n.L;
    if (MODE != kGroup && n.segs > 1) {
        q.off = (int)min((q.run - q.b * n.segs) * n.seg, (int64_t)n.L);
        q.L = min(n.L - q.off, n.seg);
    }
    q.d = q.tile * kTile + q.lane * 2;
    q.has0 = q.d < n.D;
    q.has1 = q.d + 1 < n.D;
    if (MODE == kPacked && n.runs > 1) {
        // from the first start at or after run * L / runs to that at or after (run + 1) * L / runs
        int at[2] = {0, n.L};
        for (int k = 0; k < 2; ++k) {
            const int64_t edge = (q.run + k) * n.L / n.runs;
            if (edge > 0 && edge < n.L) at[k] = min(max(cu[seq_of(cu, (int)n.n, (int)edge - 1) + 1], 0), n.L);
        }
        q.off = at[0];
        q.L = max(at[1] - at[0], 0);
    }
    return q;
}

// ---- rows in shared memory -----------------------------------------------------
// A row of a tile is 64 elements from the tile's first feature on.  kRows16: every
// row starts on 16 bytes and arrives by 16-byte copies.  kRows4: on 4 bytes, every
// lane copies its own two features.  kRows2 (16-bit types): the copy starts at the
// 16-byte granule that holds the row's first element and takes one granule more; it
// reads no granule without an element of the row in it.  400 x 300 x 300 bf16
// backward: 290 us by granules, 236 us by 4-byte copies (187 us since pairs between
// words are read without a branch).
enum Form { kRows2, kRows4, kRows16 };
template <typename T, int FORM>
struct Rows {
    static constexpr bool EVEN = FORM != kRows2;
    static constexpr int kGran = kTile * (int)sizeof(T) / 16 + (EVEN ? 0 : 1);
    static constexpr int kPitch = kGran * 16;

    // off: bytes of the row's first element past its granule
    static __device__ __forceinline__ float2 read(const char* row, int off) {
        const char* p = row + (threadIdx.x & 31) * 2 * sizeof(T) + (EVEN ? 0 : off);
        if constexpr (sizeof(T) == 4) {
            if (EVEN) return *reinterpret_cast<const float2*>(p);
            return make_float2(*reinterpret_cast<const float*>(p), *reinterpret_cast<const float*>(p + 4));
        } else {
            // (a row may start between two words: both words of the pair, without a branch)
            const uint32_t* q = reinterpret_cast<const uint32_t*>(EVEN ? p : p - (off & 2));
            uint32_t w = q[0];
            if (!EVEN) w = __funnelshift_r(w, q[1], (off & 2) * 8);
            T v[2];
            memcpy(v, &w, 4);
            return make_float2(to_f32<T>(v[0]), to_f32<T>(v[1]));
        }
    }
};

// One input of a warp: fetches S rows a turn, reads them back.  Where a row of the run follows the one before it by st
// elements (kDense, kPacked, and kGroup without gaps between sequences) and all S rows are there, the lane's granule
// (kRows16) only moves along.
struct Input {
    const void* p;
    int64_t sb, st;
};
template <typename T, int MODE, int FORM, int S>
struct Stream {
    using R = Rows<T, FORM>;
    static constexpr bool EVEN = FORM == kRows16;
    static constexpr int kLaneRows = 32 / R::kGran;      // rows of a warp's copy instruction
    const char* at;
    int bytes;
    uint32_t low, step;                                  // the run's first row and the distance of rows, in bytes, mod 2^32
    __device__ __forceinline__ static bool linear(const Input& in, const RecDim& n) { return MODE != kGroup || in.sb == in.st * n.Ls; }
    // elements from the run's first row to that of token t
    __device__ __forceinline__ static int64_t row(const Input& in, const RecDim& n, int t) {
        if (linear(in, n)) return (int64_t)t * in.st;
        const int k = t / n.Ls;
        return k * in.sb + (int64_t)(t - k * n.Ls) * in.st;
    }
    __device__ __forceinline__ static const T* base(const Input& in, const Place& w) {
        return static_cast<const T*>(in.p) + (MODE == kPacked ? 0 : w.b * in.sb) + w.off * in.st + (int64_t)w.tile * kTile;
    }
    __device__ __forceinline__ Stream(const Input& in, const Place& w, int t0, int width) {
        bytes = max(0, min(16, width * (int)sizeof(T) - w.lane % R::kGran * 16));
        low = (uint32_t)(uintptr_t)base(in, w);
        step = (uint32_t)(in.st * (int)sizeof(T));
        at = reinterpret_cast<const char*>(base(in, w) + (int64_t)(t0 + w.lane / R::kGran) * in.st);
        if (EVEN) at += w.lane % R::kGran * 16;          // (kRows2: the row's start, its granules move with it)
        if (FORM == kRows4) {
            at = reinterpret_cast<const char*>(base(in, w) + (int64_t)t0 * in.st + w.lane * 2);
            bytes = max(0, min(2, width - w.lane * 2)) * (int)sizeof(T);
        }
    }
    // t0: the first row; advance: tokens from this fetch to the next; rows and features that are not there become zeros
    __device__ __forceinline__ void fetch(char* dst, const Input& in, const Place& w, const RecDim& n, int t0, int advance, int width) {
        const uint32_t to = smem_addr(dst);
        if constexpr (FORM == kRows4) {
            auto copy = [&](int j, const char* src, int size) {
                const uint32_t d = to + j * R::kPitch + w.lane * 2 * (int)sizeof(T);
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(d), "l"(src), "r"(min(size, 4)) : "memory");
                if (sizeof(T) == 4)
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(d + 4), "l"(size > 4 ? src + 4 : src), "r"(max(size - 4, 0)) : "memory");
            };
            if (t0 + S <= w.L && linear(in, n)) {
                const char* src = at;
#pragma unroll
                for (int j = 0; j < S; ++j) {
                    copy(j, src, bytes);
                    src += in.st * (int)sizeof(T);
                }
            } else {
                const T* from0 = base(in, w);
#pragma unroll 1
                for (int j = 0; j < S; ++j) {
                    const bool there = t0 + j < w.L && bytes > 0;
                    copy(j, reinterpret_cast<const char*>(there ? from0 + row(in, n, t0 + j) + w.lane * 2 : from0), there ? bytes : 0);
                }
            }
        } else if (EVEN && t0 + S <= w.L && linear(in, n)) {
#pragma unroll
            for (int k = 0; k < S / kLaneRows; ++k)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + w.lane * 16 + k * 512),
                             "l"(at + (int64_t)(k * kLaneRows) * in.st * (int)sizeof(T)), "r"(bytes)
                             : "memory");
        } else if (FORM == kRows2 && t0 + S <= w.L && linear(in, n)) {
            const int j0 = w.lane / R::kGran, g = w.lane - j0 * R::kGran;
            const char* first = at;
#pragma unroll
            for (int j = 0; j < S; j += kLaneRows) {
                const uintptr_t from = ((uintptr_t)first & ~(uintptr_t)15) + g * 16;
                const int left = (int)((int64_t)((uintptr_t)first + width * sizeof(T)) - (int64_t)from);
                if (j0 < kLaneRows && j0 + j < S)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + (j0 + j) * R::kPitch + g * 16),
                                 "l"(left > 0 ? from : (uintptr_t)first & ~(uintptr_t)15), "r"(max(0, min(16, left)))
                                 : "memory");
                first += (int64_t)kLaneRows * in.st * (int)sizeof(T);
            }
        } else {
            const T* from0 = base(in, w);
#pragma unroll 1
            for (int q = w.lane; q < S * R::kGran; q += 32) {
                const int j = q / R::kGran, g = q - j * R::kGran;
                int bytes = 0;
                uintptr_t src = reinterpret_cast<uintptr_t>(from0) & ~(uintptr_t)15;
                if (t0 + j < w.L) {
                    const uintptr_t first = reinterpret_cast<uintptr_t>(from0 + row(in, n, t0 + j)), end = first + width * sizeof(T);
                    const uintptr_t from = (first & ~(uintptr_t)15) + g * 16;
                    if (from < end) {
                        src = from;
                        bytes = (int)min((uintptr_t)16, end - from);
                    }
                }
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + j * R::kPitch + g * 16), "l"(src), "r"(bytes) : "memory");
            }
        }
        at += (int64_t)advance * in.st * (int)sizeof(T);
    }
    // the lane's two features of token t, in slot j of the fetched rows
    __device__ __forceinline__ float2 read(const char* from, const Input& in, const RecDim& n, int j, int t) const {
        uint32_t off = 0;
        if (FORM == kRows2) off = (low + (linear(in, n) ? (uint32_t)t * step : (uint32_t)row(in, n, t) * (uint32_t)sizeof(T))) & 15u;
        return R::read(from + j * R::kPitch, (int)off);
    }
};

// one row's two features; pair: both exist and lie on 2 * sizeof(T)
template <typename T>
__device__ __forceinline__ void store_row(T* p, float2 v, bool pair, bool one) {
    if (pair) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float2*>(p) = v;
        } else {
            const T e[2] = {from_f32<T>(v.x), from_f32<T>(v.y)};
            uint32_t w;
            memcpy(&w, e, 4);
            *reinterpret_cast<uint32_t*>(p) = w;
        }
    } else if (one) {
        p[0] = from_f32<T>(v.x);
    }
}
template <typename T, bool EVEN>
__device__ __forceinline__ void store_pair(T* p, float2 v, bool even_rows, bool has0, bool has1) {
    if (EVEN || even_rows) {
        store_row<T>(p, v, has0, false);
    } else if (((uintptr_t)p & (2 * sizeof(T) - 1)) == 0) {      // (every other row of an odd number of features)
        store_row<T>(p, v, has1, has0);
    } else {
        if (has0) p[0] = from_f32<T>(v.x);
        if (has1) p[1] = from_f32<T>(v.y);
    }
}

__device__ __forceinline__ float2 load_state(const float* p, int64_t row, int D, int d, bool has0, bool has1) {
    if (p == nullptr) return f2(0.0f);
    return make_float2(has0 ? p[row * D + d] : 0.0f, has1 ? p[row * D + d + 1] : 0.0f);
}
__device__ __forceinline__ void store_state(float* p, int64_t row, int D, int d, float2 v, bool has0, bool has1) {
    if (has0) p[row * D + d] = v.x;
    if (has1) p[row * D + d + 1] = v.y;
}

// The run's first row of kept states.
template <int MODE>
__device__ __forceinline__ int64_t ckpt_row(const Place& w, const RecDim& n) {
    return MODE == kPacked ? w.off / kCkpt + w.run : (MODE == kDense ? w.b : w.run) * ((n.L + kCkpt - 1) / kCkpt) + w.off / kCkpt;
}

// Bit j: a sequence starts at token t0 + j.
template <int MODE, int S>
__device__ __forceinline__ unsigned starts_in(const Seq<MODE>& seq, int t0, int L) {
    if (MODE == kDense || t0 >= L || (seq.beg != t0 && seq.end >= t0 + S)) return 0u;
    unsigned m = 0;
    Seq<MODE> q = seq;
    for (int j = 0; j < S && t0 + j < L; ++j) {
        q.at(t0 + j);
        if (t0 + j == q.beg) m |= 1u << j;
    }
    return m;
}

// The sequences' offsets of a packed run, in shared memory where they fit.
constexpr int kCuMax = 1024;
template <int MODE>
__device__ __forceinline__ const int32_t* stage_cu(const RecDim& n, int32_t* room) {
    if (MODE != kPacked || n.n >= kCuMax) return n.cu;
    for (int k = threadIdx.x; k <= (int)n.n; k += kWarps * 32) room[k] = n.cu[k];
    __syncthreads();
    return room;
}

template <typename T, int S, int FORM, int ARRAYS>
constexpr int stage_bytes() { return kWarps * ARRAYS * S * Rows<T, FORM>::kPitch; }
// turns of rows in shared memory, as many as let two blocks share an SM
template <typename T>
constexpr int stages_fwd() { return sizeof(T) == 4 ? 2 : 3; }
template <typename T>
constexpr int stages_bwd() { return sizeof(T) == 4 ? 2 : 3; }

// A block's (A, H) or (A, K) of a turn goes to every block of the cluster.  Two turns' slots: a block writes those of
// turn k + 2 only after every block has arrived for turn k + 1, hence has read those of turn k.
template <bool CLUSTER>
struct Pub {
    float4 v[CLUSTER ? 2 : 1][CLUSTER ? kMaxCluster : 1][CLUSTER ? 32 : 1];
};

template <typename T, int MODE, int FORM, bool CLUSTER, bool SUM>
__global__ void __launch_bounds__(kWarps * 32, 2)
rec_fwd_kernel(const __grid_constant__ RecPtr p, const __grid_constant__ RecOut o, const __grid_constant__ RecDim n,
               const float* __restrict__ lam, float c) {
    constexpr bool CUTS = MODE != kDense;
    constexpr int S = kStepsFwd, kChunk = kWarps * S, ST = stages_fwd<T>();
    using In = Stream<T, MODE, FORM, S>;
    using R = Rows<T, FORM>;
    __shared__ float4 ex[2][kWarps][32];
    __shared__ Pub<CLUSTER> pub;
    __shared__ int32_t cus[MODE == kPacked ? kCuMax : 1];
    extern __shared__ __align__(16) char rows[];
    const int32_t* cu = stage_cu<MODE>(n, cus);
    const Place w = place<MODE, CLUSTER>(n, cu);
    const int D = n.D, L = w.L, P = CLUSTER ? n.P : 1, width = min(kTile, D - w.tile * kTile);
    T* y = static_cast<T*>(o.y) + ((MODE == kPacked ? 0 : w.b * n.Ls) + w.off) * D + w.d;
    const bool even_rows = (D & 1) == 0 && (uintptr_t)o.y % (2 * sizeof(T)) == 0;
    const int turns = (((MODE == kGroup ? n.L : L) + kChunk - 1) / kChunk + P - 1) / P;
    float* ck = o.ckpt ? o.ckpt + ckpt_row<MODE>(w, n) * D : nullptr;
    const float2 l = load_state(lam, 0, D, w.d, w.has0, w.has1);
    const float2 cs = make_float2(w.has0 ? c * softplus_(l.x) : kPolyEnd, w.has1 ? c * softplus_(l.y) : kPolyEnd);
    const bool small = __all_sync(kFull, cs.x >= kCsLow && cs.x <= kPolyEnd && cs.y >= kCsLow && cs.y <= kPolyEnd);
    const Consts consts;
    const int first = w.rank * kChunk + w.warp * S;
    const Input ix = {p.x, p.xb, p.xt}, ir = {p.r, p.rb, p.rt}, ii = {p.i, p.ib, p.it};
    In sx(ix, w, first, width), sr(ir, w, first, width), si(ii, w, first, width);
    char* mine = rows + w.warp * (3 * S * R::kPitch);
    auto fetch = [&](int turn) {
        if (turn < turns) {
            char* at = mine + (turn % ST) * stage_bytes<T, S, FORM, 3>();
            const int t0 = turn * P * kChunk + first;
            sr.fetch(at, ir, w, n, t0, P * kChunk, width);
            si.fetch(at + S * R::kPitch, ii, w, n, t0, P * kChunk, width);
            sx.fetch(at + 2 * S * R::kPitch, ix, w, n, t0, P * kChunk, width);
        }
        cp_commit();
    };
#pragma unroll 1
    for (int k = 0; k < ST - 1; ++k) fetch(k);
    Seq<MODE> seq{cu, (int)n.n, n.Ls, w.off, w.b, 0, 0, 0};
    float2 run = MODE == kDense && !SUM ? load_state(o.h0, w.b, D, w.d, w.has0, w.has1) : f2(0.0f), runA = f2(1.0f);
    if (!SUM && o.seg) run = load_state(o.seg, w.run, D, w.d, w.has0, w.has1);

    // gates and composition of a turn: h -> a_j h + e_j token by token, h -> A h + H together
    auto prepare = [&](int turn, float2 (&a)[S], float2 (&e)[S], unsigned& starts) {
        const int t0 = turn * P * kChunk + first;
        fetch(turn + ST - 1);
        float2 own[S];                    // the states that enter with the sequences that start here
        if (CUTS) {
            if (t0 < L) seq.at(t0);
            starts = starts_in<MODE, S>(seq, t0, L);
            if (starts) {
                Seq<MODE> q = seq;
#pragma unroll
                for (int j = 0; j < S; ++j)
                    if (starts >> j & 1u) {
                        q.at(t0 + j);
                        own[j] = load_state(o.h0, q.s, D, w.d, w.has0, w.has1);
                    }
            }
        }
        cp_wait<ST - 1>();
        __syncwarp();
        const char* at = mine + (turn % ST) * stage_bytes<T, S, FORM, 3>();
        float prod = 0.0f;
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const Gates g = gates<true>(sr.read(at, ir, n, j, t0 + j), si.read(at, ii, n, S + j, t0 + j), cs, consts, prod);
            a[j] = g.a;
            e[j] = mul(mul(g.m, g.si), sx.read(at, ix, n, 2 * S + j, t0 + j));
        }
        if (!__all_sync(kFull, small && prod < kProdEnd)) {
#pragma unroll
            for (int j = 0; j < S; ++j) {
                const Gates g = gates<false>(sr.read(at, ir, n, j, t0 + j), si.read(at, ii, n, S + j, t0 + j), cs, consts, prod);
                a[j] = g.a;
                e[j] = mul(mul(g.m, g.si), sx.read(at, ix, n, 2 * S + j, t0 + j));
            }
        }
        if (t0 + S > L)                   // tokens past the end change nothing
#pragma unroll
            for (int j = 0; j < S; ++j)
                if (t0 + j >= L) {
                    a[j] = f2(1.0f);
                    e[j] = f2(0.0f);
                }
        float2 A = f2(1.0f), H = f2(0.0f);
        if (CUTS && starts) {
#pragma unroll
            for (int j = 0; j < S; ++j) {
                if (starts >> j & 1u) {
                    e[j] = fma(a[j], own[j], e[j]);
                    A = f2(kCut);
                    H = e[j];
                } else {
                    then<CUTS>(A, H, a[j], e[j]);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < S; ++j) then<false>(A, H, a[j], e[j]);
        }
        ex[turn & 1][w.warp][w.lane] = make_float4(A.x, A.y, H.x, H.y);
        __syncthreads();
    };
    // the composition of the block's warps before this one, and the block's, which goes to the cluster
    auto publish = [&](int turn, float2& preA, float2& preH) {
        float2 tA = f2(1.0f), tH = f2(0.0f);
        for (int k = 0; k < w.warp; ++k) {
            const float4 f = ex[turn & 1][k][w.lane];
            then<CUTS>(tA, tH, make_float2(f.x, f.y), make_float2(f.z, f.w));
        }
        preA = tA;
        preH = tH;
        for (int k = w.warp; k < kWarps; ++k) {
            const float4 f = ex[turn & 1][k][w.lane];
            then<CUTS>(tA, tH, make_float2(f.x, f.y), make_float2(f.z, f.w));
        }
        if constexpr (CLUSTER)
            if (w.warp < P) st_cluster(smem_addr(&pub.v[turn & 1][w.rank][w.lane]), w.warp, make_float4(tA.x, tA.y, tH.x, tH.y));
    };
    // the state that enters the warp's tokens; run moves on to the next turn
    auto enter = [&](const float4 (&from)[CLUSTER ? kMaxCluster : kWarps][32], int count, int here) -> float2 {
        float2 h = run;
#pragma unroll
        for (int k = 0; k < (CLUSTER ? kMaxCluster : kWarps); ++k) {
            if (k >= count) break;
            if (k == here) h = run;
            const float4 f = from[k][w.lane];
            run = apply<CUTS>(make_float2(f.x, f.y), make_float2(f.z, f.w), run);
        }
        return h;
    };
    auto replay = [&](int turn, float2 (&a)[S], float2 (&e)[S], unsigned starts, float2 h) {
        const int t0 = turn * P * kChunk + first;
        if (ck && w.warp % (kCkpt / S) == 0 && t0 < L) store_state(ck, t0 / kCkpt, D, w.d, h, w.has0, w.has1);
        T* out = y + (int64_t)t0 * D;
        Seq<MODE> q = seq;
        if (CUTS && t0 < L) q.at(t0);
        if (t0 + S <= L && (!CUTS || (starts == 0 && q.end > t0 + S))) {
#pragma unroll
            for (int j = 0; j < S; ++j) {
                h = fma(a[j], h, e[j]);
                store_pair<T, FORM == kRows16>(out, h, even_rows, w.has0, w.has1);
                out += D;
            }
        } else {
#pragma unroll
            for (int j = 0; j < S; ++j) {
                const int t = t0 + j;
                h = CUTS && (starts >> j & 1u) ? e[j] : fma(a[j], h, e[j]);
                if (t < L) {
                    store_pair<T, FORM == kRows16>(out, h, even_rows, w.has0, w.has1);
                    if (CUTS) q.at(t);
                    if (CUTS && t == q.end - 1) store_state(o.h_last, q.s, D, w.d, h, w.has0, w.has1);
                }
                out += D;
            }
        }
    };

    if (CLUSTER) {                        // every block of the cluster runs before its shared memory is written to
        cluster_arrive();
        cluster_wait();
    }
    for (int turn = 0; turn < turns; ++turn) {
        float2 a[S], e[S], h;
        unsigned starts = 0;
        prepare(turn, a, e, starts);
        if constexpr (CLUSTER) {
            float2 preA, preH;
            publish(turn, preA, preH);
            cluster_arrive();
            cluster_wait();
            if constexpr (SUM) {
                for (int k = 0; k < P; ++k) {
                    const float4 f = pub.v[turn & 1][k][w.lane];
                    then<CUTS>(runA, run, make_float2(f.x, f.y), make_float2(f.z, f.w));
                }
                continue;
            }
            h = apply<CUTS>(preA, preH, enter(pub.v[turn & 1], P, w.rank));
        } else {
            h = enter(ex[turn & 1], kWarps, w.warp);
        }
        replay(turn, a, e, starts, h);
    }
    if (SUM) {
        if (w.rank == 0 && w.warp == 0) {
            store_state(o.sum, w.run * 2, D, w.d, runA, w.has0, w.has1);
            store_state(o.sum, w.run * 2 + 1, D, w.d, run, w.has0, w.has1);
        }
        return;
    }
    if (w.rank != 0 || (MODE == kPacked && w.run != 0)) return;
    if (MODE == kDense) {
        if (w.warp == 0 && L > 0 && w.off + L == n.L) store_state(o.h_last, w.b, D, w.d, run, w.has0, w.has1);
    } else if (MODE == kPacked) {
        for (int64_t s = w.warp; s < n.n; s += kWarps)       // empty sequences keep their state
            if (seq.cu[s] >= seq.cu[s + 1])
                store_state(o.h_last, s, D, w.d, load_state(o.h0, s, D, w.d, w.has0, w.has1), w.has0, w.has1);
    }
}

// Chunks from the last to the first.  The states that enter a chunk come from
// the forward; back_t = a_t G_t passes from right to left by the same products
// of decays, back -> A back + K.
template <typename T, int MODE, int FORM, bool CLUSTER, bool SUM>
__global__ void __launch_bounds__(kWarps * 32, 2)
rec_bwd_kernel(const __grid_constant__ RecPtr p, const __grid_constant__ RecOut o, const __grid_constant__ RecDim n,
               const float* __restrict__ lam, float c) {
    constexpr bool CUTS = MODE != kDense;
    constexpr int S = kStepsBwd, kChunk = kWarps * S, ST = stages_bwd<T>();
    using In = Stream<T, MODE, FORM, S>;
    using R = Rows<T, FORM>;
    __shared__ float4 ex[2][kWarps][32];          // (A, K)
    __shared__ float2 exh[2][kWarps][32];         // H
    __shared__ Pub<CLUSTER> pub;
    __shared__ int32_t cus[MODE == kPacked ? kCuMax : 1];
    extern __shared__ __align__(16) char rows[];
    const int32_t* cu = stage_cu<MODE>(n, cus);
    const Place w = place<MODE, CLUSTER>(n, cu);
    const int D = n.D, L = w.L, P = CLUSTER ? n.P : 1, width = min(kTile, D - w.tile * kTile);
    const int64_t base = ((MODE == kPacked ? 0 : w.b * n.Ls) + w.off) * D + w.d;
    const bool even_rows = (D & 1) == 0 && ((uintptr_t)o.dx | (uintptr_t)o.dr | (uintptr_t)o.di) % (2 * sizeof(T)) == 0;
    const int turns = (((MODE == kGroup ? n.L : L) + kChunk - 1) / kChunk + P - 1) / P;
    const float* ck = o.ckpt + ckpt_row<MODE>(w, n) * D;
    const float2 l = load_state(lam, 0, D, w.d, w.has0, w.has1);
    const float2 cs = make_float2(w.has0 ? c * softplus_(l.x) : kPolyEnd, w.has1 ? c * softplus_(l.y) : kPolyEnd);
    const bool small = __all_sync(kFull, cs.x >= kCsLow && cs.x <= kPolyEnd && cs.y >= kCsLow && cs.y <= kPolyEnd);
    const Consts consts;
    const int first = w.rank * kChunk + w.warp * S, last = (turns - 1) * P * kChunk + first;
    // (without dy: rows of no width, zeros)
    const Input ix = {p.x, p.xb, p.xt}, ir = {p.r, p.rb, p.rt}, ii = {p.i, p.ib, p.it}, ig = {p.dy ? p.dy : p.x, p.gb, p.gt};
    In sx(ix, w, last, width), sr(ir, w, last, width), si(ii, w, last, width), sg(ig, w, last, p.dy ? width : 0);
    char* mine = rows + w.warp * (4 * S * R::kPitch);
    auto fetch = [&](int turn) {
        if (turn >= 0) {
            char* at = mine + (turn % ST) * stage_bytes<T, S, FORM, 4>();
            const int t0 = turn * P * kChunk + first;
            sr.fetch(at, ir, w, n, t0, -P * kChunk, width);
            si.fetch(at + S * R::kPitch, ii, w, n, t0, -P * kChunk, width);
            sx.fetch(at + 2 * S * R::kPitch, ix, w, n, t0, -P * kChunk, width);
            sg.fetch(at + 3 * S * R::kPitch, ig, w, n, t0, -P * kChunk, p.dy ? width : 0);
        }
        cp_commit();
    };
    constexpr int kAhead = ST - 1;                // turns in flight beyond the one being prepared
#pragma unroll 1
    for (int k = 1; k <= kAhead; ++k) fetch(turns - k);
    Seq<MODE> seq{cu, (int)n.n, n.Ls, w.off, w.b, 0, 0, 0};
    if (L > 0) seq.at(L - 1);
    float2 run = load_state(SUM ? nullptr : o.dh_last, CUTS ? seq.s : w.b, D, w.d, w.has0, w.has1), sum = f2(0.0f), runA = f2(1.0f);
    if (!SUM && o.seg) run = load_state(o.seg, w.run, D, w.d, w.has0, w.has1);
    auto state0 = [&](int t) -> float2 {          // the state that enters the sequence of token t
        Seq<MODE> q = seq;
        q.at(t);
        return load_state(o.h0, q.s, D, w.d, w.has0, w.has1);
    };
    auto back0 = [&](int t) -> float2 {           // what enters, from the right, the sequence of token t
        if (t + w.off < 0) return f2(0.0f);
        Seq<MODE> q = seq;
        q.at(t);
        return load_state(o.dh_last, q.s, D, w.d, w.has0, w.has1);
    };
    const float2 nones = pinned(-1.0f);
    struct Turn {
        float2 sr[S], si[S], a[S], rs[S], msi[S], x[S], g[S], h, sufA, sufK, back;      // (msi: m sigmoid(i), g: dy)
        unsigned starts;
    };

    auto prepare = [&](int turn, Turn& q) {
        const int chunk = turn * P + w.rank, t0 = turn * P * kChunk + first;
        fetch(turn - kAhead);
        q.h = chunk * kChunk < L ? load_state(ck, chunk, D, w.d, w.has0, w.has1) : f2(0.0f);
        q.starts = 0;
        float2 own[S], beyond[S];                 // states and back states of the sequences that start here, end before here
        if (CUTS) {
            if (t0 < L) seq.at(t0);
            q.starts = starts_in<MODE, S>(seq, t0, L);
            if (q.starts)
#pragma unroll
                for (int j = 0; j < S; ++j)
                    if (q.starts >> j & 1u) {
                        own[j] = state0(t0 + j);
                        beyond[j] = back0(t0 + j - 1);
                    }
        }
        cp_wait<kAhead>();
        __syncwarp();
        const char* at = mine + (turn % ST) * stage_bytes<T, S, FORM, 4>();
        float prod = 0.0f;
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const Gates g = gates<true>(sr.read(at, ir, n, j, t0 + j), si.read(at, ii, n, S + j, t0 + j), cs, consts, prod);
            q.sr[j] = g.sr; q.si[j] = g.si; q.a[j] = g.a; q.rs[j] = g.rs; q.msi[j] = mul(g.m, g.si);
        }
        if (!__all_sync(kFull, small && prod < kProdEnd)) {
#pragma unroll
            for (int j = 0; j < S; ++j) {
                const Gates g = gates<false>(sr.read(at, ir, n, j, t0 + j), si.read(at, ii, n, S + j, t0 + j), cs, consts, prod);
                q.sr[j] = g.sr; q.si[j] = g.si; q.a[j] = g.a; q.rs[j] = g.rs; q.msi[j] = mul(g.m, g.si);
            }
        }
        if (t0 + S > L)                           // tokens past the end change nothing (their x and dy are zero)
#pragma unroll
            for (int j = 0; j < S; ++j)
                if (t0 + j >= L) {
                    q.a[j] = f2(1.0f);
                    q.rs[j] = q.msi[j] = q.sr[j] = f2(0.0f);
                }
        // forward composition (A, H), backward composition (A, K) of the warp's tokens
        float2 A = f2(1.0f), H = f2(0.0f), K = f2(0.0f);
#pragma unroll
        for (int j = 0; j < S; ++j) {
            q.x[j] = sx.read(at, ix, n, 2 * S + j, t0 + j);
            q.g[j] = sg.read(at, ig, n, 3 * S + j, t0 + j);
            const float2 e = mul(q.msi[j], q.x[j]);
            if (CUTS && (q.starts >> j & 1u)) {
                A = f2(kCut);
                H = fma(q.a[j], own[j], e);
            } else if (CUTS && q.starts) {
                then<CUTS>(A, H, q.a[j], e);
            } else {
                then<false>(A, H, q.a[j], e);
            }
        }
#pragma unroll
        for (int j = S - 1; j >= 0; --j) {
            if (CUTS && (q.starts >> j & 1u)) K = beyond[j];
            else K = mul(q.a[j], add(q.g[j], K));
        }
        ex[turn & 1][w.warp][w.lane] = make_float4(A.x, A.y, K.x, K.y);
        exh[turn & 1][w.warp][w.lane] = H;
        __syncthreads();
        for (int k = 0; k < w.warp; ++k) {
            const float4 f = ex[turn & 1][k][w.lane];
            q.h = apply<CUTS>(make_float2(f.x, f.y), exh[turn & 1][k][w.lane], q.h);
        }
    };
    auto publish = [&](int turn, Turn& q) {
        float2 tA = f2(1.0f), tK = f2(0.0f);
        for (int k = kWarps - 1; k > w.warp; --k) {
            const float4 f = ex[turn & 1][k][w.lane];
            then<CUTS>(tA, tK, make_float2(f.x, f.y), make_float2(f.z, f.w));
        }
        q.sufA = tA;
        q.sufK = tK;
        for (int k = w.warp; k >= 0; --k) {
            const float4 f = ex[turn & 1][k][w.lane];
            then<CUTS>(tA, tK, make_float2(f.x, f.y), make_float2(f.z, f.w));
        }
        if constexpr (CLUSTER)
            if (w.warp < P) st_cluster(smem_addr(&pub.v[turn & 1][w.rank][w.lane]), w.warp, make_float4(tA.x, tA.y, tK.x, tK.y));
    };
    auto enter = [&](const float4 (&from)[CLUSTER ? kMaxCluster : kWarps][32], int count, int here) -> float2 {
        float2 back = run;
#pragma unroll
        for (int k = (CLUSTER ? kMaxCluster : kWarps) - 1; k >= 0; --k) {
            if (k >= count) continue;
            if (k == here) back = run;
            const float4 f = from[k][w.lane];
            run = apply<CUTS>(make_float2(f.x, f.y), make_float2(f.z, f.w), run);
        }
        return back;
    };
    auto replay = [&](int turn, Turn& q) {
        const int t0 = turn * P * kChunk + first;
        float2 prev[S];
        const bool cuts = CUTS && q.starts != 0;
#pragma unroll
        for (int j = 0; j < S; ++j) {
            if (cuts && (q.starts >> j & 1u)) q.h = state0(t0 + j);
            prev[j] = q.h;
            q.h = fma(q.a[j], q.h, mul(q.msi[j], q.x[j]));
        }
#pragma unroll
        for (int j = S - 1; j >= 0; --j) {        // dy becomes G
            q.g[j] = add(q.g[j], q.back);
            q.back = mul(q.a[j], q.g[j]);         // (past the end a is 1 and dy 0)
            if (cuts && (q.starts >> j & 1u)) {
                Seq<MODE> z = seq;
                z.at(t0 + j);
                if (o.dh0) store_state(o.dh0, z.s, D, w.d, q.back, w.has0, w.has1);
                q.back = back0(t0 + j - 1);
            }
        }
        const int64_t out = base + (int64_t)t0 * D;
        T *px = static_cast<T*>(o.dx) + out, *pr = static_cast<T*>(o.dr) + out, *pi = static_cast<T*>(o.di) + out;
        const bool full = t0 + S <= L;
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const float2 vx = mul(q.g[j], q.msi[j]);
            const float2 vi = mul(mul(vx, q.x[j]), fma(q.si[j], nones, consts.one));
            // du = G a (prev - (a / m) sigmoid(i) x)
            const float2 slope = mul(mul(q.a[j], q.rs[j]), mul(q.si[j], q.x[j]));
            const float2 du = mul(mul(q.g[j], q.a[j]), fma(slope, nones, prev[j]));
            const float2 ds = mul(du, q.sr[j]);
            const float2 vr = mul(mul(ds, cs), add(q.sr[j], nones));
            if (full || t0 + j < L) {
                sum = add(sum, ds);
                store_pair<T, FORM == kRows16>(px, vx, even_rows, w.has0, w.has1);
                store_pair<T, FORM == kRows16>(pr, vr, even_rows, w.has0, w.has1);
                store_pair<T, FORM == kRows16>(pi, vi, even_rows, w.has0, w.has1);
            }
            px += D;
            pr += D;
            pi += D;
        }
    };

    if (CLUSTER) {
        cluster_arrive();
        cluster_wait();
    }
    for (int turn = turns - 1; turn >= 0; --turn) {
        Turn q;
        prepare(turn, q);
        if constexpr (CLUSTER) {
            publish(turn, q);
            cluster_arrive();
            cluster_wait();
            if constexpr (SUM) {
                for (int k = P - 1; k >= 0; --k) {
                    const float4 f = pub.v[turn & 1][k][w.lane];
                    then<CUTS>(runA, run, make_float2(f.x, f.y), make_float2(f.z, f.w));
                }
                continue;
            }
            q.back = apply<CUTS>(q.sufA, q.sufK, enter(pub.v[turn & 1], P, w.rank));
        } else {
            q.back = enter(ex[turn & 1], kWarps, w.warp);
        }
        replay(turn, q);
    }
    if (SUM) {
        if (w.rank == 0 && w.warp == 0) {
            store_state(o.sum, w.run * 2, D, w.d, runA, w.has0, w.has1);
            store_state(o.sum, w.run * 2 + 1, D, w.d, run, w.has0, w.has1);
        }
        return;
    }
    __syncthreads();
    exh[0][w.warp][w.lane] = sum;
    __syncthreads();
    if (w.warp == 0) {
        float2 s = f2(0.0f);
        for (int k = 0; k < kWarps; ++k) s = add(s, exh[0][k][w.lane]);
        store_state(o.part, w.run * P + w.rank, D, w.d, s, w.has0, w.has1);
    }
    if (w.rank != 0 || !o.dh0 || (MODE == kPacked && w.run != 0)) return;
    if (MODE == kDense) {
        if (w.warp == 0 && w.off == 0) store_state(o.dh0, w.b, D, w.d, run, w.has0, w.has1);
    } else if (MODE == kPacked) {
        for (int64_t s = w.warp; s < n.n; s += kWarps)
            if (seq.cu[s] >= seq.cu[s + 1])
                store_state(o.dh0, s, D, w.d, load_state(o.dh_last, s, D, w.d, w.has0, w.has1), w.has0, w.has1);
    }
}

// ---- many sequences: a warp has its own ------------------------------------------
// Where the sequences and tiles give the GPU warps enough, a warp takes `per`
// consecutive sequences token by token and nothing is exchanged: one pass, the state
// in a register (2000 x 17 x 512 bf16: forward 86 -> 54 us, backward 150 -> 89 us).
// The forward keeps the state before every kCkptSerial tokens.
constexpr int kCkptSerial = kStepsBwd;

__device__ __forceinline__ bool place_serial(const RecDim& n, Place& q) {
    q.lane = threadIdx.x & 31;
    q.warp = threadIdx.x >> 5;
    const int tiles = (n.D + kTile - 1) / kTile;
    const int64_t unit = (int64_t)blockIdx.x * kWarps + q.warp;
    q.rank = q.off = 0;
    q.run = unit / tiles;
    q.tile = (int)(unit - q.run * tiles);
    q.b = q.run * n.per;
    q.L = q.run < n.runs ? (int)min((int64_t)n.per, n.n - q.b) * n.Ls : 0;
    q.d = q.tile * kTile + q.lane * 2;
    q.has0 = q.d < n.D;
    q.has1 = q.d + 1 < n.D;
    return q.run < n.runs;
}

template <typename T, int FORM>
__global__ void __launch_bounds__(kWarps * 32, 2)
rec_fwd_serial(const __grid_constant__ RecPtr p, const __grid_constant__ RecOut o, const __grid_constant__ RecDim n,
               const float* __restrict__ lam, float c) {
    constexpr int S = kStepsFwd, ST = stages_fwd<T>();
    using In = Stream<T, kGroup, FORM, S>;
    using R = Rows<T, FORM>;
    extern __shared__ __align__(16) char rows[];
    Place w;
    if (!place_serial(n, w)) return;
    const int D = n.D, L = w.L, width = min(kTile, D - w.tile * kTile), turns = (L + S - 1) / S;
    T* out = static_cast<T*>(o.y) + w.b * n.Ls * D + w.d;
    const bool even_rows = (D & 1) == 0 && (uintptr_t)o.y % (2 * sizeof(T)) == 0;
    float* ck = o.ckpt ? o.ckpt + w.run * ((n.L + kCkptSerial - 1) / kCkptSerial) * D : nullptr;
    const Input ix = {p.x, p.xb, p.xt}, ir = {p.r, p.rb, p.rt}, ii = {p.i, p.ib, p.it};
    In sx(ix, w, 0, width), sr(ir, w, 0, width), si(ii, w, 0, width);
    char* mine = rows + w.warp * (3 * S * R::kPitch);
    auto fetch = [&](int turn) {
        if (turn < turns) {
            char* at = mine + (turn % ST) * stage_bytes<T, S, FORM, 3>();
            sr.fetch(at, ir, w, n, turn * S, S, width);
            si.fetch(at + S * R::kPitch, ii, w, n, turn * S, S, width);
            sx.fetch(at + 2 * S * R::kPitch, ix, w, n, turn * S, S, width);
        }
        cp_commit();
    };
#pragma unroll 1
    for (int k = 0; k < ST - 1; ++k) fetch(k);
    const float2 l = load_state(lam, 0, D, w.d, w.has0, w.has1);
    const float2 cs = make_float2(w.has0 ? c * softplus_(l.x) : kPolyEnd, w.has1 ? c * softplus_(l.y) : kPolyEnd);
    const bool small = __all_sync(kFull, cs.x >= kCsLow && cs.x <= kPolyEnd && cs.y >= kCsLow && cs.y <= kPolyEnd);
    const Consts consts;
    float2 h = f2(0.0f);
    int start = 0;                        // the next token that starts a sequence, and its sequence
    int64_t seq = w.b;
    for (int turn = 0; turn < turns; ++turn) {
        const int t0 = turn * S;
        fetch(turn + ST - 1);
        unsigned starts = 0;
        float2 own[S];
        const int64_t seq0 = seq;
        while (start < t0 + S && start < L) {
            starts |= 1u << (start - t0);
            start += n.Ls;
            ++seq;
        }
        if (starts) {
            int64_t q = seq0;
#pragma unroll
            for (int j = 0; j < S; ++j)
                if (starts >> j & 1u) own[j] = load_state(o.h0, q++, D, w.d, w.has0, w.has1);
        }
        cp_wait<ST - 1>();
        __syncwarp();
        const char* at = mine + (turn % ST) * stage_bytes<T, S, FORM, 3>();
        float2 a[S], e[S];
        float prod = 0.0f;
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const Gates g = gates<true>(sr.read(at, ir, n, j, t0 + j), si.read(at, ii, n, S + j, t0 + j), cs, consts, prod);
            a[j] = g.a;
            e[j] = mul(mul(g.m, g.si), sx.read(at, ix, n, 2 * S + j, t0 + j));
        }
        if (!__all_sync(kFull, small && prod < kProdEnd)) {
#pragma unroll
            for (int j = 0; j < S; ++j) {
                const Gates g = gates<false>(sr.read(at, ir, n, j, t0 + j), si.read(at, ii, n, S + j, t0 + j), cs, consts, prod);
                a[j] = g.a;
                e[j] = mul(mul(g.m, g.si), sx.read(at, ix, n, 2 * S + j, t0 + j));
            }
        }
        int64_t ended = seq0 - 1;
#pragma unroll
        for (int j = 0; j < S; ++j) {
            if (j % kCkptSerial == 0 && ck && t0 + j < L) store_state(ck, (t0 + j) / kCkptSerial, D, w.d, h, w.has0, w.has1);
            if (starts >> j & 1u) {
                if (t0 + j > 0) store_state(o.h_last, ended, D, w.d, h, w.has0, w.has1);
                ++ended;
                h = own[j];
            }
            if (t0 + j < L) {
                h = fma(a[j], h, e[j]);
                store_pair<T, FORM == kRows16>(out, h, even_rows, w.has0, w.has1);
            }
            out += D;
        }
        __syncwarp();                     // the rows are read before they are fetched over
    }
    store_state(o.h_last, w.b + L / n.Ls - 1, D, w.d, h, w.has0, w.has1);
}

template <typename T, int FORM>
__global__ void __launch_bounds__(kWarps * 32, 2)
rec_bwd_serial(const __grid_constant__ RecPtr p, const __grid_constant__ RecOut o, const __grid_constant__ RecDim n,
               const float* __restrict__ lam, float c) {
    constexpr int S = kStepsBwd, ST = stages_bwd<T>();
    using In = Stream<T, kGroup, FORM, S>;
    using R = Rows<T, FORM>;
    extern __shared__ __align__(16) char rows[];
    Place w;
    if (!place_serial(n, w)) return;
    const int D = n.D, L = w.L, width = min(kTile, D - w.tile * kTile), turns = (L + S - 1) / S;
    const int64_t base = w.b * n.Ls * D + w.d;
    const bool even_rows = (D & 1) == 0 && ((uintptr_t)o.dx | (uintptr_t)o.dr | (uintptr_t)o.di) % (2 * sizeof(T)) == 0;
    const float* ck = o.ckpt + w.run * ((n.L + kCkptSerial - 1) / kCkptSerial) * D;
    const Input ix = {p.x, p.xb, p.xt}, ir = {p.r, p.rb, p.rt}, ii = {p.i, p.ib, p.it}, ig = {p.dy ? p.dy : p.x, p.gb, p.gt};
    const int last = (turns - 1) * S;
    In sx(ix, w, last, width), sr(ir, w, last, width), si(ii, w, last, width), sg(ig, w, last, p.dy ? width : 0);
    char* mine = rows + w.warp * (4 * S * R::kPitch);
    auto fetch = [&](int turn) {
        if (turn >= 0) {
            char* at = mine + (turn % ST) * stage_bytes<T, S, FORM, 4>();
            sr.fetch(at, ir, w, n, turn * S, -S, width);
            si.fetch(at + S * R::kPitch, ii, w, n, turn * S, -S, width);
            sx.fetch(at + 2 * S * R::kPitch, ix, w, n, turn * S, -S, width);
            sg.fetch(at + 3 * S * R::kPitch, ig, w, n, turn * S, -S, p.dy ? width : 0);
        }
        cp_commit();
    };
#pragma unroll 1
    for (int k = 1; k < ST; ++k) fetch(turns - k);
    const float2 l = load_state(lam, 0, D, w.d, w.has0, w.has1);
    const float2 cs = make_float2(w.has0 ? c * softplus_(l.x) : kPolyEnd, w.has1 ? c * softplus_(l.y) : kPolyEnd);
    const bool small = __all_sync(kFull, cs.x >= kCsLow && cs.x <= kPolyEnd && cs.y >= kCsLow && cs.y <= kPolyEnd);
    const Consts consts;
    const float2 nones = pinned(-1.0f);
    int64_t seq = w.b + L / n.Ls - 1;                       // the sequence of the tokens at hand, and its first token
    int start = L - n.Ls;
    float2 back = load_state(o.dh_last, seq, D, w.d, w.has0, w.has1), sum = f2(0.0f);
    for (int turn = turns - 1; turn >= 0; --turn) {
        const int t0 = turn * S;
        fetch(turn - ST + 1);
        float2 h = load_state(ck, turn, D, w.d, w.has0, w.has1);
        unsigned starts = 0;
        float2 own[S], beyond[S];
        const int64_t seq0 = seq;
        while (start >= t0) {
            starts |= 1u << (start - t0);
            start -= n.Ls;
            --seq;
        }
        if (starts) {
            int64_t q = seq0;
#pragma unroll
            for (int j = S - 1; j >= 0; --j)
                if (starts >> j & 1u) {
                    own[j] = load_state(o.h0, q, D, w.d, w.has0, w.has1);
                    beyond[j] = q > w.b ? load_state(o.dh_last, q - 1, D, w.d, w.has0, w.has1) : f2(0.0f);
                    --q;
                }
        }
        cp_wait<ST - 1>();
        __syncwarp();
        const char* at = mine + (turn % ST) * stage_bytes<T, S, FORM, 4>();
        float2 sgr[S], sgi[S], a[S], rs[S], msi[S];
        float prod = 0.0f;
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const Gates g = gates<true>(sr.read(at, ir, n, j, t0 + j), si.read(at, ii, n, S + j, t0 + j), cs, consts, prod);
            sgr[j] = g.sr; sgi[j] = g.si; a[j] = g.a; rs[j] = g.rs; msi[j] = mul(g.m, g.si);
        }
        if (!__all_sync(kFull, small && prod < kProdEnd)) {
#pragma unroll
            for (int j = 0; j < S; ++j) {
                const Gates g = gates<false>(sr.read(at, ir, n, j, t0 + j), si.read(at, ii, n, S + j, t0 + j), cs, consts, prod);
                sgr[j] = g.sr; sgi[j] = g.si; a[j] = g.a; rs[j] = g.rs; msi[j] = mul(g.m, g.si);
            }
        }
        float2 prev[S], xv[S];
#pragma unroll
        for (int j = 0; j < S; ++j) {
            xv[j] = sx.read(at, ix, n, 2 * S + j, t0 + j);
            if (starts >> j & 1u) h = own[j];
            prev[j] = h;
            h = fma(a[j], h, mul(msi[j], xv[j]));
        }
        const int64_t at0 = base + (int64_t)t0 * D;
        T *px = static_cast<T*>(o.dx) + at0, *pr = static_cast<T*>(o.dr) + at0, *pi = static_cast<T*>(o.di) + at0;
        int64_t q = seq0;
#pragma unroll
        for (int j = S - 1; j >= 0; --j) {
            if (t0 + j < L) {
                const float2 G = add(sg.read(at, ig, n, 3 * S + j, t0 + j), back);
                back = mul(a[j], G);
                const float2 vx = mul(G, msi[j]);
                const float2 vi = mul(mul(vx, xv[j]), fma(sgi[j], nones, consts.one));
                // du = G a (prev - (a / m) sigmoid(i) x)
                const float2 slope = mul(mul(a[j], rs[j]), mul(sgi[j], xv[j]));
                const float2 du = mul(back, fma(slope, nones, prev[j]));
                const float2 ds = mul(du, sgr[j]);
                const float2 vr = mul(mul(ds, cs), add(sgr[j], nones));
                sum = add(sum, ds);
                store_pair<T, FORM == kRows16>(px + (int64_t)j * D, vx, even_rows, w.has0, w.has1);
                store_pair<T, FORM == kRows16>(pr + (int64_t)j * D, vr, even_rows, w.has0, w.has1);
                store_pair<T, FORM == kRows16>(pi + (int64_t)j * D, vi, even_rows, w.has0, w.has1);
            }
            if (starts >> j & 1u) {
                if (o.dh0) store_state(o.dh0, q, D, w.d, back, w.has0, w.has1);
                --q;
                back = beyond[j];
            }
        }
        __syncwarp();
    }
    store_state(o.part, w.run, D, w.d, sum, w.has0, w.has1);
}

// What enters every segment of a sequence (blockIdx.y; packed: of all), from the first on or (REVERSE) from the last on.
template <bool REVERSE>
__global__ void rec_join_kernel(const float* __restrict__ sum, const float* __restrict__ init, RecDim n, float* __restrict__ state) {
    const int d = blockIdx.x * blockDim.x + threadIdx.x;
    if (d >= n.D) return;
    const int64_t first = (int64_t)blockIdx.y * n.segs;
    float h = 0.0f;
    if (n.cu == nullptr) {
        if (init) h = init[(int64_t)blockIdx.y * n.D + d];
    } else if (REVERSE && init) {                 // the last token's sequence
        int64_t lo = 0, hi = n.n - 1;
        while (lo < hi) {
            const int64_t mid = (lo + hi + 1) / 2;
            if (n.cu[mid] <= n.L - 1) lo = mid;
            else hi = mid - 1;
        }
        h = init[lo * n.D + d];
    }
    for (int k = 0; k < n.segs; ++k) {
        const int64_t run = first + (REVERSE ? n.segs - 1 - k : k);
        state[run * n.D + d] = h;
        const float A = sum[run * 2 * n.D + d], H = sum[(run * 2 + 1) * n.D + d];
        h = A < 0.0f ? H : fmaf(A, h, H);
    }
}

// dlam[d] = -c sigmoid(lam[d]) * sum of the n partials of feature d: a block takes
// 32 features, a warp every 32nd partial, then the warps' sums in order.
__global__ void __launch_bounds__(1024)
rec_dlam_kernel(const float* __restrict__ part, int64_t n, int64_t D, const float* __restrict__ lam, float c, float* __restrict__ dlam) {
    __shared__ float sums[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t d = (int64_t)blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (d < D)
        for (int64_t k = warp; k < n; k += 32) s += part[k * D + d];
    sums[warp][lane] = s;
    __syncthreads();
    if (warp != 0 || d >= D) return;
    s = 0.0f;
    for (int k = 0; k < 32; ++k) s += sums[k][lane];
    dlam[d] = -c * sigmoid_(lam[d]) * s;
}

// One token of every sequence: reads 3 values and a state, writes a value and a state.  A thread keeps one pair of
// features (its decay parameters are computed once) and walks the sequences of its block row; PAIR: rows lie on pairs.
// 256 x 4096 bf16: 4.5 us (16.8 MB; L2 warm, in a graph), a single row 1.8 us.
template <typename T, bool PAIR>
__global__ void __launch_bounds__(128)
rec_step_kernel(RecPtr p, int64_t B, int D, const float* __restrict__ lam, float c, float* __restrict__ h, T* __restrict__ y) {
    const int d = ((int)blockIdx.x * 128 + (int)threadIdx.x) * 2;
    if (d >= D) return;
    const bool two = PAIR || d + 1 < D;
    const Consts consts;
    auto load = [&](const void* from, int64_t at) -> float2 {
        const T* e = static_cast<const T*>(from) + at + d;
        if constexpr (PAIR) {
            T v[2];
            if constexpr (sizeof(T) == 4) {
                const float2 w = *reinterpret_cast<const float2*>(e);
                return w;
            } else {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(e);
                memcpy(v, &w, 4);
                return make_float2(to_f32<T>(v[0]), to_f32<T>(v[1]));
            }
        } else {
            return make_float2(to_f32<T>(e[0]), two ? to_f32<T>(e[1]) : 0.0f);
        }
    };
    float2 cs = f2(0.0f);
    for (int64_t b = blockIdx.y; b < B; b += gridDim.y) {
        const float2 x = load(p.x, b * p.xb), r = load(p.r, b * p.rb), i = load(p.i, b * p.ib);
        float2 s;
        float* hb = h + b * D + d;
        if (PAIR) s = *reinterpret_cast<const float2*>(hb);
        else s = make_float2(hb[0], two ? hb[1] : 0.0f);
        if (b == blockIdx.y) cs = make_float2(c * softplus_(lam[d]), two ? c * softplus_(lam[d + 1]) : 0.0f);
        float prod;
        const Gates g = gates<false>(r, i, cs, consts, prod);
        s = fma(g.a, s, mul(mul(g.m, g.si), x));
        if (PAIR) {
            *reinterpret_cast<float2*>(hb) = s;
        } else {
            hb[0] = s.x;
            if (two) hb[1] = s.y;
        }
        store_pair<T, PAIR>(y + b * D + d, s, PAIR, true, two);
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
    int mode, per, L, P;
    int64_t runs, tiles;
    bool serial;
    int segs, seg;
};

Plan rec_plan(const bcm_gated_rec_args* a) {
    constexpr int kChunk = kWarps * kStepsFwd;
    Plan pl = {kDense, 1, (int)a->seqlen, 1, a->batch, rec_parts(a->dim, kTile), false, 1, 0};
    if (a->cu_seqlens) {
        // Runs need no exchange, but a long sequence leaves them uneven: one for every four sequences at most, and no
        // more than two blocks per SM take; clusters fill the rest.
        pl.mode = kPacked;
        pl.runs = 1;
        while (pl.runs * 8 <= a->batch && pl.tiles * pl.runs <= (int64_t)sm_count() && pl.runs * 2 * kChunk <= a->seqlen) pl.runs *= 2;
    } else if (a->batch * pl.tiles >= 12 * (int64_t)sm_count()) {
        // Sequences enough for 12 warps per SM and more: each warp has its own, and takes the fewest that keep its last
        // turn an eighth empty at most (or that fill the GPU's 16 warps per SM eight times over).
        pl.mode = kGroup;
        pl.serial = true;
        const int64_t full = (a->batch * pl.tiles + 8 * 16 * (int64_t)sm_count() - 1) / (8 * 16 * (int64_t)sm_count());
        const int64_t some = std::min<int64_t>((8 * kStepsFwd + a->seqlen - 1) / a->seqlen, a->batch * pl.tiles / (12 * (int64_t)sm_count()));
        pl.per = (int)std::min<int64_t>(std::max<int64_t>(std::max<int64_t>(full, some), 1), std::max<int64_t>((1ll << 30) / a->seqlen, 1));
        pl.L = (int)(pl.per * a->seqlen);
        pl.runs = rec_parts(a->batch, pl.per);
        return pl;
    } else if (a->seqlen < 4 * kChunk && a->batch > 1) {
        // runs of about 8 chunks (an eighth of the last one empty at most), fewer where that leaves SMs without a block
        pl.mode = kGroup;
        int64_t per = (8 * kChunk + a->seqlen - 1) / a->seqlen;
        while (per > 1 && per * a->seqlen > kChunk && rec_parts(a->batch, (int)per) * pl.tiles < 4 * (int64_t)sm_count()) per = (per + 1) / 2;
        pl.per = (int)std::min<int64_t>(per, a->batch);
        pl.L = (int)(pl.per * a->seqlen);
        pl.runs = rec_parts(a->batch, pl.per);
    }
    // blocks of a cluster: as many as the chunks allow and two blocks per SM hold at once
    while (pl.P < kMaxCluster && pl.runs * pl.tiles * pl.P <= (int64_t)sm_count() && 2 * pl.P <= rec_parts(pl.mode == kPacked ? pl.L / pl.runs : pl.L, kChunk)) pl.P *= 2;
    // Segments where full clusters still leave most of the GPU empty: they take their tokens twice, so three at least,
    // of four turns or more.
    const int64_t room = 2 * (int64_t)sm_count() / (pl.runs * pl.tiles * pl.P), turns = rec_parts(pl.L, kChunk * kMaxCluster);
    if (pl.P == kMaxCluster && pl.mode != kGroup && (pl.mode == kDense || pl.runs == 1) && std::min(room, turns / 4) >= 3) {
        pl.seg = (int)rec_parts(rec_parts(pl.L, (int)std::min(room, turns / 4)), kChunk) * kChunk;
        pl.segs = (int)rec_parts(pl.L, pl.seg);
        pl.runs *= pl.segs;
    }
    return pl;
}

// What every row of every input starts on (and, for 16 bytes, the outputs' rows on two features).
int rec_form(const bcm_gated_rec_args* a, bool bwd) {
    const int64_t s = (int64_t)dtype_size(a->dtype);
    int64_t bits = 0;
    auto see = [&](const void* p, int64_t sb, int64_t st) {
        bits |= (int64_t)(uintptr_t)p | (a->cu_seqlens || a->batch == 1 ? 0 : sb * s) | (a->seqlen == 1 ? 0 : st * s);
    };
    see(a->x, a->x_stride_b, a->x_stride_t);
    see(a->r, a->r_stride_b, a->r_stride_t);
    see(a->i, a->i_stride_b, a->i_stride_t);
    if (bwd && a->dy) see(a->dy, a->dy_stride_b, a->dy_stride_t);
    if ((bits & 3) != 0 || (s == 2 && a->dim % 2 != 0)) return kRows2;
    bits |= (int64_t)(bwd ? (uintptr_t)a->dx | (uintptr_t)a->dr | (uintptr_t)a->di : (uintptr_t)a->y);
    return (bits & 15) == 0 && a->dim % 2 == 0 ? kRows16 : kRows4;
}

RecDim rec_dim(const bcm_gated_rec_args* a, const Plan& pl) {
    return {a->cu_seqlens, a->batch, pl.L, (int)a->seqlen, pl.per, pl.segs > 1 ? 1 : (int)pl.runs, (int)a->dim, pl.P, pl.segs, pl.seg};
}

template <typename F>
bcm_status rec_launch_as(F* kernel, int smem, const bcm_gated_rec_args* a, const RecOut& o, const Plan& pl, cudaStream_t stream) {
    const int64_t blocks = pl.serial ? rec_parts(pl.tiles * pl.runs, kWarps) : pl.tiles * pl.runs * pl.P;
    BCM_REQUIRE(blocks < (1ll << 31), "gated_rec: batch x dim too large");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)pl.P;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pl.P > 1 ? 1 : 0;
    BCM_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    const RecDim n = rec_dim(a, pl);
    BCM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, rec_ptr(a), o, n, a->lam, a->decay_scale));
    return BCM_OK;
}

template <bool BWD, typename T, int MODE, int FORM>
bcm_status rec_launch_p(const bcm_gated_rec_args* a, const RecOut& o, const Plan& pl, cudaStream_t stream) {
    if constexpr (BWD) {
        constexpr int smem = stages_bwd<T>() * stage_bytes<T, kStepsBwd, FORM, 4>();
        if constexpr (MODE == kGroup)
            if (pl.serial) return rec_launch_as(rec_bwd_serial<T, FORM>, smem, a, o, pl, stream);
        if constexpr (MODE != kGroup)
            if (o.sum) return rec_launch_as(rec_bwd_kernel<T, MODE, FORM, true, true>, smem, a, o, pl, stream);
        return pl.P > 1 ? rec_launch_as(rec_bwd_kernel<T, MODE, FORM, true, false>, smem, a, o, pl, stream)
                        : rec_launch_as(rec_bwd_kernel<T, MODE, FORM, false, false>, smem, a, o, pl, stream);
    } else {
        constexpr int smem = stages_fwd<T>() * stage_bytes<T, kStepsFwd, FORM, 3>();
        if constexpr (MODE == kGroup)
            if (pl.serial) return rec_launch_as(rec_fwd_serial<T, FORM>, smem, a, o, pl, stream);
        if constexpr (MODE != kGroup)
            if (o.sum) return rec_launch_as(rec_fwd_kernel<T, MODE, FORM, true, true>, smem, a, o, pl, stream);
        return pl.P > 1 ? rec_launch_as(rec_fwd_kernel<T, MODE, FORM, true, false>, smem, a, o, pl, stream)
                        : rec_launch_as(rec_fwd_kernel<T, MODE, FORM, false, false>, smem, a, o, pl, stream);
    }
}

template <bool BWD, typename T, int FORM>
bcm_status rec_launch_m(const bcm_gated_rec_args* a, const RecOut& o, const Plan& pl, cudaStream_t stream) {
    if (pl.mode == kDense) return rec_launch_p<BWD, T, kDense, FORM>(a, o, pl, stream);
    if (pl.mode == kGroup) return rec_launch_p<BWD, T, kGroup, FORM>(a, o, pl, stream);
    return rec_launch_p<BWD, T, kPacked, FORM>(a, o, pl, stream);
}

template <bool BWD>
bcm_status rec_launch_form(const bcm_gated_rec_args* a, const RecOut& o, const Plan& pl, cudaStream_t stream) {
    return dispatch_dtype(a->dtype, [&](auto tag) -> bcm_status {
        using T = decltype(tag);
        const int form = rec_form(a, BWD);
        if (form == kRows16) return rec_launch_m<BWD, T, kRows16>(a, o, pl, stream);
        if constexpr (sizeof(T) == 2)
            if (form == kRows2) return rec_launch_m<BWD, T, kRows2>(a, o, pl, stream);
        return rec_launch_m<BWD, T, kRows4>(a, o, pl, stream);
    });
}

template <bool BWD>
bcm_status rec_launch(const bcm_gated_rec_args* a, const RecOut& o, const Plan& pl, cudaStream_t stream) {
    if (pl.segs > 1 && o.sum) {                   // compose the segments, join them, then start each from its own state
        if (bcm_status st = rec_launch_form<BWD>(a, o, pl, stream); st != BCM_OK) return st;
        float* state = o.sum + 2 * pl.runs * a->dim;
        const dim3 grid((unsigned)ceil_div(a->dim, 64), (unsigned)(pl.runs / pl.segs));
        rec_join_kernel<BWD><<<grid, 64, 0, stream>>>(o.sum, BWD ? a->dh_last : a->h0, rec_dim(a, pl), state);
        BCM_LAUNCH_CHECK();
        RecOut next = o;
        next.sum = nullptr;
        next.seg = state;
        return rec_launch_form<BWD>(a, next, pl, stream);
    }
    return rec_launch_form<BWD>(a, o, pl, stream);
}

}  // namespace
}  // namespace bcm

using namespace bcm;

extern "C" size_t bcm_gated_rec_ckpt_bytes(const bcm_gated_rec_args* a) {
    if (!a || a->batch < 0 || a->seqlen < 0 || a->dim < 1) return 0;
    if (rec_rows(a) == 0) return 0;
    const Plan pl = rec_plan(a);
    const int64_t states = pl.mode == kPacked ? rec_parts(pl.L, kCkpt) + pl.runs + 1 : pl.runs / pl.segs * rec_parts(pl.L, pl.serial ? kCkptSerial : kCkpt);
    return align_up((size_t)states * (size_t)a->dim * sizeof(float), 256);
}

static size_t rec_segment_bytes(const bcm_gated_rec_args* a, const Plan& pl) {
    return pl.segs > 1 ? align_up((size_t)pl.runs * (size_t)a->dim * 3 * sizeof(float), 256) : 0;
}

extern "C" size_t bcm_gated_rec_fwd_workspace_bytes(const bcm_gated_rec_args* a) {
    if (!a || a->batch < 0 || a->seqlen < 0 || a->dim < 1 || rec_rows(a) == 0) return 0;
    return rec_segment_bytes(a, rec_plan(a));
}

extern "C" size_t bcm_gated_rec_bwd_workspace_bytes(const bcm_gated_rec_args* a) {
    if (!a || a->batch < 0 || a->seqlen < 0 || a->dim < 1 || rec_rows(a) == 0) return 0;
    const Plan pl = rec_plan(a);
    return align_up((size_t)pl.runs * (size_t)pl.P * (size_t)a->dim * sizeof(float), 256) + rec_segment_bytes(a, pl);
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
    const Plan pl = rec_plan(a);
    if (pl.segs > 1) {
        if (!a->workspace || a->workspace_bytes < rec_segment_bytes(a, pl)) {
            set_error("gated_rec_fwd: workspace of %zu bytes < required %zu", a->workspace_bytes, rec_segment_bytes(a, pl));
            return BCM_ERR_WORKSPACE;
        }
        o.sum = static_cast<float*>(a->workspace);
    }
    return rec_launch<false>(a, o, pl, stream);
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
    const Plan pl = rec_plan(a);
    if (pl.segs > 1) o.sum = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + need - rec_segment_bytes(a, pl));
    if (bcm_status st = rec_launch<true>(a, o, pl, stream); st != BCM_OK) return st;
    rec_dlam_kernel<<<(unsigned)ceil_div(a->dim, 32), 1024, 0, stream>>>(o.part, pl.runs * pl.P, a->dim, a->lam, a->decay_scale,
                                                                        a->dlam);
    BCM_LAUNCH_CHECK();
    return BCM_OK;
}

extern "C" bcm_status bcm_gated_rec_step(const void* x, int64_t x_stride_b, const void* r, int64_t r_stride_b, const void* i,
                                         int64_t i_stride_b, bcm_dtype dtype, int64_t batch, int64_t dim, const float* lam,
                                         float decay_scale, float* h, void* y, cudaStream_t stream) {
    clear_error();
    BCM_REQUIRE(dtype_ok(dtype), "gated_rec_step: unsupported dtype %d", (int)dtype);
    BCM_REQUIRE(batch >= 0 && dim >= 1 && batch < (1ll << 31) && dim < (1ll << 30), "gated_rec_step: bad sizes");
    BCM_REQUIRE(decay_scale >= 0.0f, "gated_rec_step: decay_scale must not be negative");
    if (batch == 0) return BCM_OK;
    BCM_REQUIRE(x && r && i && lam && h && y, "gated_rec_step: null pointer");
    RecPtr p = {};
    p.x = x; p.r = r; p.i = i;
    p.xb = x_stride_b; p.rb = r_stride_b; p.ib = i_stride_b;
    const int64_t el = (int64_t)dtype_size(dtype);
    const bool pair = dim % 2 == 0 && (uintptr_t)h % 8 == 0 &&
                      (((int64_t)((uintptr_t)x | (uintptr_t)r | (uintptr_t)i | (uintptr_t)y) |
                        (batch == 1 ? 0 : (x_stride_b | r_stride_b | i_stride_b) * el)) & (2 * el - 1)) == 0;
    // a block row walks several sequences once the blocks fill the GPU eight times over
    const int64_t cols = (dim + 255) / 256;
    const dim3 grid((unsigned)cols, (unsigned)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(batch, 65535), (int64_t)sm_count() * 8 / cols)));
    return dispatch_dtype(dtype, [&](auto tag) -> bcm_status {
        using T = decltype(tag);
        auto kernel = pair ? rec_step_kernel<T, true> : rec_step_kernel<T, false>;
        kernel<<<grid, 128, 0, stream>>>(p, batch, (int)dim, lam, decay_scale, h, static_cast<T*>(y));
        BCM_LAUNCH_CHECK();
        return BCM_OK;
    });
}
