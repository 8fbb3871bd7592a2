#include <algorithm>
#include <cstring>

#include "common.cuh"

namespace bcm {
namespace {

// A block, or a cluster of C blocks, has a row, in 16-byte granules (rows may start
// anywhere); each pass reads it again, from L2 (keeping it in a cluster's shared
// memory left fewer rows in flight and measured slower: 264 against 191 us at 512 x
// 131072 bf16, top-k 50).  One pass finds the maximum, one counts the tokens in
// buckets of s; the buckets bound the mass above every cut, so that one more pass
// leaves a short list of tokens around the cut: the rest is certainly kept or
// certainly not.  The first block sorts the list and finds the cut exactly; the block
// whose tokens hold the target walks them.
// Where more than kListMax tokens lie around the cut (equal or close logits, top-k
// beyond the list together with top-p), the range of s is narrowed, by buckets of
// its bits and exact sums above them, until the list takes what it holds or one
// value is left.
constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBuckets = 4096;
constexpr int kListMax = 4096;                   // tokens around the cut
constexpr float kInf = __builtin_huge_valf();
constexpr float kOne = 1099511627776.0f;         // 2^40
constexpr float kEnd = 27.75f;                   // e^-27.75 2^40 < 1: further down tokens weigh nothing
constexpr float kTop = 3.402823466e38f;

typedef unsigned long long u64;

__device__ __forceinline__ int bucket_of(float d) { return min((int)(d * ((float)kBuckets / kEnd)), kBuckets - 1); }
// The smallest distance, as bits, whose bucket is at least bk.
__device__ uint32_t bucket_edge(uint32_t bk) {
    uint32_t lo = 0, hi = __float_as_uint(kEnd);          // the answer lies in [lo, hi]; distances from kEnd on have no bucket
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2;
        if (bucket_of(__uint_as_float(mid)) >= (int)bk) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}
__device__ __forceinline__ float rel_weight(float s) { return expf(s); }
__device__ __forceinline__ u64 weight_of(float e) { return (u64)(e * kOne); }

// Sums of weights in two 32-bit limbs of 20 bits (adding 2^23 with rounding down leaves the integer in the mantissa);
// exact for fewer than 4096 terms.  The n terms include those that weigh nothing.
struct Sum {
    uint32_t hi = 0, lo = 0;
    __device__ __forceinline__ void add(float2 e) {
        const float2 big = make_float2(8388608.0f, 8388608.0f), scale = make_float2(1048576.0f, 1048576.0f);
        const float2 t = __ffma2_rd(e, scale, big);                                 // 2^23 + floor(e 2^20)
        const float2 rest = __ffma2_rn(e, scale, __fadd2_rn(big, make_float2(-t.x, -t.y)));   // exact, in [0, 1)
        const float2 r = __ffma2_rd(rest, scale, big);
        hi += __float_as_uint(t.x) + __float_as_uint(t.y);
        lo += __float_as_uint(r.x) + __float_as_uint(r.y);
    }
    __device__ __forceinline__ u64 take(uint32_t n) {
        const u64 v = ((u64)(hi - n * 0x4b000000u) << 20) + (u64)(lo - n * 0x4b000000u);
        hi = lo = 0;
        return v;
    }
};
constexpr uint32_t kSumMax = 4000;

template <typename V>
__device__ V block_sum_u(V v, V* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
    for (int k = 0; k < kWarps; ++k) v += red[k];
    return v;
}

// ---- the cluster's shared memory --------------------------------------------------
__device__ __forceinline__ uint32_t remote(const void* p, int rank) {
    uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}
__device__ __forceinline__ void st_remote(uint32_t a, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }
__device__ __forceinline__ void st_remote(uint32_t a, u64 v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory"); }
__device__ __forceinline__ void red_remote(uint32_t a, uint32_t v) { asm volatile("red.shared::cluster.add.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory"); }
__device__ __forceinline__ uint32_t add_remote(uint32_t a, uint32_t v) {
    uint32_t o;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(o) : "r"(a), "r"(v) : "memory");
    return o;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

struct Shared {
    float tops[kMaxCluster];
    float fred[kWarps];
    u64 red[kWarps];
    // per warp of the cluster, at rank 0: the weight above the window, all of it and what min-p keeps, and that below it
    u64 kept[kMaxCluster * kWarps], all[kMaxCluster * kWarps], rest[kMaxCluster * kWarps];
    // from rank 0 to all: the window of buckets (first, end), what to do, then the cut and the target
    uint32_t win_lo, win_hi, mode, list_n, list_at;
    uint32_t nar_lo, nar_hi;                     // the narrowed range of -s (as bits), the count or weight above it,
    u64 nar_base, nar_goal;                      // and which one of them, from 1, is the last kept
    uint32_t k_left;                             // how many of the list's tokens top-k leaves (rank 0)
    uint32_t cut_d, cut_v, seg;                  // the last kept token (-s, index); the warp that holds the target
    u64 target, total;                           // the target within that warp's tokens; the kept weight
};
enum { kSet, kNarrow };                          // whether [nar_lo, nar_hi) is the list's range already

// Granule g of the row: its elements as floats, those outside the row -inf; then their distances -s from the maximum.
template <typename T>
struct Granule {
    static constexpr int N = 16 / (int)sizeof(T);
    float f[N];
    __device__ __forceinline__ void unpack(uint4 w) {
        T t[N];
        memcpy(t, &w, 16);
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = to_f32<T>(t[e]);
    }
    __device__ __forceinline__ void trim(int64_t g, int64_t last, int shift, int64_t V) {
        if (g == 0 || g == last)
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (g * N + e < shift || g * N + e - shift >= V) f[e] = -kInf;
    }
    // (a NaN, or -inf at 1/T = 0, becomes a NaN: its bits lie above every distance that counts)
    __device__ __forceinline__ void distances(float top, float it) {
        if (top > kTop)                                  // +inf: its equals at 0, the rest far away
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = f[e] == top ? 0.0f : kInf;
        else
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = (top - f[e]) * it;
    }
};

// The list in ascending order (bitonic network over the next power of two, rest ~0).  A warp takes consecutive pairs:
// steps within its own elements need no block barrier.
__device__ void sort_list(u64* list, int n) {
    int m = 1;
    while (m < n) m <<= 1;
    for (int k = n + threadIdx.x; k < m; k += kThreads) list[k] = ~0ull;
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, own = max(m / 2 / kWarps, 32);   // pairs of a warp
    for (int size = 2; size <= m; size <<= 1)
        for (int step = size >> 1; step > 0; step >>= 1) {
            for (int k = warp * own + lane; k < min((warp + 1) * own, m / 2); k += 32) {
                const int i = 2 * k - (k & (step - 1)), j = i + step;
                const u64 x = list[i], y = list[j];
                if ((x > y) == ((i & size) == 0)) {
                    list[i] = y;
                    list[j] = x;
                }
            }
            // what comes next reads other warps' elements when this step or the next one leaves the warp's own
            const int next = step > 1 ? step >> 1 : size;
            if (max(step, next) > own) __syncthreads();
            else __syncwarp();
        }
    __syncthreads();
}

// Exclusive prefixes of a thread's counts and bounds over the block, and their totals.
struct Prefix {
    uint32_t n, tn;
    float lo, hi, tl, th;
};
__device__ Prefix block_prefix(uint32_t n, float lo, float hi) {
    __shared__ uint32_t pn[kWarps];
    __shared__ float pl[kWarps], ph[kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t cn = n;
    float cl = lo, ch = hi;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t vn = __shfl_up_sync(kFull, cn, o);
        const float vl = __shfl_up_sync(kFull, cl, o), vh = __shfl_up_sync(kFull, ch, o);
        if (lane >= o) {
            cn += vn;
            cl += vl;
            ch += vh;
        }
    }
    __syncthreads();
    if (lane == 31) {
        pn[warp] = cn;
        pl[warp] = cl;
        ph[warp] = ch;
    }
    __syncthreads();
    Prefix r = {cn - n, 0, cl - lo, ch - hi, 0.0f, 0.0f};
    for (int j = 0; j < kWarps; ++j) {
        if (j < warp) {
            r.n += pn[j];
            r.lo += pl[j];
            r.hi += ph[j];
        }
        r.tn += pn[j];
        r.tl += pl[j];
        r.th += ph[j];
    }
    return r;
}
// What n tokens with -s in [from, to) weigh at least and at most, over 2^40.  1e-5 covers rounded edges and 2^-40 the
// rounding down; the sums of up to 4096 fp32 terms, added in blocks, are within 1e-5 too.
__device__ __forceinline__ float weighs_least(uint32_t n, float to) { return (float)n * fmaxf(expf(-to - 1e-5f) - 1.0f / kOne, 0.0f) * (1.0f - 4e-5f); }
__device__ __forceinline__ float weighs_most(uint32_t n, float from) { return (float)n * expf(-from + 1e-5f) * (1.0f + 4e-5f); }

// Plain, top-k 50 and top-p 0.9: 512 x 131072 bf16 161, 169 and 360 us, bound by instructions (issue slots 76, 60 and
// 73 % busy, DRAM 12 % or less; 1.7 waves of blocks); 1 x 32000 fp32 17, 30 and 36 us, a chain of dependent phases.
template <typename T>
__global__ void __launch_bounds__(kThreads, 2)
sample_kernel(const __grid_constant__ bcm_sample_args a, int C) {
    using Gr = Granule<T>;
    extern __shared__ __align__(16) char dyn[];
    __shared__ Shared sh;
    u64* list = reinterpret_cast<u64*>(dyn);                         // after the buckets are done
    uint32_t* hist = reinterpret_cast<uint32_t*>(dyn);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = blockIdx.x % C;
    const int64_t b = blockIdx.x / C, V = a.vocab;
    const T* x = static_cast<const T*>(a.logits) + b * a.logits_stride;
    const int shift = (int)((uintptr_t)x & 15) / (int)sizeof(T);
    const uint4* row = reinterpret_cast<const uint4*>((uintptr_t)x & ~(uintptr_t)15);
    const int64_t grans = (shift + V + Gr::N - 1) / Gr::N, last = grans - 1;
    const int64_t per = (grans + C - 1) / C, wper = (per + kWarps - 1) / kWarps;
    // the warp's granules: a contiguous range, so that warps follow one another in index order
    const int64_t g0 = rank * per + warp * wper, g1 = min(min(g0 + wper, (rank + 1) * per), grans);
    const float temp = a.temperature ? a.temperature[b] : a.temperature_all;
    const float inv = 1.0f / temp;
    const bool warm = temp > 0.0f && inv < kInf;
    const float it = warm ? inv : 1.0f;
    int64_t k = warm ? (a.top_k ? a.top_k[b] : a.top_k_all) : 1;
    if (k <= 0 || k > V) k = V;
    const float p = a.top_p ? a.top_p[b] : a.top_p_all;
    const float mp = a.min_p ? a.min_p[b] : a.min_p_all;
    const float least = mp > 0.0f ? fminf(mp, 1.0f) : 0.0f;
    const bool use_k = k < V, use_p = p < 1.0f;

    // the row comes in; its maximum
    float top = -kInf;
#pragma unroll 4
    for (int64_t g = g0 + lane; g < g1; g += 32) {
        const uint4 w = row[g];
        Gr q;
        q.unpack(w);
        q.trim(g, last, shift, V);
#pragma unroll
        for (int e = 0; e < Gr::N; ++e) top = fmaxf(top, q.f[e]);
    }
    for (int j = tid; j < kBuckets; j += kThreads) hist[j] = 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
    if (lane == 0) sh.fred[warp] = top;
    if (tid == 0) sh.list_n = 0;
    __syncthreads();
    for (int j = 0; j < kWarps; ++j) top = fmaxf(top, sh.fred[j]);
    if (C > 1) {
        cluster_sync();                                   // every block runs before its shared memory is written to
        if (tid < C) st_remote(remote(&sh.tops[rank], tid), __float_as_uint(top));
        cluster_sync();
        for (int j = 0; j < C; ++j) top = fmaxf(top, sh.tops[j]);
    }
    if (top == -kInf) {
        if (rank == 0 && tid == 0) {
            a.tokens[b] = -1;
            a.logprob[b] = -kInf;
        }
        return;
    }
    auto each = [&](auto&& f) {                           // f(index of the first element, distances) over the warp's granules
        for (int64_t g = g0 + lane; g - lane < g1; g += 32) {      // (the whole warp)
            Gr q;
            if (g < g1) {
                q.unpack(row[g]);
                q.trim(g, last, shift, V);
                q.distances(top, it);
            } else {
#pragma unroll
                for (int e = 0; e < Gr::N; ++e) q.f[e] = kInf;
            }
            f(g * Gr::N - shift, q);
        }
    };

    // buckets of s, counted; the first block finds the window of buckets that holds the cut
    if (use_k || use_p) {
        each([&](int64_t, Gr& q) {
#pragma unroll
            for (int e = 0; e < Gr::N; ++e) {
                if (q.f[e] < kEnd) atomicAdd(&hist[bucket_of(q.f[e])], 1u);
            }
        });
        __syncthreads();
        if (C > 1) {
            if (rank != 0)
                for (int j = tid; j < kBuckets; j += kThreads)
                    if (hist[j]) red_remote(remote(&hist[j], 0), hist[j]);
            cluster_sync();
        }
        if (rank == 0) {
            constexpr int kEach = kBuckets / kThreads;
            uint32_t n[kEach], below = 0;
            float lo[kEach], hi[kEach], slo = 0.0f, shi = 0.0f;
            const float width = kEnd / (float)kBuckets;
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const int bk = tid * kEach + j;
                n[j] = hist[bk];
                below += n[j];
                lo[j] = use_p ? weighs_least(n[j], (float)(bk + 1) * width) : 0.0f;
                hi[j] = use_p ? weighs_most(n[j], (float)bk * width) : 0.0f;
                slo += lo[j];
                shi += hi[j];
            }
            if (tid == 0) {
                sh.win_lo = 0;
                sh.win_hi = kBuckets;
                sh.mode = kSet;
                sh.k_left = 0xffffffffu;
            }
            const Prefix pre = block_prefix(below, slo, shi);
            uint32_t bn = pre.n;
            const uint32_t tn = pre.tn;
            float bl = pre.lo, bh = pre.hi;
            const float tl = pre.tl, th = pre.th;
            // a k-th token beyond the last bucket weighs nothing: no cut by count
            const bool by_k = use_k && (uint64_t)k < tn;
            const float p_lo = p * tl * (1.0f - 2e-5f), p_hi = p * th * (1.0f + 2e-5f) + 1e-9f;
            for (int j = 0; j < kEach; ++j) {
                const uint32_t bk = tid * kEach + j, an = bn + n[j];
                const float al = bl + lo[j], ah = bh + hi[j];
                if (by_k) {
                    if (bn < k && k <= an) {
                        // with top-p the list has to hold all of the first k
                        const bool whole = an <= kListMax;
                        sh.win_lo = whole ? 0 : bk;
                        sh.win_hi = bk + 1;
                        sh.k_left = (uint32_t)k - (whole ? 0u : bn);
                        sh.mode = whole || (n[j] <= kListMax && !use_p) ? kSet : kNarrow;
                    }
                } else if (use_p) {
                    if ((bh < p_lo || bk == 0) && ah >= p_lo) sh.win_lo = bk;
                    if ((bl < p_hi || bk == 0) && al >= p_hi) sh.win_hi = bk + 1;
                }
                bn = an;
                bl = al;
                bh = ah;
            }
            __syncthreads();
            if (!by_k && use_p) {                          // how many tokens that window holds
                u64 in = 0;
#pragma unroll
                for (int j = 0; j < kEach; ++j)
                    if (tid * kEach + j >= sh.win_lo && tid * kEach + j < sh.win_hi) in += n[j];
                in = block_sum_u<u64>(in, sh.red);
                if (tid == 0 && in > kListMax) sh.mode = kNarrow;
            }
            __syncthreads();
            if (warp == 0 && lane < 2) {                   // the window's edges
                const bool any = by_k || use_p;
                const uint32_t edge = !any ? __float_as_uint(kEnd) : bucket_edge(lane ? sh.win_hi : sh.win_lo);
                for (int c = 0; c < C; ++c) st_remote(remote(lane ? &sh.nar_hi : &sh.nar_lo, c), edge);
            }
            if (tid < C && tid > 0) {
                st_remote(remote(&sh.mode, tid), sh.mode);
                st_remote(remote(&sh.k_left, tid), sh.k_left);
            }
        }
        if (C > 1) cluster_sync();
        else __syncthreads();
    } else {
        if (tid == 0) {
            sh.nar_lo = sh.nar_hi = __float_as_uint(kEnd);
            sh.mode = kSet;
            sh.k_left = 0xffffffffu;
        }
        __syncthreads();
    }
    u64 limit = 0x7f7fffffffffffffull;                    // (-s, index) of the last token that is still in
    auto token_of = [&](float d, int64_t v) -> u64 { return ((u64)__float_as_uint(d) << 32) | (u64)(uint32_t)v; };
    if (sh.mode == kNarrow) {
        const uint32_t end = __float_as_uint(kEnd);
        auto sync = [&]() {
            if (C > 1) cluster_sync();
            else __syncthreads();
        };
        // weight of the tokens that are still in with -s in [from, mid) and in [mid, to), at rank 0 (through sh.all, sh.rest)
        u64 front = 0, back = 0;
        auto weigh = [&](uint32_t from, uint32_t mid, uint32_t to) {
            Sum sf, sb;
            uint32_t terms = 0;
            front = back = 0;
            each([&](int64_t v0, Gr& q) {
#pragma unroll
                for (int e0 = 0; e0 < Gr::N; e0 += 2) {
                    float in_front[2], behind[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const u64 at = token_of(q.f[e0 + j], v0 + e0 + j);
                        const uint32_t d = (uint32_t)(at >> 32);
                        const float r = d >= from && d < to && at <= limit ? rel_weight(-q.f[e0 + j]) : 0.0f;
                        in_front[j] = d < mid ? r : 0.0f;
                        behind[j] = d < mid ? 0.0f : r;
                    }
                    sf.add(make_float2(in_front[0], in_front[1]));
                    sb.add(make_float2(behind[0], behind[1]));
                }
                terms += Gr::N;
                if (terms > kSumMax) {
                    front += sf.take(terms);
                    back += sb.take(terms);
                    terms = 0;
                }
            });
            front += sf.take(terms);
            back += sb.take(terms);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                front += __shfl_xor_sync(kFull, front, o);
                back += __shfl_xor_sync(kFull, back, o);
            }
            if (lane == 0) {
                st_remote(remote(&sh.all[rank * kWarps + warp], 0), front);
                st_remote(remote(&sh.rest[rank * kWarps + warp], 0), back);
            }
            sync();
            if (rank == 0) {
                front = back = 0;
                for (int j = tid; j < C * kWarps; j += kThreads) {
                    front += sh.all[j];
                    back += sh.rest[j];
                }
                front = block_sum_u<u64>(front, sh.red);
                back = block_sum_u<u64>(back, sh.red);
            }
            sync();
        };
        for (int by_weight = 0; by_weight < 2; ++by_weight) {
            if (by_weight ? !use_p : sh.k_left == 0xffffffffu) continue;
            // rank 0 keeps the range [nar_lo, nar_hi) of -s that holds the last kept token, and tells the others
            uint32_t lo0 = 0, hi0 = end;
            if (by_weight) {
                if (sh.k_left == 0xffffffffu) {           // (without top-k the window of buckets holds it)
                    lo0 = sh.nar_lo;
                    hi0 = sh.nar_hi;
                }
                weigh(0, lo0, end);
            }
            if (rank == 0 && tid == 0) {
                sh.nar_lo = lo0;
                sh.nar_hi = hi0;
                sh.nar_base = front;
                const double lim = ceil((double)p * (double)(front + back));
                sh.nar_goal = by_weight ? (lim >= 1.0 ? (u64)lim : 1ull) : (u64)k;
            }
            for (int round = 0; round < 64; ++round) {    // (each narrows a thousandfold; 64 only bounds the loop)
                for (int j = tid; j < kBuckets; j += kThreads) hist[j] = 0;
                if (rank == 0) {
                    __syncthreads();
                    if (tid < C && tid > 0) {
                        st_remote(remote(&sh.nar_lo, tid), sh.nar_lo);
                        st_remote(remote(&sh.nar_hi, tid), sh.nar_hi);
                        st_remote(remote(&sh.mode, tid), sh.mode);
                        st_remote(remote(&sh.k_left, tid), sh.k_left);
                    }
                }
                sync();
                const uint32_t from = sh.nar_lo, span = sh.nar_hi - from;
                if (span == 1 || sh.mode == kSet) break;
                const int cut = max(0, 32 - __clz((span - 1) >> 12));      // buckets of 2^cut values
                each([&](int64_t v0, Gr& q) {
#pragma unroll
                    for (int e = 0; e < Gr::N; ++e) {
                        const u64 at = token_of(q.f[e], v0 + e);
                        const uint32_t d = (uint32_t)(at >> 32) - from;
                        if (d < span && at <= limit) atomicAdd(&hist[d >> cut], 1u);
                    }
                });
                __syncthreads();
                if (C > 1) {
                    if (rank != 0)
                        for (int j = tid; j < kBuckets; j += kThreads)
                            if (hist[j]) red_remote(remote(&hist[j], 0), hist[j]);
                    cluster_sync();
                }
                uint32_t first = from, next = from;                        // the bucket that may hold the token first
                if (rank == 0) {
                    constexpr int kEach = kBuckets / kThreads;
                    uint32_t n[kEach], below = 0;
                    float lo[kEach], hi[kEach], slo = 0.0f, shi = 0.0f;
#pragma unroll
                    for (int j = 0; j < kEach; ++j) {
                        const uint32_t bk = tid * kEach + j;
                        n[j] = hist[bk];
                        below += n[j];
                        lo[j] = hi[j] = 0.0f;
                        if (by_weight && n[j]) {
                            lo[j] = weighs_least(n[j], __uint_as_float(from + ((bk + 1) << cut)));
                            hi[j] = weighs_most(n[j], __uint_as_float(from + (bk << cut)));
                        }
                        slo += lo[j];
                        shi += hi[j];
                    }
                    const Prefix pre = block_prefix(below, slo, shi);
                    uint32_t bn = pre.n;
                    float bl = pre.lo, bh = pre.hi;
                    // (float differences of 64-bit weights: 2^-24 of the goal, in both directions)
                    const float left = (float)((double)(sh.nar_goal - sh.nar_base) / (double)kOne);
                    const u64 count_left = sh.nar_goal - sh.nar_base;
                    if (tid == 0) {
                        sh.win_lo = 0xffffffffu;
                        sh.win_hi = (span - 1) >> cut;
                    }
                    __syncthreads();
#pragma unroll
                    for (int j = 0; j < kEach; ++j) {
                        const uint32_t bk = tid * kEach + j;
                        if (n[j]) {
                            if (!by_weight && bn < count_left && count_left <= (u64)bn + n[j]) {
                                sh.win_lo = sh.win_hi = bk;
                                sh.nar_base += bn;
                            }
                            if (by_weight && bh + hi[j] >= left * (1.0f - 2e-5f)) atomicMin(&sh.win_lo, bk);
                            if (by_weight && bl + lo[j] >= left * (1.0f + 2e-5f)) atomicMin(&sh.win_hi, bk);
                        }
                        bn += n[j];
                        bl += lo[j];
                        bh += hi[j];
                    }
                    __syncthreads();
                    u64 in = 0;                           // tokens in what is left: enough for the list to take over?
#pragma unroll
                    for (int j = 0; j < kEach; ++j)
                        if (tid * kEach + j >= sh.win_lo && tid * kEach + j <= sh.win_hi) in += n[j];
                    in = block_sum_u<u64>(in, sh.red);
                    if (tid == 0) {
                        if (in <= kListMax && sh.win_lo != 0xffffffffu && (by_weight || !use_p)) {
                            sh.mode = kSet;
                            sh.k_left = by_weight ? 0xffffffffu : (uint32_t)(sh.nar_goal - sh.nar_base);
                        }
                        first = from + ((sh.win_lo == 0xffffffffu ? 0u : sh.win_lo) << cut);
                        sh.nar_lo = first;
                        sh.nar_hi = min(sh.nar_hi, from + ((sh.win_hi + 1) << cut));
                    }
                    __syncthreads();
                    first = sh.nar_lo;
                }
                if (by_weight) {
                    if (rank == 0 && tid < C && tid > 0) {
                        st_remote(remote(&sh.nar_lo, tid), first);
                        st_remote(remote(&sh.mode, tid), sh.mode);
                    }
                    sync();
                    if (sh.mode == kSet) continue;
                    // exactly: the weight above that bucket and in it
                    first = sh.nar_lo;
                    next = first + (1u << cut);
                    weigh(from, first, next);
                    if (rank == 0 && tid == 0) {
                        sh.nar_base += front;
                        if (sh.nar_base + back >= sh.nar_goal) {
                            sh.nar_hi = min(sh.nar_hi, next);
                        } else {
                            sh.nar_base += back;
                            sh.nar_lo = next;
                            sh.nar_hi = max(sh.nar_hi, next + 1);
                        }
                    }
                }
            }
            if (sh.mode == kSet) break;
            // one value is left: of the tokens that have it, the first ones by index
            const uint32_t value = sh.nar_lo;
            u64 mine = 0;
            each([&](int64_t v0, Gr& q) {
#pragma unroll
                for (int e = 0; e < Gr::N; ++e) {
                    const u64 at = token_of(q.f[e], v0 + e);
                    mine += (uint32_t)(at >> 32) == value && at <= limit;
                }
            });
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(kFull, mine, o);
            if (lane == 0) st_remote(remote(&sh.all[rank * kWarps + warp], 0), mine);
            sync();
            if (rank == 0 && tid == 0) {
                const u64 w = by_weight ? max(weight_of(rel_weight(-__uint_as_float(value))), 1ull) : 1ull;
                u64 left = (sh.nar_goal - sh.nar_base + w - 1) / w;
                int q = 0;
                while (q < C * kWarps - 1 && left > sh.all[q]) left -= sh.all[q++];
                for (int c = 0; c < C; ++c) {
                    st_remote(remote(&sh.seg, c), (uint32_t)q);
                    st_remote(remote(&sh.target, c), left);
                }
            }
            sync();
            if ((int)sh.seg == rank * kWarps + warp) {    // that warp finds it
                u64 before = 0;
                for (int64_t gb = g0; gb < g1; gb += 32) {
                    const int64_t g = gb + lane;
                    Gr q;
                    uint32_t here = 0;
                    if (g < g1) {
                        q.unpack(row[g]);
                        q.trim(g, last, shift, V);
                        q.distances(top, it);
#pragma unroll
                        for (int e = 0; e < Gr::N; ++e) {
                            const u64 at = token_of(q.f[e], g * Gr::N - shift + e);
                            here |= ((uint32_t)(at >> 32) == value && at <= limit ? 1u : 0u) << e;
                        }
                    }
                    const u64 upto = before + warp_inclusive_sum<u64>((u64)__popc(here));
                    u64 run = upto - __popc(here);
                    if (run < sh.target && sh.target <= upto)
#pragma unroll
                        for (int e = 0; e < Gr::N; ++e)
                            if ((here >> e & 1u) && ++run == sh.target)
                                for (int c = 0; c < C; ++c) {
                                    st_remote(remote(&sh.cut_d, c), value);
                                    st_remote(remote(&sh.cut_v, c), (uint32_t)(g * Gr::N - shift + e));
                                }
                    before = __shfl_sync(kFull, upto, 31);
                }
            }
            sync();
            limit = ((u64)sh.cut_d << 32) | sh.cut_v;
            sync();
        }
    }
    // (a cut that is known needs no list: everything up to the limit)
    const uint32_t list_lo = sh.mode == kSet ? sh.nar_lo : __float_as_uint(kEnd), list_hi = sh.mode == kSet ? sh.nar_hi : __float_as_uint(kEnd);
    // what lies above the list's range is summed (all of it, and what min-p keeps), what lies in it goes to the list
    {
        const uint32_t end = __float_as_uint(kEnd);
        // top-p's share is of every token's weight, or, after top-k, of the weight that top-k leaves
        const bool some_above = list_lo > 0, want_all = use_p && least > 0.0f, limited = limit != 0x7f7fffffffffffffull;
        const bool want_rest = use_p && list_hi > list_lo && sh.k_left == 0xffffffffu, listed = list_hi > list_lo;
        u64 kept = 0, all = 0, rest = 0;
        Sum sk, sa, sr;
        uint32_t terms = 0;
        each([&](int64_t v0, Gr& q) {
            uint32_t to_list = 0;
            if (some_above || want_rest) {
#pragma unroll
                for (int e0 = 0; e0 < Gr::N; e0 += 2) {
                    float wk[2], wa[2], wr[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t d = __float_as_uint(q.f[e0 + j]);
                        float w = d < end ? rel_weight(-q.f[e0 + j]) : 0.0f;
                        if (limited && token_of(q.f[e0 + j], v0 + e0 + j) > limit) w = 0.0f;
                        wa[j] = d < list_lo ? w : 0.0f;
                        wk[j] = wa[j] >= least ? wa[j] : 0.0f;
                        wr[j] = d >= list_hi ? w : 0.0f;
                    }
                    sk.add(make_float2(wk[0], wk[1]));
                    if (want_all) sa.add(make_float2(wa[0], wa[1]));
                    if (want_rest) sr.add(make_float2(wr[0], wr[1]));
                }
                terms += Gr::N;
                if (terms > kSumMax) {
                    kept += sk.take(terms);
                    if (want_all) all += sa.take(terms);
                    if (want_rest) rest += sr.take(terms);
                    terms = 0;
                }
            }
            if (listed) {
#pragma unroll
                for (int e = 0; e < Gr::N; ++e) {
                    const uint32_t d = __float_as_uint(q.f[e]);
                    if (d >= list_lo && d < list_hi && (!limited || token_of(q.f[e], v0 + e) <= limit)) to_list |= 1u << e;
                }
                // the warp's tokens go to consecutive places
                if (__any_sync(kFull, to_list != 0)) {
                    const uint32_t mine = __popc(to_list), upto = warp_inclusive_sum<uint32_t>(mine);
                    uint32_t slot = 0;
                    if (lane == 31) slot = atomicAdd(&sh.list_n, upto);
                    slot = __shfl_sync(kFull, slot, 31) + upto - mine;
#pragma unroll
                    for (int e = 0; e < Gr::N; ++e)
                        if (to_list >> e & 1u) {
                            if (slot < kListMax) list[slot] = token_of(q.f[e], v0 + e);
                            ++slot;
                        }
                }
            }
        });
        kept += sk.take(terms);
        if (want_all) all += sa.take(terms);
        else all = kept;                                  // (without min-p the same; not asked for without top-p)
        if (want_rest) rest += sr.take(terms);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            kept += __shfl_xor_sync(kFull, kept, o);
            all += __shfl_xor_sync(kFull, all, o);
            rest += __shfl_xor_sync(kFull, rest, o);
        }
        if (lane == 0) {
            st_remote(remote(&sh.rest[rank * kWarps + warp], 0), rest);
            st_remote(remote(&sh.kept[rank * kWarps + warp], 0), kept);
            st_remote(remote(&sh.all[rank * kWarps + warp], 0), all);
        }
    }
    if (C > 1) {                                          // the other blocks' lists go behind the first one's
        cluster_sync();
        if (rank != 0) {
            const uint32_t n = min(sh.list_n, (uint32_t)kListMax);
            if (tid == 0) sh.list_at = n ? add_remote(remote(&sh.list_n, 0), n) : 0;
            __syncthreads();
            for (uint32_t j = tid; j < n; j += kThreads)
                if (sh.list_at + j < kListMax) st_remote(remote(list + sh.list_at + j, 0), list[j]);
        }
        cluster_sync();
    } else {
        __syncthreads();
    }
    if (rank == 0) {
        const int n = min((int)sh.list_n, kListMax), nk = (int)min((uint32_t)n, sh.k_left), segs = C * kWarps;
        u64 above = 0, rest = 0;
        for (int j = tid; j < segs; j += kThreads) {
            above += sh.all[j];
            rest += sh.rest[j];
        }
        above = block_sum_u<u64>(above, sh.red);
        rest = block_sum_u<u64>(rest, sh.red);
        if (tid == 0) {
            sh.cut_d = (uint32_t)(limit >> 32);           // without a list everything up to the limit is kept
            sh.cut_v = (uint32_t)limit;
        }
        if (n > 0) {
            sort_list(list, n);
            // a thread takes consecutive entries of the first nk; prefix sums of their weights
            constexpr int kEach = kListMax / kThreads;
            const int each_n = (nk + kThreads - 1) / kThreads, e0 = min(tid * each_n, nk), e1 = min(e0 + each_n, nk);
            u64 w[kEach], mine = 0;
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                w[j] = e0 + j < e1 ? weight_of(rel_weight(-__uint_as_float((uint32_t)(list[e0 + j] >> 32)))) : 0ull;
                mine += w[j];
            }
            u64 run = warp_inclusive_sum<u64>(mine);
            __syncthreads();
            if (lane == 31) sh.red[warp] = run;
            __syncthreads();
            u64 in_list = 0;
            run -= mine;
            for (int j = 0; j < kWarps; ++j) {
                if (j < warp) run += sh.red[j];
                in_list += sh.red[j];
            }
            u64 most = ~0ull;
            if (use_p) {
                const double lim = ceil((double)p * (double)(above + in_list + rest));
                most = lim >= 1.0 ? (u64)lim : 1ull;
            }
            run += above;
#pragma unroll
            for (int j = 0; j < kEach; ++j)
                if (e0 + j < e1) {
                    const u64 at = list[e0 + j], next = run + w[j];
                    if (run < most) {                     // kept: its weight goes to its warp
                        const uint32_t d = (uint32_t)(at >> 32), v = (uint32_t)at;
                        if (e0 + j + 1 == nk || next >= most) {
                            sh.cut_d = d;
                            sh.cut_v = v;
                        }
                        if (rel_weight(-__uint_as_float(d)) >= least) {
                            const int64_t g = ((int64_t)v + shift) / Gr::N, r = g / per;
                            atomicAdd(&sh.kept[r * kWarps + (g - r * per) / wper], w[j]);
                        }
                    }
                    run = next;
                }
        }
        __syncthreads();
        if (warp == 0) {                                  // the target and the warp that holds it: 4 warps' sums a lane
            u64 part[kMaxCluster * kWarps / 32], mine = 0;
#pragma unroll
            for (int j = 0; j < kMaxCluster * kWarps / 32; ++j) {
                const int q = lane * (kMaxCluster * kWarps / 32) + j;
                part[j] = q < segs ? sh.kept[q] : 0ull;
                mine += part[j];
            }
            const u64 upto = warp_inclusive_sum<u64>(mine), total = __shfl_sync(kFull, upto, 31);
            const double want = floor((double)a.u[b] * (double)total);
            u64 target = want > 0.0 ? (u64)want : 0ull;
            if (target >= total) target = total - 1;
            u64 run = upto - mine;
#pragma unroll
            for (int j = 0; j < kMaxCluster * kWarps / 32; ++j) {
                if (run <= target && target < run + part[j]) {
                    const int q = lane * (kMaxCluster * kWarps / 32) + j, r = q / kWarps;
                    st_remote(remote(&sh.cut_d, r), sh.cut_d);
                    st_remote(remote(&sh.cut_v, r), sh.cut_v);
                    st_remote(remote(&sh.target, r), target - run);
                    st_remote(remote(&sh.total, r), total);
                    for (int c = 0; c < C; ++c) st_remote(remote(&sh.seg, c), (uint32_t)q);
                }
                run += part[j];
            }
        }
    }
    if (C > 1) cluster_sync();
    else __syncthreads();
    // The block that holds the target walks that warp's tokens in index order: every warp sums a part of them, the one
    // whose part holds the target finds it.
    if ((int)sh.seg / kWarps != rank) return;
    const u64 cut = ((u64)sh.cut_d << 32) | sh.cut_v;
    const int64_t w0 = rank * per + sh.seg % kWarps * wper, w1 = min(min(w0 + wper, (rank + 1) * per), grans), part = (wper + kWarps - 1) / kWarps;
    const int64_t p0 = min(w0 + warp * part, w1), p1 = min(p0 + part, w1);
    auto kept_in = [&](int64_t g, Gr& q, u64 (&w)[Gr::N]) -> u64 {
        u64 mine = 0;
#pragma unroll
        for (int e = 0; e < Gr::N; ++e) w[e] = 0;
        if (g < p1) {
            q.unpack(row[g]);
            q.trim(g, last, shift, V);
            q.distances(top, it);
#pragma unroll
            for (int e = 0; e < Gr::N; ++e) {
                const float r = rel_weight(-q.f[e]);
                if (token_of(q.f[e], g * Gr::N - shift + e) <= cut && r >= least) w[e] = weight_of(r);
                mine += w[e];
            }
        }
        return mine;
    };
    Gr q;
    u64 w[Gr::N], sum = 0;
    for (int64_t g = p0 + lane; g < p1; g += 32) sum += kept_in(g, q, w);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    if (lane == 0) sh.red[warp] = sum;
    __syncthreads();
    u64 before = 0;
    for (int j = 0; j < warp; ++j) before += sh.red[j];
    if (!(before <= sh.target && sh.target < before + sum)) return;
    for (int64_t gb = p0; gb < p1; gb += 32) {
        const int64_t g = gb + lane;
        const u64 mine = kept_in(g, q, w);
        const u64 upto = before + warp_inclusive_sum<u64>(mine);
        u64 run = upto - mine;
        if (run <= sh.target && sh.target < upto)
#pragma unroll
            for (int e = 0; e < Gr::N; ++e) {
                if (run <= sh.target && sh.target < run + w[e]) {
                    a.tokens[b] = g * Gr::N - shift + e;
                    a.logprob[b] = -q.f[e] - (float)log((double)sh.total / (double)kOne);
                }
                run += w[e];
            }
        before = __shfl_sync(kFull, upto, 31);
        if (before > sh.target) return;
    }
}

}  // namespace
}  // namespace bcm

using namespace bcm;

extern "C" bcm_status bcm_sample_tokens(const bcm_sample_args* a, cudaStream_t stream) {
    clear_error();
    BCM_REQUIRE(a != nullptr, "sample_tokens: null arguments");
    BCM_REQUIRE(dtype_ok(a->dtype), "sample_tokens: unsupported dtype %d", (int)a->dtype);
    BCM_REQUIRE(a->batch >= 0 && a->batch < (1ll << 31) && a->vocab >= 1 && a->vocab <= BCM_SAMPLE_MAX_VOCAB,
                "sample_tokens: vocab must be in [1, %d], batch below 2^31", BCM_SAMPLE_MAX_VOCAB);
    if (a->batch == 0) return BCM_OK;
    BCM_REQUIRE(a->logits && a->u && a->tokens && a->logprob, "sample_tokens: null pointer");
    // Blocks of a row: one where the batch fills the GPU (two blocks per SM), more below (down to slices of 4 KB).
    const int64_t bytes = a->vocab * (int64_t)dtype_size(a->dtype);
    int C = 1;
    while (C < kMaxCluster && a->batch * C <= sm_count() && bytes / C > 4096) C *= 2;
    return dispatch_dtype(a->dtype, [&](auto tag) -> bcm_status {
        using T = decltype(tag);
        auto kernel = sample_kernel<T>;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(a->batch * C));
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = kListMax * 8;
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)C;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = C > 1 ? 1 : 0;
        BCM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, *a, C));
        return BCM_OK;
    });
}
