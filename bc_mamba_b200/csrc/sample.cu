// sample.cu — one token per row from its logits and a given uniform number,
// with temperature, top-k, top-p and min-p.
//
// Row b, T = temperature[b]; T <= 0 (or NaN, or so small that 1/T overflows)
// means greedy: 1/T is taken as 1 and top_k as 1.
//   s_v = (logit_v - max logit) * (1/T)  (fp32, 0 at the maximum; a NaN logit
//         counts as -inf; s = -inf is never taken)
//   e_v = exp(s_v),  w_v = floor(e_v 2^40)   (integer weight)
// In descending order of s (equal s in ascending order of index):
//   top-k  keeps the first k (k <= 0: all);
//   top-p  keeps of these the tokens whose preceding weight is below
//          ceil(p * total weight of these), the first always (p >= 1: all);
//   min-p  keeps of these the tokens with e_v >= min(min_p, 1).
// The token is the first, in ascending order of index, whose inclusive kept
// weight exceeds floor(u * total kept weight).  Weights are integers, so sums
// are exact and no order of summation changes a token.
#include <algorithm>

#include "common.cuh"

namespace bcm {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr float kInf = __builtin_huge_valf();
constexpr float kOne = 1099511627776.0f;   // 2^40

typedef unsigned long long u64;

// Order-preserving key of s <= 0 (larger s, larger key); 0 for -inf.
__device__ __forceinline__ uint32_t key_of(float s) { return 0x7f800000u - __float_as_uint(-s); }
__device__ __forceinline__ float from_key(uint32_t k) { return -__uint_as_float(0x7f800000u - k); }

template <typename T>
__device__ __forceinline__ float scaled(const T* x, int64_t v, float top, float it) {
    const float l = to_f32<T>(x[v]);
    const float s = l == top ? 0.0f : (l - top) * it;
    return s <= 0.0f ? fabsf(s) * -1.0f : -kInf;   // -0 for 0; NaN to -inf
}

__device__ __forceinline__ float rel_weight(float s) { return expf(s); }
__device__ __forceinline__ u64 weight_of(float e) { return (u64)(e * kOne); }

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

// The largest key whose keys-at-or-above hold more than `skip` of what count
// (or, BY_WEIGHT, weight) adds up over the tokens with key > lo_key, or key ==
// lo_key (whose tokens count `lo_ties` times).  above: what lies above that key.
template <typename T, bool BY_WEIGHT>
__device__ uint32_t select_key(const T* x, int64_t V, float top, float it, u64 skip, uint32_t lo_key, u64* above_out, u64* hist) {
    uint32_t prefix = 0, mask = 0;
    u64 above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int k = threadIdx.x; k < 256; k += kThreads) hist[k] = 0;
        __syncthreads();
        for (int64_t v = threadIdx.x; v < V; v += kThreads) {
            const float s = scaled<T>(x, v, top, it);
            const uint32_t key = key_of(s);
            if (key == 0u || key < lo_key || (key & mask) != prefix) continue;
            atomicAdd(&hist[(key >> shift) & 255u], BY_WEIGHT ? weight_of(rel_weight(s)) : 1ull);
        }
        __syncthreads();
        int digit = 255;
        for (; digit > 0; --digit) {
            if (above + hist[digit] > skip) break;
            above += hist[digit];
        }
        prefix |= (uint32_t)digit << shift;
        mask |= 255u << shift;
    }
    __syncthreads();
    *above_out = above;
    return prefix;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
sample_kernel(const bcm_sample_args a) {
    __shared__ u64 red[kWarps];
    __shared__ u64 hist[256];
    __shared__ float fred[kWarps];
    __shared__ int64_t s_cut;
    const int64_t b = blockIdx.x;
    const int64_t V = a.vocab;
    const T* x = static_cast<const T*>(a.logits) + b * a.logits_stride;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float temp = a.temperature ? a.temperature[b] : a.temperature_all;
    const float inv = 1.0f / temp;
    const bool warm = temp > 0.0f && inv < kInf;
    const float it = warm ? inv : 1.0f;
    int64_t k = warm ? (a.top_k ? a.top_k[b] : a.top_k_all) : 1;
    if (k <= 0 || k > V) k = V;
    const float p = a.top_p ? a.top_p[b] : a.top_p_all;
    const float mp = a.min_p ? a.min_p[b] : a.min_p_all;
    const float least = mp > 0.0f ? fminf(mp, 1.0f) : 0.0f;

    float top = -kInf;
    for (int64_t v = threadIdx.x; v < V; v += kThreads) top = fmaxf(top, to_f32<T>(x[v]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
    if (lane == 0) fred[warp] = top;
    __syncthreads();
    for (int j = 0; j < kWarps; ++j) top = fmaxf(top, fred[j]);
    if (top == -kInf) {
        if (threadIdx.x == 0) {
            a.tokens[b] = -1;
            a.logprob[b] = -kInf;
        }
        return;
    }
    u64 n_valid = 0;
    for (int64_t v = threadIdx.x; v < V; v += kThreads) n_valid += key_of(scaled<T>(x, v, top, it)) != 0u;
    n_valid = block_sum_u<u64>(n_valid, red);
    // kept so far: key > cut, or key == cut and among the first `ties` of its equals by index
    uint32_t cut = 1u;
    u64 ties = (u64)V;
    if ((u64)k < n_valid) {
        u64 above;
        cut = select_key<T, false>(x, V, top, it, (u64)k - 1, 1u, &above, hist);
        ties = (u64)k - above;
    }
    if (p < 1.0f) {
        u64 sum = 0, at_cut = 0;
        for (int64_t v = threadIdx.x; v < V; v += kThreads) {
            const float s = scaled<T>(x, v, top, it);
            const uint32_t key = key_of(s);
            if (key > cut) sum += weight_of(rel_weight(s));
            else if (key == cut) ++at_cut;
        }
        sum = block_sum_u<u64>(sum, red);
        at_cut = block_sum_u<u64>(at_cut, red);
        const u64 w_cut = weight_of(rel_weight(from_key(cut)));
        const u64 total = sum + (at_cut < ties ? at_cut : ties) * (cut == 1u ? 0ull : w_cut);
        const double lim = ceil((double)p * (double)total);
        const u64 most = lim >= 1.0 ? (u64)lim : 1ull;
        // the last kept token in descending order is the one holding weight unit most - 1
        u64 above;
        const uint32_t pk = select_key<T, true>(x, V, top, it, most - 1, cut, &above, hist);
        const u64 wp = weight_of(rel_weight(from_key(pk)));
        const u64 pt = wp ? (most - above + wp - 1) / wp : (u64)V;
        if (pk > cut) {
            cut = pk;
            ties = pt;
        } else if (pt < ties) {
            ties = pt;
        }
    }
    // the index of the last kept token among those at the cut
    const int64_t seg = ((V + kWarps - 1) / kWarps + 31) / 32 * 32;
    const int64_t lo = warp * seg < V ? warp * seg : V, hi = lo + seg < V ? lo + seg : V;
    if (threadIdx.x == 0) s_cut = V;
    u64 mine = 0;
    for (int64_t v = lo + lane; v < hi; v += 32) mine += key_of(scaled<T>(x, v, top, it)) == cut;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(kFull, mine, o);
    __syncthreads();
    if (lane == 0) red[warp] = mine;
    __syncthreads();
    u64 before = 0;
    for (int j = 0; j < warp; ++j) before += red[j];
    if (before < ties && before + mine >= ties) {
        for (int64_t v0 = lo; v0 < hi; v0 += 32) {
            const int64_t v = v0 + lane;
            const bool at = v < hi && key_of(scaled<T>(x, v, top, it)) == cut;
            const unsigned m = __ballot_sync(kFull, at);
            if (at && before + __popc(m & ((2u << lane) - 1u)) == ties) s_cut = v;
            before += __popc(m);
        }
    }
    __syncthreads();
    const int64_t last = s_cut;
    // integer prefix sums in index order: one contiguous segment per warp
    auto kept = [&](int64_t v, float& s) -> u64 {
        s = scaled<T>(x, v, top, it);
        const uint32_t key = key_of(s);
        if (key < cut || (key == cut && v > last)) return 0ull;
        const float e = rel_weight(s);
        return e >= least ? weight_of(e) : 0ull;
    };
    u64 sum = 0;
    for (int64_t v = lo + lane; v < hi; v += 32) {
        float s;
        sum += kept(v, s);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
    __syncthreads();
    if (lane == 0) red[warp] = sum;
    __syncthreads();
    u64 total = 0, start = 0;
    for (int j = 0; j < kWarps; ++j) {
        if (j == warp) start = total;
        total += red[j];
    }
    const double want = floor((double)a.u[b] * (double)total);
    u64 target = want > 0.0 ? (u64)want : 0ull;
    if (target >= total) target = total - 1;
    if (start <= target && target < start + sum) {
        for (int64_t v0 = lo; v0 < hi; v0 += 32) {
            const int64_t v = v0 + lane;
            float s = 0.0f;
            const u64 w = v < hi ? kept(v, s) : 0ull;
            const u64 run = warp_inclusive_sum<u64>(w);
            if (start + run > target && start + run - w <= target) {
                a.tokens[b] = v;
                a.logprob[b] = s - (float)log((double)total / (double)kOne);
            }
            start += __shfl_sync(kFull, run, 31);
            if (start > target) break;
        }
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
    return dispatch_dtype(a->dtype, [&](auto tag) -> bcm_status {
        using T = decltype(tag);
        sample_kernel<T><<<(unsigned)a->batch, kThreads, 0, stream>>>(*a);
        BCM_LAUNCH_CHECK();
        return BCM_OK;
    });
}
