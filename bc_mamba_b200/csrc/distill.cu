// distill.cu — distillation loss on a teacher's top logits, and its gradient.
//
// Row t: p = softmax over the row's teacher logits q/tau (entries whose token
// id lies outside [0, V) or whose logit is -inf are absent), s = softmax(z/tau)
// over the whole vocabulary:
//   loss = w tau^2 sum_k p_k (ln p_k - ln s_{id_k}),
//   dz_v = g w tau (s_v - sum_{k: id_k = v} p_k).
// A row without teacher entries, or with w = 0, has loss 0 and gradient 0
// whatever its logits hold.
#include <algorithm>

#include "common.cuh"

namespace bcm {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr float kInf = __builtin_huge_valf();

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

// Block reductions: every thread gets the result; red holds kWarps floats.
__device__ float block_max(float v, float* red) {
    v = warp_max(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
    for (int k = 1; k < kWarps; ++k) v = fmaxf(v, red[k]);
    return v;
}
__device__ float block_sum(float v, float* red) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
    for (int k = 1; k < kWarps; ++k) v += red[k];
    return v;
}

__device__ __forceinline__ int64_t load_id(const void* ids, int wide, int64_t k) {
    return wide ? static_cast<const int64_t*>(ids)[k] : (int64_t) static_cast<const int32_t*>(ids)[k];
}

// The row's teacher distribution: s_id[k] (-1: absent) and s_p[k]; returns the
// logarithm of the normaliser plus the maximum, -inf for an empty row.
template <typename TQ>
__device__ float teacher_row(const TQ* q, const void* ids, int wide, int64_t off, int K, int64_t V, float itau, int* s_id,
                             float* s_p, float* red) {
    float top = -kInf;
    for (int k = threadIdx.x; k < K; k += kThreads) {
        const int64_t id = load_id(ids, wide, off + k);
        const float v = to_f32<TQ>(q[k]) * itau;
        const bool there = id >= 0 && id < V && v != -kInf;
        s_id[k] = there ? (int)id : -1;
        s_p[k] = v;
        if (there) top = v > top || isnan(v) ? v : top;
    }
    float any = block_sum(isnan(top) ? 1.0f : 0.0f, red);
    top = block_max(top, red);
    if (any > 0.0f) top = __int_as_float(0x7fffffff);
    if (top == -kInf) return -kInf;
    float sum = 0.0f;
    for (int k = threadIdx.x; k < K; k += kThreads)
        if (s_id[k] >= 0) sum += expf(s_p[k] - top);
    sum = block_sum(sum, red);
    const float lg = logf(sum);
    for (int k = threadIdx.x; k < K; k += kThreads) s_p[k] = s_id[k] >= 0 ? expf(s_p[k] - top) / sum : 0.0f;
    __syncthreads();
    return top + lg;
}

// stats[2t] = max of z/tau, stats[2t+1] = sum of exp(z/tau - max).
template <typename T>
__device__ float2 row_stats(const T* z, int64_t V, float itau, float* red) {
    float m = -kInf, s = 0.0f;
    for (int64_t v = threadIdx.x; v < V; v += kThreads) {
        const float x = to_f32<T>(z[v]) * itau;
        if (x > m) {
            s = s * expf(m - x) + 1.0f;
            m = x;
        } else if (x != -kInf) {
            s += expf(x - m);
        }
    }
    const float top = block_max(m, red);
    s = block_sum(m == top ? s : (m == -kInf && !isnan(s) ? 0.0f : s * expf(m - top)), red);
    return make_float2(top, s);
}

template <typename T, typename TQ, bool FWD, bool GRAD>
__global__ void __launch_bounds__(kThreads)
distill_kernel(const T* __restrict__ z, int64_t z_stride, const TQ* __restrict__ q, const void* __restrict__ ids, int wide,
               int64_t V, int K, const float* __restrict__ weight, float itau, float tau, float* __restrict__ loss,
               float2* __restrict__ stats, const float* __restrict__ dloss, T* __restrict__ dz) {
    extern __shared__ float smem[];
    __shared__ float red[kWarps];
    int* s_id = reinterpret_cast<int*>(smem);
    float* s_p = smem + K;
    const int64_t t = blockIdx.x;
    const T* zr = z + t * z_stride;
    T* dr = GRAD ? dz + t * V : nullptr;
    const float w = weight ? weight[t] : 1.0f;
    const float lse_q = w != 0.0f ? teacher_row<TQ>(q + t * K, ids, wide, t * K, K, V, itau, s_id, s_p, red) : -kInf;
    if (lse_q == -kInf) {
        if (FWD && threadIdx.x == 0) {
            loss[t] = 0.0f;
            stats[t] = make_float2(0.0f, 1.0f);
        }
        if (GRAD)
            for (int64_t v = threadIdx.x; v < V; v += kThreads) dr[v] = from_f32<T>(0.0f);
        return;
    }
    const float2 st = FWD ? row_stats<T>(zr, V, itau, red) : stats[t];
    if (FWD) {
        const float lse = st.x + logf(st.y);
        float sum = 0.0f;
        for (int k = threadIdx.x; k < K; k += kThreads)
            if (s_p[k] > 0.0f || isnan(s_p[k]))
                sum += s_p[k] * (to_f32<TQ>(q[t * K + k]) * itau - lse_q - to_f32<T>(zr[s_id[k]]) * itau + lse);
        sum = block_sum(sum, red);
        if (threadIdx.x == 0) {
            loss[t] = w * tau * tau * sum;
            stats[t] = st;
        }
    }
    if (GRAD) {
        const float scale = (dloss ? dloss[t] : 1.0f) * w * tau, inv = 1.0f / st.y;
        for (int64_t v = threadIdx.x; v < V; v += kThreads)
            dr[v] = from_f32<T>(expf(to_f32<T>(zr[v]) * itau - st.x) * inv * scale);
        __syncthreads();
        for (int k = threadIdx.x; k < K; k += kThreads) {
            const int id = s_id[k];
            if (id < 0) continue;
            bool first = true;
            float p = s_p[k];
            for (int j = 0; j < K; ++j)
                if (j != k && s_id[j] == id) {
                    if (j < k) { first = false; break; }
                    p += s_p[j];
                }
            if (first) dr[id] = from_f32<T>((expf(to_f32<T>(zr[id]) * itau - st.x) * inv - p) * scale);
        }
    }
}

bcm_status distill_validate(const bcm_distill_args* a, const char* what) {
    BCM_REQUIRE(a != nullptr, "%s: null arguments", what);
    BCM_REQUIRE(dtype_ok(a->dtype) && dtype_ok(a->teacher_dtype), "%s: unsupported dtype", what);
    BCM_REQUIRE(a->rows >= 0 && a->rows < (1ll << 31) && a->vocab >= 1 && a->vocab < (1ll << 31), "%s: bad sizes", what);
    BCM_REQUIRE(a->k >= 1 && a->k <= BCM_DISTILL_MAX_K, "%s: k must be in [1, %d]", what, BCM_DISTILL_MAX_K);
    BCM_REQUIRE(a->temperature > 0.0f && a->temperature < kInf, "%s: temperature must be positive and finite", what);
    BCM_REQUIRE(a->rows == 0 || (a->logits && a->teacher_logits && a->teacher_ids && a->loss && a->stats),
                "%s: null pointer", what);
    return BCM_OK;
}

template <bool FWD, bool GRAD>
bcm_status distill_launch(const bcm_distill_args* a, cudaStream_t stream) {
    return dispatch_dtype(a->dtype, [&](auto tag) -> bcm_status {
        using T = decltype(tag);
        return dispatch_dtype(a->teacher_dtype, [&](auto qtag) -> bcm_status {
            using TQ = decltype(qtag);
            distill_kernel<T, TQ, FWD, GRAD><<<(unsigned)a->rows, kThreads, (size_t)a->k * 8, stream>>>(
                static_cast<const T*>(a->logits), a->logits_stride, static_cast<const TQ*>(a->teacher_logits), a->teacher_ids,
                a->ids_are_int64, a->vocab, (int)a->k, a->weight, 1.0f / a->temperature, a->temperature, a->loss,
                reinterpret_cast<float2*>(a->stats), a->dloss, static_cast<T*>(a->dlogits));
            BCM_LAUNCH_CHECK();
            return BCM_OK;
        });
    });
}

}  // namespace
}  // namespace bcm

using namespace bcm;

extern "C" bcm_status bcm_distill_fwd(const bcm_distill_args* a, cudaStream_t stream) {
    clear_error();
    if (bcm_status st = distill_validate(a, "distill_fwd"); st != BCM_OK) return st;
    if (a->rows == 0) return BCM_OK;
    return distill_launch<true, false>(a, stream);
}

extern "C" bcm_status bcm_distill_bwd(const bcm_distill_args* a, cudaStream_t stream) {
    clear_error();
    if (bcm_status st = distill_validate(a, "distill_bwd"); st != BCM_OK) return st;
    if (a->rows == 0) return BCM_OK;
    BCM_REQUIRE(a->dlogits && a->dloss, "distill_bwd: null pointer");
    return distill_launch<false, true>(a, stream);
}

extern "C" bcm_status bcm_distill_fwd_grad(const bcm_distill_args* a, cudaStream_t stream) {
    clear_error();
    if (bcm_status st = distill_validate(a, "distill_fwd_grad"); st != BCM_OK) return st;
    if (a->rows == 0) return BCM_OK;
    BCM_REQUIRE(a->dlogits, "distill_fwd_grad: null pointer");
    return distill_launch<true, true>(a, stream);
}
