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
#include <cstring>

#include "common.cuh"

namespace bcm {
namespace {

// C blocks of a cluster share a row, in 16-byte granules (rows may start anywhere).
// The forward is one pass with a running maximum and sum; the backward one pass that
// writes; loss and gradient in one call are both by the same block, the second from
// L2 as far as it holds.  (8192 x 131072 bf16: clusters of four, which leave few
// enough rows in flight for L2, take 1110 against 991 us, since a block's fixed work -
// teacher, reductions, the places written again - then recurs for every part.  A row
// kept in a cluster's shared memory in between was only measured with granules loaded
// straight into registers, 1545 us, not with the rings below.)
// Granules arrive by cyclic cp.async buffers of each thread's own.  The teacher's
// entries and the loss are the work of a warp of their own meanwhile; the K places
// of the gradient that they touch are written again at the end.
constexpr int kMaxCluster = 8;
constexpr int kBatch = 4, kStages = 3;           // granules a thread takes at a time; batches in flight or in use
constexpr int kShortRow = 24 * 1024;             // bytes of a row up to which a block has 64 threads, not 256
constexpr float kInf = __builtin_huge_valf();
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2_(float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }

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

__device__ __forceinline__ int64_t load_id(const void* ids, int wide, int64_t k) {
    return wide ? static_cast<const int64_t*>(ids)[k] : (int64_t) static_cast<const int32_t*>(ids)[k];
}

__host__ __device__ __forceinline__ int list_len(int K) { return (K + 3) / 4 * 4; }

// The row's teacher distribution, by one warp: s_id[k] (-1: absent, up to a multiple of 4), s_p[k] and the student's
// logit s_z[k].  Returns its largest logit (-inf for an empty row) and the logarithm of the sum of exp((q - top) / tau).
// The difference comes before the factor 1 / tau: an offset of the row loses no digits, and no finite logit becomes -inf.
struct Teacher {
    float top, lsum;
};
template <typename T, typename TQ>
__device__ Teacher teacher_row(const T* z, const TQ* q, const void* ids, int wide, int64_t off, int K, int64_t V, float itau, int* s_id,
                               float* s_p, float* s_z) {
    const int lane = threadIdx.x & 31;
    float top = -kInf;
    bool nan = false;
    if (lane < 4 && K + lane < list_len(K)) s_id[K + lane] = -1;
    for (int k = lane; k < K; k += 32) {
        const int64_t id = load_id(ids, wide, off + k);
        const float v = to_f32<TQ>(q[k]);
        const bool there = id >= 0 && id < V && v != -kInf;
        s_id[k] = there ? (int)id : -1;
        s_p[k] = v;
        s_z[k] = there ? to_f32<T>(z[id]) : 0.0f;
        if (there) {
            top = fmaxf(top, v);
            nan |= isnan(v);
        }
    }
    top = warp_max(top);
    if (__any_sync(kFull, nan)) top = __int_as_float(0x7fffffff);
    if (top == -kInf) return {-kInf, 0.0f};
    float sum = 0.0f;
    for (int k = lane; k < K; k += 32)
        if (s_id[k] >= 0) sum += expf((s_p[k] - top) * itau);
    sum = warp_sum(sum);
    for (int k = lane; k < K; k += 32) s_p[k] = s_id[k] >= 0 ? expf((s_p[k] - top) * itau) / sum : 0.0f;
    return {top, logf(sum)};
}

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
    // exp2((f - m) c): the difference first, so that large logits lose nothing; packed, two elements an instruction
    __device__ __forceinline__ void exponentials(float m, float c) {
        const float2 nm = m == -kInf ? make_float2(0.0f, 0.0f) : make_float2(-m, -m), cc = make_float2(c, c);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            const float2 v = __fmul2_rn(__fadd2_rn(make_float2(f[e], f[e + 1]), nm), cc);
            f[e] = ex2_(v.x);
            f[e + 1] = ex2_(v.y);
        }
    }
    __device__ __forceinline__ uint4 pack() const {
        T t[N];
        uint4 w;
#pragma unroll
        for (int e = 0; e < N; ++e) t[e] = from_f32<T>(f[e]);
        memcpy(&w, t, 16);
        return w;
    }
};

// A row of V elements at x as 16-byte granules: the first holds `shift` foreign elements in front.
template <typename T>
struct RowOf {
    static constexpr int N = 16 / (int)sizeof(T);
    const uint4* at;
    int shift;
    int64_t grans;
    __device__ __forceinline__ RowOf(const T* x, int64_t V)
        : at(reinterpret_cast<const uint4*>((uintptr_t)x & ~(uintptr_t)15)), shift((int)((uintptr_t)x & 15) / (int)sizeof(T)),
          grans((shift + V + N - 1) / N) {}
};

// Sum of exp2(c (f - m)) with its maximum m; c > 0 is log2(e) / tau.
struct Soft {
    float m, s;
    __device__ __forceinline__ void join(float m2, float s2, float c) {
        const float top = fmaxf(m, m2);
        if (top == -kInf) {
            s += s2;                             // (0, or NaN)
            return;
        }
        s = (m == top ? s : (m == -kInf && s == 0.0f ? 0.0f : s * ex2_((m - top) * c))) +
            (m2 == top ? s2 : (m2 == -kInf && s2 == 0.0f ? 0.0f : s2 * ex2_((m2 - top) * c)));
        m = top;
    }
};

__device__ __forceinline__ uint32_t remote(const void* p, int rank) {
    uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Granules g, g + kThreads, ... of a thread, in order.
template <int kThreads>
struct Feed {
    uint4* ring;
    const uint4* at;
    int64_t end;
    __device__ __forceinline__ Feed(uint4* room, const uint4* from, int64_t begin, int64_t end_) : ring(room + threadIdx.x), at(from), end(end_) {
#pragma unroll
        for (int k = 0; k < kStages - 1; ++k) issue(begin + threadIdx.x + (int64_t)k * kBatch * kThreads, k);
    }
    __device__ __forceinline__ void issue(int64_t g, int stage) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
            if (g + j * kThreads < end)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(ring + (stage * kBatch + j) * kThreads)),
                             "l"(at + g + j * kThreads)
                             : "memory");
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    // f(granule, its 16 bytes) for every granule of the thread from g on
    template <typename F>
    __device__ __forceinline__ void run(int64_t g, F&& f) {
        int stage = 0;
        for (; g < end; g += kBatch * kThreads) {
            issue(g + (int64_t)(kStages - 1) * kBatch * kThreads, stage == 0 ? kStages - 1 : stage - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
                if (g + j * kThreads < end) f(g + j * kThreads, ring[(stage * kBatch + j) * kThreads]);
            stage = stage == kStages - 1 ? 0 : stage + 1;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
};

// 8192 x 131072 bf16: forward 407 us (5.3 TB/s), backward 674 us (6.4 TB/s of reads and writes, memory's rate), both in one call 991 us;
// 4096 x 50257 bf16: forward 106 us, bound by instructions (issue slots 78 % busy), backward 137 us (6.0 TB/s), one call 188 us.
template <typename T, typename TQ, bool FWD, bool GRAD, int kThreads>
__global__ void __launch_bounds__(kThreads + 32, kThreads == 64 ? 12 : 4)
distill_kernel(const __grid_constant__ bcm_distill_args a, int C) {
    constexpr int kWarps = kThreads / 32;        // that stream the row; one more is the teacher's
    using Gr = Granule<T>;
    constexpr int N = Gr::N;
    extern __shared__ __align__(16) char dyn[];
    __shared__ float wm[kWarps], ws[kWarps];
    __shared__ float2 parts[kMaxCluster];
    __shared__ Teacher s_teacher;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, K = (int)a.k;
    int* s_id = reinterpret_cast<int*>(dyn);
    float *s_p = reinterpret_cast<float*>(dyn) + list_len(K), *s_z = s_p + list_len(K);
    uint4* ring = reinterpret_cast<uint4*>(s_z + list_len(K));
    const bool teacher = warp == kWarps;
    const int rank = blockIdx.x % C;
    const int64_t t = blockIdx.x / C, V = a.vocab;
    const T* z = static_cast<const T*>(a.logits) + t * a.logits_stride;
    const TQ* q = static_cast<const TQ*>(a.teacher_logits) + t * K;
    const float w = a.weight ? a.weight[t] : 1.0f;
    const float tau = a.temperature, itau = 1.0f / tau, c = kLog2e * itau;
    const RowOf<T> row(z, V);
    const int64_t per = (row.grans + C - 1) / C, g0 = rank * per, g1 = min(g0 + per, row.grans);
    auto trim = [&](int64_t g, Gr& x) {          // elements outside the row
        if (g == 0 || g == row.grans - 1)
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (g * N + e < row.shift || g * N + e - row.shift >= V) x.f[e] = -kInf;
    };
    bool live = w != 0.0f;
    Soft soft = {-kInf, 0.0f};
    if (!FWD) {
        soft = {a.stats[2 * t], a.stats[2 * t + 1]};
        live = soft.s >= 0.0f || isnan(soft.s);  // (the forward marks rows without a target)
    }
    if (live) {
        if (FWD) {
            if (teacher) {
                const Teacher l = teacher_row<T, TQ>(z, q, a.teacher_ids, a.ids_are_int64, t * K, K, V, itau, s_id, s_p, s_z);
                if (lane == 0) s_teacher = l;
            } else {
                Feed<kThreads> feed(ring, row.at, g0, g1);
                feed.run(g0 + tid, [&](int64_t g, uint4 in) {
                    Gr x;
                    x.unpack(in);
                    trim(g, x);
                    float top = x.f[0];
#pragma unroll
                    for (int e = 1; e < N; ++e) top = fmaxf(top, x.f[e]);
                    if (top > soft.m) {
                        if (soft.m != -kInf) soft.s *= ex2_((soft.m - top) * c);
                        soft.m = top;
                    }
                    x.exponentials(soft.m, c);
#pragma unroll
                    for (int step = 1; step < N; step <<= 1)
#pragma unroll
                        for (int e = 0; e < N; e += 2 * step) x.f[e] += x.f[e + step];
                    soft.s += x.f[0];
                });
#pragma unroll
                for (int o = 16; o > 0; o >>= 1)
                    soft.join(__shfl_xor_sync(kFull, soft.m, o), __shfl_xor_sync(kFull, soft.s, o), c);
                if (lane == 0) {
                    wm[warp] = soft.m;
                    ws[warp] = soft.s;
                }
            }
            __syncthreads();
            soft = {wm[0], ws[0]};
            for (int k = 1; k < kWarps; ++k) soft.join(wm[k], ws[k], c);
            if (C > 1) {
                cluster_sync();                  // every block runs before its shared memory is written to
                if (tid < C) {
                    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(remote(&parts[rank], tid)), "f"(soft.m), "f"(soft.s) : "memory");
                }
                cluster_sync();
                soft = {parts[0].x, parts[0].y};
                for (int k = 1; k < C; ++k) soft.join(parts[k].x, parts[k].y, c);
            }
            live = s_teacher.top != -kInf;
            if (rank == 0 && teacher) {
                // tau (ln p - ln s), both from differences to their maxima: logits with a common offset lose no digits, and
                // nothing on the way is larger than the difference of a logit and its maximum
                const float lsum = tau * (logf(soft.s) - s_teacher.lsum), top_q = s_teacher.top;
                float sum = 0.0f;
                if (live)
                    for (int k = lane; k < K; k += 32)
                        if (s_p[k] > 0.0f || isnan(s_p[k])) sum += s_p[k] * ((to_f32<TQ>(q[k]) - top_q) + (soft.m - s_z[k]) + lsum);
                sum = warp_sum(sum);
                if (lane == 0) {
                    a.loss[t] = live ? w * tau * sum : 0.0f;
                    a.stats[2 * t] = live ? soft.m : 0.0f;
                    a.stats[2 * t + 1] = live ? soft.s : -1.0f;
                }
            }
        }
    } else if (FWD && rank == 0 && tid == 0) {
        a.loss[t] = 0.0f;
        a.stats[2 * t] = 0.0f;
        a.stats[2 * t + 1] = -1.0f;
    }
    if (!GRAD) return;
    // the gradient by granules of its own row, which may lie differently from the logits'
    T* d = static_cast<T*>(a.dlogits) + t * V;
    const RowOf<T> out(d, V);
    const bool alike = out.shift == row.shift;
    const int64_t oper = alike ? per : (out.grans + C - 1) / C, o0 = rank * oper, o1 = min(o0 + oper, out.grans);
    const float scale = live ? (a.dloss ? a.dloss[t] : 1.0f) * w * tau : 0.0f, k_out = scale / soft.s;
    auto put = [&](int64_t g, const Gr& x) {
        const int64_t v0 = g * N - out.shift;
        if (v0 >= 0 && v0 + N <= V) {
            __stcs(const_cast<uint4*>(out.at) + g, x.pack());
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (v0 + e >= 0 && v0 + e < V) d[v0 + e] = from_f32<T>(x.f[e]);
        }
    };
    auto gradient = [&](Gr& x) {
        x.exponentials(soft.m, c);
        const float2 k2 = make_float2(k_out, k_out);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
            const float2 v = __fmul2_rn(make_float2(x.f[e], x.f[e + 1]), k2);
            x.f[e] = v.x;
            x.f[e + 1] = v.y;
        }
    };
    if (live && alike) {
        if (teacher) {
            if (!FWD) teacher_row<T, TQ>(z, q, a.teacher_ids, a.ids_are_int64, t * K, K, V, itau, s_id, s_p, s_z);
        } else {
            Feed<kThreads> feed(ring, row.at, o0, o1);
            feed.run(o0 + tid, [&](int64_t g, uint4 in) {
            Gr x;
            x.unpack(in);
            gradient(x);
            put(g, x);
        });
        }
    } else {
        // Rows without a target, and logits whose rows lie differently on 16 bytes than the gradient's (columns of a wider
        // buffer): element by element, 4096 x 50257 of 50304 bf16 backward 270 us against 137.
        if (!FWD && live && teacher) teacher_row<T, TQ>(z, q, a.teacher_ids, a.ids_are_int64, t * K, K, V, itau, s_id, s_p, s_z);
        for (int64_t g = o0 + tid; g < o1; g += kThreads + 32) {
            const int64_t v0 = g * N - out.shift;
            Gr x;
#pragma unroll
            for (int e = 0; e < N; ++e) x.f[e] = live && v0 + e >= 0 && v0 + e < V ? to_f32<T>(z[v0 + e]) : 0.0f;
            if (live) gradient(x);
            put(g, x);
        }
    }
    if (!live) return;
    // the teacher's tokens among this block's: the first entry of a token takes its later ones' shares too
    __syncthreads();
    for (int k = tid; k < K; k += kThreads + 32) {
        const int id = s_id[k];
        const int64_t g = ((int64_t)id + out.shift) / N;
        if (id < 0 || g < o0 || g >= o1) continue;
        bool first = true;
        float p = s_p[k];
        for (int j = 0; j < K; j += 4) {
            const int4 at = reinterpret_cast<const int4*>(s_id)[j / 4];
            if (at.x != id && at.y != id && at.z != id && at.w != id) continue;
            const int who[4] = {at.x, at.y, at.z, at.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (who[e] == id && j + e != k) {
                    first = first && j + e > k;
                    p += s_p[j + e];
                }
        }
        if (first) d[id] = from_f32<T>((ex2_((s_z[k] - soft.m) * c) / soft.s - p) * scale);
    }
}

bcm_status distill_validate(const bcm_distill_args* a, const char* what, bool fwd) {
    BCM_REQUIRE(a != nullptr, "%s: null arguments", what);
    BCM_REQUIRE(dtype_ok(a->dtype) && dtype_ok(a->teacher_dtype), "%s: unsupported dtype", what);
    BCM_REQUIRE(a->rows >= 0 && a->rows < (1ll << 31) && a->vocab >= 1 && a->vocab < (1ll << 31), "%s: bad sizes", what);
    BCM_REQUIRE(a->k >= 1 && a->k <= BCM_DISTILL_MAX_K, "%s: k must be in [1, %d]", what, BCM_DISTILL_MAX_K);
    // (of a smaller one every exponent would be a difference, 0 among them, times infinity)
    BCM_REQUIRE(a->temperature > 0.0f && a->temperature < kInf && kLog2e / a->temperature < kInf,
                "%s: temperature must be positive and finite, and its reciprocal a float32", what);
    BCM_REQUIRE(a->rows == 0 || (a->logits && a->teacher_logits && a->teacher_ids && (a->loss || !fwd) && a->stats),
                "%s: null pointer", what);
    return BCM_OK;
}

template <typename F>
bcm_status distill_launch_as(F* kernel, const bcm_distill_args* a, int threads, cudaStream_t stream) {
    // one block a row, and more where the rows leave SMs without a block (down to slices of 8 KB)
    const int64_t bytes = a->vocab * (int64_t)dtype_size(a->dtype);
    int C = 1;
    while (C < kMaxCluster && a->rows * C < 2 * (int64_t)sm_count() && bytes / C > 8192) C *= 2;
    BCM_REQUIRE(a->rows * C < (1ll << 31), "distill: too many rows");
    const int smem = list_len((int)a->k) * 12 + kStages * kBatch * threads * 16;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a->rows * C));
    cfg.blockDim = dim3((unsigned)threads + 32);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)C;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = C > 1 ? 1 : 0;
    BCM_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    BCM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, *a, C));
    return BCM_OK;
}

template <bool FWD, bool GRAD>
bcm_status distill_launch(const bcm_distill_args* a, cudaStream_t stream) {
    const bool small = a->vocab * (int64_t)dtype_size(a->dtype) <= kShortRow;
    return dispatch_dtype(a->dtype, [&](auto tag) -> bcm_status {
        using T = decltype(tag);
        return dispatch_dtype(a->teacher_dtype, [&](auto qtag) -> bcm_status {
            using TQ = decltype(qtag);
            return small ? distill_launch_as(distill_kernel<T, TQ, FWD, GRAD, 64>, a, 64, stream)
                         : distill_launch_as(distill_kernel<T, TQ, FWD, GRAD, 256>, a, 256, stream);
        });
    });
}

}  // namespace
}  // namespace bcm

using namespace bcm;

extern "C" bcm_status bcm_distill_fwd(const bcm_distill_args* a, cudaStream_t stream) {
    clear_error();
    if (bcm_status st = distill_validate(a, "distill_fwd", true); st != BCM_OK) return st;
    if (a->rows == 0) return BCM_OK;
    return distill_launch<true, false>(a, stream);
}

extern "C" bcm_status bcm_distill_bwd(const bcm_distill_args* a, cudaStream_t stream) {
    clear_error();
    if (bcm_status st = distill_validate(a, "distill_bwd", false); st != BCM_OK) return st;
    if (a->rows == 0) return BCM_OK;
    BCM_REQUIRE(a->dlogits && a->dloss, "distill_bwd: null pointer");
    return distill_launch<false, true>(a, stream);
}

extern "C" bcm_status bcm_distill_fwd_grad(const bcm_distill_args* a, cudaStream_t stream) {
    clear_error();
    if (bcm_status st = distill_validate(a, "distill_fwd_grad", true); st != BCM_OK) return st;
    if (a->rows == 0) return BCM_OK;
    BCM_REQUIRE(a->dlogits, "distill_fwd_grad: null pointer");
    return distill_launch<true, true>(a, stream);
}
