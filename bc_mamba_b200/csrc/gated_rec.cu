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

#include "common.cuh"

namespace bcm {
namespace {

__device__ __forceinline__ float sigmoid_(float v) { return 1.0f / (1.0f + expf(-v)); }
__device__ __forceinline__ float softplus_(float v) { return v > 20.0f ? v : log1pf(expf(v)); }

struct Gates {
    float sr, si, u, a, m;
};

__device__ __forceinline__ Gates gates(float r, float i, float cs) {
    Gates g;
    g.sr = sigmoid_(r);
    g.si = sigmoid_(i);
    g.u = -cs * g.sr;
    const float w = expm1f(g.u);       // a - 1 without cancellation
    g.a = 1.0f + w;
    g.m = sqrtf(-w * (2.0f + w));      // 1 - a^2
    return g;
}

struct RecPtr {
    const void* x; const void* r; const void* i; const void* dy;
    int64_t xb, xt, rb, rt, ib, it, gb, gt;
};

// Rows of sequence b: dense [b*L, (b+1)*L); packed [cu[b], cu[b+1]) within [0, L).
__device__ __forceinline__ void rows_of(const int32_t* cu, int64_t b, int64_t L, int64_t& t0, int64_t& n) {
    if (cu == nullptr) {
        t0 = 0;
        n = L;
        return;
    }
    const int64_t lo = cu[b], hi = cu[b + 1];
    t0 = lo < 0 ? 0 : (lo > L ? L : lo);
    const int64_t e = hi < t0 ? t0 : (hi > L ? L : hi);
    n = e - t0;
}

template <typename T>
__global__ void rec_fwd_kernel(RecPtr p, const int32_t* __restrict__ cu, int64_t L, int64_t D, const float* __restrict__ lam,
                               float c, const float* __restrict__ h0, T* __restrict__ y, float* __restrict__ h_last,
                               float* __restrict__ hs) {
    const int64_t d = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t b = blockIdx.y;
    if (d >= D) return;
    int64_t t0, n;
    rows_of(cu, b, L, t0, n);
    const T* x = static_cast<const T*>(p.x) + (cu ? 0 : b * p.xb) + t0 * p.xt + d;
    const T* r = static_cast<const T*>(p.r) + (cu ? 0 : b * p.rb) + t0 * p.rt + d;
    const T* i = static_cast<const T*>(p.i) + (cu ? 0 : b * p.ib) + t0 * p.it + d;
    const int64_t o = ((cu ? 0 : b * L) + t0) * D + d;
    const float cs = c * softplus_(lam[d]);
    float h = h0 ? h0[b * D + d] : 0.0f;
    for (int64_t t = 0; t < n; ++t) {
        const Gates g = gates(to_f32<T>(r[t * p.rt]), to_f32<T>(i[t * p.it]), cs);
        if (hs) hs[o + t * D] = h;
        h = fmaf(g.a, h, g.m * g.si * to_f32<T>(x[t * p.xt]));
        y[o + t * D] = from_f32<T>(h);
    }
    h_last[b * D + d] = h;
}

template <typename T>
__global__ void rec_bwd_kernel(RecPtr p, const int32_t* __restrict__ cu, int64_t L, int64_t D, const float* __restrict__ lam,
                               float c, const float* __restrict__ hs, const float* __restrict__ dh_last, T* __restrict__ dx,
                               T* __restrict__ dr, T* __restrict__ di, float* __restrict__ part, float* __restrict__ dh0) {
    const int64_t d = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t b = blockIdx.y;
    if (d >= D) return;
    int64_t t0, n;
    rows_of(cu, b, L, t0, n);
    const T* x = static_cast<const T*>(p.x) + (cu ? 0 : b * p.xb) + t0 * p.xt + d;
    const T* r = static_cast<const T*>(p.r) + (cu ? 0 : b * p.rb) + t0 * p.rt + d;
    const T* i = static_cast<const T*>(p.i) + (cu ? 0 : b * p.ib) + t0 * p.it + d;
    const T* dy = p.dy ? static_cast<const T*>(p.dy) + (cu ? 0 : b * p.gb) + t0 * p.gt + d : nullptr;
    const int64_t o = ((cu ? 0 : b * L) + t0) * D + d;
    const float cs = c * softplus_(lam[d]);
    float back = dh_last ? dh_last[b * D + d] : 0.0f, sum = 0.0f;
    for (int64_t t = n - 1; t >= 0; --t) {
        const Gates g = gates(to_f32<T>(r[t * p.rt]), to_f32<T>(i[t * p.it]), cs);
        const float xv = to_f32<T>(x[t * p.xt]);
        const float G = back + (dy ? to_f32<T>(dy[t * p.gt]) : 0.0f);
        const float dxv = G * g.m * g.si;
        dx[o + t * D] = from_f32<T>(dxv);
        di[o + t * D] = from_f32<T>(dxv * xv * (1.0f - g.si));
        const float slope = g.m == 0.0f ? 0.0f : g.a * g.a / g.m;
        const float du = G * (g.a * hs[o + t * D] - slope * g.si * xv);
        dr[o + t * D] = from_f32<T>(du * g.u * (1.0f - g.sr));
        sum = fmaf(du, g.sr, sum);
        back = g.a * G;
    }
    if (dh0) dh0[b * D + d] = back;
    part[b * D + d] = sum;
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
        const Gates g = gates(to_f32<T>(static_cast<const T*>(p.r)[b * p.rb + d]),
                              to_f32<T>(static_cast<const T*>(p.i)[b * p.ib + d]), c * softplus_(lam[d]));
        const float v = fmaf(g.a, h[k], g.m * g.si * to_f32<T>(static_cast<const T*>(p.x)[b * p.xb + d]));
        h[k] = v;
        y[k] = from_f32<T>(v);
    }
}

bcm_status rec_validate(const bcm_gated_rec_args* a, const char* what) {
    BCM_REQUIRE(a != nullptr, "%s: null arguments", what);
    BCM_REQUIRE(dtype_ok(a->dtype), "%s: unsupported dtype %d", what, (int)a->dtype);
    BCM_REQUIRE(a->batch >= 0 && a->seqlen >= 0 && a->dim >= 1, "%s: bad sizes", what);
    BCM_REQUIRE(a->batch < 65536 && a->seqlen < (1ll << 31) && a->dim < (1ll << 31),
                "%s: batch must be below 65536, seqlen and dim below 2^31", what);
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

}  // namespace
}  // namespace bcm

using namespace bcm;

extern "C" size_t bcm_gated_rec_ckpt_bytes(const bcm_gated_rec_args* a) {
    if (!a || a->batch < 0 || a->seqlen < 0 || a->dim < 1) return 0;
    return align_up((size_t)rec_rows(a) * (size_t)a->dim * sizeof(float), 256);
}

extern "C" size_t bcm_gated_rec_bwd_workspace_bytes(const bcm_gated_rec_args* a) {
    if (!a || a->batch < 0 || a->seqlen < 0 || a->dim < 1) return 0;
    return align_up((size_t)a->batch * (size_t)a->dim * sizeof(float), 256);
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
    const dim3 grid((unsigned)ceil_div(a->dim, 128), (unsigned)a->batch);
    return dispatch_dtype(a->dtype, [&](auto tag) -> bcm_status {
        using T = decltype(tag);
        rec_fwd_kernel<T><<<grid, 128, 0, stream>>>(rec_ptr(a), a->cu_seqlens, a->seqlen, a->dim, a->lam, a->decay_scale, a->h0,
                                                    static_cast<T*>(a->y), a->h_last, static_cast<float*>(a->ckpt));
        BCM_LAUNCH_CHECK();
        return BCM_OK;
    });
}

extern "C" bcm_status bcm_gated_rec_bwd(const bcm_gated_rec_args* a, cudaStream_t stream) {
    clear_error();
    if (bcm_status st = rec_validate(a, "gated_rec_bwd"); st != BCM_OK) return st;
    BCM_REQUIRE(a->lam && a->dlam, "gated_rec_bwd: null pointer");
    if (a->batch == 0) {
        BCM_CUDA_TRY(cudaMemsetAsync(a->dlam, 0, sizeof(float) * a->dim, stream));
        return BCM_OK;
    }
    BCM_REQUIRE(rec_rows(a) == 0 || (a->x && a->r && a->i && a->dx && a->dr && a->di && a->ckpt), "gated_rec_bwd: null pointer");
    const size_t need = bcm_gated_rec_bwd_workspace_bytes(a), ck = bcm_gated_rec_ckpt_bytes(a);
    if (!a->workspace || a->workspace_bytes < need || a->ckpt_bytes < ck) {
        set_error("gated_rec_bwd: workspace of %zu bytes or ckpt of %zu bytes < required %zu and %zu", a->workspace_bytes,
                  a->ckpt_bytes, need, ck);
        return BCM_ERR_WORKSPACE;
    }
    float* part = static_cast<float*>(a->workspace);
    const dim3 grid((unsigned)ceil_div(a->dim, 128), (unsigned)a->batch);
    bcm_status st = dispatch_dtype(a->dtype, [&](auto tag) -> bcm_status {
        using T = decltype(tag);
        rec_bwd_kernel<T><<<grid, 128, 0, stream>>>(rec_ptr(a), a->cu_seqlens, a->seqlen, a->dim, a->lam, a->decay_scale,
                                                    static_cast<const float*>(a->ckpt), a->dh_last, static_cast<T*>(a->dx),
                                                    static_cast<T*>(a->dr), static_cast<T*>(a->di), part, a->dh0);
        BCM_LAUNCH_CHECK();
        return BCM_OK;
    });
    if (st != BCM_OK) return st;
    rec_dlam_kernel<<<(unsigned)ceil_div(a->dim, 128), 128, 0, stream>>>(part, a->batch, a->dim, a->lam, a->decay_scale, a->dlam);
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
