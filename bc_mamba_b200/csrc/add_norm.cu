// add_norm.cu — the residual addition of a block's output and the norm before the next block, in one pass.
//
// v = residual + s branch (s per feature, or 1), out = v r w with r = (mean v^2 + eps)^(-1/2).  Backward, with
// dn = dout w and dres the gradient of v from the stream itself:  dv = dres + r (dn - v r^2 mean(dn v)),
// dbranch = s dv,  dw = sum over rows of dout v r,  ds = sum over rows of dv branch.
// v is formed anew from its two inputs, which the scale's gradient reads anyway: its rounding to the stream's type
// does not enter the gradients.
#include "row_norm.cuh"

namespace bcm {
namespace row_norm {

struct AddArgs {
    int64_t rows;
    int dim;
    float eps;
    const void *res, *branch, *dres, *dout;
    int64_t res_st, branch_st, dres_st, dout_st;
    const float *weight, *scale;
    void *res_out, *out, *dresidual, *dbranch;      // contiguous
    float *dw, *ds;                                 // [blocks][dim]
};

constexpr int kAddFwdPerSm = 1024, kAddBwdPerSm = 512;     // threads that fit with the registers they need

// 65536 x 2048 bf16 with a scale: forward 167 us (98 % of a copy's bandwidth), backward 283 us (87 %); rows off 16 bytes
// (30011 x 1001 float16 beside a float32 stream) 69 and 108 us (80 and 76 %).
// In both directions the next row's operands are on their way while this one's are used.  Backward the weight is read
// again for each row, which spilled otherwise.
template <typename R, typename T, typename G>
__global__ void __launch_bounds__(G::threads, resident(G::threads, kAddFwdPerSm)) add_fwd_kernel(const __grid_constant__ AddArgs p) {
    __shared__ float room[2][32][2];
    int turn = 0;
    float w[G::n], s[G::n];
    typename G::template Raw<R> next_res;
    typename G::template Raw<T> next_branch;
    auto fetch = [&](int64_t row) {
        const int in = row < p.rows ? p.dim : 0;
        G::fetch((const R*)p.res + row * p.res_st, in, next_res);
        G::fetch((const T*)p.branch + row * p.branch_st, in, next_branch);
    };
    const int64_t across = (int64_t)gridDim.x * G::teams;
    fetch((int64_t)blockIdx.x * G::teams + G::id());
    G::load(p.weight, p.dim, w);
    if (p.scale) G::load(p.scale, p.dim, s);
    for (int64_t base = (int64_t)blockIdx.x * G::teams; base < p.rows; base += across, turn ^= 1) {
        const int64_t row = base + G::id();
        const bool live = row < p.rows;
        float v[G::n], b[G::n];
        G::values(next_res, v);
        G::values(next_branch, b);
        fetch(row + across);
#pragma unroll
        for (int j = 0; j < G::n; ++j) v[j] = p.scale ? fmaf(s[j], b[j], v[j]) : v[j] + b[j];
        if (live) G::store((R*)p.res_out + row * p.dim, p.dim, v);
        float sq = 0.0f, none = 0.0f;
#pragma unroll
        for (int j = 0; j < G::n; ++j) sq = fmaf(v[j], v[j], sq);
        G::sum(sq, none, room, turn);
        const float r = rsqrtf(sq / p.dim + p.eps);
#pragma unroll
        for (int j = 0; j < G::n; ++j) v[j] *= r * w[j];
        if (live) G::store((T*)p.out + row * p.dim, p.dim, v);
    }
}

template <typename R, typename T, typename G, bool SCALED>
__global__ void __launch_bounds__(G::threads, resident(G::threads, kAddBwdPerSm)) add_bwd_kernel(const __grid_constant__ AddArgs p) {
    extern __shared__ float cols_room[];
    __shared__ float room[2][32][2];
    float dw[G::n] = {}, ds[SCALED ? G::n : 1] = {}, s[SCALED ? G::n : 1];
    int turn = 0;
    typename G::template Raw<R> next_res, next_dres;
    typename G::template Raw<T> next_branch, next_dout;
    auto fetch = [&](int64_t row) {
        const int in = row < p.rows ? p.dim : 0;
        G::fetch((const R*)p.res + row * p.res_st, in, next_res);
        G::fetch((const T*)p.branch + row * p.branch_st, in, next_branch);
        G::fetch((const T*)p.dout + row * p.dout_st, p.dout ? in : 0, next_dout);
        G::fetch((const R*)p.dres + row * p.dres_st, p.dres ? in : 0, next_dres);
    };
    const int64_t across = (int64_t)gridDim.x * G::teams;
    if (G::ahead_back) fetch((int64_t)blockIdx.x * G::teams + G::id());
    if constexpr (SCALED) G::load(p.scale, p.dim, s);
    for (int64_t base = (int64_t)blockIdx.x * G::teams; base < p.rows; base += across, turn ^= 1) {
        const int64_t row = base + G::id();
        const bool live = row < p.rows;
        float v[G::n], b[G::n], d[G::n], dv[G::n], w[G::n];
        if (!G::ahead_back) fetch(row);
        G::values(next_res, v);
        G::values(next_branch, b);
        G::values(next_dout, d);
        G::values(next_dres, dv);
        if (G::ahead_back) fetch(row + across);
        G::load(p.weight, p.dim, w);
#pragma unroll
        for (int j = 0; j < G::n; ++j) {
            if constexpr (SCALED) v[j] = fmaf(s[j], b[j], v[j]);
            else v[j] += b[j];
        }
        float sq = 0.0f, dot = 0.0f;
#pragma unroll
        for (int j = 0; j < G::n; ++j) {
            sq = fmaf(v[j], v[j], sq);
            w[j] *= d[j];
            dot = fmaf(w[j], v[j], dot);
        }
        G::sum(sq, dot, room, turn);
        const float r = rsqrtf(sq / p.dim + p.eps), m = r * (r * (dot / p.dim));       // (r r of a tiny eps alone may be infinite)
#pragma unroll
        for (int j = 0; j < G::n; ++j) {
            dw[j] = fmaf(d[j] * v[j], r, dw[j]);
            dv[j] = fmaf(r, w[j] - v[j] * m, dv[j]);
            if constexpr (SCALED) ds[j] = fmaf(dv[j], b[j], ds[j]);
        }
        if (live) G::store((R*)p.dresidual + row * p.dim, p.dim, dv);
        if constexpr (SCALED) {
#pragma unroll
            for (int j = 0; j < G::n; ++j) dv[j] *= s[j];
        }
        if (live && p.dbranch) G::store((T*)p.dbranch + row * p.dim, p.dim, dv);
    }
    G::columns(dw, p.dim, cols_room, p.dw + (int64_t)blockIdx.x * p.dim);
    if constexpr (SCALED) G::columns(ds, p.dim, cols_room, p.ds + (int64_t)blockIdx.x * p.dim);
}

bcm_status check(const bcm_add_norm_args* a, const char* what) {
    BCM_REQUIRE(a != nullptr, "%s: null arguments", what);
    BCM_REQUIRE(dtype_ok(a->dtype), "%s: unsupported dtype %d", what, (int)a->dtype);
    BCM_REQUIRE(a->residual_dtype == a->dtype || a->residual_dtype == BCM_F32, "%s: the residual must have the branch's dtype or be float32", what);
    BCM_REQUIRE(a->rows >= 0 && a->dim >= 1, "%s: bad sizes", what);
    BCM_REQUIRE(a->dim <= kMostWidth, "%s: a norm over more than %d features", what, (int)kMostWidth);
    BCM_REQUIRE(a->eps > 0.0f && a->eps <= 3.4028234e38f, "%s: eps must be positive and finite", what);
    return BCM_OK;
}

// calls f(R, T, team) for the argument's types and the rows' alignment
template <typename F>
bcm_status dispatch(const bcm_add_norm_args* a, bool vec, F&& f) {
    return dispatch_dtype(a->dtype, [&](auto type) -> bcm_status {
        using T = decltype(type);
        auto go = [&](auto res) -> bcm_status {
            auto team = [&](auto t) -> bcm_status { return f(res, type, t); };
            return vec ? by_width<true>(a->dim, team) : by_width<false>(a->dim, team);
        };
        if constexpr (!std::is_same<T, float>::value) {
            if (a->residual_dtype == BCM_F32) return go(float{});
        }
        return go(type);
    });
}

AddArgs args_of(const bcm_add_norm_args* a) {
    AddArgs p{a->rows, (int)a->dim, a->eps, a->residual, a->branch, a->dresidual_out, a->dout, a->residual_stride, a->branch_stride,
              a->dresidual_out_stride, a->dout_stride, a->weight, a->scale, a->residual_out, a->out, a->dresidual, a->dbranch,
              (float*)a->workspace, nullptr};
    return p;
}

}  // namespace row_norm
}  // namespace bcm

using namespace bcm;
using namespace bcm::row_norm;

extern "C" bcm_status bcm_add_norm_fwd(const bcm_add_norm_args* a, cudaStream_t stream) {
    clear_error();
    const bcm_status st = check(a, "add_norm_fwd");
    if (st != BCM_OK || a->rows == 0) return st;
    BCM_REQUIRE(a->residual && a->branch && a->weight && a->residual_out && a->out, "add_norm_fwd: null pointer");
    const AddArgs p = args_of(a);
    const int64_t size = (int64_t)dtype_size(a->dtype), res = (int64_t)dtype_size(a->residual_dtype);
    const bool vec = a->dim % 8 == 0 && on_16(p.res, p.res_st * res) && on_16(p.branch, p.branch_st * size) && on_16(p.weight, 0) &&
                     on_16(p.scale, 0) && on_16(p.res_out, 0) && on_16(p.out, 0);
    return row_norm::dispatch(a, vec, [&](auto r, auto t, auto team) -> bcm_status {
        using G = decltype(team);
        add_fwd_kernel<decltype(r), decltype(t), G><<<(unsigned)row_blocks(a->rows, 1, G::teams, G::threads, kAddFwdPerSm), G::threads, 0, stream>>>(p);
        BCM_LAUNCH_CHECK();
        return BCM_OK;
    });
}

extern "C" size_t bcm_add_norm_bwd_workspace_bytes(const bcm_add_norm_args* a) {
    if (check(a, "add_norm") != BCM_OK) return 0;
    return (a->scale ? 2 : 1) * sizeof(float) * (size_t)most_row_blocks(1, 256, kAddBwdPerSm) * a->dim;
}

extern "C" bcm_status bcm_add_norm_bwd(const bcm_add_norm_args* a, cudaStream_t stream) {
    clear_error();
    bcm_status st = check(a, "add_norm_bwd");
    if (st != BCM_OK) return st;
    BCM_REQUIRE(a->dweight && (!a->scale || a->dscale), "add_norm_bwd: null pointer");
    BCM_REQUIRE(a->rows == 0 || (a->residual && a->branch && a->weight && a->dresidual), "add_norm_bwd: null pointer");
    BCM_REQUIRE(a->rows == 0 || a->dbranch || (!a->scale && a->residual_dtype == a->dtype), "add_norm_bwd: dbranch differs from dresidual");
    BCM_REQUIRE(a->workspace && a->workspace_bytes >= bcm_add_norm_bwd_workspace_bytes(a), "add_norm_bwd: workspace too small");
    AddArgs p = args_of(a);
    const int64_t size = (int64_t)dtype_size(a->dtype), res = (int64_t)dtype_size(a->residual_dtype);
    const bool vec = a->dim % 8 == 0 && on_16(p.res, p.res_st * res) && on_16(p.branch, p.branch_st * size) && on_16(p.weight, 0) &&
                     on_16(p.scale, 0) && on_16(p.dres, p.dres_st * res) && on_16(p.dout, p.dout_st * size) && on_16(p.dresidual, 0) &&
                     on_16(p.dbranch, 0);
    int64_t blocks = 0;
    st = row_norm::dispatch(a, vec, [&](auto r, auto t, auto team) -> bcm_status {
        using G = decltype(team);
        blocks = row_blocks(a->rows, 1, G::teams, G::threads, kAddBwdPerSm);
        p.ds = p.dw + blocks * a->dim;
        const size_t smem = G::teams > 1 ? sizeof(float) * G::teams * a->dim : 0;
        if (p.scale) add_bwd_kernel<decltype(r), decltype(t), G, true><<<(unsigned)blocks, G::threads, smem, stream>>>(p);
        else add_bwd_kernel<decltype(r), decltype(t), G, false><<<(unsigned)blocks, G::threads, smem, stream>>>(p);
        BCM_LAUNCH_CHECK();
        return BCM_OK;
    });
    if (st != BCM_OK) return st;
    add_blocks_kernel<<<dim3(ceil_div(a->dim, 32), p.scale ? 2 : 1), 1024, 0, stream>>>(p.dw, (int)blocks, a->dim, a->dweight, a->dscale);
    BCM_LAUNCH_CHECK();
    return BCM_OK;
}
