// gated_norm.cu — norm of a mixer's output by groups of features (its heads), times weight and silu(gate).
//
// Per row and group of W features: r = (mean x^2 + eps)^(-1/2), out = x r w silu(z).  Backward, with
// dn = dout w silu(z):  dx = r (dn - x r^2 mean(dn x)),  dz = dout x r w silu'(z),  dw = sum over rows of dout x r silu(z).
// Both means of a row are found in one pass over it, so x, z and dout are read once.
#include "row_norm.cuh"

namespace bcm {
namespace row_norm {

struct GatedArgs {
    int64_t rows;
    int width, groups;
    float eps;
    const void *x, *gate, *dout;
    int64_t x_st, gate_st, dout_st;
    const float* weight;
    void *out, *dx, *dgate;     // contiguous
    float* dw;                  // [row blocks][dim]
};

// silu(z) and its slope
__device__ __forceinline__ float silu(float z, float& slope) {
    const float s = __fdividef(1.0f, 1.0f + expf(-z));       // 2 units in the last place; an infinite divisor gives 0
    slope = s * (1.0f + z * (1.0f - s));
    return z * s;
}

template <bool BACK>
constexpr int kGatedPerSm = BACK ? 768 : 1024;              // threads that fit with the registers they need

// 512000 x 256 bf16 in 4 groups: forward 146 us (82 % of a copy's bandwidth, issue slots 67 % busy), backward 244 us (82 %, 70 %).
// The next row's operands are on their way while this one's are used.  The weight stays in registers forward; backward
// it is read again for each row, which spilled otherwise.
template <typename T, typename G, bool BACK>
__global__ void __launch_bounds__(G::threads, resident(G::threads, kGatedPerSm<BACK>)) gated_kernel(const __grid_constant__ GatedArgs p) {
    extern __shared__ float cols_room[];
    __shared__ float room[2][32][2];
    const int group = blockIdx.x % p.groups, width = p.width;
    const int64_t block = blockIdx.x / p.groups, blocks = gridDim.x / p.groups, dim = (int64_t)p.groups * width;
    const int64_t at = (int64_t)group * width;
    float dw[G::n] = {}, weight[G::n];
    int turn = 0;
    typename G::template Raw<T> next[BACK ? 3 : 2];
    auto fetch = [&](int64_t row) {
        const int in = row < p.rows ? width : 0;
        G::fetch((const T*)p.x + row * p.x_st + at, in, next[0]);
        G::fetch((const T*)p.gate + row * p.gate_st + at, in, next[1]);
        if constexpr (BACK) G::fetch((const T*)p.dout + row * p.dout_st + at, in, next[2]);
    };
    constexpr bool ahead = !BACK || G::ahead_back;
    if (ahead) fetch(block * G::teams + G::id());
    if (!BACK) G::load(p.weight + at, width, weight);
    for (int64_t base = block * G::teams; base < p.rows; base += blocks * G::teams, turn ^= 1) {
        const int64_t row = base + G::id();
        const bool live = row < p.rows;
        float x[G::n], z[G::n], d[G::n], w[G::n];
        if (!ahead) fetch(row);
        G::values(next[0], x);
        G::values(next[1], z);
        if constexpr (BACK) G::values(next[2], d);
        if (ahead) fetch(row + blocks * G::teams);
        if (BACK) G::load(p.weight + at, width, weight);
#pragma unroll
        for (int j = 0; j < G::n; ++j) w[j] = weight[j];
        float sq = 0.0f, dot = 0.0f;
#pragma unroll
        for (int j = 0; j < G::n; ++j) {
            sq = fmaf(x[j], x[j], sq);
            if (BACK) {
                // d becomes dout x silu(z), z becomes dout x w silu'(z), w becomes dn
                float slope;
                const float g = silu(z[j], slope);
                z[j] = d[j] * x[j] * w[j] * slope;
                w[j] *= d[j] * g;
                d[j] *= x[j] * g;
                dot = fmaf(w[j], x[j], dot);
            }
        }
        G::sum(sq, dot, room, turn);
        const float r = rsqrtf(sq / width + p.eps);
        if (BACK) {
            const float m = r * (r * (dot / width));           // (r r of a tiny eps alone may be infinite)
#pragma unroll
            for (int j = 0; j < G::n; ++j) {
                dw[j] = fmaf(d[j], r, dw[j]);
                x[j] = r * (w[j] - x[j] * m);
                z[j] *= r;
            }
            if (live) {
                G::store((T*)p.dx + row * dim + at, width, x);
                G::store((T*)p.dgate + row * dim + at, width, z);
            }
        } else {
#pragma unroll
            for (int j = 0; j < G::n; ++j) {
                float slope;
                x[j] = x[j] * r * w[j] * silu(z[j], slope);
            }
            if (live) G::store((T*)p.out + row * dim + at, width, x);
        }
    }
    if (BACK) G::columns(dw, width, cols_room, p.dw + block * dim + at);
}

bcm_status check(const bcm_gated_norm_args* a, const char* what) {
    BCM_REQUIRE(a != nullptr, "%s: null arguments", what);
    BCM_REQUIRE(dtype_ok(a->dtype), "%s: unsupported dtype %d", what, (int)a->dtype);
    BCM_REQUIRE(a->rows >= 0 && a->dim >= 1 && a->groups >= 1 && a->dim % a->groups == 0, "%s: bad sizes", what);
    BCM_REQUIRE(a->dim / a->groups <= kMostWidth, "%s: a norm over more than %d features", what, (int)kMostWidth);
    BCM_REQUIRE(a->groups <= (1 << 20), "%s: too many groups", what);
    BCM_REQUIRE(a->eps > 0.0f && a->eps <= 3.4028234e38f, "%s: eps must be positive and finite", what);
    return BCM_OK;
}

template <bool BACK>
bcm_status run(const bcm_gated_norm_args* a, cudaStream_t stream) {
    GatedArgs p{a->rows, (int)(a->dim / a->groups), (int)a->groups, a->eps, a->x, a->gate, a->dout, a->x_stride, a->gate_stride,
                a->dout_stride, a->weight, a->out, a->dx, a->dgate, (float*)a->workspace};
    const int64_t size = (int64_t)dtype_size(a->dtype);
    const bool vec = p.width % 8 == 0 && on_16(a->x, a->x_stride * size) && on_16(a->gate, a->gate_stride * size) && on_16(a->weight, 0) &&
                     (BACK ? on_16(a->dout, a->dout_stride * size) && on_16(a->dx, 0) && on_16(a->dgate, 0) : on_16(a->out, 0));
    int64_t blocks = 0;
    bcm_status st = dispatch_dtype(a->dtype, [&](auto type) -> bcm_status {
        using T = decltype(type);
        auto go = [&](auto team) -> bcm_status {
            using G = decltype(team);
            blocks = row_blocks(a->rows, a->groups, G::teams, G::threads, kGatedPerSm<BACK>);
            const size_t smem = BACK && G::teams > 1 ? sizeof(float) * G::teams * p.width : 0;
            gated_kernel<T, G, BACK><<<(unsigned)(blocks * a->groups), G::threads, smem, stream>>>(p);
            BCM_LAUNCH_CHECK();
            return BCM_OK;
        };
        return vec ? by_width<true>(p.width, go) : by_width<false>(p.width, go);
    });
    if (!BACK || st != BCM_OK) return st;
    add_blocks_kernel<<<ceil_div(a->dim, 32), 1024, 0, stream>>>(p.dw, (int)blocks, a->dim, a->dweight, nullptr);
    BCM_LAUNCH_CHECK();
    return BCM_OK;
}

}  // namespace row_norm
}  // namespace bcm

using namespace bcm;
using namespace bcm::row_norm;

extern "C" bcm_status bcm_gated_norm_fwd(const bcm_gated_norm_args* a, cudaStream_t stream) {
    clear_error();
    const bcm_status st = check(a, "gated_norm_fwd");
    if (st != BCM_OK || a->rows == 0) return st;
    BCM_REQUIRE(a->x && a->gate && a->weight && a->out, "gated_norm_fwd: null pointer");
    return run<false>(a, stream);
}

extern "C" size_t bcm_gated_norm_bwd_workspace_bytes(const bcm_gated_norm_args* a) {
    if (check(a, "gated_norm") != BCM_OK) return 0;
    return sizeof(float) * (size_t)most_row_blocks(a->groups, 256, kGatedPerSm<true>) * a->dim;
}

extern "C" bcm_status bcm_gated_norm_bwd(const bcm_gated_norm_args* a, cudaStream_t stream) {
    clear_error();
    const bcm_status st = check(a, "gated_norm_bwd");
    if (st != BCM_OK) return st;
    BCM_REQUIRE(a->dweight, "gated_norm_bwd: null pointer");
    BCM_REQUIRE(a->rows == 0 || (a->x && a->gate && a->weight && a->dout && a->dx && a->dgate), "gated_norm_bwd: null pointer");
    BCM_REQUIRE(a->workspace && a->workspace_bytes >= bcm_gated_norm_bwd_workspace_bytes(a), "gated_norm_bwd: workspace too small");
    return run<true>(a, stream);
}
