// decay_attn_bwd.cu — backward of the linear attention with a decay for each head.
//
// With dS the gradient of the state behind a chunk, W_ij = (q_i . k_j) D_ij (dy_i . v_j):
//   dQ = ((dY V^T) o D) K + diag(exp G) dY S_in^T          dV = ((Q K^T) o D)^T dY + diag(exp(G_64 - G)) K dS
//   dK = ((dY V^T) o D)^T Q + diag(exp(G_64 - G)) V dS^T   dS_in = exp(G_64) dS + sum_i exp(G_i) q_i dy_i^T
//   dg_t = sum_(i >= t > j) W_ij + sum_(i >= t) (exp(G_i) q_i . S_in dy_i) + sum_(j < t) (exp(G_64 - G_j) k_j . dS v_j)
//          + exp(G_64) <S_in, dS>,
// every term of dg_t holds the factor a_t, and none cancels against another: the gradient of a strong decay, which is
// proportional to it, keeps its digits.
#include "decay_attn.cuh"

namespace bcm {
namespace decay_attn {

struct BwdArgs {
    Sizes z;
    Rows q, k, v, dy;          // dy.p NULL: zeros
    const float* g;
    int64_t g_sb, g_st, g_sh;
    const float* ckpt;         // states that enter the chunks, from the forward
    const float* dh_last;      // or NULL
    const float* enter;        // gradients of the states behind the items, where sequences are cut
    void* dq;                  // contiguous; of `shares` blocks a float32 part each where there is more than one
    void* dk;
    void* dv;
    float* dg;                 // of `slices` blocks a part each
    float* dh0;
    int shares;
};

// Four groups of four warps: dv and dg's pairs; dk; dq; the state's gradient.  The first three take 16 tokens a warp.
// Where there is room for it the pieces of the next chunk's gradient go to a second buffer.
constexpr int kBwdThreads = 512;

template <typename T, int NT, int PT>
struct BwdSmem {
    static constexpr int NS = Pieces<T>::in, MS = Pieces<T>::out;
    struct Tiles {
        bf16 q[NS][kChunk][NT + 8], k[NS][kChunk][NT + 8], v[NS][kChunk][PT + 8], dy[NS][kChunk][PT + 8];
        bf16 s[kFull3][NT][PT + 8];
    } tiles;
    static constexpr int buffers = sizeof(Tiles) + 2 * sizeof(bf16[kFull3][NT][PT + 8]) <= 222 * 1024 ? 2 : 1;
    bf16 ds[buffers][kFull3][NT][PT + 8];
    Decays d;
    float pairs[4][kChunk];    // sum over i >= t, j < t of W_ij, j of one warp
    float of_q[kChunk], of_k[kChunk];
    float across[4];           // <S_in, dS> of the warps
};

// where a block's rows of dq and dk go
template <typename T>
struct RowsOut {
    T* whole;
    float* part;
    int64_t st;
    __device__ __forceinline__ void put(int64_t row, int c, float x) const {
        if (part) part[row * st + c] = x;
        else whole[row * st + c] = from_f32<T>(x);
    }
    __device__ __forceinline__ void put2(int64_t row, int c, int cols, float x, float y, bool pair) const {
        if (c + 1 < cols && pair) {
            if (part) {
                *(float2*)(part + row * st + c) = make_float2(x, y);
            } else {
                struct alignas(2 * sizeof(T)) Two { T x, y; };
                *(Two*)(whole + row * st + c) = Two{from_f32<T>(x), from_f32<T>(y)};
            }
        } else {
            if (c < cols) put(row, c, x);
            if (c + 1 < cols) put(row, c + 1, y);
        }
    }
    __device__ __forceinline__ bool pairs() const {
        return part ? (((uintptr_t)part | (uintptr_t)(st * 4)) & 7) == 0
                    : (((uintptr_t)whole | (uintptr_t)(st * sizeof(T))) & (2 * sizeof(T) - 1)) == 0;
    }
};

// A chunk with a value that is not finite, token by token from its last: a state is run up anew for each.
// `f` (shared): the state's gradient NT x PT, then sums.
template <typename T, int NT, int PT>
__device__ __noinline__ void back_tokens(const BwdArgs& p, const T* q, const T* k, const T* v, const T* dy, const float* g, const float* s_in,
                                         const RowsOut<T>& dq, const RowsOut<T>& dk, T* dv, int64_t dv_st, float* dg, int64_t dg_st,
                                         int rows, int cols, int64_t row0, float* f) {
    constexpr int parts = kBwdThreads / PT, warps = PT / 32, all_warps = kBwdThreads / 32;
    const int c = threadIdx.x % PT, part = threadIdx.x / PT, w = threadIdx.x >> 5, l = lane_id();
    float* const sq = f + NT * PT;                 // [warps][NT]
    float* const sk = sq + 2 * NT;
    float* const sv = sk + 2 * NT;                 // [kBwdThreads]
    float* const sg = sv + kBwdThreads;            // [all_warps]
    const bool in = c < cols;
    for (int t = rows - 1; t >= 0; --t) {
        const float a = expf(g[t * p.g_st]);
        const float gy = in && dy ? to_f32(dy[t * p.dy.st + c]) : 0.0f, x = in ? to_f32(v[t * p.v.st + c]) : 0.0f;
        float gv = 0.0f, gg = 0.0f;
        for (int n = part; n < p.z.n; n += parts) {
            float s = in ? s_in[(int64_t)n * p.z.p + c] : 0.0f;
            if (in)
                for (int u = 0; u < t; ++u) s = fmaf(expf(g[u * p.g_st]), s, to_f32(k[u * p.k.st + n]) * to_f32(v[u * p.v.st + c]));
            const float kn = to_f32(k[t * p.k.st + n]), now = fmaf(a, s, kn * x);
            const float ds = f[n * PT + c] + (dy ? to_f32(q[t * p.q.st + n]) * gy : 0.0f);
            float gq = in ? now * gy : 0.0f, gk = in ? ds * x : 0.0f;
            gv = fmaf(ds, kn, gv);
            const float back = a * ds;
            gg += in ? back * s : 0.0f;
            f[n * PT + c] = in ? back : 0.0f;
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                gq += __shfl_xor_sync(kFull, gq, o);
                gk += __shfl_xor_sync(kFull, gk, o);
            }
            if (l == 0) {
                sq[w % warps * NT + n] = gq;
                sk[w % warps * NT + n] = gk;
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) gg += __shfl_xor_sync(kFull, gg, o);
        if (l == 0) sg[w] = gg;
        sv[threadIdx.x] = gv;
        __syncthreads();
        for (int n = threadIdx.x; n < p.z.n; n += kBwdThreads) {
            float x0 = sq[n], x1 = sk[n];
            if (warps > 1) {
                x0 += sq[NT + n];
                x1 += sk[NT + n];
            }
            dq.put(row0 + t, n, x0);
            dk.put(row0 + t, n, x1);
        }
        if (part == 0 && in) {
            for (int r = 1; r < parts; ++r) gv += sv[r * PT + c];
            dv[t * dv_st + c] = from_f32<T>(gv);
        }
        if (threadIdx.x == 0) {
            for (int r = 1; r < all_warps; ++r) gg += sg[r];
            dg[t * dg_st] = gg;
        }
        __syncthreads();
    }
}

template <typename T, int NT, int PT>
__global__ void __launch_bounds__(kBwdThreads) bwd_kernel(const __grid_constant__ BwdArgs p) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    using Smem = BwdSmem<T, NT, PT>;
    Smem& sm = *(Smem*)smem_raw;
    constexpr int NS = Smem::NS, MS = Smem::MS, LN = NT + 8, LP = PT + 8;
    const Sizes& z = p.z;
    const int across = z.heads * z.slices, share = z.heads / z.qk_heads;
    const int item = blockIdx.x / across, hs = blockIdx.x % across, h = hs / z.slices, slice = hs % z.slices, col = slice * PT;
    const int cols = min(PT, z.p - col), hq = h / share;
    const int64_t rows_all = (z.cu ? 1 : (int64_t)z.batch) * z.seqlen;
    const int64_t qk_st = (int64_t)z.qk_heads * z.n, v_st = (int64_t)z.heads * z.p;
    const int mine = h % share * z.slices + slice;            // of the blocks that share a row of dq
    RowsOut<T> dq{(T*)p.dq + (int64_t)hq * z.n, nullptr, qk_st}, dk{(T*)p.dk + (int64_t)hq * z.n, nullptr, qk_st};
    if (p.shares > 1) {
        dq.part = (float*)p.dq + mine * rows_all * qk_st + (int64_t)hq * z.n;
        dk.part = (float*)p.dk + mine * rows_all * qk_st + (int64_t)hq * z.n;
    }
    float* const dg_all = p.dg + slice * rows_all * z.heads + h;
    if (z.cu) {
        const int end = z.tables.seq_item[z.batch + 1];
        zero_rows((T*)p.dv + (int64_t)h * z.p + col, end, z.seqlen, v_st, cols, item, z.items);
        zero_rows(dg_all, end, z.seqlen, z.heads, 1, item, z.items);
        if (dq.part) {
            zero_rows(dq.part, end, z.seqlen, qk_st, z.n, item, z.items);
            zero_rows(dk.part, end, z.seqlen, qk_st, z.n, item, z.items);
        } else {
            zero_rows(dq.whole, end, z.seqlen, qk_st, z.n, item, z.items);
            zero_rows(dk.whole, end, z.seqlen, qk_st, z.n, item, z.items);
        }
    }
    const Item it = item_of(z, item);
    if (it.seq < 0) return;
    const T* q = row_ptr<T>(p.q, z, it.seq, it.t0, hq);
    const T* k = row_ptr<T>(p.k, z, it.seq, it.t0, hq);
    const T* v = row_ptr<T>(p.v, z, it.seq, it.t0, h) + col;
    const T* dy = p.dy.p ? row_ptr<T>(p.dy, z, it.seq, it.t0, h) + col : nullptr;
    const float* g = p.g + (z.cu ? 0 : it.seq * p.g_sb) + it.t0 * p.g_st + h * p.g_sh;
    const int64_t row_at = (z.cu ? 0 : (int64_t)it.seq * z.seqlen) + it.t0;
    T* const dv = (T*)p.dv + row_at * v_st + (int64_t)h * z.p + col;
    float* const dg = dg_all + row_at * z.heads;
    const bool vq = on_16(q, p.q.st), vk = on_16(k, p.k.st), vv = on_16(v, p.v.st), vy = dy && on_16(dy, p.dy.st);
    const bool pair_v = (((uintptr_t)dv | (uintptr_t)(v_st * sizeof(T))) & (2 * sizeof(T) - 1)) == 0, pair_qk = dq.pairs() && dk.pairs();
    const int np = z.n * z.p;
    const int len = it.t1 - it.t0, nc = (len + kChunk - 1) / kChunk;
    const int l = lane_id(), group = threadIdx.x >> 7, w = (threadIdx.x >> 5) & 3, row = w * 16 + (l >> 2), lq = l & 3;
    const bool decay_warp = threadIdx.x >= 384 && threadIdx.x < 416;
    bf16* const tq = &sm.tiles.q[0][0][0];
    bf16* const tk = &sm.tiles.k[0][0][0];
    bf16* const tv = &sm.tiles.v[0][0][0];
    bf16* const ty = &sm.tiles.dy[0][0][0];
    bf16* const ts = &sm.tiles.s[0][0][0];
    constexpr int piece_n = kChunk * LN, piece_p = kChunk * LP, piece_s = NT * LP;

    Pending<T, kChunk, NT, kBwdThreads> pq, pk;
    Pending<T, kChunk, PT, kBwdThreads> pv, py;
    Pending<float, NT, PT, kBwdThreads> ps;
    float g0 = 0.0f, g1 = 0.0f;
    const bool vs = (z.p & 3) == 0 && (col & 3) == 0 && ((uintptr_t)p.ckpt & 15) == 0;
    auto state_in = [&](int c) { return p.ckpt + ((int64_t)(it.chunk + c) * z.heads + h) * np + col; };
    auto fetch = [&](int c) {
        const int t = c * kChunk, rows = min(kChunk, len - t);
        pq.fetch(q + t * p.q.st, p.q.st, rows, z.n, vq);
        pk.fetch(k + t * p.k.st, p.k.st, rows, z.n, vk);
        pv.fetch(v + t * p.v.st, p.v.st, rows, cols, vv);
        py.fetch(dy + t * p.dy.st, p.dy.st, dy ? rows : 0, cols, vy);
        ps.fetch(state_in(c), z.p, z.n, cols, vs);
        if (decay_warp) {
            g0 = 2 * l < rows ? g[(int64_t)(t + 2 * l) * p.g_st] : 0.0f;
            g1 = 2 * l + 1 < rows ? g[(int64_t)(t + 2 * l + 1) * p.g_st] : 0.0f;
        }
    };
    auto put = [&]() {
        bool bad = pq.put(tq, LN);
        bad |= pk.put(tk, LN);
        bad |= pv.put(tv, LP);
        bad |= py.put(ty, LP);
        bad |= ps.put(ts, LP);
        if (decay_warp) {
            bad |= !(g0 <= 3.38e38f && g1 <= 3.38e38f);
            decays_of(sm.d, g0, g1);
        }
        return bad;
    };
    auto walk = [&](int c) {
        const int t = c * kChunk;
        back_tokens<T, NT, PT>(p, q + t * p.q.st, k + t * p.k.st, v + t * p.v.st, dy ? dy + t * p.dy.st : nullptr, g + t * p.g_st, state_in(c), dq, dk,
                               dv + t * v_st, v_st, dg + (int64_t)t * z.heads, z.heads, min(kChunk, len - t), cols, row_at + t, (float*)&sm.tiles);
    };
    if (nc > 0) fetch(nc - 1);

    if (group == 3) {
        // dg of chunk c from what its walk left in shared memory (one warp)
        auto finish_dg = [&](int c) {
            const int t = 2 * l, rows = min(kChunk, len - c * kChunk);
            const float q0 = sm.of_q[t], q1 = sm.of_q[t + 1], k0 = sm.of_k[t], k1 = sm.of_k[t + 1];
            float behind = q0 + q1, before = k0 + k1;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const float a = __shfl_down_sync(kFull, behind, off), b = __shfl_up_sync(kFull, before, off);
                if (l + off < 32) behind += a;
                if (l >= off) before += b;
            }
            float rest = __shfl_down_sync(kFull, behind, 1), past = __shfl_up_sync(kFull, before, 1);
            if (l == 31) rest = 0.0f;
            if (l == 0) past = 0.0f;
            const float through = sm.d.whole * ((sm.across[0] + sm.across[1]) + (sm.across[2] + sm.across[3]));
            float d0 = 0.0f, d1 = 0.0f;
            for (int k2 = 0; k2 <= t / 16; ++k2) {
                d0 += sm.pairs[k2][t];
                d1 += sm.pairs[k2][t + 1];
            }
            d0 += (rest + q1 + q0) + past + through;
            d1 += (rest + q1) + (past + k0) + through;
            if (t < rows) dg[(int64_t)(c * kChunk + t) * z.heads] = d0;
            if (t + 1 < rows) dg[(int64_t)(c * kChunk + t + 1) * z.heads] = d1;
        };
        State<NT, PT> ds;
        const float* from = it.last ? (p.dh_last ? p.dh_last + ((int64_t)it.seq * z.heads + h) * np : nullptr)
                                    : p.enter + ((int64_t)item * z.heads + h) * np;
        if (from) ds.load(from + col, z.n, z.p - col, z.p);
        else ds.zero();
        bool bad = false, pending = false;                    // pending: the chunk behind has its dg still to be finished
        if (Smem::buffers > 1) bad = ds.template put<kFull3>(&sm.ds[(nc - 1) & 1 & (Smem::buffers - 1)][0][0][0]);
        for (int c = nc - 1; c >= 0; --c) {
            __syncthreads();                                  // the chunk behind is done with the tiles
            if (pending && decay_warp) finish_dg(c + 1);
            bad |= put();
            if (Smem::buffers == 1) bad |= ds.template put<kFull3>(&sm.ds[0][0][0][0]);
            const bool slow = __syncthreads_or(bad);
            if (c > 0) fetch(c - 1);
            pending = !slow;
            if (slow) {
                float* f = (float*)&sm.tiles;
                ds.pairs([&](float& x0, float& x1, int r, int cc) {
                    f[r * PT + cc] = x0;
                    f[r * PT + cc + 1] = x1;
                });
                __syncthreads();
                walk(c);
                ds.pairs([&](float& x0, float& x1, int r, int cc) {
                    x0 = f[r * PT + cc];
                    x1 = f[r * PT + cc + 1];
                });
            } else {
                float x = 0.0f;
                ds.pairs([&](float& x0, float& x1, int r, int cc) {
                    const float2 in = from_pieces<kFull3>(ts + r * LP + cc, piece_s);
                    x = fmaf(in.x, x0, fmaf(in.y, x1, x));
                });
#pragma unroll
                for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(kFull, x, o);
                if (l == 0) sm.across[w] = x;
                ds.template advance<NS>(tq, ty, sm.d.since, sm.d.whole);
            }
            bad = false;
            if (Smem::buffers > 1) bad = ds.template put<kFull3>(&sm.ds[(c + 1) & 1 & (Smem::buffers - 1)][0][0][0]);
        }
        __syncthreads();
        if (pending && decay_warp) finish_dg(0);
        if (it.first) ds.store(p.dh0 + ((int64_t)it.seq * z.heads + h) * np + col, z.n, z.p - col, z.p);
        return;
    }

    for (int c = nc - 1; c >= 0; --c) {
        const int t = c * kChunk, rows = min(kChunk, len - t);
        __syncthreads();
        const bool bad = put();
        const bool slow = __syncthreads_or(bad);
        if (c > 0) fetch(c - 1);
        if (slow) {
            __syncthreads();
            walk(c);
            continue;
        }
        const bf16* tds = &sm.ds[c & 1 & (Smem::buffers - 1)][0][0][0];
        const float hi0 = sm.d.hi[row], lo0 = sm.d.lo[row], hi1 = sm.d.hi[row + 8], lo1 = sm.d.lo[row + 8];
        auto keys = [&](uint32_t(&a)[4], int s, int kk) { load_a(a, tk + s * piece_n, LN, w * 16, kk * 16); };
        auto values = [&](uint32_t(&a)[4], int s, int kk) { load_a(a, tv + s * piece_p, LP, w * 16, kk * 16); };
        auto ups = [&](uint32_t(&a)[4], int s, int kk) { load_a(a, ty + s * piece_p, LP, w * 16, kk * 16); };
        // x D of 16 rows by 16 columns: rows as the earlier tokens (keys) or as the later ones (queries)
        auto decayed = [&](float(&x)[2][4], int block, bool as_keys) {
#pragma unroll
            for (int q2 = 0; q2 < 2; ++q2) {
                const int o = block * 16 + q2 * 8 + 2 * lq;
                const float2 h2 = *(const float2*)&sm.d.hi[o], l2 = *(const float2*)&sm.d.lo[o];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = o + (e & 1), r = row + (e & 2) * 4;
                    const float ho = e & 1 ? h2.y : h2.x, lo = e & 1 ? l2.y : l2.x, hr = e & 2 ? hi1 : hi0, lr = e & 2 ? lo1 : lo0;
                    if (as_keys) x[q2][e] = i >= r ? x[q2][e] * between(ho, lo, hr, lr) : 0.0f;
                    else x[q2][e] = i <= r ? x[q2][e] * between(hr, lr, ho, lo) : 0.0f;
                }
            }
        };
        // a row's dot with `tile`'s, into out[row]
        auto dots = [&](float(&x)[NT / 8][4], const bf16* tile, float* out) {
            float dot0 = 0.0f, dot1 = 0.0f;
#pragma unroll
            for (int nb = 0; nb < NT / 8; ++nb) {
                const float2 k0 = from_pieces<NS>(tile + row * LN + nb * 8 + 2 * lq, piece_n);
                const float2 k1 = from_pieces<NS>(tile + (row + 8) * LN + nb * 8 + 2 * lq, piece_n);
                dot0 = fmaf(k0.x, x[nb][0], fmaf(k0.y, x[nb][1], dot0));
                dot1 = fmaf(k1.x, x[nb][2], fmaf(k1.y, x[nb][3], dot1));
            }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                dot0 += __shfl_xor_sync(kFull, dot0, o);
                dot1 += __shfl_xor_sync(kFull, dot1, o);
            }
            if (lq == 0) {
                out[row] = dot0;
                out[row + 8] = dot1;
            }
        };
        if (group == 0) {
            // dv of 16 tokens, and the sums of W
            float gv[PT / 8][4] = {};
            gemm<NS, MS, MS, NT / 16, PT / 16, true>(gv, keys, tds, LP, piece_s, 0, 0);
            const float u0 = sm.d.until[row], u1 = sm.d.until[row + 8];
#pragma unroll
            for (int pb = 0; pb < PT / 8; ++pb) {
                gv[pb][0] *= u0;
                gv[pb][1] *= u0;
                gv[pb][2] *= u1;
                gv[pb][3] *= u1;
            }
            float run[2] = {0.0f, 0.0f};                      // sums of W over the queries behind the block
#pragma unroll 1
            for (int ib = 3; ib >= w; --ib) {
                float at[2][4] = {}, dt[2][4] = {};
                gemm<NS, NS, kFull3, NT / 16, 1, false>(at, keys, tq, LN, piece_n, 0, ib * 16);
                gemm<NS, NS, kFull3, PT / 16, 1, false>(dt, values, ty, LP, piece_p, 0, ib * 16);
                decayed(at, ib, true);
                float sum[2][2] = {};                         // of the four columns, over this warp's keys before them
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int j = row + 8 * half;
                    float W[2][2], ex[2], all[2];
#pragma unroll
                    for (int q2 = 0; q2 < 2; ++q2) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) W[q2][e] = at[q2][2 * half + e] * dt[q2][2 * half + e];
                        float s = W[q2][0] + W[q2][1];
                        float o = __shfl_down_sync(kFull, s, 1, 4);
                        if (lq < 3) s += o;
                        o = __shfl_down_sync(kFull, s, 2, 4);
                        if (lq < 2) s += o;
                        o = __shfl_down_sync(kFull, s, 1, 4);
                        ex[q2] = lq < 3 ? o : 0.0f;
                        all[q2] = __shfl_sync(kFull, s, 0, 4);
                    }
                    float u = run[half] + ex[1] + W[1][1];
                    const int i = ib * 16 + 2 * lq;
                    if (j < i + 9) sum[1][1] += u;
                    u += W[1][0];
                    if (j < i + 8) sum[1][0] += u;
                    u = run[half] + all[1] + ex[0] + W[0][1];
                    if (j < i + 1) sum[0][1] += u;
                    u += W[0][0];
                    if (j < i) sum[0][0] += u;
                    run[half] += all[1] + all[0];
                }
#pragma unroll
                for (int q2 = 0; q2 < 2; ++q2)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) sum[q2][e] += __shfl_xor_sync(kFull, sum[q2][e], o);
                        if (l < 4) sm.pairs[w][ib * 16 + q2 * 8 + 2 * lq + e] = sum[q2][e];
                    }
                uint32_t a[MS][4];
                split_a<MS>(at[0], at[1], a);
                gemm<MS, NS, MS, 1, PT / 16, true>(gv, [&](uint32_t(&r)[4], int s, int) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) r[e] = a[s][e];
                }, ty, LP, piece_p, ib * 16, 0);
            }
            const RowsOut<T> ov{dv + t * v_st, nullptr, v_st};
#pragma unroll
            for (int half = 0; half < 2; ++half)
                if (row + 8 * half < rows)
#pragma unroll
                    for (int pb = 0; pb < PT / 8; ++pb)
                        ov.put2(row + 8 * half, pb * 8 + 2 * lq, cols, gv[pb][2 * half], gv[pb][2 * half + 1], pair_v);
        } else {
            // dk (rows as keys) and dq (rows as queries) are one form:  (dP o D) X + decay (V or dY) times the state's
            // gradient or the state; the far part's dot with the row itself is its share of dg
            const bool as_keys = group == 1;
            float gx[NT / 8][4] = {};
            const bf16* const own = as_keys ? tv : ty;
            const bf16* const other = as_keys ? ty : tv;
            const bf16* const mate = as_keys ? tq : tk;
            auto lines = [&](uint32_t(&a)[4], int s, int kk) { load_a(a, own + s * piece_p, LP, w * 16, kk * 16); };
            gemm<NS, kFull3, kFull3, PT / 16, NT / 16, false>(gx, lines, as_keys ? tds : ts, LP, piece_s, 0, 0);
            const float* decay = as_keys ? sm.d.until : sm.d.since;
            const float u0 = decay[row], u1 = decay[row + 8];
#pragma unroll
            for (int nb = 0; nb < NT / 8; ++nb) {
                gx[nb][0] *= u0;
                gx[nb][1] *= u0;
                gx[nb][2] *= u1;
                gx[nb][3] *= u1;
            }
            dots(gx, as_keys ? tk : tq, as_keys ? sm.of_k : sm.of_q);
            const int from = as_keys ? w : 0, to = as_keys ? 4 : w + 1;
#pragma unroll 1
            for (int b = from; b < to; ++b) {
                float dt[2][4] = {};
                gemm<NS, NS, MS, PT / 16, 1, false>(dt, lines, other, LP, piece_p, 0, b * 16);
                decayed(dt, b, as_keys);
                uint32_t a[MS][4];
                split_a<MS>(dt[0], dt[1], a);
                gemm<MS, NS, MS, 1, NT / 16, true>(gx, [&](uint32_t(&r)[4], int s, int) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) r[e] = a[s][e];
                }, mate, LN, piece_n, b * 16, 0);
            }
            const RowsOut<T>& out = as_keys ? dk : dq;
#pragma unroll
            for (int half = 0; half < 2; ++half)
                if (row + 8 * half < rows)
#pragma unroll
                    for (int nb = 0; nb < NT / 8; ++nb)
                        out.put2(row_at + t + row + 8 * half, nb * 8 + 2 * lq, z.n, gx[nb][2 * half], gx[nb][2 * half + 1], pair_qk);
        }
    }
    __syncthreads();
}

template <typename T, int NT, int PT>
bcm_status launch_bwd(const BwdArgs& p, cudaStream_t stream) {
    using Smem = BwdSmem<T, NT, PT>;
    static_assert(sizeof(Smem) <= 227 * 1024, "shared memory of a block");
    static_assert(sizeof(typename Smem::Tiles) >= sizeof(float) * (NT * PT + 4 * NT + kBwdThreads + kBwdThreads / 32), "the state of back_tokens");
    auto kernel = bwd_kernel<T, NT, PT>;
    bcm_status st = allow_smem(kernel, sizeof(Smem));
    if (st != BCM_OK) return st;
    kernel<<<(unsigned)(p.z.items * p.z.heads * p.z.slices), kBwdThreads, sizeof(Smem), stream>>>(p);
    BCM_LAUNCH_CHECK();
    return BCM_OK;
}

// out[e] = sum over the parts, in their order
template <typename T>
__global__ void __launch_bounds__(256) add_parts_kernel(const float* part, int parts, int64_t n, T* out) {
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < n; e += (int64_t)gridDim.x * 256) {
        float s = 0.0f;
#pragma unroll 4
        for (int k = 0; k < parts; ++k) s += part[k * n + e];
        out[e] = from_f32<T>(s);
    }
}

template <typename T>
bcm_status add_parts(const float* part, int parts, int64_t n, T* out, cudaStream_t stream) {
    if (n == 0) return BCM_OK;
    const int64_t blocks = std::min<int64_t>((n + 255) / 256, 16 * sm_count());
    add_parts_kernel<T><<<(unsigned)blocks, 256, 0, stream>>>(part, parts, n, out);
    BCM_LAUNCH_CHECK();
    return BCM_OK;
}

// The gradient of one decay for all of a head's tokens: sums over the rows (rows, heads) in float64, of each block's
// rows first, then of the blocks in their order.
constexpr int kDecayBlocks = 256;
__global__ void __launch_bounds__(256) sum_rows_kernel(const float* x, int64_t rows, int heads, double* out) {
    __shared__ double part[256];
    const int wide = min(heads, 256), deep = 256 / wide, h = threadIdx.x % wide, r0 = threadIdx.x / wide;
    const int64_t per = (rows + kDecayBlocks - 1) / kDecayBlocks, from = blockIdx.x * per, stop = min(rows, from + per);
    for (int h0 = 0; h0 < heads; h0 += wide) {
        double s = 0.0;
        if (r0 < deep && h0 + h < heads)
            for (int64_t r = from + r0; r < stop; r += deep) s += x[r * heads + h0 + h];
        part[threadIdx.x] = s;
        __syncthreads();
        if (r0 == 0 && h0 + h < heads) {
            for (int k = 1; k < deep; ++k) s += part[k * wide + h];
            out[(int64_t)blockIdx.x * heads + h0 + h] = s;
        }
        __syncthreads();
    }
}

__global__ void __launch_bounds__(256) sum_blocks_kernel(const double* x, int heads, float* out) {
    const int h = blockIdx.x * 256 + threadIdx.x;
    if (h >= heads) return;
    double s = 0.0;
    for (int k = 0; k < kDecayBlocks; ++k) s += x[(int64_t)k * heads + h];
    out[h] = (float)s;
}

// What the backward keeps beside the plan's: parts of dq and dk, of dg, and the sums of a fixed decay
struct BwdRoom {
    size_t dq, dk, dg, rows, sums, bytes;
    int shares;
    bool fixed;
};

BwdRoom room_of(const bcm_decay_attn_args* a, const Plan& plan) {
    BwdRoom r{};
    const Sizes& z = plan.z;
    const size_t tokens = (size_t)(z.cu ? 1 : z.batch) * z.seqlen;
    r.shares = z.heads / z.qk_heads * z.slices;
    r.fixed = a->fixed_decay != 0;
    size_t at = plan.bytes;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at = align_up(at + bytes, 256);
        return here;
    };
    if (r.shares > 1) {
        r.dq = take(sizeof(float) * r.shares * tokens * z.qk_heads * z.n);
        r.dk = take(sizeof(float) * r.shares * tokens * z.qk_heads * z.n);
    }
    if (z.slices > 1 || r.fixed) r.dg = take(sizeof(float) * z.slices * tokens * z.heads);
    if (z.slices > 1 && r.fixed) r.rows = take(sizeof(float) * tokens * z.heads);
    if (r.fixed) r.sums = take(sizeof(double) * kDecayBlocks * z.heads);
    r.bytes = at;
    return r;
}

}  // namespace decay_attn
}  // namespace bcm

using namespace bcm;
using namespace bcm::decay_attn;

extern "C" size_t bcm_decay_attn_bwd_workspace_bytes(const bcm_decay_attn_args* a) {
    return check(a, "decay_attn") == BCM_OK ? room_of(a, plan_of(a, true)).bytes : 0;
}

extern "C" bcm_status bcm_decay_attn_bwd(const bcm_decay_attn_args* a, cudaStream_t stream) {
    clear_error();
    bcm_status st = check(a, "decay_attn_bwd");
    if (st != BCM_OK) return st;
    if (a->batch == 0) return BCM_OK;
    Plan plan = plan_of(a, true);
    const Sizes& z = plan.z;
    const BwdRoom room = room_of(a, plan);
    BCM_REQUIRE(a->seqlen == 0 || (a->q && a->k && a->v && a->log_decay && a->dq && a->dk && a->dv && a->ckpt), "decay_attn_bwd: null pointer");
    BCM_REQUIRE(a->dh0 && a->dlog_decay, "decay_attn_bwd: null pointer");
    BCM_REQUIRE(room.bytes == 0 || (a->workspace && a->workspace_bytes >= room.bytes), "decay_attn_bwd: workspace too small");
    BCM_REQUIRE(a->ckpt_bytes >= bcm_decay_attn_ckpt_bytes(a), "decay_attn_bwd: ckpt too small");
    BCM_REQUIRE((int64_t)z.items * z.heads * z.slices < INT32_MAX, "decay_attn_bwd: too many blocks");
    if ((st = fill_tables(plan, a->workspace, stream)) != BCM_OK) return st;
    const Parts parts = parts_of(plan, a->workspace);
    char* const ws = (char*)a->workspace;
    const Rows q = rows_of(a->q, a->q_stride_b, a->q_stride_t, a->q_stride_h), k = rows_of(a->k, a->k_stride_b, a->k_stride_t, a->k_stride_h),
               v = rows_of(a->v, a->v_stride_b, a->v_stride_t, a->v_stride_h), dy = rows_of(a->dy, a->dy_stride_b, a->dy_stride_t, a->dy_stride_h);
    const bool apart = room.shares > 1, dg_parts = z.slices > 1 || room.fixed;
    const int64_t tokens = (int64_t)(z.cu ? 1 : z.batch) * z.seqlen;
    return dispatch(a->dtype, padded_n(a->dim_k), plan.pt, [&](auto type, auto n, auto pt) -> bcm_status {
        using T = decltype(type);
        bcm_status r = BCM_OK;
        if constexpr (sizeof(T) == 4 && n == 128 && pt == 64) {
            set_error("decay_attn_bwd: unplanned tile");
            return BCM_ERR_INVALID_ARGUMENT;
        } else {
            if (plan.cut) {
                // without dy an item's own part is 0: its rows count as none
                PartArgs pa{plan.z, q, dy, a->log_decay, a->g_stride_b, a->g_stride_t, a->g_stride_h, parts};
                if ((r = launch_part<T, n, pt, true>(pa, stream)) != BCM_OK) return r;
                if ((r = join(plan, parts, a->dh_last, true, stream)) != BCM_OK) return r;
            }
            const BwdArgs ba{plan.z, q, k, v, dy, a->log_decay, a->g_stride_b, a->g_stride_t, a->g_stride_h, (const float*)a->ckpt,
                             a->dh_last, parts.state, apart ? (void*)(ws + room.dq) : a->dq, apart ? (void*)(ws + room.dk) : a->dk,
                             a->dv, dg_parts ? (float*)(ws + room.dg) : a->dlog_decay, a->dh0, room.shares};
            if ((r = launch_bwd<T, n, pt>(ba, stream)) != BCM_OK) return r;
            if (apart) {
                const int64_t count = tokens * z.qk_heads * z.n;
                if ((r = add_parts((const float*)(ws + room.dq), room.shares, count, (T*)a->dq, stream)) != BCM_OK) return r;
                if ((r = add_parts((const float*)(ws + room.dk), room.shares, count, (T*)a->dk, stream)) != BCM_OK) return r;
            }
            if (!dg_parts) return BCM_OK;
            const float* rows = (const float*)(ws + room.dg);
            if (z.slices > 1) {
                float* to = room.fixed ? (float*)(ws + room.rows) : a->dlog_decay;
                if ((r = add_parts(rows, z.slices, tokens * z.heads, to, stream)) != BCM_OK) return r;
                rows = to;
            }
            if (room.fixed) {
                sum_rows_kernel<<<kDecayBlocks, 256, 0, stream>>>(rows, tokens, z.heads, (double*)(ws + room.sums));
                BCM_LAUNCH_CHECK();
                sum_blocks_kernel<<<ceil_div(z.heads, 256), 256, 0, stream>>>((const double*)(ws + room.sums), z.heads, a->dlog_decay);
                BCM_LAUNCH_CHECK();
            }
            return BCM_OK;
        }
    });
}
