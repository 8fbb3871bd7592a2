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
    const float* ckpt;         // [chunks][heads][slices][64][NT] transposed states that enter the chunks
    const float* dh_last;      // or NULL
    const float* enter;        // gradients of the states behind the items, where sequences are cut
    void* dq;                  // contiguous; of `shares` blocks a float32 part each where there is more than one
    void* dk;
    void* dv;
    float* dg;                 // of `slices` blocks a part each
    float* dh0;
    int shares;
};

// Four groups of four warps; a warp takes 16 keys (or queries).  The first three decay both products of scores, blocks of
// 16 queries dealt among them, put the pieces of (Q K^T o D)^T into tensor memory and those of (dY V^T o D)^T into shared
// memory (where they serve dk by rows and dq by columns) and sum W for dg; then they finish dv, dk and dq: the far part
// of each is decayed in place and the near part added on top.  The fourth holds the state's gradient and advances it
// meanwhile.
// Bound by the chain of one chunk with one block on an SM (registers, shared and tensor memory are full): 16 x 2048 tokens
// of 8 heads of 64 x 64 bf16 195 us, 11000 clocks a chunk, of which the tensor pipe is active for 2550 (23 %, DRAM 18 %);
// float32 keys of 128 features share one place for the state and its gradient, three more barriers a chunk.
constexpr int kBwdThreads = 512;

template <typename T, int NT>
struct BwdSmem {
    static constexpr int NS = Pieces<T>::in, MS = Pieces<T>::out;
    // Keys of 128 leave no room in tensor memory for the state's increase beside the other sums: there it is formed last,
    // in the scores' place, and its operand takes the place of the scores' pieces.
    static constexpr bool late = NT > 64;
    // and in float32 the state takes the place of its gradient once that has been read
    static constexpr bool one_state = late && NS == 3;
    // Tiles of several pieces or of 128 features are fetched when their chunk begins; held in registers through the chunk
    // behind it they spilled (training of 1 x 30011 tokens of 12 heads of 128 x 64 float16 1373 us, so 1241; 16 x 2048 of 8
    // heads of 64 x 64 float32 473 and 461, float16 389 and 371).  One piece of 64 is fetched ahead (16 x 4096 tokens of
    // such heads bf16 538 us, else 585).
    static constexpr bool now = late || NS > 1;
    struct Tiles {
        bf16 q[NS][Wide<NT>::elements], k[NS][Wide<NT>::elements], v[NS][Wide<kP>::elements], dy[NS][Wide<kP>::elements];
        bf16 ds[kFull3][Wide<NT>::elements], dyw[kFull3][Wide<kP>::elements];
        bf16 s[one_state ? 1 : kFull3][one_state ? 8 : Wide<NT>::elements], dp[late ? 1 : MS][late ? 8 : Wide<kP>::elements];
        __device__ __forceinline__ bf16* state() { return one_state ? ds[0] : s[0]; }
        __device__ __forceinline__ bf16* scores() { return late ? dyw[0] : dp[0]; }
    } tiles;
    Decays d[2];
    // of two chunks
    float pairs[2][4][kChunk]; // [key block][query t]: sum over i >= t in t's block, j < t of W_ij
    float rows[2][4][kChunk];  // [query block][key j]: sum over i of W_ij, blocks behind j's own
    float of_q[2][kChunk], of_k[2][kChunk];
    float across[2][4];        // <S_in, dS> of the warps
    float across_whole[2];     // the chunks' decays (those of the chunk before take their place early)
    Sync<8> sync;

    // tensor memory: both scores, dv, dk, dq, the state's increase, the pieces of the keys' decayed scores (32 columns
    // each).  In float32 with keys of 128 the pieces have to take the scores' place.
    static constexpr bool over = late && MS == 3;
    static constexpr uint32_t at = 0, dt = 64, gv = 128, gk = 192, gq = gk + NT, inc = late ? 0 : gq + NT;
    static constexpr uint32_t piece = over ? 0 : late ? gq + NT : inc + NT, cols = 512;
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
};

// A chunk with an input that is not finite, token by token from its last: a state is run up anew for each (1.75 ms a chunk of
// 64 x 64; forward 0.17 ms).
// `f` (shared): the state's gradient NT x kP, then sums.
template <typename T, int NT>
__device__ __noinline__ void back_tokens(const BwdArgs& p, const T* q, const T* k, const T* v, const T* dy, const float* g, const float* s_in,
                                         const RowsOut<T> dq, const RowsOut<T> dk, T* dv, int64_t dv_st, float* dg, int64_t dg_st,
                                         int rows, int cols, float* f) {
    constexpr int parts = kBwdThreads / kP, warps = kP / 32, all_warps = kBwdThreads / 32;
    const int c = threadIdx.x % kP, part = threadIdx.x / kP, w = threadIdx.x >> 5, l = lane_id();
    float* const sq = f + NT * kP;                 // [warps][NT]
    float* const sk = sq + 2 * NT;
    float* const sv = sk + 2 * NT;                 // [kBwdThreads]
    float* const sg = sv + kBwdThreads;            // [all_warps]
    const bool in = c < cols;
    for (int t = rows - 1; t >= 0; --t) {
        const float a = expf(g[t * p.g_st]);
        const float gy = in && dy ? to_f32(dy[t * p.dy.st + c]) : 0.0f, x = in ? to_f32(v[t * p.v.st + c]) : 0.0f;
        float gv = 0.0f, gg = 0.0f;
        for (int n = part; n < p.z.n; n += parts) {
            float s = in ? s_in[c * NT + n] : 0.0f;
            if (in)
                for (int u = 0; u < t; ++u) s = fmaf(expf(g[u * p.g_st]), s, to_f32(k[u * p.k.st + n]) * to_f32(v[u * p.v.st + c]));
            const float kn = to_f32(k[t * p.k.st + n]), now = fmaf(a, s, kn * x);
            const float ds = f[n * kP + c] + (dy ? to_f32(q[t * p.q.st + n]) * gy : 0.0f);
            float gq = in ? now * gy : 0.0f, gk = in ? ds * x : 0.0f;
            gv = fmaf(ds, kn, gv);
            const float back = a * ds;
            gg += in ? back * s : 0.0f;
            f[n * kP + c] = in ? back : 0.0f;
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
            dq.put(t, n, x0);
            dk.put(t, n, x1);
        }
        if (part == 0 && in) {
            for (int r = 1; r < parts; ++r) gv += sv[r * kP + c];
            dv[t * dv_st + c] = from_f32<T>(gv);
        }
        if (threadIdx.x == 0) {
            for (int r = 1; r < all_warps; ++r) gg += sg[r];
            dg[t * dg_st] = gg;
        }
        __syncthreads();
    }
}

// HALF: float32 copies of float16 operands.  Their third pieces are 0 and dv, dk and dq are rounded to 11 bits
// afterwards, so products with the third pieces are left out (35 of 54 in a chunk remain).
template <typename T, int NT, bool VEC, bool HALF>
__global__ void __launch_bounds__(kBwdThreads) bwd_kernel(const __grid_constant__ BwdArgs p) {
    extern __shared__ unsigned char smem_raw[];
    using Smem = BwdSmem<T, NT>;
    Smem& sm = *(Smem*)tiles_base(smem_raw);
    constexpr int NS = Smem::NS, MS = Smem::MS, NI = HALF ? 2 : NS, MI = HALF ? 2 : MS;       // pieces; those that products take
    const Sizes& z = p.z;
    const int across = z.heads * z.slices, share = z.heads / z.qk_heads;
    const int item = blockIdx.x / across, hs = blockIdx.x % across, h = hs / z.slices, slice = hs % z.slices, col = slice * kP;
    const int cols = min(kP, z.p - col), hq = h / share;
    const int64_t rows_all = (z.cu ? 1 : (int64_t)z.batch) * z.seqlen;
    const int64_t qk_st = (int64_t)z.qk_heads * z.n, v_st = (int64_t)z.heads * z.p;
    const int part = h % share * z.slices + slice;            // of the blocks that share a row of dq
    // rows of dq or dk from `row` on, whole or this block's part of them
    auto rows_out = [&](void* all, int64_t row) {
        RowsOut<T> o{(T*)all + row * qk_st + (int64_t)hq * z.n, nullptr, qk_st};
        if (p.shares > 1) o.part = (float*)all + (part * rows_all + row) * qk_st + (int64_t)hq * z.n;
        return o;
    };
    float* const dg_all = p.dg + slice * rows_all * z.heads + h;
    if (z.cu) {
        const int end = z.tables.seq_item[z.batch + 1];
        zero_rows((T*)p.dv + (int64_t)h * z.p + col, end, z.seqlen, v_st, cols, item, z.items);
        zero_rows(dg_all, end, z.seqlen, z.heads, 1, item, z.items);
        for (void* all : {p.dq, p.dk}) {
            const RowsOut<T> o = rows_out(all, 0);
            if (o.part) zero_rows(o.part, end, z.seqlen, qk_st, z.n, item, z.items);
            else zero_rows(o.whole, end, z.seqlen, qk_st, z.n, item, z.items);
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
    const int np = z.n * z.p;
    const int len = it.t1 - it.t0, nc = (len + kChunk - 1) / kChunk;
    const int warp = t5::warp_id(), l = lane_id(), group = warp >> 2, w = warp & 3, row = w * 16 + (l >> 2), lq = l & 3;
    const bool decay_warp = warp == 13, dg_warp = warp == 14;
    const int p16 = (cols + 15) / 16, n16 = (z.n + 15) / 16;

    const float* const ckpt = p.ckpt + (((int64_t)it.chunk * z.heads + h) * z.slices + slice) * (NT * kP);
    const int64_t ckpt_st = (int64_t)z.heads * z.slices * (NT * kP);
    Pending<T, NT, kBwdThreads, VEC> pq, pk;
    Pending<T, kP, kBwdThreads, VEC> pv, py;
    Pending<float, NT, kBwdThreads, true> ps;
    Logs logs{g, p.g_st};
    sm.sync.init(Smem::cols, 2);
    const uint32_t tm = __shfl_sync(kFull, sm.sync.tmem, 0), lanes = (uint32_t)w << 21;
    enum { kScores, kFarV, kFarK, kFarQ, kInc, kNearV, kNearK, kNearQ };

    // dg of chunk c from what its walk left in shared memory (one warp, tokens 2 lane and 2 lane + 1)
    auto finish_dg = [&](int c) {
        const int t = 2 * l, block = t / 16, rows = min(kChunk, len - c * kChunk);
        const float q0 = sm.of_q[c & 1][t], q1 = sm.of_q[c & 1][t + 1], k0 = sm.of_k[c & 1][t], k1 = sm.of_k[c & 1][t + 1];
        float behind = q0 + q1, before = k0 + k1;
        float r[3];                                           // of the keys up to these two, over a block of queries
#pragma unroll
        for (int ib = 1; ib < 4; ++ib) r[ib - 1] = block < ib ? sm.rows[c & 1][ib][t] + sm.rows[c & 1][ib][t + 1] : 0.0f;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const float a = __shfl_down_sync(kFull, behind, off), b = __shfl_up_sync(kFull, before, off);
            if (l + off < 32) behind += a;
            if (l >= off) before += b;
#pragma unroll
            for (int ib = 0; ib < 3; ++ib) {
                const float e = __shfl_up_sync(kFull, r[ib], off);
                if (l >= off) r[ib] += e;
            }
        }
        float rest = __shfl_down_sync(kFull, behind, 1), past = __shfl_up_sync(kFull, before, 1);
        if (l == 31) rest = 0.0f;
        if (l == 0) past = 0.0f;
        const float through = sm.across_whole[c & 1] * ((sm.across[c & 1][0] + sm.across[c & 1][1]) + (sm.across[c & 1][2] + sm.across[c & 1][3]));
        float d0 = sm.sync.poison(), d1 = d0;                 // (where a wait ran out all gradients are NaN)
        for (int k2 = 0; k2 <= block; ++k2) {
            d0 += sm.pairs[c & 1][k2][t];
            d1 += sm.pairs[c & 1][k2][t + 1];
        }
#pragma unroll
        for (int ib = 1; ib < 4; ++ib) {
            float e = __shfl_up_sync(kFull, r[ib - 1], 1);
            if (l == 0) e = 0.0f;
            if (ib > block) {
                d0 += e;
                d1 += e + sm.rows[c & 1][ib][t];
            }
        }
        d0 += (rest + q1 + q0) + past + through;
        d1 += (rest + q1) + (past + k0) + through;
        if (t < rows) dg[(int64_t)(c * kChunk + t) * z.heads] = d0;
        if (t + 1 < rows) dg[(int64_t)(c * kChunk + t + 1) * z.heads] = d1;
    };
    // a far part: 16 rows of an accumulator times their decays, in place
    auto decay_far = [&](uint32_t acc, int blocks, float f0, float f1, auto&& each) {
#pragma unroll 1
        for (int nb = 0; nb < blocks; ++nb) {
            float x[2][4];
            t5::ld16(x, acc + 16 * nb);
#pragma unroll
            for (int q2 = 0; q2 < 2; ++q2)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[q2][e] *= e < 2 ? f0 : f1;
            each(x, nb);
            t5::st_acc16(acc + 16 * nb, x);
        }
    };

    // Puts chunk c's tiles down, starts the products that need no other and the way of the chunk before it; whether the
    // chunk has to be taken token by token.
    auto start = [&](int c, bool bad, uint32_t phase) {
        const int t = c * kChunk;
        bool slow = false;
        if (c < nc) {
            if (Smem::now) {
                const int r = min(kChunk, len - t);
                pq.fetch(q + t * p.q.st, p.q.st, r, z.n);
                pk.fetch(k + t * p.k.st, p.k.st, r, z.n);
                pv.fetch(v + t * p.v.st, p.v.st, r, cols);
                py.fetch(dy + t * p.dy.st, p.dy.st, dy ? r : 0, cols);
                ps.fetch(ckpt + c * ckpt_st, NT, cols, NT);
            }
            __syncthreads();                                  // decays are there; the chunk behind is done with the tiles
            bad |= pq.bad() | pk.bad() | pv.bad() | py.bad();
            pq.put(sm.tiles.q[0]);
            pk.put(sm.tiles.k[0]);
            pv.put(sm.tiles.v[0]);
            py.put(sm.tiles.dy[0]);
            if (!Smem::one_state) ps.put(sm.tiles.state());
            if (!Smem::late) py.put_weighted(sm.tiles.dyw[0], sm.d[c & 1].since);
            t5::fence_smem();
            t5::fence_before();
            slow = __syncthreads_or(bad);
            if (!slow) {
                // (issuing takes as long as the products: the fourth group has the time for those that are needed later)
                if (w == 0 && t5::elect()) {
                    t5::fence_after();
                    const Operand<NT, true> Q(sm.tiles.q), K(sm.tiles.k), Sk(sm.tiles.ds);
                    const Operand<NT, false> Qt(sm.tiles.q), dS(sm.tiles.ds), S(sm.tiles.state());
                    const Operand<kP, true> V(sm.tiles.v), Y(sm.tiles.dy);
                    if (group == 0) {
                        products<NI, NI, kFull3, NT / 16>(tm + Smem::at, K, Q, t5::instr(kChunk, false, false), false);
                        t5::commit(&sm.sync.bars[kScores]);
                    } else if (group == 1) {
                        products<NI, NI, kFull3, kP / 16>(tm + Smem::dt, V, Y, t5::instr(kChunk, false, false), false);
                        t5::commit(&sm.sync.bars[kScores]);
                    } else if (group == 3) {
                        products<NI, MI, MI, NT / 16>(tm + Smem::gv, K, Sk, t5::instr(p16 * 16, false, false), false);
                        t5::commit(&sm.sync.bars[kFarV]);
                        products<NI, kFull3, kFull3, kP / 16>(tm + Smem::gk, V, dS, t5::instr(n16 * 16, false, true), false);
                        t5::commit(&sm.sync.bars[kFarK]);
                        if (!Smem::one_state) {
                            products<NI, kFull3, kFull3, kP / 16>(tm + Smem::gq, Y, S, t5::instr(n16 * 16, false, true), false);
                            t5::commit(&sm.sync.bars[kFarQ]);
                        }
                        if (!Smem::late) {
                            products<kFull3, NI, kFull3, kChunk / 16>(tm + Smem::inc, Operand<kP, false>(sm.tiles.dyw), Qt, t5::instr(NT, true, true), false);
                            t5::commit(&sm.sync.bars[kInc]);
                        }
                    }
                }
                __syncwarp();
                if (Smem::one_state) {
                    // the state in the place of its gradient, which all products have read by then
                    sm.sync.wait(kFarV, phase);
                    sm.sync.wait(kFarK, phase);
                    ps.put(sm.tiles.state());
                    t5::fence_smem();
                    t5::fence_before();
                    __syncthreads();
                    if (warp == 8 && t5::elect()) {
                        t5::fence_after();
                        const Operand<NT, false> S(sm.tiles.state());
                        const Operand<kP, true> Y(sm.tiles.dy);
                        products<NI, kFull3, kFull3, kP / 16>(tm + Smem::gq, Y, S, t5::instr(n16 * 16, false, true), false);
                        t5::commit(&sm.sync.bars[kFarQ]);
                    }
                    __syncwarp();
                }
            }
        }
        if (!Smem::now && c > 0) {
            const int t2 = t - kChunk, r2 = min(kChunk, len - t2);
            pq.fetch(q + t2 * p.q.st, p.q.st, r2, z.n);
            pk.fetch(k + t2 * p.k.st, p.k.st, r2, z.n);
            pv.fetch(v + t2 * p.v.st, p.v.st, r2, cols);
            py.fetch(dy + t2 * p.dy.st, p.dy.st, dy ? r2 : 0, cols);
            ps.fetch(ckpt + (c - 1) * ckpt_st, NT, cols, NT);
        }
        return slow;
    };
    auto walk = [&](int c) {
        const int t = c * kChunk;
        back_tokens<T, NT>(p, q + t * p.q.st, k + t * p.k.st, v + t * p.v.st, dy ? dy + t * p.dy.st : nullptr, g + t * p.g_st, ckpt + c * ckpt_st,
                           rows_out(p.dq, row_at + t), rows_out(p.dk, row_at + t), dv + t * v_st, v_st, dg + (int64_t)t * z.heads, z.heads,
                           min(kChunk, len - t), cols, (float*)&sm.tiles);
    };
    uint32_t phase = 0;
    if (group == 3) {
        State<NT, 1> ds(0);
        bool bad_logs = false, pending = false;               // pending: the chunk behind has its dg still to be finished
        const float* from = it.last ? (p.dh_last ? p.dh_last + ((int64_t)it.seq * z.heads + h) * np : nullptr)
                                    : p.enter + ((int64_t)item * z.heads + h) * np;
        if (decay_warp) logs.fetch((nc - 1) * kChunk, len);
        if (from) ds.load(from + col, z.n, cols, z.p);
        else ds.zero();
        ds.template put<kFull3, !Smem::late>(sm.tiles.ds[0]);
        if (decay_warp) {
            bad_logs = logs.bad();
            decays_of(sm.d[(nc - 1) & 1], logs.a, logs.b);
            logs.fetch((nc - 2) * kChunk, len);
        }
        for (int c = nc; c >= 0; --c) {
            const int t = c * kChunk;
            const bool slow = start(c, bad_logs, phase);
            if (c == nc) continue;
            if (pending && dg_warp) finish_dg(c + 1);
            pending = !slow;
            const Decays& d = sm.d[c & 1];
            if (slow) {
                // token by token, through shared memory
                float* f = (float*)&sm.tiles;
                const float none = sm.sync.poison();
                ds.pairs([&](float& x0, float& x1, int pp, int n) {
                    f[n * kP + pp] = x0 + none;
                    f[(n + 1) * kP + pp] = x1 + none;
                });
                __syncthreads();
                walk(c);
                ds.pairs([&](float& x0, float& x1, int pp, int n) {
                    x0 = f[n * kP + pp];
                    x1 = f[(n + 1) * kP + pp];
                });
                __syncthreads();                              // all have theirs back before the pieces take the place
            }
            if (decay_warp && c > 0) {
                bad_logs = logs.bad();
                decays_of(sm.d[(c - 1) & 1], logs.a, logs.b);
                logs.fetch((c - 2) * kChunk, len);
            }
            if (!slow) {
                float x = 0.0f;
                ds.pairs([&](float& x0, float& x1, int pp, int n) {
                    const float2 in = from_pieces<kFull3>(sm.tiles.state() + Wide<NT>::at(pp, n), Wide<NT>::elements);
                    x = fmaf(in.x, x0, fmaf(in.y, x1, x));
                });
#pragma unroll
                for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(kFull, x, o);
                if (l == 0) sm.across[c & 1][w] = x;
                if (threadIdx.x == 384) sm.across_whole[c & 1] = d.whole;
                if (Smem::late) {
                    // behind all other products of the chunk
                    for (int b = kNearV; b <= kNearQ; ++b) sm.sync.wait(b, phase);
                    for (int i = threadIdx.x - 384; i < 64 * 8; i += 128) {
                        const int r = i / 8, e = Wide<kP>::at(r, i % 8 * 8);
                        uint32_t a[4][kFull3];
#pragma unroll
                        for (int k2 = 0; k2 < 4; ++k2) {
                            const float2 in = from_pieces<NS>(sm.tiles.dy[0] + e + 2 * k2, Wide<kP>::elements);
                            split<kFull3>(in.x * d.since[r], in.y * d.since[r], a[k2]);
                        }
#pragma unroll
                        for (int s = 0; s < kFull3; ++s) *(uint4*)(sm.tiles.dyw[s] + e) = make_uint4(a[0][s], a[1][s], a[2][s], a[3][s]);
                    }
                    t5::fence_smem();
                    t5::fence_before();
                    named_sync(2, 128);
                    if (warp == 12 && t5::elect()) {
                        t5::fence_after();
                        const Operand<kP, false> Yw(sm.tiles.dyw);
                        const Operand<NT, false> Qt(sm.tiles.q);
                        products<kFull3, NI, kFull3, kChunk / 16>(tm + Smem::inc, Yw, Qt, t5::instr(NT, true, true), false);
                        t5::commit(&sm.sync.bars[kInc]);
                    }
                    __syncwarp();
                }
                sm.sync.wait(kInc, phase);
                ds.advance(tm + Smem::inc + lanes, d.whole);
                sm.sync.wait(kFarV, phase);                   // the products with the gradient (and the state) have read it
                sm.sync.wait(kFarK, phase);
                if (Smem::one_state) sm.sync.wait(kFarQ, phase);
                t5::fence_before();
                if (Smem::one_state) named_sync(2, 128);      // (and this group the state, for its dot)
                phase ^= 1;
            }
            ds.template put<kFull3, !Smem::late>(sm.tiles.ds[0]);
        }
        __syncthreads();
        if (pending && dg_warp) finish_dg(0);
        if (sm.sync.failed) ds.pairs([](float& x, float& y1, int, int) { x = y1 = __int_as_float(0x7fc00000); });
        if (it.first) ds.store(p.dh0 + ((int64_t)it.seq * z.heads + h) * np + col, z.n, cols, z.p);
        sm.sync.end(Smem::cols);
        return;
    }

    for (int c = nc; c >= 0; --c) {
        const int t = c * kChunk, rows = min(kChunk, len - t);
        const bool slow = start(c, false, phase);
        if (c == nc) continue;
        if (slow) {
            __syncthreads();
            walk(c);
            __syncthreads();
            continue;
        }
        const Decays& d = sm.d[c & 1];
        // ---- scores: this warp's block of queries, and a block of zeros before the keys
        const float hi0 = d.hi[row], lo0 = d.lo[row], hi1 = d.hi[row + 8], lo1 = d.lo[row + 8], u0 = d.until[row], u1 = d.until[row + 8];
        bf16* const dp = sm.tiles.scores();
        auto put_block = [&](int ib, const uint32_t(&r)[2][2][MS], const uint32_t(&r2)[2][2][MS]) {
#pragma unroll
            for (int m = 0; m < MS; ++m) {
                t5::st16(tm + Smem::piece + lanes + 32 * m + 8 * ib, r[0][0][m], r[0][1][m], r[1][0][m], r[1][1][m]);
#pragma unroll
                for (int q2 = 0; q2 < 2; ++q2)
#pragma unroll
                    for (int half = 0; half < 2; ++half)
                        *(uint32_t*)(dp + m * Wide<kP>::elements + Wide<kP>::at(row + 8 * half, ib * 16 + q2 * 8 + 2 * lq)) = r2[q2][half][m];
            }
        };
        auto block = [&](int ib, float(&at)[2][4], float(&dt)[2][4]) {
            uint32_t r[2][2][MS], r2[2][2][MS];
            float W[2][2][2], sum[2][2] = {};                 // sum: of the four columns, over this warp's keys before them
#pragma unroll
            for (int q2 = 0; q2 < 2; ++q2) {
                const int i = ib * 16 + q2 * 8 + 2 * lq;
                const float2 hi = *(const float2*)&d.hi[i], lo = *(const float2*)&d.lo[i];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool in = i + (e & 1) >= row + (e & 2) * 4;
                    const float f = between(e & 1 ? hi.y : hi.x, e & 1 ? lo.y : lo.x, e & 2 ? hi1 : hi0, e & 2 ? lo1 : lo0);
                    float &a = at[q2][e], &b = dt[q2][e];
                    a = in ? a * f : 0.0f;
                    W[e >> 1][q2][e & 1] = in ? a * b : 0.0f;
                    b = in ? b * f : 0.0f;
                }
                split<MS>(at[q2][0], at[q2][1], r[q2][0]);
                split<MS>(at[q2][2], at[q2][3], r[q2][1]);
                split<MS>(dt[q2][0], dt[q2][1], r2[q2][0]);
                split<MS>(dt[q2][2], dt[q2][3], r2[q2][1]);
            }
            put_block(ib, r, r2);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int j = row + 8 * half, i = ib * 16 + 2 * lq;
                float ex[2], all[2];                          // of the lanes behind this one, of all four
#pragma unroll
                for (int q2 = 0; q2 < 2; ++q2) {
                    float s = W[half][q2][0] + W[half][q2][1];
                    float o = __shfl_down_sync(kFull, s, 1, 4);
                    if (lq < 3) s += o;
                    o = __shfl_down_sync(kFull, s, 2, 4);
                    if (lq < 2) s += o;
                    o = __shfl_down_sync(kFull, s, 1, 4);
                    ex[q2] = lq < 3 ? o : 0.0f;
                    all[q2] = __shfl_sync(kFull, s, 0, 4);
                }
                float u = ex[1] + W[half][1][1];
                if (j < i + 9) sum[1][1] += u;
                u += W[half][1][0];
                if (j < i + 8) sum[1][0] += u;
                u = all[1] + ex[0] + W[half][0][1];
                if (j < i + 1) sum[0][1] += u;
                u += W[half][0][0];
                if (j < i) sum[0][0] += u;
                if (lq == 0) sm.rows[c & 1][ib][j] = all[0] + all[1];
            }
#pragma unroll
            for (int q2 = 0; q2 < 2; ++q2)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) sum[q2][e] += __shfl_xor_sync(kFull, sum[q2][e], o);
                    if (l < 4) sm.pairs[c & 1][w][ib * 16 + q2 * 8 + 2 * lq + e] = sum[q2][e];
                }
        };
        // the first quarter has four blocks for three warps
        const int blocks_here = w + group > 3 ? 0 : w == 0 && group == 0 ? 2 : 1;
        auto load = [&](int ib, float(&at)[2][4], float(&dt)[2][4]) {
            t5::ld16x2(at, tm + Smem::at + lanes + 16 * ib, dt, tm + Smem::dt + lanes + 16 * ib);
        };
        sm.sync.wait(kScores, phase);
        if constexpr (Smem::over) {
            float at[2][4], dt[2][4], at2[2][4], dt2[2][4];
            if (blocks_here > 0) load(w + group, at, dt);
            if (blocks_here > 1) load(3, at2, dt2);
            t5::fence_before();
            named_sync(1, 384);
            t5::fence_after();
            if (blocks_here > 0) block(w + group, at, dt);
            if (blocks_here > 1) block(3, at2, dt2);
        } else {
#pragma unroll 1
            for (int n = 0; n < blocks_here; ++n) {
                const int ib = n ? 3 : w + group;
                float at[2][4], dt[2][4];
                load(ib, at, dt);
                block(ib, at, dt);
            }
        }
        if (group < w) {
            const uint32_t none[2][2][MS] = {};
            put_block(group, none, none);
        }
        t5::fence_smem();

        // ---- far parts; those of dk and dq leave their dots with the row itself for dg
        float dot0 = 0.0f, dot1 = 0.0f;
        const uint32_t acc = tm + (group == 0 ? Smem::gv : group == 1 ? Smem::gk : Smem::gq) + lanes;
        sm.sync.wait(kFarV + group, phase);
        if (group == 0) {
            decay_far(acc, p16, u0, u1, [](float(&)[2][4], int) {});
        } else {
            const bf16* const self = group == 1 ? sm.tiles.k[0] : sm.tiles.q[0];
            decay_far(acc, n16, group == 1 ? u0 : d.since[row], group == 1 ? u1 : d.since[row + 8], [&](float(&x)[2][4], int nb) {
#pragma unroll
                for (int q2 = 0; q2 < 2; ++q2) {
                    const int n = 16 * nb + 8 * q2 + 2 * lq;
                    const float2 k0 = from_pieces<NS>(self + Wide<NT>::at(row, n), Wide<NT>::elements);
                    const float2 k1 = from_pieces<NS>(self + Wide<NT>::at(row + 8, n), Wide<NT>::elements);
                    dot0 = fmaf(k0.x, x[q2][0], fmaf(k0.y, x[q2][1], dot0));
                    dot1 = fmaf(k1.x, x[q2][2], fmaf(k1.y, x[q2][3], dot1));
                }
            });
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                dot0 += __shfl_xor_sync(kFull, dot0, o);
                dot1 += __shfl_xor_sync(kFull, dot1, o);
            }
            if (lq == 0) {
                float* out = group == 1 ? sm.of_k[c & 1] : sm.of_q[c & 1];
                out[row] = dot0;
                out[row + 8] = dot1;
            }
        }
        t5::wait_st();
        t5::fence_before();
        named_sync(1, 384);
        if (w == 0 && t5::elect()) {
            t5::fence_after();
            const Operand<NT, false> Qt(sm.tiles.q), Kt(sm.tiles.k);
            const Operand<kP, true> P(sm.tiles.scores());
            const Operand<kP, false> Yt(sm.tiles.dy), Pt(sm.tiles.scores());
            if (group == 0)
                products<MI, NI, MI, kChunk / 16>(tm + Smem::gv, [&](int s, int i) { return tm + Smem::piece + 32 * s + 8 * i; }, Yt,
                                                  t5::instr(p16 * 16, false, true), true);
            else if (group == 1)
                products<MI, NI, MI, kChunk / 16>(tm + Smem::gk, P, Qt, t5::instr(n16 * 16, false, true), true);
            else
                products<MI, NI, MI, kChunk / 16>(tm + Smem::gq, Pt, Kt, t5::instr(n16 * 16, true, true), true);
            t5::commit(&sm.sync.bars[kNearV + group]);
        }
        __syncwarp();
        sm.sync.wait(kNearV + group, phase);
        // (a wait lost by another warp is known by now: what it held up is awaited behind the barrier above)
        const float none = sm.sync.poison();
        // ---- out: dv, or (whole or as a part) dk and dq
        const RowsOut<T> o = group == 0 ? RowsOut<T>{dv + t * v_st, nullptr, v_st} : rows_out(group == 1 ? p.dk : p.dq, row_at + t);
        const int width = group == 0 ? cols : z.n, blocks = group == 0 ? p16 : n16;
#pragma unroll 1
        for (int nb = 0; nb < blocks; nb += 2) {
            float x[2][4], x2[2][4];
            t5::ld16x2(x, acc + 16 * nb, x2, acc + 16 * min(nb + 1, blocks - 1));
            if (none != 0.0f) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e >> 2][e & 3] = x2[e >> 2][e & 3] = none;
            }
            if (o.part) {
                store_rows<VEC>(o.part, o.st, rows, width, row, 16 * nb, x[0], x[1]);
                store_rows<VEC>(o.part, o.st, rows, width, row, 16 * nb + 16, x2[0], x2[1]);
            } else {
                store_rows<VEC>(o.whole, o.st, rows, width, row, 16 * nb, x[0], x[1]);
                store_rows<VEC>(o.whole, o.st, rows, width, row, 16 * nb + 16, x2[0], x2[1]);
            }
        }
        t5::fence_before();
        phase ^= 1;
    }
    __syncthreads();
    sm.sync.end(Smem::cols);
}

template <typename T, int NT, bool HALF>
bcm_status launch_bwd(const BwdArgs& p, bool vec, cudaStream_t stream) {
    using Smem = BwdSmem<T, NT>;
    constexpr size_t smem = sizeof(Smem) + 1024;
    static_assert(smem <= 227 * 1024, "shared memory of a block");
    static_assert(sizeof(typename Smem::Tiles) >= sizeof(float) * (NT * kP + 4 * NT + kBwdThreads + kBwdThreads / 32), "the state of back_tokens");
    static_assert(Smem::gq + NT <= 512 && Smem::piece + 32 * Smem::MS <= 512, "tensor memory of a block");
    auto kernel = vec ? bwd_kernel<T, NT, true, HALF> : bwd_kernel<T, NT, false, HALF>;
    bcm_status st = allow_smem(kernel, smem);
    if (st != BCM_OK) return st;
    kernel<<<(unsigned)(p.z.items * p.z.heads * p.z.slices), kBwdThreads, smem, stream>>>(p);
    BCM_LAUNCH_CHECK();
    return BCM_OK;
}

// out[e] = sum over the parts, in their order; V elements at a time
template <typename T, int V>
__global__ void __launch_bounds__(256) add_parts_kernel(const float* part, int parts, int64_t n, T* out) {
    for (int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V; e < n; e += (int64_t)gridDim.x * 256 * V) {
        float s[V] = {};
#pragma unroll 4
        for (int k = 0; k < parts; ++k) {
            float x[V];
            if constexpr (V == 4) *(float4*)x = *(const float4*)(part + k * n + e);
            else x[0] = part[k * n + e];
#pragma unroll
            for (int i = 0; i < V; ++i) s[i] += x[i];
        }
        struct alignas(V * sizeof(T)) Out { T v[V]; } o;
#pragma unroll
        for (int i = 0; i < V; ++i) o.v[i] = from_f32<T>(s[i]);
        *(Out*)(out + e) = o;
    }
}

template <typename T>
bcm_status add_parts(const float* part, int parts, int64_t n, T* out, cudaStream_t stream) {
    if (n == 0) return BCM_OK;
    const bool four = n % 4 == 0 && (((uintptr_t)part | (uintptr_t)out) & 15) == 0;
    const int64_t turns = four ? n / 4 : n, blocks = std::min<int64_t>((turns + 255) / 256, 16 * sm_count());
    if (four) add_parts_kernel<T, 4><<<(unsigned)blocks, 256, 0, stream>>>(part, parts, n, out);
    else add_parts_kernel<T, 1><<<(unsigned)blocks, 256, 0, stream>>>(part, parts, n, out);
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

// float32 copies of strided float16 rows (tokens, heads, width), contiguous: a warp per token, V elements a lane
template <int V>
__global__ void __launch_bounds__(256) widen_kernel(const __grid_constant__ Rows in, int64_t tokens, int64_t seqlen, int heads, int width, float* out) {
    const int per = width / V, n = heads * per;
    for (int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); t < tokens; t += (int64_t)gridDim.x * 8) {
        const int64_t b = t / seqlen;
        const __half* from = (const __half*)in.p + b * in.sb + (t - b * seqlen) * in.st;
        float* to = out + t * heads * width;
#pragma unroll 4
        for (int i = lane_id(); i < n; i += 32) {
            const int h = i / per, c = (i - h * per) * V;
            struct alignas(V * 2) In { __half v[V]; };
            const In x = *(const In*)(from + h * in.sh + c);
            struct alignas(V * 4 < 16 ? V * 4 : 16) Out { float v[V]; } y;
#pragma unroll
            for (int e = 0; e < V; ++e) y.v[e] = to_f32(x.v[e]);
            *(Out*)(to + (int64_t)h * width + c) = y;
        }
    }
}

// What the backward keeps beside the plan's: parts of dq and dk, of dg, and the sums of a fixed decay
struct BwdRoom {
    size_t dq, dk, dg, rows, sums, wide[5], bytes;
    int shares;
    bool fixed, widen;
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
    if (r.shares > 1 || (a->dtype == BCM_F16 && z.n > 64)) {
        r.dq = take(sizeof(float) * r.shares * tokens * z.qk_heads * z.n);
        r.dk = take(sizeof(float) * r.shares * tokens * z.qk_heads * z.n);
    }
    if (z.slices > 1 || r.fixed) r.dg = take(sizeof(float) * z.slices * tokens * z.heads);
    if (z.slices > 1 && r.fixed) r.rows = take(sizeof(float) * tokens * z.heads);
    if (r.fixed) r.sums = take(sizeof(double) * kDecayBlocks * z.heads);
    // float16 keys of more than 64 features are taken as float32, whose operands share places in shared memory: two
    // pieces of every operand beside two whole states would take all of it
    r.widen = a->dtype == BCM_F16 && z.n > 64;
    if (r.widen) {
        for (int i = 0; i < 2; ++i) r.wide[i] = take(sizeof(float) * tokens * z.qk_heads * z.n);
        for (int i = 2; i < 5; ++i) r.wide[i] = take(sizeof(float) * tokens * z.heads * z.p);
    }
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
    if (a->batch == 0) {
        if (a->fixed_decay && a->dlog_decay) BCM_CUDA_TRY(cudaMemsetAsync(a->dlog_decay, 0, sizeof(float) * a->heads, stream));
        return BCM_OK;
    }
    Plan plan = plan_of(a, true);
    const Sizes& z = plan.z;
    const BwdRoom room = room_of(a, plan);
    BCM_REQUIRE(a->seqlen == 0 || (a->q && a->k && a->v && a->log_decay && a->dq && a->dk && a->dv && a->ckpt), "decay_attn_bwd: null pointer");
    BCM_REQUIRE(a->dh0 && (a->dlog_decay || (a->seqlen == 0 && !a->fixed_decay)), "decay_attn_bwd: null pointer");   // (empty: no address)
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
    const bool vec = aligned(a, true);
    return dispatch(a->dtype, a->dim_k, [&](auto type, auto n) -> bcm_status {
        using T = decltype(type);
        bcm_status r = BCM_OK;
        constexpr bool widen = std::is_same<T, __half>::value && n > 64;
        using K = typename std::conditional<widen, float, T>::type;         // what the walk reads and writes
        Rows in[4] = {q, k, v, dy};
        void* dv = a->dv;
        if constexpr (widen) {
            for (int i = 0; i < (dy.p ? 4 : 3); ++i) {                          // (no dy stays none)
                const int heads = i < 2 ? z.qk_heads : z.heads, width = i < 2 ? z.n : z.p;
                float* const to = (float*)(ws + room.wide[i]);
                if (tokens > 0) {
                    const unsigned blocks = (unsigned)std::min<int64_t>((tokens + 7) / 8, 8 * sm_count());
                    if (vec) widen_kernel<8><<<blocks, 256, 0, stream>>>(in[i], tokens, z.seqlen, heads, width, to);
                    else widen_kernel<1><<<blocks, 256, 0, stream>>>(in[i], tokens, z.seqlen, heads, width, to);
                    BCM_LAUNCH_CHECK();
                }
                in[i] = rows_of(ws + room.wide[i], (int64_t)z.seqlen * heads * width, (int64_t)heads * width, width);
            }
            dv = ws + room.wide[4];
        }
        const bool in_ws = apart || widen;
        if (plan.cut) {
            // without dy an item's own part is 0: its rows count as none
            PartArgs pa{plan.z, in[0], in[3], a->log_decay, a->g_stride_b, a->g_stride_t, a->g_stride_h, parts};
            if ((r = launch_part<K, n, true>(pa, widen ? a->dim_k % 8 == 0 && a->dim_v % 8 == 0 : vec, stream)) != BCM_OK) return r;
            if ((r = join(plan, parts, a->dh_last, true, stream)) != BCM_OK) return r;
        }
        const BwdArgs ba{plan.z, in[0], in[1], in[2], in[3], a->log_decay, a->g_stride_b, a->g_stride_t, a->g_stride_h, (const float*)a->ckpt,
                         a->dh_last, parts.state, in_ws ? (void*)(ws + room.dq) : a->dq, in_ws ? (void*)(ws + room.dk) : a->dk, dv,
                         dg_parts ? (float*)(ws + room.dg) : a->dlog_decay, a->dh0, room.shares};
        if ((r = launch_bwd<K, n, widen>(ba, widen ? a->dim_k % 8 == 0 && a->dim_v % 8 == 0 : vec, stream)) != BCM_OK) return r;
        if (in_ws) {
            const int64_t count = tokens * z.qk_heads * z.n;
            if ((r = add_parts((const float*)(ws + room.dq), room.shares, count, (T*)a->dq, stream)) != BCM_OK) return r;
            if ((r = add_parts((const float*)(ws + room.dk), room.shares, count, (T*)a->dk, stream)) != BCM_OK) return r;
        }
        if constexpr (widen) {
            if ((r = add_parts((const float*)dv, 1, tokens * z.heads * z.p, (T*)a->dv, stream)) != BCM_OK) return r;
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
    });
}
