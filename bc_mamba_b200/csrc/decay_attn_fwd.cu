// decay_attn_fwd.cu — linear attention with a decay for each head: plan of a call, forward walk, one-token step.
#include "decay_attn.cuh"

namespace bcm {
namespace decay_attn {

bcm_status check(const bcm_decay_attn_args* a, const char* what) {
    BCM_REQUIRE(a != nullptr, "%s: null arguments", what);
    BCM_REQUIRE(dtype_ok(a->dtype), "%s: unsupported dtype %d", what, (int)a->dtype);
    BCM_REQUIRE(a->batch >= 0 && a->seqlen >= 0 && a->heads >= 1 && a->qk_heads >= 1 && a->dim_k >= 1 && a->dim_v >= 1,
                "%s: bad sizes", what);
    BCM_REQUIRE(a->dim_k <= BCM_DECAY_ATTN_MAX_DIM_K, "%s: a query of more than %d features", what, BCM_DECAY_ATTN_MAX_DIM_K);
    BCM_REQUIRE(a->batch > 0 || a->seqlen == 0 || !a->cu_seqlens, "%s: offsets of no sequence with tokens", what);
    BCM_REQUIRE(a->heads % a->qk_heads == 0, "%s: heads must be a multiple of the queries' heads", what);
    BCM_REQUIRE(a->dim_v <= (1 << 20) && a->heads <= (1 << 20) && a->batch < (1 << 24) && a->seqlen < INT32_MAX - 4096, "%s: sizes too large", what);
    BCM_REQUIRE(on_16(a->ckpt, 0) && on_16(a->workspace, 0), "%s: ckpt and workspace must be aligned to 16 bytes", what);
    BCM_REQUIRE(a->heads * a->dim_v <= (1 << 24) && a->batch * (a->seqlen / kChunk + 1) < INT32_MAX, "%s: sizes too large", what);
    return BCM_OK;
}

// Blocks are (item, head, 64 columns of the values) and walk their item's chunks one after another.  Sequences are cut
// into items only where whole ones leave much of the GPU without a block: an item costs one more pass over two inputs
// and states to join.  The border, half a block to an SM, is that of training (16 x 4096 tokens of 8 heads of 64 x 64 bf16,
// 128 blocks, uncut 537 us with its backward, cut in two 674; 12 x 4096, 96 blocks, 532 and 648).  A forward alone, whose
// walks are two to an SM, loses by it behind the border: 1 x 65536 tokens of 75, 80, 112 and 148 such heads take 2610 us
// uncut and would take 1418, 1426, 1968 and 2363 cut; 1 x 4096 tokens 178 us uncut and 133, 135, 166 and 193.  An item has
// 256 tokens at least.  `room` blocks are two turns of the walks, whose blocks one or two to an SM hold, and one of the
// parts', four to an SM (one turn of the walks against two: 1 x 65536 tokens of 32 such heads 627 and 574 us, forward and
// backward of 1 x 30011 of 12 heads 518 and 488 us).  A packed batch is cut by its total, since only the device knows its
// lengths: of many short sequences none has a second item, the parts' blocks end at once and the join copies entering
// states that nothing reads.
Plan plan_of(const bcm_decay_attn_args* a, bool backward) {
    Plan plan{};
    Sizes& z = plan.z;
    z.batch = (int)a->batch;
    z.heads = (int)a->heads;
    z.qk_heads = (int)a->qk_heads;
    z.n = (int)a->dim_k;
    z.p = (int)a->dim_v;
    z.seqlen = (int)a->seqlen;
    z.cu = a->cu_seqlens;
    z.slices = ceil_div(z.p, kP);
    const int64_t across = (int64_t)z.heads * z.slices, room = (backward ? 2 : 4) * sm_count();
    const int64_t tokens = a->seqlen;
    auto chunks_up = [](int64_t v) { return std::max<int64_t>(256, (v + kChunk - 1) / kChunk * kChunk); };
    if (!z.cu) {
        const int64_t blocks = std::max<int64_t>(1, z.batch * across), segs = blocks * 2 > sm_count() ? 1 : room / blocks;
        z.span = (int)chunks_up((tokens + segs - 1) / segs);
        z.per_seq = std::max(1, ceil_div(tokens, z.span));
        z.items = z.batch * z.per_seq;
        z.chunks = z.batch * ceil_div(tokens, kChunk);
        plan.cut = z.per_seq > 1;
    } else {
        z.span = (int)chunks_up((tokens * across + 2 * room - 1) / (2 * room));
        z.per_seq = 0;
        z.items = z.batch + (int)(tokens / z.span);
        z.chunks = z.batch + (int)(tokens / kChunk);
        plan.cut = tokens > z.span;
    }
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at = align_up(at + bytes, 256);
        return here;
    };
    if (z.cu) {
        plan.items_at = take(sizeof(Item) * (size_t)z.items);
        plan.seq_at = take(sizeof(int) * ((size_t)z.batch + 2));
    }
    if (plan.cut) {
        plan.state_at = take(sizeof(float) * (size_t)z.items * z.heads * z.n * z.p);
        plan.whole_at = take(sizeof(float) * (size_t)z.items * z.heads);
    }
    plan.bytes = at;
    return plan;
}

bool aligned(const bcm_decay_attn_args* a, bool backward) {
    const int64_t size = (int64_t)dtype_size(a->dtype);
    auto in = [&](const void* p, int64_t sb, int64_t st, int64_t sh) { return on_16(p, sb * size) && on_16(p, st * size) && on_16(p, sh * size); };
    if (a->dim_k % 8 || a->dim_v % 8 || !in(a->q, a->q_stride_b, a->q_stride_t, a->q_stride_h) ||
        !in(a->k, a->k_stride_b, a->k_stride_t, a->k_stride_h) || !in(a->v, a->v_stride_b, a->v_stride_t, a->v_stride_h))
        return false;
    if (!backward) return on_16(a->y, 0);
    return in(a->dy, a->dy_stride_b, a->dy_stride_t, a->dy_stride_h) && on_16(a->dq, 0) && on_16(a->dk, 0) && on_16(a->dv, 0);
}

Parts parts_of(const Plan& plan, void* workspace) {
    char* ws = (char*)workspace;
    return plan.cut ? Parts{(float*)(ws + plan.state_at), (float*)(ws + plan.whole_at)} : Parts{nullptr, nullptr};
}

// One block.  Offsets are bounded to the rows and made ascending (a maximum over those before), so that tables of any
// offsets hold rows that exist, and not more items than there is room for.
__global__ void __launch_bounds__(1024) tables_kernel(Sizes z) {
    __shared__ int part[3][32];
    __shared__ int carry[3];
    const int l = lane_id(), w = threadIdx.x >> 5;
    if (threadIdx.x < 3) carry[threadIdx.x] = 0;
    __syncthreads();
    for (int base = 0; base < z.batch; base += 1024) {
        const int s = base + threadIdx.x;
        const bool in = s < z.batch;
        // the highest offset up to this sequence's end
        int end = in ? min(max(z.cu[s + 1], 0), z.seqlen) : 0;
        end = warp_inclusive_max(end);
        if (l == 31) part[0][w] = end;
        __syncthreads();
        int before = carry[0];
        if (base == 0) before = max(before, min(max(z.cu[0], 0), z.seqlen));
        for (int k = 0; k < w; ++k) before = max(before, part[0][k]);
        const int up = __shfl_up_sync(kFull, end, 1);
        const int start = max(before, l ? up : 0);
        end = max(before, end);
        const int len = end - start;
        const int items = in ? (len > 0 ? (len - 1) / z.span + 1 : 1) : 0, chunks = in ? (len + kChunk - 1) / kChunk : 0;
        const int si = warp_inclusive_sum(items), sc = warp_inclusive_sum(chunks);
        if (l == 31) {
            part[1][w] = si;
            part[2][w] = sc;
        }
        __syncthreads();
        int item = carry[1] + si - items, chunk = carry[2] + sc - chunks;
        for (int k = 0; k < w; ++k) {
            item += part[1][k];
            chunk += part[2][k];
        }
        if (in) {
            z.tables.seq_item[s] = item;
            for (int k = 0; k < items; ++k) {
                const int t0 = start + k * z.span;
                z.tables.items[item + k] = Item{s, t0, t0 + min(z.span, end - t0), chunk + k * (z.span / kChunk), k == 0, k == items - 1};
            }
        }
        __syncthreads();
        if (threadIdx.x == 1023) {
            carry[0] = end;
            carry[1] = item + items;
            carry[2] = chunk + chunks;
        }
        __syncthreads();
    }
    for (int i = carry[1] + threadIdx.x; i < z.items; i += 1024) z.tables.items[i].seq = -1;
    if (threadIdx.x == 0) {
        z.tables.seq_item[z.batch] = carry[1];
        z.tables.seq_item[z.batch + 1] = carry[0];
    }
}

bcm_status fill_tables(Plan& plan, void* workspace, cudaStream_t stream) {
    if (!plan.z.cu) return BCM_OK;
    char* ws = (char*)workspace;
    plan.z.tables = Tables{(Item*)(ws + plan.items_at), (int*)(ws + plan.seq_at)};
    tables_kernel<<<1, 1024, 0, stream>>>(plan.z);
    BCM_LAUNCH_CHECK();
    return BCM_OK;
}

// A thread per element of a head's state goes along the items of its sequence.
__global__ void __launch_bounds__(256) join_kernel(Sizes z, Parts parts, const float* end, bool backward) {
    const int np = z.n * z.p, blocks = (np + 255) / 256;
    const int sh = blockIdx.x / blocks, e = blockIdx.x % blocks * 256 + threadIdx.x;
    const int seq = sh / z.heads, h = sh % z.heads;
    if (e >= np) return;
    const int first = z.cu ? z.tables.seq_item[seq] : seq * z.per_seq, stop = z.cu ? z.tables.seq_item[seq + 1] : first + z.per_seq;
    float s = end ? end[(int64_t)sh * np + e] : 0.0f;
    const int count = stop - first;
    // the last of the walk has no part.  Eight items' loads are under way together: one after another they took 34 us
    // for 9 items of 32 heads of 64 x 64.
    constexpr int kAhead = 8;
    for (int k0 = 0; k0 < count - 1; k0 += kAhead) {
        float own[kAhead], whole[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (k0 + j < count - 1) {
                const int64_t at = (int64_t)(backward ? stop - 1 - k0 - j : first + k0 + j) * z.heads + h;
                own[j] = parts.state[at * np + e];
                whole[j] = parts.whole[at];
            }
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            if (k0 + j < count - 1) {
                const int64_t at = (int64_t)(backward ? stop - 1 - k0 - j : first + k0 + j) * z.heads + h;
                parts.state[at * np + e] = s;
                s = fmaf(whole[j], s, own[j]);
            }
        }
    }
    if (count > 0) parts.state[((int64_t)(backward ? first : stop - 1) * z.heads + h) * np + e] = s;
}

bcm_status join(const Plan& plan, const Parts& parts, const float* end, bool backward, cudaStream_t stream) {
    const Sizes& z = plan.z;
    const int64_t blocks = (int64_t)z.batch * z.heads * ceil_div(z.n * z.p, 256);
    join_kernel<<<(unsigned)blocks, 256, 0, stream>>>(z, parts, end, backward);
    BCM_LAUNCH_CHECK();
    return BCM_OK;
}

// -------------------------------------------------------------------- forward ----
struct FwdArgs {
    Sizes z;
    Rows q, k, v;
    const float* g;
    int64_t g_sb, g_st, g_sh;
    const float* h0;
    const float* enter;        // [items][heads][n][p], or NULL where items are whole sequences
    void* y;                   // contiguous
    float* h_last;
    float* ckpt;               // [chunks][heads][slices][64][NT] transposed states that enter each chunk, or NULL
};

// Two threads issue the products of a chunk that need no other: Q K^T, and Q S with the state's V'^T K (V' the values
// times their decays until the chunk's end).  Warps 0 to 3 take 16 queries each: they mask and decay the scores, put their
// pieces back into tensor memory as an operand, and add the two parts of y.  Warps 4 to 7 hold the state and advance it
// meanwhile.  The next chunk's tiles are on their way to registers during all of that.
// Bound by the chain of one chunk (tiles down, scores, their decay, the second product, rows out), 5300 clocks with one
// block on an SM, of which the tensor pipe is active for 1060: 16 x 2048 tokens of 8 heads of 64 x 64 bf16 93 us (tensor
// pipe 20 %, DRAM 22 %), 1 x 32768 of 32 heads, two blocks on an SM, 214 us behind 99 for the items' parts (32 and 30 %).
// Twice the threads, with the rows dealt to eight warps, were slower: the barriers wait for more.
constexpr int kFwdThreads = 256;

template <typename T, int NT>
struct FwdSmem {
    static constexpr int NS = Pieces<T>::in, MS = Pieces<T>::out;
    struct Tiles {
        bf16 q[NS][Wide<NT>::elements], k[NS][Wide<NT>::elements], v[NS][Wide<kP>::elements];
        bf16 vw[kFull3][Wide<kP>::elements];
    } tiles;
    bf16 s[MS][Wide<NT>::elements];
    Decays d[2];
    Sync<4> sync;

    // tensor memory: scores, then their pieces (32 columns each); the near and the far part of y; the state's increase.
    // Beside a state of 128 there is no room for both parts: the far one is decayed in place and the near one added to it.
    static constexpr bool apart = NT <= 64;
    static constexpr uint32_t scores = 0, near = MS > 2 ? 96 : 64, far = apart ? near + 64 : near, inc = far + 64;
    static constexpr uint32_t cols = inc + NT <= 256 ? 256 : 512;
    static constexpr int resident = cols == 256 && sizeof(Tiles) + sizeof(bf16[MS][Wide<NT>::elements]) <= 108 * 1024 ? 2 : 1;   // blocks on an SM
};

// A chunk with an input that is not finite, token by token: 0 times such a value would spread it to tokens before it.
// `s` (shared, NT x kP) holds the state before and after, `sum` a float for each thread.
template <typename T>
__device__ __noinline__ void walk_tokens(const FwdArgs& p, const T* q, const T* k, const T* v, const float* g, T* y, int rows, int cols,
                                         float* s, float* sum) {
    constexpr int parts = kFwdThreads / kP;
    const int c = threadIdx.x % kP, part = threadIdx.x / kP;
    for (int t = 0; t < rows; ++t) {
        const float a = expf(g[(int64_t)t * p.g_st]), x = c < cols ? to_f32(v[(int64_t)t * p.v.st + c]) : 0.0f;
        float got = 0.0f;
        for (int n = part; n < p.z.n; n += parts) {
            const float now = fmaf(a, s[n * kP + c], to_f32(k[(int64_t)t * p.k.st + n]) * x);
            s[n * kP + c] = now;
            got = fmaf(to_f32(q[(int64_t)t * p.q.st + n]), now, got);
        }
        sum[threadIdx.x] = got;
        __syncthreads();
        if (part == 0 && c < cols) {
            for (int k2 = 1; k2 < parts; ++k2) got += sum[k2 * kP + c];
            y[(int64_t)t * p.z.heads * p.z.p + c] = from_f32<T>(got);
        }
        __syncthreads();
    }
}

// All that this block has written becomes NaN (of its own item: the others begin with states from elsewhere).  Finds them
// anew, so that the walk holds nothing for it in registers.
template <typename T, int NT>
__device__ __noinline__ void nan_item(const FwdArgs& p) {
    const Sizes& z = p.z;
    const int across = z.heads * z.slices, item = blockIdx.x / across, hs = blockIdx.x % across, h = hs / z.slices, slice = hs % z.slices;
    const Item it = item_of(z, item);
    const int len = it.t1 - it.t0;
    const int64_t y_st = (int64_t)z.heads * z.p, row_at = (z.cu ? 0 : (int64_t)it.seq * z.seqlen) + it.t0;
    nan_rows((T*)p.y + row_at * y_st + (int64_t)h * z.p + slice * kP, y_st, len, min(kP, z.p - slice * kP));
    if (p.ckpt)
        nan_rows(p.ckpt + (((int64_t)it.chunk * z.heads + h) * z.slices + slice) * (NT * kP), (int64_t)z.heads * z.slices * (NT * kP),
                 (len + kChunk - 1) / kChunk, NT * kP);
    if (it.last) nan_rows(p.h_last + ((int64_t)it.seq * z.heads + h) * z.n * z.p + slice * kP, z.p, z.n, min(kP, z.p - slice * kP));
}

template <typename T, int NT, bool VEC>
__global__ void __launch_bounds__(kFwdThreads, FwdSmem<T, NT>::resident) fwd_kernel(const __grid_constant__ FwdArgs p) {
    extern __shared__ unsigned char smem_raw[];
    using Smem = FwdSmem<T, NT>;
    Smem& sm = *(Smem*)tiles_base(smem_raw);
    constexpr int NS = Smem::NS, MS = Smem::MS;
    const Sizes& z = p.z;
    const int across = z.heads * z.slices;
    const int item = blockIdx.x / across, hs = blockIdx.x % across, h = hs / z.slices, col = hs % z.slices * kP;
    const int64_t y_st = (int64_t)z.heads * z.p;
    const int cols = min(kP, z.p - col), hq = h / (z.heads / z.qk_heads);
    if (z.cu)
        zero_rows((T*)p.y + (int64_t)h * z.p + col, z.tables.seq_item[z.batch + 1], z.seqlen, y_st, cols, item, z.items);
    const Item it = item_of(z, item);
    if (it.seq < 0) return;
    // the rows of the item's token t
    auto rows_of_token = [&](const Rows& r, int t, int head, int c0) { return row_ptr<T>(r, z, it.seq, it.t0 + t, head) + c0; };
    const float* g = p.g + (z.cu ? 0 : it.seq * p.g_sb) + it.t0 * p.g_st + h * p.g_sh;
    auto y_of_token = [&](int t) { return (T*)p.y + ((z.cu ? 0 : (int64_t)it.seq * z.seqlen) + it.t0 + t) * y_st + (int64_t)h * z.p + col; };
    const int np = z.n * z.p;
    const int len = it.t1 - it.t0, nc = (len + kChunk - 1) / kChunk;
    const int warp = t5::warp_id(), w = warp & 3;
    const bool state_warp = warp >= 4, decay_warp = warp == 5;
    const int p16 = (cols + 15) / 16;

    Pending<T, NT, kFwdThreads, VEC> pq, pk;
    Pending<T, kP, kFwdThreads, VEC> pv;
    Logs logs{g, p.g_st};
    State<NT, 1> st(0);                                       // (warps 4 to 7)
    bool bad_logs = false;
    sm.sync.init(Smem::cols);
    const uint32_t tm = __shfl_sync(kFull, sm.sync.tmem, 0), lanes = (uint32_t)w << 21;
    if (state_warp) {
        const float* from = it.first ? (p.h0 ? p.h0 + ((int64_t)it.seq * z.heads + h) * np : nullptr)
                                     : p.enter + ((int64_t)item * z.heads + h) * np;
        if (decay_warp) logs.fetch(0, len);
        if (from) st.load(from + col, z.n, cols, z.p);
        else st.zero();
        st.template put<MS, true>(sm.s[0]);
        if (decay_warp) {
            bad_logs = logs.bad();
            decays_of(sm.d[0], logs.a, logs.b);
            logs.fetch(kChunk, len);
        }
    }
    // with 128 features and 128 registers the next chunk's tiles are fetched when it begins: held through this one they
    // spilled (1 x 65536 tokens of 16 heads of 128 x 128 bf16 1289 us, so 1100)
    constexpr bool now = NT > 64 && Smem::resident == 2;
    uint32_t phase = 0;
    for (int c = -1; c < nc; ++c) {
        const int t = c * kChunk, rows = min(kChunk, len - t);
        bool slow = false;
        if (c >= 0) {
            if (state_warp && p.ckpt) {
                float* to = p.ckpt + (((int64_t)(it.chunk + c) * z.heads + h) * z.slices + hs % z.slices) * (NT * kP);
                st.pairs([&](float& x, float& y1, int pp, int n) {
                    if (pp < cols) *(float2*)(to + pp * NT + n) = make_float2(x, y1);
                });
            }
            if (now) {
                pq.fetch(rows_of_token(p.q, t, hq, 0), p.q.st, rows, z.n);
                pk.fetch(rows_of_token(p.k, t, hq, 0), p.k.st, rows, z.n);
                pv.fetch(rows_of_token(p.v, t, h, col), p.v.st, rows, cols);
            }
            __syncthreads();                                  // decays are there; the chunk before is done with the tiles
            const bool bad = bad_logs | pq.bad() | pk.bad() | pv.bad();
            pq.put(sm.tiles.q[0]);
            pk.put(sm.tiles.k[0]);
            pv.put(sm.tiles.v[0]);
            pv.put_weighted(sm.tiles.vw[0], sm.d[c & 1].until);
            t5::fence_smem();
            t5::fence_before();
            slow = __syncthreads_or(bad);
            // (issuing takes as long as the products: the state's warps have the time for the long ones)
            if (!slow && warp == 0 && t5::elect()) {
                t5::fence_after();
                products<NS, NS, MS, NT / 16>(tm + Smem::scores, Operand<NT, true>(sm.tiles.q), Operand<NT, true>(sm.tiles.k),
                                              t5::instr(kChunk, false, false), false);
                t5::commit(&sm.sync.bars[0]);
            }
            if (!slow && warp == 4 && t5::elect()) {
                t5::fence_after();
                products<NS, MS, MS, NT / 16>(tm + Smem::far, Operand<NT, true>(sm.tiles.q), Operand<NT, true>(sm.s),
                                              t5::instr(p16 * 16, false, false), false);
                t5::commit(&sm.sync.bars[1]);
                products<kFull3, NS, kFull3, kChunk / 16>(tm + Smem::inc, Operand<kP, false>(sm.tiles.vw), Operand<NT, false>(sm.tiles.k),
                                                          t5::instr(NT, true, true), false);
                t5::commit(&sm.sync.bars[2]);
            }
            __syncwarp();
        }
        if (!now && c + 1 < nc) {
            const int t2 = t + kChunk, r2 = min(kChunk, len - t2);
            pq.fetch(rows_of_token(p.q, t2, hq, 0), p.q.st, r2, z.n);
            pk.fetch(rows_of_token(p.k, t2, hq, 0), p.k.st, r2, z.n);
            pv.fetch(rows_of_token(p.v, t2, h, col), p.v.st, r2, cols);
        }
        if (c < 0) continue;
        if (slow) {
            // token by token, the state through shared memory
            float* f = (float*)&sm.tiles;
            if (state_warp)
                st.pairs([&](float& x, float& x1, int pp, int n) {
                    f[n * kP + pp] = x;
                    f[(n + 1) * kP + pp] = x1;
                });
            __syncthreads();
            walk_tokens<T>(p, rows_of_token(p.q, t, hq, 0), rows_of_token(p.k, t, hq, 0), rows_of_token(p.v, t, h, col), g + t * p.g_st, y_of_token(t),
                           rows, cols, f, f + NT * kP);
            if (state_warp) {
                st.pairs([&](float& x, float& x1, int pp, int n) {
                    x = f[n * kP + pp];
                    x1 = f[(n + 1) * kP + pp];
                });
            }
        }
        if (state_warp) {
            if (decay_warp && c + 1 < nc) {
                bad_logs = logs.bad();
                decays_of(sm.d[(c + 1) & 1], logs.a, logs.b);
                logs.fetch(t + 2 * kChunk, len);
            }
            if (!slow) {
                const float whole = sm.d[c & 1].whole;
                sm.sync.wait(2, phase);
                st.advance(tm + Smem::inc + lanes, whole);
                sm.sync.wait(1, phase);                       // the products with the entering state have read it
                t5::fence_before();
                phase ^= 1;
            }
            st.template put<MS, true>(sm.s[0]);
            continue;
        }
        if (slow) continue;
        const Decays& d = sm.d[c & 1];
        const int l = lane_id(), row = w * 16 + (l >> 2);
        const float hi0 = d.hi[row], lo0 = d.lo[row], hi1 = d.hi[row + 8], lo1 = d.lo[row + 8], since0 = d.since[row], since1 = d.since[row + 8];
        sm.sync.wait(0, phase);
        float sc[4][2][4];
#pragma unroll
        for (int jb = 0; jb < 4; ++jb)
            if (jb <= w) t5::ld16(sc[jb], tm + Smem::scores + lanes + 16 * jb);
#pragma unroll
        for (int jb = 0; jb < 4; ++jb) {
            uint32_t r[2][2][MS] = {};                        // [tile][half]
            if (jb <= w)
#pragma unroll
                for (int q2 = 0; q2 < 2; ++q2) {
                    const int j = jb * 16 + q2 * 8 + 2 * (l & 3);
                    const float2 hj = *(const float2*)&d.hi[j], lj = *(const float2*)&d.lo[j];
                    float(&x)[4] = sc[jb][q2];
                    x[0] = j <= row ? x[0] * between(hi0, lo0, hj.x, lj.x) : 0.0f;
                    x[1] = j + 1 <= row ? x[1] * between(hi0, lo0, hj.y, lj.y) : 0.0f;
                    x[2] = j <= row + 8 ? x[2] * between(hi1, lo1, hj.x, lj.x) : 0.0f;
                    x[3] = j + 1 <= row + 8 ? x[3] * between(hi1, lo1, hj.y, lj.y) : 0.0f;
                    split<MS>(x[0], x[1], r[q2][0]);
                    split<MS>(x[2], x[3], r[q2][1]);
                }
#pragma unroll
            for (int m = 0; m < MS; ++m) t5::st16(tm + Smem::scores + lanes + 32 * m + 8 * jb, r[0][0][m], r[0][1][m], r[1][0][m], r[1][1][m]);
        }
        if (!Smem::apart) {
            sm.sync.wait(1, phase);
            for (int pb = 0; pb < p16; ++pb) {
                float x[2][4];
                t5::ld16(x, tm + Smem::far + lanes + 16 * pb);
#pragma unroll
                for (int q2 = 0; q2 < 2; ++q2)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[q2][e] *= e < 2 ? since0 : since1;
                t5::st_acc16(tm + Smem::far + lanes + 16 * pb, x);
            }
        }
        t5::wait_st();
        t5::fence_before();
        named_sync(1, 128);
        if (warp == 0 && t5::elect()) {
            t5::fence_after();
            const Operand<kP, false> V(sm.tiles.v);
            products<MS, NS, MS, kChunk / 16>(tm + Smem::near, [&](int s, int i) { return tm + Smem::scores + 32 * s + 8 * i; }, V,
                                              t5::instr(p16 * 16, false, true), !Smem::apart);
            t5::commit(&sm.sync.bars[3]);
        }
        __syncwarp();
        sm.sync.wait(3, phase);
        sm.sync.wait(1, phase);
        T* const out = y_of_token(t);
#pragma unroll
        for (int pb = 0; pb < kP / 16; ++pb) {
            if (pb >= p16) break;
            float x[2][4];
            if constexpr (Smem::apart) {
                float f[2][4];
                t5::ld16x2(x, tm + Smem::near + lanes + 16 * pb, f, tm + Smem::far + lanes + 16 * pb);
#pragma unroll
                for (int q2 = 0; q2 < 2; ++q2)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[q2][e] = fmaf(e < 2 ? since0 : since1, f[q2][e], x[q2][e]);
            } else {
                t5::ld16(x, tm + Smem::near + lanes + 16 * pb);
            }
            store_rows<VEC>(out, y_st, rows, cols, row, 16 * pb, x[0], x[1]);
        }
        t5::fence_before();
        phase ^= 1;
    }
    if (state_warp && it.last) st.store(p.h_last + ((int64_t)it.seq * z.heads + h) * np + col, z.n, cols, z.p);
    if (sm.sync.lost()) nan_item<T, NT>(p);
    sm.sync.end(Smem::cols);
}

template <typename T, int NT>
bcm_status launch_fwd(const FwdArgs& p, bool vec, cudaStream_t stream) {
    using Smem = FwdSmem<T, NT>;
    constexpr size_t smem = sizeof(Smem) + 1024;
    static_assert(smem <= 227 * 1024, "shared memory of a block");
    static_assert(sizeof(typename Smem::Tiles) >= sizeof(float) * (NT * kP + kFwdThreads), "the state of walk_tokens");
    auto kernel = vec ? fwd_kernel<T, NT, true> : fwd_kernel<T, NT, false>;
    bcm_status st = allow_smem(kernel, smem);
    if (st != BCM_OK) return st;
    kernel<<<(unsigned)(p.z.items * p.z.heads * p.z.slices), kFwdThreads, smem, stream>>>(p);
    BCM_LAUNCH_CHECK();
    return BCM_OK;
}

// ----------------------------------------------------------------- one token ----
struct StepArgs {
    Rows q, k, v;
    const float* g;
    int64_t g_sb, g_st, g_sh;
    int heads, qk_heads, n, p, tokens;
    const float* from;         // states before the first token (the step: h), or NULL for zeros
    float* h;                  // and behind the last
    void* y;
};

// A block per sequence and head: its threads hold V neighbouring columns each, and the rows of the state are dealt to
// groups of threads, whose sums of q_n S_n meet in shared memory.  Bound by memory, the state read and written once:
// one token of 256 x 64 heads of 64 x 64 92 to 97 us, 85 to 90 % of a copy's bandwidth (125 us when the state was read behind the
// queries' barrier).
// ONE: one token in place (as a token of many 104 us).
template <typename T, int V, bool ONE>
__global__ void __launch_bounds__(256) step_kernel(const __grid_constant__ StepArgs a) {
    constexpr int kAhead = 4;
    __shared__ float part[8][32 * V];                     // sums of a warp's rows, by columns
    __shared__ float sq[128], sk[128];
    const int b = blockIdx.x / a.heads, h = blockIdx.x % a.heads, hq = h / (a.heads / a.qk_heads), tid = threadIdx.x;
    float* const s = a.h + (int64_t)blockIdx.x * a.n * a.p;
    // threads side by side over the columns: a power of two, so that the others form whole groups
    int wide = 1;
    while (wide < 32 && wide * V < a.p) wide *= 2;
    const int rows = blockDim.x / wide, row = tid / wide, lane = tid % wide;
    float now[kAhead][V];
    // the state's rows n0, n0 + rows, .. of columns from c: under way before the queries and keys are waited for
    auto fetch = [&](const float* from, int c, int n0) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int n = n0 + i * rows;
#pragma unroll
            for (int e = 0; !ONE && e < V; ++e) now[i][e] = 0.0f;
            if ((ONE || from) && c < a.p && n < a.n) {
                const float* at = from + (int64_t)n * a.p + c;
                if constexpr (V == 4) *(float4*)now[i] = *(const float4*)at;
                else now[i][0] = at[0];
            }
        }
    };
    for (int t = 0; t < (ONE ? 1 : a.tokens); ++t) {
        // (a thread meets its own elements of the state again with every token)
        const float* const from = ONE || t ? s : a.from ? a.from + (int64_t)blockIdx.x * a.n * a.p : nullptr;
        const T* q = (const T*)a.q.p + b * a.q.sb + t * a.q.st + hq * a.q.sh;
        const T* k = (const T*)a.k.p + b * a.k.sb + t * a.k.st + hq * a.k.sh;
        const T* v = (const T*)a.v.p + b * a.v.sb + t * a.v.st + h * a.v.sh;
        T* y = (T*)a.y + (ONE ? (int64_t)blockIdx.x : ((int64_t)b * a.tokens + t) * a.heads + h) * a.p;
        fetch(from, lane * V, row);
        if (tid < a.n) {
            sq[tid] = to_f32(q[tid]);
            sk[tid] = to_f32(k[tid]);
        }
        const float decay = expf(a.g[b * a.g_sb + t * a.g_st + h * a.g_sh]);
        for (int c0 = 0; c0 < a.p; c0 += wide * V) {
            const int c = c0 + lane * V;
            float x[V], sum[V] = {};
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = c < a.p ? to_f32(v[c + e]) : 0.0f;
            __syncthreads();                                  // queries and keys are there; the last turn's sums are read
            for (int n0 = row; n0 < a.n; n0 += kAhead * rows) {
                if (c0 || n0 != row) fetch(from, c, n0);
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const int n = n0 + i * rows;
                    if (c < a.p && n < a.n) {
                        float* at = s + (int64_t)n * a.p + c;
                        const float kn = sk[n], qn = sq[n];
#pragma unroll
                        for (int e = 0; e < V; ++e) {
                            now[i][e] = fmaf(decay, now[i][e], kn * x[e]);
                            sum[e] = fmaf(qn, now[i][e], sum[e]);
                        }
                        if constexpr (V == 4) *(float4*)at = *(const float4*)now[i];
                        else at[0] = now[i][0];
                    }
                }
            }
            for (int o = 16; o >= wide; o >>= 1) {
#pragma unroll
                for (int e = 0; e < V; ++e) sum[e] += __shfl_xor_sync(kFull, sum[e], o);
            }
            if ((tid & 31) < wide) {
#pragma unroll
                for (int e = 0; e < V; ++e) part[tid >> 5][lane * V + e] = sum[e];
            }
            __syncthreads();
            if (tid < wide * V && c0 + tid < a.p) {
                float got = 0.0f;
#pragma unroll
                for (int r = 0; r < 8; ++r) got += part[r][tid];
                y[c0 + tid] = from_f32<T>(got);
            }
        }
    }
}

// Sequences of few tokens without a backward are not worth a chunk of 64 each: 2000 of 4 heads of 64 x 64 with 2, 4, 6, 8 and
// 12 tokens take 78, 133, 186, 241 and 350 us one by one in every type; as chunks bf16 takes 196 us, float16 244, float32 372.
// One border for all types, where the quickest as chunks still gains; float16 would up to 8 tokens, float32 up to 12.
constexpr int kFewTokens = 4;
// every sequence's tokens one by one, states from `from` (NULL: zeros) to h
bcm_status launch_step(const bcm_decay_attn_args* a, const float* from, float* h, cudaStream_t stream) {
    const StepArgs sa{rows_of(a->q, a->q_stride_b, a->q_stride_t, a->q_stride_h), rows_of(a->k, a->k_stride_b, a->k_stride_t, a->k_stride_h),
                      rows_of(a->v, a->v_stride_b, a->v_stride_t, a->v_stride_h), a->log_decay, a->g_stride_b, a->g_stride_t, a->g_stride_h,
                      (int)a->heads, (int)a->qk_heads, (int)a->dim_k, (int)a->dim_v, (int)a->seqlen, from, h, a->y};
    const bool four = a->dim_v % 4 == 0 && (((uintptr_t)h | (uintptr_t)from) & 15) == 0;
    const unsigned blocks = (unsigned)(a->batch * a->heads);
    return dispatch_dtype(a->dtype, [&](auto type) -> bcm_status {
        using T = decltype(type);
        const bool one = a->seqlen == 1 && from == h;
        auto kernel = four ? (one ? step_kernel<T, 4, true> : step_kernel<T, 4, false>) : one ? step_kernel<T, 1, true> : step_kernel<T, 1, false>;
        kernel<<<blocks, 256, 0, stream>>>(sa);
        BCM_LAUNCH_CHECK();
        return BCM_OK;
    });
}

}  // namespace decay_attn
}  // namespace bcm

using namespace bcm;
using namespace bcm::decay_attn;

extern "C" size_t bcm_decay_attn_ckpt_bytes(const bcm_decay_attn_args* a) {
    if (check(a, "decay_attn") != BCM_OK) return 0;
    const Plan plan = plan_of(a, false);
    const int nt = plan.z.n <= 16 ? 16 : plan.z.n <= 32 ? 32 : plan.z.n <= 64 ? 64 : 128;
    return sizeof(float) * (size_t)plan.z.chunks * plan.z.heads * plan.z.slices * kP * nt;
}

extern "C" size_t bcm_decay_attn_fwd_workspace_bytes(const bcm_decay_attn_args* a) {
    return check(a, "decay_attn") == BCM_OK ? plan_of(a, false).bytes : 0;
}

extern "C" bcm_status bcm_decay_attn_fwd(const bcm_decay_attn_args* a, cudaStream_t stream) {
    clear_error();
    bcm_status st = check(a, "decay_attn_fwd");
    if (st != BCM_OK) return st;
    if (a->batch == 0) return BCM_OK;
    Plan plan = plan_of(a, false);
    BCM_REQUIRE(a->seqlen == 0 || (a->q && a->k && a->v && a->log_decay && a->y), "decay_attn_fwd: null pointer");
    BCM_REQUIRE(a->h_last, "decay_attn_fwd: null pointer");
    BCM_REQUIRE(plan.bytes == 0 || (a->workspace && a->workspace_bytes >= plan.bytes), "decay_attn_fwd: workspace too small");
    BCM_REQUIRE(!a->ckpt || a->ckpt_bytes >= bcm_decay_attn_ckpt_bytes(a), "decay_attn_fwd: ckpt too small");
    BCM_REQUIRE((int64_t)plan.z.items * plan.z.heads * plan.z.slices < INT32_MAX, "decay_attn_fwd: too many blocks");
    if (!a->cu_seqlens && !a->ckpt && a->seqlen >= 1 && a->seqlen <= kFewTokens) return launch_step(a, a->h0, a->h_last, stream);
    if ((st = fill_tables(plan, a->workspace, stream)) != BCM_OK) return st;
    const Parts parts = parts_of(plan, a->workspace);
    const Rows q = rows_of(a->q, a->q_stride_b, a->q_stride_t, a->q_stride_h), k = rows_of(a->k, a->k_stride_b, a->k_stride_t, a->k_stride_h),
               v = rows_of(a->v, a->v_stride_b, a->v_stride_t, a->v_stride_h);
    const bool vec = aligned(a, false);
    return dispatch(a->dtype, a->dim_k, [&](auto type, auto n) -> bcm_status {
        using T = decltype(type);
        if (plan.cut) {
            const PartArgs pa{plan.z, k, v, a->log_decay, a->g_stride_b, a->g_stride_t, a->g_stride_h, parts};
            bcm_status r = launch_part<T, n, false>(pa, vec, stream);
            if (r != BCM_OK) return r;
            if ((r = join(plan, parts, a->h0, false, stream)) != BCM_OK) return r;
        }
        const FwdArgs fa{plan.z, q, k, v, a->log_decay, a->g_stride_b, a->g_stride_t, a->g_stride_h, a->h0, parts.state,
                         a->y, a->h_last, (float*)a->ckpt};
        return launch_fwd<T, n>(fa, vec, stream);
    });
}

extern "C" bcm_status bcm_decay_attn_step(const bcm_decay_attn_args* a, float* h, cudaStream_t stream) {
    clear_error();
    bcm_status st = check(a, "decay_attn_step");
    if (st != BCM_OK) return st;
    BCM_REQUIRE(a->seqlen == 1 && !a->cu_seqlens, "decay_attn_step: one token of every sequence");
    if (a->batch == 0) return BCM_OK;
    BCM_REQUIRE(a->q && a->k && a->v && a->log_decay && a->y && h, "decay_attn_step: null pointer");
    BCM_REQUIRE(a->batch * a->heads < INT32_MAX, "decay_attn_step: too many blocks");
    return launch_step(a, h, h, stream);
}
