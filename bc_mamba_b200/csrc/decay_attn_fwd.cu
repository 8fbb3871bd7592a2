// decay_attn_fwd.cu — linear attention with a decay for each head: plan of a call, forward walk, one-token step.
#include "decay_attn.cuh"

namespace bcm {
namespace decay_attn {

int padded_n(int64_t n) { return n <= 16 ? 16 : n <= 32 ? 32 : n <= 64 ? 64 : 128; }

bcm_status check(const bcm_decay_attn_args* a, const char* what) {
    BCM_REQUIRE(a != nullptr, "%s: null arguments", what);
    BCM_REQUIRE(dtype_ok(a->dtype), "%s: unsupported dtype %d", what, (int)a->dtype);
    BCM_REQUIRE(a->batch >= 0 && a->seqlen >= 0 && a->heads >= 1 && a->qk_heads >= 1 && a->dim_k >= 1 && a->dim_v >= 1,
                "%s: bad sizes", what);
    BCM_REQUIRE(a->dim_k <= BCM_DECAY_ATTN_MAX_DIM_K, "%s: a query of more than %d features", what, BCM_DECAY_ATTN_MAX_DIM_K);
    BCM_REQUIRE(a->heads % a->qk_heads == 0, "%s: heads must be a multiple of the queries' heads", what);
    BCM_REQUIRE(a->dim_v <= (1 << 20) && a->heads <= (1 << 20) && a->batch < (1 << 24) && a->seqlen < INT32_MAX - 4096, "%s: sizes too large", what);
    BCM_REQUIRE(a->batch == 0 || a->heads * a->dim_v <= (1 << 24), "%s: sizes too large", what);
    return BCM_OK;
}

// Blocks are (item, head, 64 columns of the values) and walk their item's chunks one after another.  Sequences are cut
// into items only where whole ones leave the GPU short of blocks: an item costs one more pass over two inputs and
// states to join.  An item has 256 tokens at least.
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
    // shared memory of the backward walk: two tiles of 128 x 64 in three pieces do not fit beside the others
    const bool narrow = z.p <= 32 || (backward && a->dtype == BCM_F32 && z.n > 64);
    plan.pt = narrow ? 32 : 64;
    z.slices = ceil_div(z.p, plan.pt);
    const int64_t across = (int64_t)z.heads * z.slices, want = 4 * sm_count();
    const int64_t tokens = a->seqlen;
    auto chunks_up = [](int64_t v) { return std::max<int64_t>(256, (v + kChunk - 1) / kChunk * kChunk); };
    if (!z.cu) {
        const int64_t blocks = std::max<int64_t>(1, z.batch * across);
        const int64_t segs = blocks >= 2 * sm_count() ? 1 : (want + blocks - 1) / blocks;
        z.span = (int)chunks_up((tokens + segs - 1) / std::max<int64_t>(1, segs));
        z.per_seq = std::max(1, ceil_div(tokens, z.span));
        z.items = z.batch * z.per_seq;
        z.chunks = z.batch * ceil_div(tokens, kChunk);
        plan.cut = z.per_seq > 1;
    } else {
        z.span = (int)chunks_up((tokens * across + want - 1) / want);
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
        const int items = in ? max(1, (len + z.span - 1) / z.span) : 0, chunks = in ? (len + kChunk - 1) / kChunk : 0;
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
                z.tables.items[item + k] = Item{s, t0, min(end, t0 + z.span), chunk + k * (z.span / kChunk), k == 0, k == items - 1};
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
    for (int k = 0; k < count - 1; ++k) {              // the last of the walk has no part
        const int64_t at = (int64_t)(backward ? stop - 1 - k : first + k) * z.heads + h;
        const float own = parts.state[at * np + e];
        parts.state[at * np + e] = s;
        s = fmaf(parts.whole[at], s, own);
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
    float* ckpt;               // [chunks][heads][n][p] states that enter each chunk, or NULL
};

// Warps 0 to 3 form the outputs of 16 tokens each, warps 4 to 7 hold the state and advance it meanwhile.  Where there is
// room for it the pieces of the next chunk's entering state go to a second buffer.
constexpr int kFwdThreads = 256;

template <typename T, int NT, int PT>
struct FwdSmem {
    static constexpr int NS = Pieces<T>::in, MS = Pieces<T>::out;
    struct Tiles {
        bf16 q[NS][kChunk][NT + 8], k[NS][kChunk][NT + 8], v[NS][kChunk][PT + 8];
    } tiles;
    static constexpr int buffers = sizeof(Tiles) + 2 * sizeof(bf16[MS][NT][PT + 8]) <= 110 * 1024 ? 2 : 1;
    bf16 s[buffers][MS][NT][PT + 8];
    Decays d;
};

// A chunk with a value that is not finite, token by token: 0 times such a value would spread it to tokens before it.
// `s` (shared, NT x PT) holds the state before and after, `sum` a float for each thread.
template <typename T, int NT, int PT>
__device__ __noinline__ void walk_tokens(const FwdArgs& p, const T* q, const T* k, const T* v, const float* g, T* y, int rows, int cols,
                                         float* s, float* sum) {
    constexpr int parts = kFwdThreads / PT;
    const int c = threadIdx.x % PT, part = threadIdx.x / PT;
    for (int t = 0; t < rows; ++t) {
        const float a = expf(g[(int64_t)t * p.g_st]), x = c < cols ? to_f32(v[(int64_t)t * p.v.st + c]) : 0.0f;
        float got = 0.0f;
        for (int n = part; n < p.z.n; n += parts) {
            const float now = fmaf(a, s[n * PT + c], to_f32(k[(int64_t)t * p.k.st + n]) * x);
            s[n * PT + c] = now;
            got = fmaf(to_f32(q[(int64_t)t * p.q.st + n]), now, got);
        }
        sum[threadIdx.x] = got;
        __syncthreads();
        if (part == 0 && c < cols) {
            for (int k2 = 1; k2 < parts; ++k2) got += sum[k2 * PT + c];
            y[(int64_t)t * p.z.heads * p.z.p + c] = from_f32<T>(got);
        }
        __syncthreads();
    }
}

template <typename T, int NT, int PT>
__global__ void __launch_bounds__(kFwdThreads, FwdSmem<T, NT, PT>::buffers) fwd_kernel(const __grid_constant__ FwdArgs p) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    using Smem = FwdSmem<T, NT, PT>;
    Smem& sm = *(Smem*)smem_raw;
    constexpr int NS = Smem::NS, MS = Smem::MS, LN = NT + 8, LP = PT + 8;
    const Sizes& z = p.z;
    const int across = z.heads * z.slices;
    const int item = blockIdx.x / across, hs = blockIdx.x % across, h = hs / z.slices, col = hs % z.slices * PT;
    const int64_t y_st = (int64_t)z.heads * z.p;
    const int cols = min(PT, z.p - col), hq = h / (z.heads / z.qk_heads);
    if (z.cu)
        zero_rows((T*)p.y + (int64_t)h * z.p + col, z.tables.seq_item[z.batch + 1], z.seqlen, y_st, cols, item, z.items);
    const Item it = item_of(z, item);
    if (it.seq < 0) return;
    const T* q = row_ptr<T>(p.q, z, it.seq, it.t0, hq);
    const T* k = row_ptr<T>(p.k, z, it.seq, it.t0, hq);
    const T* v = row_ptr<T>(p.v, z, it.seq, it.t0, h) + col;
    const float* g = p.g + (z.cu ? 0 : it.seq * p.g_sb) + it.t0 * p.g_st + h * p.g_sh;
    T* y = (T*)p.y + ((z.cu ? 0 : (int64_t)it.seq * z.seqlen) + it.t0) * y_st + (int64_t)h * z.p + col;
    const bool vq = on_16(q, p.q.st), vk = on_16(k, p.k.st), vv = on_16(v, p.v.st);
    const bool pair_y = (((uintptr_t)y | (uintptr_t)(y_st * sizeof(T))) & (2 * sizeof(T) - 1)) == 0;
    const int np = z.n * z.p;
    const int len = it.t1 - it.t0, nc = (len + kChunk - 1) / kChunk;
    const int l = lane_id(), w = (threadIdx.x >> 5) & 3, row = w * 16 + (l >> 2);
    const bool state_warp = threadIdx.x >= 128, decay_warp = threadIdx.x >= 128 && threadIdx.x < 160;
    bf16* const tq = &sm.tiles.q[0][0][0];
    bf16* const tk = &sm.tiles.k[0][0][0];
    bf16* const tv = &sm.tiles.v[0][0][0];

    Pending<T, kChunk, NT, kFwdThreads> pq, pk;
    Pending<T, kChunk, PT, kFwdThreads> pv;
    float g0 = 0.0f, g1 = 0.0f;
    auto fetch = [&](int c) {
        const int t = c * kChunk, rows = min(kChunk, len - t);
        pq.fetch(q + t * p.q.st, p.q.st, rows, z.n, vq);
        pk.fetch(k + t * p.k.st, p.k.st, rows, z.n, vk);
        pv.fetch(v + t * p.v.st, p.v.st, rows, cols, vv);
        if (decay_warp) {
            g0 = 2 * l < rows ? g[(int64_t)(t + 2 * l) * p.g_st] : 0.0f;
            g1 = 2 * l + 1 < rows ? g[(int64_t)(t + 2 * l + 1) * p.g_st] : 0.0f;
        }
    };
    // the tiles of the fetched chunk; whether a value was not finite
    auto put = [&]() {
        bool bad = pq.put(tq, LN);
        bad |= pk.put(tk, LN);
        bad |= pv.put(tv, LP);
        if (decay_warp) {
            bad |= !(g0 <= 3.38e38f && g1 <= 3.38e38f);
            decays_of(sm.d, g0, g1);
        }
        return bad;
    };
    // token by token, the state through shared memory
    auto walk = [&](int c) {
        const int t = c * kChunk;
        float* f = (float*)&sm.tiles;
        walk_tokens<T, NT, PT>(p, q + t * p.q.st, k + t * p.k.st, v + t * p.v.st, g + t * p.g_st, y + t * y_st, min(kChunk, len - t), cols, f,
                               f + NT * PT);
    };
    if (nc > 0) fetch(0);

    if (state_warp) {
        State<NT, PT> st;
        const float* from = it.first ? (p.h0 ? p.h0 + ((int64_t)it.seq * z.heads + h) * np : nullptr)
                                     : p.enter + ((int64_t)item * z.heads + h) * np;
        if (from) st.load(from + col, z.n, z.p - col, z.p);
        else st.zero();
        bool bad = false;
        if (Smem::buffers > 1) bad = st.template put<MS>(&sm.s[0][0][0][0]);
        for (int c = 0; c < nc; ++c) {
            if (p.ckpt) st.store(p.ckpt + ((int64_t)(it.chunk + c) * z.heads + h) * np + col, z.n, z.p - col, z.p);
            __syncthreads();
            bad |= put();
            if (Smem::buffers == 1) bad |= st.template put<MS>(&sm.s[0][0][0][0]);
            const bool slow = __syncthreads_or(bad);
            if (c + 1 < nc) fetch(c + 1);
            if (slow) {
                float* f = (float*)&sm.tiles;
                st.pairs([&](float& x, float& x1, int r, int cc) {
                    f[r * PT + cc] = x;
                    f[r * PT + cc + 1] = x1;
                });
                __syncthreads();
                walk(c);
                st.pairs([&](float& x, float& x1, int r, int cc) {
                    x = f[r * PT + cc];
                    x1 = f[r * PT + cc + 1];
                });
            } else {
                st.template advance<NS>(tk, tv, sm.d.until, sm.d.whole);
            }
            bad = false;
            if (Smem::buffers > 1) bad = st.template put<MS>(&sm.s[(c + 1) % Smem::buffers][0][0][0]);
        }
        if (it.last) st.store(p.h_last + ((int64_t)it.seq * z.heads + h) * np + col, z.n, z.p - col, z.p);
        return;
    }
    for (int c = 0; c < nc; ++c) {
        const int t = c * kChunk, rows = min(kChunk, len - t);
        __syncthreads();                                      // the chunk before is done with the tiles
        const bool bad = put();
        const bool slow = __syncthreads_or(bad);
        if (c + 1 < nc) fetch(c + 1);
        if (slow) {
            __syncthreads();
            walk(c);
            continue;
        }
        // 16 queries: the entering state's part, then those of the keys up to their own
        float acc[PT / 8][4] = {};
        const bf16* ts = &sm.s[c % Smem::buffers][0][0][0];
        auto queries = [&](uint32_t(&a)[4], int s, int kk) { load_a(a, tq + s * kChunk * LN, LN, w * 16, kk * 16); };
        gemm<NS, MS, MS, NT / 16, PT / 16, true>(acc, queries, ts, LP, NT * LP, 0, 0);
        const float since0 = sm.d.since[row], since1 = sm.d.since[row + 8];
#pragma unroll
        for (int pb = 0; pb < PT / 8; ++pb) {
            acc[pb][0] *= since0;
            acc[pb][1] *= since0;
            acc[pb][2] *= since1;
            acc[pb][3] *= since1;
        }
        const float hi0 = sm.d.hi[row], lo0 = sm.d.lo[row], hi1 = sm.d.hi[row + 8], lo1 = sm.d.lo[row + 8];
#pragma unroll 1
        for (int jb = 0; jb <= w; ++jb) {
            float sc[2][4] = {};
            gemm<NS, NS, MS, NT / 16, 1, false>(sc, queries, tk, LN, kChunk * LN, 0, jb * 16);
#pragma unroll
            for (int q2 = 0; q2 < 2; ++q2) {
                const int j = jb * 16 + q2 * 8 + 2 * (l & 3);
                const float2 hj = *(const float2*)&sm.d.hi[j], lj = *(const float2*)&sm.d.lo[j];
                sc[q2][0] = j <= row ? sc[q2][0] * between(hi0, lo0, hj.x, lj.x) : 0.0f;
                sc[q2][1] = j + 1 <= row ? sc[q2][1] * between(hi0, lo0, hj.y, lj.y) : 0.0f;
                sc[q2][2] = j <= row + 8 ? sc[q2][2] * between(hi1, lo1, hj.x, lj.x) : 0.0f;
                sc[q2][3] = j + 1 <= row + 8 ? sc[q2][3] * between(hi1, lo1, hj.y, lj.y) : 0.0f;
            }
            uint32_t a[MS][4];
            split_a<MS>(sc[0], sc[1], a);
            gemm<MS, NS, MS, 1, PT / 16, true>(acc, [&](uint32_t(&r)[4], int s, int) {
#pragma unroll
                for (int e = 0; e < 4; ++e) r[e] = a[s][e];
            }, tv, LP, kChunk * LP, jb * 16, 0);
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int r = row + 8 * half;
            if (r < rows) {
                T* out = y + (int64_t)(t + r) * y_st;
#pragma unroll
                for (int pb = 0; pb < PT / 8; ++pb) {
                    const int cc = pb * 8 + 2 * (l & 3);
                    struct alignas(2 * sizeof(T)) Two { T x, y; };
                    const T x0 = from_f32<T>(acc[pb][2 * half]), x1 = from_f32<T>(acc[pb][2 * half + 1]);
                    if (pair_y && cc + 1 < cols) {
                        *(Two*)(out + cc) = Two{x0, x1};
                    } else {
                        if (cc < cols) out[cc] = x0;
                        if (cc + 1 < cols) out[cc + 1] = x1;
                    }
                }
            }
        }
    }
}

template <typename T, int NT, int PT>
bcm_status launch_fwd(const FwdArgs& p, cudaStream_t stream) {
    constexpr size_t smem = sizeof(FwdSmem<T, NT, PT>);
    static_assert(smem <= 227 * 1024, "shared memory of a block");
    static_assert(sizeof(typename FwdSmem<T, NT, PT>::Tiles) >= sizeof(float) * (NT * PT + kFwdThreads), "the state of walk_tokens");
    auto kernel = fwd_kernel<T, NT, PT>;
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
    int64_t g_sb, g_sh;
    int heads, qk_heads, n, p;
    float* h;
    void* y;
};

// A block per sequence and head: its threads hold V neighbouring columns each, and the rows of the state are dealt to
// `parts` groups of threads, whose sums of q_n S_n meet in shared memory.
template <typename T, int V>
__global__ void __launch_bounds__(256) step_kernel(const __grid_constant__ StepArgs a) {
    extern __shared__ float part[];                       // [parts][columns of the block's turn]
    __shared__ float sq[128], sk[128];
    const int b = blockIdx.x / a.heads, h = blockIdx.x % a.heads, hq = h / (a.heads / a.qk_heads);
    const T* q = (const T*)a.q.p + b * a.q.sb + hq * a.q.sh;
    const T* k = (const T*)a.k.p + b * a.k.sb + hq * a.k.sh;
    const T* v = (const T*)a.v.p + b * a.v.sb + h * a.v.sh;
    if (threadIdx.x < a.n) {
        sq[threadIdx.x] = to_f32(q[threadIdx.x]);
        sk[threadIdx.x] = to_f32(k[threadIdx.x]);
    }
    const float decay = expf(a.g[b * a.g_sb + h * a.g_sh]);
    float* s = a.h + (int64_t)blockIdx.x * a.n * a.p;
    T* y = (T*)a.y + (int64_t)blockIdx.x * a.p;
    __syncthreads();
    // threads side by side over the columns: a power of two, so that the others form whole groups
    int wide = 1;
    while (wide < 32 && wide * V < a.p) wide *= 2;
    const int parts = blockDim.x / wide, part_id = threadIdx.x / wide, lane = threadIdx.x % wide;
    for (int c0 = 0; c0 < a.p; c0 += wide * V) {
        const int c = c0 + lane * V;
        float x[V], sum[V] = {};
        if (c < a.p) {
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = to_f32(v[c + e]);
#pragma unroll 4
            for (int n = part_id; n < a.n; n += parts) {
                float now[V];
                float* at = s + (int64_t)n * a.p + c;
                if (V == 4) *(float4*)now = *(const float4*)at;
                else now[0] = at[0];
                const float kn = sk[n], qn = sq[n];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    now[e] = fmaf(decay, now[e], kn * x[e]);
                    sum[e] = fmaf(qn, now[e], sum[e]);
                }
                if (V == 4) *(float4*)at = *(const float4*)now;
                else at[0] = now[0];
            }
        }
#pragma unroll
        for (int e = 0; e < V; ++e) part[(part_id * wide + lane) * V + e] = sum[e];
        __syncthreads();
        for (int e = threadIdx.x; e < wide * V && c0 + e < a.p; e += blockDim.x) {
            float got = 0.0f;
            for (int r = 0; r < parts; ++r) got += part[r * wide * V + e];
            y[c0 + e] = from_f32<T>(got);
        }
        __syncthreads();
    }
}

}  // namespace decay_attn
}  // namespace bcm

using namespace bcm;
using namespace bcm::decay_attn;

extern "C" size_t bcm_decay_attn_ckpt_bytes(const bcm_decay_attn_args* a) {
    if (check(a, "decay_attn") != BCM_OK) return 0;
    const Plan plan = plan_of(a, false);
    return sizeof(float) * (size_t)plan.z.chunks * plan.z.heads * plan.z.n * plan.z.p;
}

extern "C" size_t bcm_decay_attn_fwd_workspace_bytes(const bcm_decay_attn_args* a) {
    return check(a, "decay_attn") == BCM_OK ? plan_of(a, false).bytes : 0;
}

extern "C" bcm_status bcm_decay_attn_fwd(const bcm_decay_attn_args* a, cudaStream_t stream) {
    clear_error();
    bcm_status st = check(a, "decay_attn_fwd");
    if (st != BCM_OK) return st;
    if (a->batch == 0 && a->seqlen == 0) return BCM_OK;
    if (a->batch == 0 && !a->cu_seqlens) return BCM_OK;
    Plan plan = plan_of(a, false);
    BCM_REQUIRE(a->seqlen == 0 || (a->q && a->k && a->v && a->log_decay && a->y), "decay_attn_fwd: null pointer");
    BCM_REQUIRE(a->h_last, "decay_attn_fwd: null pointer");
    BCM_REQUIRE(plan.bytes == 0 || (a->workspace && a->workspace_bytes >= plan.bytes), "decay_attn_fwd: workspace too small");
    BCM_REQUIRE(!a->ckpt || a->ckpt_bytes >= bcm_decay_attn_ckpt_bytes(a), "decay_attn_fwd: ckpt too small");
    BCM_REQUIRE((int64_t)plan.z.items * plan.z.heads * plan.z.slices < INT32_MAX, "decay_attn_fwd: too many blocks");
    if ((st = fill_tables(plan, a->workspace, stream)) != BCM_OK) return st;
    const Parts parts = parts_of(plan, a->workspace);
    const Rows q = rows_of(a->q, a->q_stride_b, a->q_stride_t, a->q_stride_h), k = rows_of(a->k, a->k_stride_b, a->k_stride_t, a->k_stride_h),
               v = rows_of(a->v, a->v_stride_b, a->v_stride_t, a->v_stride_h);
    return dispatch(a->dtype, padded_n(a->dim_k), plan.pt, [&](auto type, auto n, auto p) -> bcm_status {
        using T = decltype(type);
        if (plan.cut) {
            const PartArgs pa{plan.z, k, v, a->log_decay, a->g_stride_b, a->g_stride_t, a->g_stride_h, parts};
            bcm_status r = launch_part<T, n, p, false>(pa, stream);
            if (r != BCM_OK) return r;
            if ((r = join(plan, parts, a->h0, false, stream)) != BCM_OK) return r;
        }
        const FwdArgs fa{plan.z, q, k, v, a->log_decay, a->g_stride_b, a->g_stride_t, a->g_stride_h, a->h0, parts.state,
                         a->y, a->h_last, (float*)a->ckpt};
        return launch_fwd<T, n, p>(fa, stream);
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
    const StepArgs sa{rows_of(a->q, a->q_stride_b, 0, a->q_stride_h), rows_of(a->k, a->k_stride_b, 0, a->k_stride_h),
                      rows_of(a->v, a->v_stride_b, 0, a->v_stride_h), a->log_decay, a->g_stride_b, a->g_stride_h, (int)a->heads,
                      (int)a->qk_heads, (int)a->dim_k, (int)a->dim_v, h, a->y};
    const bool four = a->dim_v % 4 == 0 && ((uintptr_t)h & 15) == 0;
    const unsigned blocks = (unsigned)(a->batch * a->heads);
    return dispatch_dtype(a->dtype, [&](auto type) -> bcm_status {
        using T = decltype(type);
        if (four) step_kernel<T, 4><<<blocks, 256, 256 * 4 * sizeof(float), stream>>>(sa);
        else step_kernel<T, 1><<<blocks, 256, 256 * sizeof(float), stream>>>(sa);
        BCM_LAUNCH_CHECK();
        return BCM_OK;
    });
}
