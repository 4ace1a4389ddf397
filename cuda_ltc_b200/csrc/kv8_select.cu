// Which blocks of an 8-bit cache the newest tokens should read: see ltca_kv8_select in include/ltc_attn.h.
//
// One cluster of CTAs takes a pair (sequence, head of keys), each CTA a run of its blocks; scores never leave shared memory.
//   - Scores: Q in eight bits and the bounds are whole numbers, so that four channels cost a byte mask (the sign of q picks the
//     lower or the upper bound), a selection and a four-way dot product.  The sum is below 2^21 and exact.
//   - The `count` best: the score's bits in an order that whole numbers have, and a search for the count-th largest of them
//     eight bits at a time with histograms in shared memory.  Up to kGather blocks the scores go to the cluster's first CTA,
//     which searches alone, from the highest bit in which they differ on: two or three rounds.  With more blocks every CTA keeps
//     its own, and the cluster adds up the histograms (times of both at kGather).
//   - The indices come out in rising order, since it is known how many of the blocks before have been taken.
// Bound by the waits one behind another - lengths, queries, bounds, the cluster, the search - of about a microsecond each: 2048
// blocks of 8 sequences and 8 heads 15 us, of which the bounds (2 D + 4 bytes a block) take 3.8; 256 blocks of one sequence 6 us; 4096 of eight 42 us, 16384 124 us.
#include <cooperative_groups.h>

#include "kv8.cuh"

namespace ltca {

namespace {

struct SelectArgs {
    ltca_kv8_cache c;
    ltca_kv8_select_params p;
    int nb, G, R;               // blocks of tokens; heads of queries per head of keys; rows of a pair
    int ctas;                   // of a pair, one cluster
    int room;                   // scores that a CTA has room for
};

// Numbers in the order of the scores; 0 is below every score's, the largest above.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

// 0xff for each byte below zero (a selector's highest bit replicates the byte's sign).
__device__ __forceinline__ uint32_t signs(uint32_t x) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %1, 0xba98;" : "=r"(r) : "r"(x));
    return r;
}

constexpr int kThreads = 256, kSelectWarps = kThreads / 32;
constexpr int kRowsAtATime = 32;            // rows of Q in shared memory
constexpr int kMaxSelectCluster = 16;
constexpr int kGather = 4096;             // blocks whose scores one CTA goes through; from there on its rounds take longer than the cluster's
                                          // barriers (one sequence, 8 heads of 128: 2048 blocks 10.8 us, with the cluster 13.3; 8192 35.7 and 21.6,
                                          // 16384 69.9 and 35.6; eight sequences 2048 24.1 and 30.0, 4096 41.6 and 43.9, 8192 82.9 and 70.7)
constexpr int kAtOnce = 4;                  // blocks of a lane whose bounds are on their way together

template <typename T, int D, bool kGathered>
__global__ void __launch_bounds__(kThreads) kv8_select_kernel(const __grid_constant__ SelectArgs a) {
    constexpr int kLanes = D / 16;                                  // of a block: each has 16 channels of both bounds
    constexpr int kPerWarp = 32 / kLanes;
    extern __shared__ __align__(16) unsigned char smem[];
    uint32_t* key = reinterpret_cast<uint32_t*>(smem);              // [room]
    __shared__ __align__(16) int8_t sm_q[kRowsAtATime][D];
    __shared__ float sm_step[kRowsAtATime];
    __shared__ uint32_t sm_hist[kGathered ? 1 : 4][256];
    __shared__ uint32_t sm_warp[2][kSelectWarps];
    __shared__ uint32_t sm_digit, sm_above, sm_here;
    __shared__ uint32_t sm_count[2];                                // of this CTA's scores: above the threshold, at it
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    if constexpr (kGathered)
        if (a.ctas > 1) cluster.barrier_arrive();                   // the first CTA may be written to once it has started
    grid_dependency_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = (int)(blockIdx.x % a.ctas);
    const int64_t pair = blockIdx.x / a.ctas;
    const int b = (int)(pair / a.c.H), h = (int)(pair % a.c.H);
    const int live = a.p.kv_len ? min(max(a.p.kv_len[b], 0), a.c.S) : a.c.S;
    const int blocks = (live + a.c.block - 1) / a.c.block;
    const int n = new_tokens(a.p.new_len, b, a.p.Sq), rows = a.G * n;
    int32_t* out = a.p.blocks + pair * a.p.count;
    const int per = (blocks + a.ctas - 1) / a.ctas;                 // <= room
    const int j0 = min(rank * per, blocks), mine = min(per, blocks - j0);

    const int total = min(a.p.count, blocks);
    for (int i = total + rank * kThreads + tid; i < a.p.count; i += a.ctas * kThreads) out[i] = -1;
    if (blocks <= a.p.count) {                                      // all of them, in every CTA of the cluster alike
        for (int i = rank * kThreads + tid; i < blocks; i += a.ctas * kThreads) out[i] = i;
        if constexpr (kGathered)
            if (a.ctas > 1) cluster.barrier_wait();
        return;
    }
    if constexpr (!kGathered) {
        for (int i = tid; i < 4 * 256; i += kThreads) (&sm_hist[0][0])[i] = 0;
        if (tid < 2) sm_count[tid] = 0;
    }

    // ---- scores ----
    const uint32_t floor_key = order_of(-INFINITY);
    const int8_t* bounds = a.c.bounds + (pair * a.nb + j0) * 2 * D;
    const float* scale = a.c.k_scale + pair * a.nb + j0;
    const int sub = lane % kLanes, slot = lane / kLanes;
    constexpr int kTurn = kSelectWarps * kPerWarp;                  // blocks that the warps take side by side
    uint4 lo[kAtOnce], hi[kAtOnce];
    float ks[kAtOnce];
    auto load = [&](int base) {
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) {
            const int j = base + x * kTurn + slot;
            lo[x] = hi[x] = make_uint4(0, 0, 0, 0);
            ks[x] = 0.f;
            if (j < mine) {
                const uint4* p = reinterpret_cast<const uint4*>(bounds + (int64_t)j * 2 * D) + sub;
                lo[x] = __ldg(p);
                hi[x] = __ldg(p + kLanes);
                ks[x] = __ldg(scale + j);
            }
        }
    };
    load(warp * kPerWarp);
    uint32_t* to = key;
    if constexpr (kGathered) {
        if (a.ctas > 1) {
            to = cluster.map_shared_rank(key, 0);
            cluster.barrier_wait();
        }
        to += j0;
    }
    int r0 = 0;
    do {
        const int batch = min(rows - r0, kRowsAtATime);
        if (r0) __syncthreads();
        for (int r = warp; r < batch; r += kSelectWarps) {
            const int i = a.p.Sq == 1 ? 0 : (r0 + r) / a.G, g = r0 + r - i * a.G;
            const T* q = reinterpret_cast<const T*>(a.p.q) + b * a.p.q_strides.batch + (int64_t)(h * a.G + g) * a.p.q_strides.head +
                         (int64_t)i * a.p.q_strides.seq;
            float x[D / 32];
            uint32_t most = 0;
#pragma unroll
            for (int y = 0; y < D / 32; ++y) {
                x[y] = ld_value(q + lane + 32 * y);
                most = max(most, finite_abs_bits(x[y]));
            }
            const int e = int8_exponent(__reduce_max_sync(0xffffffffu, most));
            const float down = pow2(-e);
#pragma unroll
            for (int y = 0; y < D / 32; ++y) {
                const float v = x[y] * down;
                sm_q[r][lane + 32 * y] = v == v ? (int8_t)rintf(fminf(fmaxf(v, -127.f), 127.f)) : (int8_t)0;
            }
            if (lane == 0) sm_step[r] = pow2(e);
        }
        __syncthreads();
        for (int base = warp * kPerWarp; base < mine; base += kTurn * kAtOnce) {
            if (base != warp * kPerWarp || r0) load(base);
#pragma unroll
            for (int x = 0; x < kAtOnce; ++x) {
                if (base + x * kTurn >= mine) break;
                const int j = base + x * kTurn + slot;
                const bool there = j < mine;
                uint32_t best = r0 && there ? to[j] : floor_key;
                for (int r = 0; r < batch; ++r) {
                    const uint4 q = *reinterpret_cast<const uint4*>(&sm_q[r][sub * 16]);
                    int sum = 0;
                    auto four = [&](uint32_t qw, uint32_t l, uint32_t u) {
                        const uint32_t neg = signs(qw);
                        sum = __dp4a((int)qw, (int)((l & neg) | (u & ~neg)), sum);
                    };
                    four(q.x, lo[x].x, hi[x].x); four(q.y, lo[x].y, hi[x].y);
                    four(q.z, lo[x].z, hi[x].z); four(q.w, lo[x].w, hi[x].w);
#pragma unroll
                    for (int off = kLanes / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                    const float s = (float)sum * ks[x] * sm_step[r];
                    if (s == s) best = max(best, order_of(s));
                }
                if (there && sub == 0) {
                    const int at = j0 + j;
                    if (r0 + batch == rows && (at < a.p.first || at >= blocks - a.p.last)) best = 0xffffffffu;
                    to[j] = best;
                }
            }
        }
        r0 += batch;
    } while (r0 < rows);

    if constexpr (kGathered) {
        if (a.ctas > 1) {
            cluster.sync();
            if (rank) return;
        } else {
            __syncthreads();
        }
        // ---- the count-th largest: of those that are not taken anyway, from the highest bit in which they differ on ----
        uint32_t need = (uint32_t)(a.p.count - a.p.first - a.p.last), prefix = 0xffffffffu, known = 0xffffffffu;
        if (need) {
            uint32_t low = 0xffffffffu, high = 0;
            for (int i = a.p.first + tid; i < blocks - a.p.last; i += kThreads) { low = min(low, key[i]); high = max(high, key[i]); }
            low = __reduce_min_sync(0xffffffffu, low);
            high = __reduce_max_sync(0xffffffffu, high);
            if (lane == 0) { sm_warp[0][warp] = low; sm_warp[1][warp] = high; }
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kSelectWarps; ++w) { low = min(low, sm_warp[0][w]); high = max(high, sm_warp[1][w]); }
            int open = 32 - __clz(low ^ high);                      // bits that are not known
            known = open == 32 ? 0u : ~0u << open;
            prefix = low & known;
            uint32_t at_prefix = (uint32_t)(blocks - a.p.first - a.p.last);
            while (open > 0 && at_prefix != need) {
                const int bits = min(open, 8), shift = open - bits;
                __syncthreads();
                sm_hist[0][tid] = 0;
                __syncthreads();
                for (int i = a.p.first + tid; i < blocks - a.p.last; i += kThreads) {
                    const uint32_t k = key[i];
                    if ((k & known) == prefix) atomicAdd(&sm_hist[0][(k >> shift) & ((1u << bits) - 1)], 1u);
                }
                __syncthreads();
                const uint32_t mysum = sm_hist[0][tid];
                uint32_t run = mysum;                               // how many lie in this digit and those above
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const uint32_t o = __shfl_down_sync(0xffffffffu, run, off);
                    if (lane + off < 32) run += o;
                }
                if (lane == 0) sm_warp[0][warp] = run;
                __syncthreads();
                uint32_t above = run - mysum;
                for (int w = warp + 1; w < kSelectWarps; ++w) above += sm_warp[0][w];
                if (above < need && above + mysum >= need) { sm_digit = (uint32_t)tid; sm_above = above; sm_here = mysum; }
                __syncthreads();
                prefix |= sm_digit << shift;
                known |= ((1u << bits) - 1) << shift;
                need -= sm_above;
                at_prefix = sm_here;
                open = shift;
            }
        }
        // ---- the indices: a thread has a run of blocks ----
        const int run_len = (blocks + kThreads - 1) / kThreads, i0 = min(tid * run_len, blocks), i1 = min(i0 + run_len, blocks);
        auto sort_of = [&](int i) -> int {                          // 2: taken, 1: at the threshold, 0: below it
            if (i < a.p.first || i >= blocks - a.p.last) return 2;
            const uint32_t k = key[i] & known;
            return k > prefix ? 2 : k == prefix && need ? 1 : 0;
        };
        uint32_t mine_of = 0;                                       // taken, and at the threshold in the upper half
        for (int i = i0; i < i1; ++i) {
            const int c = sort_of(i);
            mine_of += c == 2 ? 1u : c == 1 ? 0x10000u : 0u;
        }
        uint32_t upto = mine_of;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const uint32_t o = __shfl_up_sync(0xffffffffu, upto, off);
            if (lane >= off) upto += o;
        }
        __syncthreads();
        if (lane == 31) sm_warp[0][warp] = upto;
        __syncthreads();
        for (int w = 0; w < warp; ++w) upto += sm_warp[0][w];
        upto -= mine_of;
        uint32_t ups = upto & 0xffffu, ats = upto >> 16;
        for (int i = i0; i < i1; ++i) {
            const int c = sort_of(i);
            if (c == 2 || (c == 1 && ats < need)) out[ups + min(ats, need)] = i;
            ups += c == 2;
            ats += c == 1;
        }
        return;
    } else {
    __syncthreads();

    // ---- the count-th largest ----
    uint32_t prefix = 0, known = 0;                                 // its leading bits, and a mask of them
    uint32_t need = (uint32_t)a.p.count;                            // how many of those that share them are wanted
    uint32_t at_prefix = 0;                                         // and how many do
#pragma unroll 1
    for (int pass = 0; pass < 4; ++pass) {
        const int shift = 24 - 8 * pass;
        for (int i = tid; i < mine; i += kThreads) {
            const uint32_t k = key[i];
            if ((k & known) == prefix) atomicAdd(&sm_hist[pass][(k >> shift) & 255], 1u);
        }
        cluster.sync();
        uint32_t mysum = 0;
        for (int k = 0; k < a.ctas; ++k) mysum += *cluster.map_shared_rank(&sm_hist[pass][tid], k);
        // how many lie in digits above this thread's
        uint32_t run = mysum;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const uint32_t o = __shfl_down_sync(0xffffffffu, run, off);
            if (lane + off < 32) run += o;
        }
        if (lane == 0) sm_warp[0][warp] = run;
        __syncthreads();
        uint32_t above = run - mysum;
        for (int w = warp + 1; w < kSelectWarps; ++w) above += sm_warp[0][w];
        if (above < need && above + mysum >= need) { sm_digit = (uint32_t)tid; sm_above = above; sm_here = mysum; }
        __syncthreads();
        prefix |= sm_digit << shift;
        known |= 255u << shift;
        need -= sm_above;
        at_prefix = sm_here;
        if (at_prefix == need) break;                               // all that share the prefix are wanted
        __syncthreads();
    }
    // ---- the indices ----
    // above: the known bits are larger; at: they are the prefix
    uint32_t n_above = 0, n_at = 0;
    for (int i = tid; i < mine; i += kThreads) {
        const uint32_t k = key[i] & known;
        n_above += k > prefix;
        n_at += k == prefix;
    }
    n_above = __reduce_add_sync(0xffffffffu, n_above);
    n_at = __reduce_add_sync(0xffffffffu, n_at);
    if (lane == 0) {
        atomicAdd(&sm_count[0], n_above);
        atomicAdd(&sm_count[1], n_at);
    }
    cluster.sync();
    uint32_t done = 0, left = need;                                 // places that are taken; how many at the threshold still may be
    for (int k = 0; k < rank; ++k) {
        const uint32_t x = *cluster.map_shared_rank(&sm_count[0], k), y = *cluster.map_shared_rank(&sm_count[1], k);
        const uint32_t take = min(y, left);
        done += x + take;
        left -= take;
    }
    for (int base = 0; base < mine; base += kThreads) {
        const int i = base + tid;
        const uint32_t k = i < mine ? key[i] & known : 0u;
        const bool up = i < mine && k > prefix, at = i < mine && k == prefix;
        const uint32_t vote_up = __ballot_sync(0xffffffffu, up), vote_at = __ballot_sync(0xffffffffu, at), below = (1u << lane) - 1;
        if (lane == 0) { sm_warp[0][warp] = __popc(vote_up); sm_warp[1][warp] = __popc(vote_at); }
        __syncthreads();
        uint32_t ups = 0, ats = 0, all_up = 0, all_at = 0;
        for (int w = 0; w < kSelectWarps; ++w) {
            if (w < warp) { ups += sm_warp[0][w]; ats += sm_warp[1][w]; }
            all_up += sm_warp[0][w];
            all_at += sm_warp[1][w];
        }
        ups += __popc(vote_up & below);
        ats += __popc(vote_at & below);
        if (up || (at && ats < left)) out[done + ups + min(ats, left)] = j0 + i;
        const uint32_t take = min(all_at, left);
        done += all_up + take;
        left -= take;
        __syncthreads();
    }
    cluster.sync();                                                 // until nobody reads this CTA's shared memory
    }
}

template <typename T, int D, bool kGathered>
int launch(ltca_ctx* ctx, const SelectArgs& a) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)((int64_t)a.c.B * a.c.H * a.ctas));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = (size_t)a.room * 4;
    cfg.stream = ctx->stream;
    static SmemOptIn once;
    if (cfg.dynamicSmemBytes > 32 * 1024)
        LTCA_CUDA_OK(ctx, opt_in_dynamic_smem(once, ctx->device, kv8_select_kernel<T, D, kGathered>, 200 * 1024));
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)a.ctas;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.ctas > 1 ? 2 : 1;
    if (a.ctas > 8) {
        static SmemOptIn wide;      // clusters of more than eight CTAs are an opt-in of a kernel on one device
        const uint64_t bit = (ctx->device >= 0 && ctx->device < 64) ? (1ull << ctx->device) : 0ull;
        if (!bit || !(wide.done.load(std::memory_order_acquire) & bit)) {
            LTCA_CUDA_OK(ctx, cudaFuncSetAttribute(kv8_select_kernel<T, D, kGathered>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
            wide.done.fetch_or(bit, std::memory_order_release);
        }
    }
    LTCA_CUDA_OK(ctx, cudaLaunchKernelEx(&cfg, kv8_select_kernel<T, D, kGathered>, a));
    return LTCA_OK;
}
template <typename T, bool kGathered>
int launch_width(ltca_ctx* ctx, const SelectArgs& a) {
    return a.c.D == 32 ? launch<T, 32, kGathered>(ctx, a) : a.c.D == 64 ? launch<T, 64, kGathered>(ctx, a) : launch<T, 128, kGathered>(ctx, a);
}
template <typename T>
int launch_blocks(ltca_ctx* ctx, const SelectArgs& a) {
    return a.nb <= kGather ? launch_width<T, true>(ctx, a) : launch_width<T, false>(ctx, a);
}

}  // namespace

int launch_kv8_select(ltca_ctx* ctx, const ltca_kv8_cache* c, const ltca_kv8_select_params* p) {
    SelectArgs a{*c, *p, (c->S + c->block - 1) / c->block, p->Hq / c->H, p->Hq / c->H * p->Sq, 1, 0};
    // About two CTAs per SM, each with 64 blocks at least.  Both sides, 8 heads of 128, 32 / 64 / 128 at least: one sequence of 256 blocks 5.7 /
    // 6.4 / 7.4 us, eight of 256 9.4 / 7.1 / 7.8, eight of 512 11.5 / 11.5 / 9.0; with 1024 blocks and more all three are alike.
    const int64_t pairs = (int64_t)c->B * c->H;
    while (a.ctas < kMaxSelectCluster && pairs * a.ctas < 2 * kPlanSms && a.nb / (2 * a.ctas) >= 64) a.ctas *= 2;
    while (a.ctas < kMaxSelectCluster && (a.nb + a.ctas - 1) / a.ctas > 48 * 1024) a.ctas *= 2;
    a.room = a.nb <= kGather ? a.nb : (a.nb + a.ctas - 1) / a.ctas;
    if (a.room > 48 * 1024) return fail(ctx, LTCA_ERR_UNSUPPORTED, "select: %d blocks of tokens are too many", a.nb);
    if (pairs * a.ctas > 0x7fffffff) return fail(ctx, LTCA_ERR_INVALID, "select: too many sequences and heads for one call");
    return p->dtype == LTCA_BF16 ? launch_blocks<__nv_bfloat16>(ctx, a) : launch_blocks<float>(ctx, a);
}

}  // namespace ltca
