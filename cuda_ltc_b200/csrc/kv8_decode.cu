// Attention of the newest tokens over an 8-bit cache: see ltca_kv8_decode in include/ltc_attn.h.
//
// The work is one pass over the codes, 2 D bytes a key for the rows (new tokens x heads of queries that share the head of
// keys) of a pair (sequence, head of keys): bound by memory as long as a byte costs the SM little.  On the FMA pipe it costs
// a multiplication per row and the conversions; so the products run on the tensor pipe, transposed, with the rows as the
// narrow side of the tile:
//     S^T [16 keys x 8 rows] = K [16 x D] Q^T [D x 8],      O^T [D x 8] += V^T [D x 16] W^T [16 x 8]
// (m16n8k16, fp16 operands, fp32 accumulators in registers).  e4m3 codes are exact in fp16, so that K and V come from the
// cache with one conversion per two codes and no scale; Q is brought to [1, 2) by a power of two per row and rounded to fp16,
// which keeps bf16's 8 bits; fp32 rows travel in two fp16 terms (22 bits), and so do their weights.  (Products of warps, not
// tcgen05's: its tiles of 64 and 128 rows would be empty but for one to sixteen, and it takes operands from shared memory as they
// lie there, while codes become fp16 on their way and four of a key's bytes have to meet four of the next.)
//
// The order of the contracted index is free as long as both operands agree.  A lane therefore takes whole pieces of rows: of
// K, D/4 bytes of two keys; of V, D/8 bytes of four keys, whose bytes a permutation brings side by side.  The rows come by TMA
// into a ring of the warp's own (a lane issues a step's copies; with cp.async the warps stood in line to issue them), all of whose steps but
// one are on their way: 96 KB of an SM with heads of 128 and 128 KB with narrower ones, up to eight rows, and 64 to 96 KB with sixteen.
//
// Softmax.  With t the score in powers of two, a row keeps a reference m (a whole number) and
//     l = sum 2^(t - m),      O = sum 2^(t - m) v_scale code.
// A weight has to go through fp16, which has 11 bits down to 2^-14, 2^-24 at the least and 2^16 at the most.
//   - bf16 rows: the products are summed on the tensor pipe, so that the scale of the values has to go with the weight.  A second
//     whole number e takes it out again, 2^(t - m) (v_scale 2^(6 - e)): weights lie around 2^6 where they matter and may rise to
//     2^14 before m and e have to move.  What weighs a row's largest weight times scale by 2^-20 and less loses bits, 2^-31 is lost.
//   - fp32 rows: each product is added by the FMA pipe, which multiplies by the scale on the way; weights are 2^(t - m + 10), of two
//     terms, with 22 bits down to 2^-13 of the largest, and 2^-35 at the least.
// So the usual step asks one vote of the warp instead of a reduction of maxima and a multiplication of O, and every factor that
// ever touches O is a power of two.
//
// Every warp works for itself.  The steps of all units (a pair and up to 8 NT of its rows) lie in one line, each unit's behind
// a blank that stands for what a unit costs beside them, and a warp takes an equal run of it, whatever the lengths; it fetches
// across the borders of units, so that the stream does not stop while a unit's queries are brought in or its sums leave.  A
// unit that one warp has seen whole is finished by it; shares of a unit go to scratch and are joined by a second kernel.
// Calls that are over in a few steps take no line: the CTAs of a cluster divide a unit's steps and join their shares through
// each other's shared memory, in one launch (3 sequences of up to 4000 keys 11.0 us; on the line, at an earlier step, 17 against 10.6).
//
// Measured: 74 full caches, 8 heads of keys, 1 / 8 / 16 rows each, bf16 rows and fp32 rows (1.24 GB, 193 us at the memory's rate):
//     8192 keys of 128     204 / 207 / 235 us    208 / 211 / 333
//     16384 keys of 64     216 / 218 / 298       254 / 256 / 394
//     32768 keys of 32     261 / 262 / 360       308 / 310 / 478
// Up to eight rows of 128 are bound by memory.  Sixteen rows are bound by the waits of the few warps that the registers leave on an SM
// (fp32 at 64 also spills), and narrow heads by the work per key, which does not shrink with a key's bytes.  Many short sequences pay
// for what a unit costs beside its steps (by stamps of an earlier step 3500 cycles, with sixteen rows 17000) and for the join: 256 of up to 1024 keys of 64, fp32 rows 47.5 us,
// bf16 rows 41.7, twice the memory's time of 21.
#include <cooperative_groups.h>

#include "kv8.cuh"
#include "kv8_shares.h"

namespace ltca {

namespace {

constexpr int kWarps = 4;                   // of a CTA
constexpr int kThreads = 32 * kWarps;
constexpr int kHead = 48;                   // a step's positions and scales
constexpr int kMaxCluster = 8;              // CTAs that join their shares through shared memory (more would be a launch's opt-in)
constexpr int kClusterSteps = 8;            // of a warp there, at most (8 rows of 128: 8000 keys 16.6 us with 4, 17.6 with 8; 16000 keys 19.3 with 8,
                                            // 26.9 with 16; 128 pairs of up to 3000 keys 22.9 with 4, 21.7 with 8)
constexpr int kMinCost = 4;                 // of a warp's run, where there is little to do (600 pairs of 64 keys of 64: 13.2 us with 2, 13.5 with 4, 17.2 with
                                            // 8; 8 of 16000 keys of 128: 20.7, 19.3, 21.2)
// What a unit costs beside its steps, in steps (1 / 3 / 5: 256 sequences of up to 1024 keys of 64, bf16 54.1 / 42.4 / 43.0 us, fp32 57.4 / 48.3 / 50.9;
// 16 rows, 32 sequences of up to 6001 keys of 128 68.8 / 57.1 / 55.9, 75 of up to 1024 54.9 / 44.8 / 44.1: nearer five there).
constexpr int kUnitCost = 3;
constexpr int kNowhere = 0x7fffffff;        // the position of a group that is not there
constexpr float kNone = -3.402823466e38f;   // the reference of a row that has seen no key
constexpr float kLimit = 16384.f;           // largest weight before the references move
// With fp32 rows: what a weight is multiplied by, and the scale of its values, so that O is 2^-24 of what it stands for and sums of
// values near the end of fp32's range stay inside (e is then 30, a constant).
constexpr float kWeight = 0x1p10f, kValue = 0x1p-34f, kFixed = 30.f;

// A warp's ring: its steps are SG groups of 16 keys, 4 to 8 KB, and all but one are in flight.
constexpr int step_groups(int D) { return D == 32 ? 4 : 2; }
template <int D> constexpr int kGroups = step_groups(D);
template <int D> constexpr int kStepBytes = kGroups<D> * 32 * D;
template <int D> constexpr int kStages = D == 128 ? 2 : 3;
// CTAs of an SM, by the registers that NT tiles of 8 rows take
// (four of 64 channels: 128 registers a thread and three stages; with three CTAs of four stages 74 long caches took 228 us for 209, 256 short
// sequences 46.6 for 42.4 with bf16 rows and 49.7 for 48.3 with fp32)
constexpr int ctas_per_sm(int D, int nt) { return nt * D >= 256 ? 2 : nt == 1 && D <= 64 ? 4 : 3; }
template <int D, int NT> constexpr int kCtas = ctas_per_sm(D, NT);
constexpr int kLens = 256;                  // lengths in shared memory

struct DecodeArgs {
    ltca_kv8_cache c;
    ltca_kv8_decode_params p;
    int nb, G, R;               // blocks of tokens; heads of queries per head of keys; rows of a pair
    int tiles, rows;            // of a pair: tiles of 8 NT rows; rows of a tile that exist (of the first one)
    int warps;                  // that share the line of steps
    int vec_q, vec_o;           // rows of q start on 16-byte boundaries, rows of o on boundaries of four values
    int mask_rows;              // rows of keep_mask that a tile's rows need
    int box;                    // keys of a copy
    int strides;                // what has a stride of its own: sequences of k (1) and v (4), heads of k (2) and v (8)
    int splits;                 // CTAs (a cluster) of a unit; 0: the warps share one line
    float* partial;             // [2 warps][rows][D + 4]
    int2* shares;               // [units]: the warp that has a unit's first step, and how many after it have others
    uint32_t* status;
};

// Steps of each unit of sequence b.
__device__ __forceinline__ int steps_for(const DecodeArgs& a, int len) {
    const int live = min(max(len, 0), a.c.S);
    if (live == 0) return 0;
    const int sg = step_groups(a.c.D);
    if (a.p.blocks) return (a.p.n_blocks * (a.c.block >> 4) + sg - 1) / sg;
    return (live + 16 * sg - 1) / (16 * sg);
}
__device__ __forceinline__ int length_of(const DecodeArgs& a, int b) { return a.p.kv_len ? a.p.kv_len[b] : a.c.S; }
// A unit's head of keys and tile; a row's new token (rows: new token first, then the heads that share).
__device__ __forceinline__ int head_of(const DecodeArgs& a, int unit) { return a.tiles == 1 ? unit : unit / a.tiles; }
__device__ __forceinline__ int tile_of(const DecodeArgs& a, int unit) { return a.tiles == 1 ? 0 : unit % a.tiles; }
__device__ __forceinline__ int token_of(const DecodeArgs& a, int gr) { return a.p.Sq == 1 ? 0 : gr / a.G; }
// Warps that get a run of the line; where warp w's begins; whose a place of the line is.
__device__ __forceinline__ int warps_of(const DecodeArgs& a, int64_t total) {
    return (int)min((int64_t)a.warps, (total + kMinCost - 1) / kMinCost);
}
__device__ __forceinline__ int64_t divided(int64_t a, int64_t b) {                            // neither below zero
    return ((uint64_t)(a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}
__device__ __forceinline__ int64_t run_begin(int64_t total, int warps, int w) { return divided(total * w, warps); }
__device__ __forceinline__ int warp_at(int64_t total, int warps, int64_t at) { return (int)divided((at + 1) * warps - 1, total); }

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d += A (B's terms, low-order first).  The tensor pipe cuts its running sums off instead of rounding them, which over the products of
// a long sequence comes to 1e-6 of the result; with fp32 rows every product is therefore summed from zero and added by the FMA
// pipe, to nearest (8 sequences of up to 16384 keys against 64 bits: 1.4e-6 without, 3.3e-7 with, for 5 to 9 % of the time with up to
// eight rows and up to 30 % with sixteen).
// `by`: a factor of the product (with two terms only).
template <int kTerms>
__device__ __forceinline__ void add_product(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint32_t (&b0)[kTerms],
                                            const uint32_t (&b1)[kTerms], float by = 1.f) {
    if constexpr (kTerms == 1) {
        mma(d, a0, a1, a2, a3, b0[0], b1[0]);
    } else {
        float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = kTerms - 1; i >= 0; --i) mma(x, a0, a1, a2, a3, b0[i], b1[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = fmaf(x[i], by, d[i]);
    }
}
// An 8 x 8 matrix of 16-bit values, two of a row in each lane, transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void codes_to_half2(uint32_t four, uint32_t& low, uint32_t& high) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(low), "=r"(high) : "r"(four));
}
template <int N>
__device__ __forceinline__ void fetch(uint32_t dst, const void* src) {
    if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}
// Four channels of a row of Q as they lie in memory: the largest magnitude so far (an infinity or NaN shows as 2^128 or more),
// the largest finite one, and the values.
struct Four32 {
    float4 v;
    __device__ __forceinline__ void largest(uint32_t& m) const {
        m = max(max(m, __float_as_uint(v.x) & 0x7fffffffu), max(__float_as_uint(v.y) & 0x7fffffffu,
            max(__float_as_uint(v.z) & 0x7fffffffu, __float_as_uint(v.w) & 0x7fffffffu)));
    }
    __device__ __forceinline__ void get(float (&x)[4]) const { x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w; }
};
struct Four16 {
    uint2 v;
    __device__ __forceinline__ void largest(uint32_t& m) const {
        const uint32_t t = __vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu);
        m = max(m, max(t << 16, t & 0xffff0000u));
    }
    __device__ __forceinline__ void get(float (&x)[4]) const {
        x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xffff0000u);
        x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xffff0000u);
    }
};
template <typename T> struct FourOf { using type = Four32; };
template <> struct FourOf<__nv_bfloat16> { using type = Four16; };
__device__ __forceinline__ void store4(float* p, bool vec, const float (&x)[4]) {
    if (vec) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    else
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = x[i];
}
__device__ __forceinline__ void store4(__nv_bfloat16* p, bool vec, const float (&x)[4]) {
    if (vec) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
        *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = __float2bfloat16_rn(x[i]);
    }
}

// How a group of 16 keys lies in the ring, rows of D bytes as TMA leaves them (128-byte swizzle for D = 128, 64-byte for 64), and
// which pieces a lane (r, c) = (lane / 4, lane % 4) takes: of K's rows r and r + 8 the 16-byte chunks c and c + 4 (D = 32: 8
// bytes), of V's rows 2c, 2c + 1, 2c + 8, 2c + 9 the D/8 bytes at r D/8.  Rows eight apart lie alike.
template <int D>
struct Group {
    static constexpr int kParts = D == 128 ? 2 : 1;               // pieces of a key's row of K
    static constexpr int kWords = D == 32 ? 2 : 4;                // words of a piece
    static constexpr int kBytes = 16 * D;                         // of K, or of V
    static __device__ __forceinline__ int swizzled(int row, int byte) {
        if (D == 128) return row * 128 + (byte ^ (row & 7) << 4);
        if (D == 64) return row * 64 + (byte ^ (row >> 1 & 3) << 4);
        return row * 32 + byte;
    }
    // channel of word w of a lane's bytes of K
    static __device__ __forceinline__ int k_dim(int c, int w) { return D == 32 ? c * 8 + 4 * w : (w >> 2) * 64 + c * 16 + 4 * (w & 3); }
};

// The shares of a row joined by a CTA whose warps take them in turn (kWide), or by a warp; a lane has D/32 channels.  part(k):
// share k's m, e, l and its sums behind them.
template <typename T, int D, bool kWide, typename Part>
__device__ __forceinline__ void join_row(int parts, Part part, float (*sm_o)[D], T* out, float* lse) {
    constexpr int E = D / 32;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // lane: a share
    float4 mine = make_float4(kNone, 0.f, 0.f, 0.f);
    if (lane < parts) mine = *reinterpret_cast<const float4*>(part(lane));
    float M = mine.x, L = 0.f, top = -INFINITY;
    for (int k = lane + 32; k < parts; k += 32) M = fmaxf(M, part(k)[0]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
    for (int k = lane; k < parts; k += 32) {
        const float4 x = k < 32 ? mine : *reinterpret_cast<const float4*>(part(k));
        L += x.z * exp2_fast(x.x - M);
        top = fmaxf(top, (x.x - M) + x.y);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        L += __shfl_xor_sync(0xffffffffu, L, off);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    }
    float sum[E];
#pragma unroll
    for (int x = 0; x < E; ++x) sum[x] = 0.f;
    for (int k0 = 0; k0 < parts; k0 += 32) {
        if (k0 && k0 + lane < parts) mine = *reinterpret_cast<const float4*>(part(k0 + lane));
        const float weight = exp2_fast((mine.x - M) + mine.y - top);
        const int n = min(parts - k0, 32);
#pragma unroll 8
        for (int k = kWide ? warp : 0; k < n; k += kWide ? kWarps : 1) {
            const float* src = part(k0 + k);
            const float by = __shfl_sync(0xffffffffu, weight, k);
            if constexpr (E == 4) {
                const float4 x = *reinterpret_cast<const float4*>(src + 4 + lane * 4);
                sum[0] = fmaf(x.x, by, sum[0]); sum[1] = fmaf(x.y, by, sum[1]); sum[2] = fmaf(x.z, by, sum[2]); sum[3] = fmaf(x.w, by, sum[3]);
            } else if constexpr (E == 2) {
                const float2 x = *reinterpret_cast<const float2*>(src + 4 + lane * 2);
                sum[0] = fmaf(x.x, by, sum[0]); sum[1] = fmaf(x.y, by, sum[1]);
            } else {
                sum[0] = fmaf(src[4 + lane], by, sum[0]);
            }
        }
    }
    if constexpr (kWide) {
#pragma unroll
        for (int x = 0; x < E; ++x) sm_o[warp][lane * E + x] = sum[x];
        __syncthreads();
    }
    const float by = L == 0.f ? 0.f : pow2((int)top - 6) / L;
    if constexpr (kWide) {
        if (tid < D) {
            float y = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) y += sm_o[w][tid];
            st_value(out + tid, L == 0.f ? 0.f : y * by);
        }
    } else {
#pragma unroll
        for (int x = 0; x < E; ++x) st_value(out + lane * E + x, L == 0.f ? 0.f : sum[x] * by);
    }
    if ((kWide ? tid : lane) == 0 && lse) *lse = L == 0.f ? -INFINITY : (M == kNone ? 0.f : M * 0.693147181f) + logf(L);
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, kCtas<D, NT>)
kv8_decode_kernel(const __grid_constant__ DecodeArgs a, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    using Gr = Group<D>;
    constexpr int W = D / 16, ROWS = 8 * NT;                      // products of a score; also tiles of 16 channels of O
    constexpr int kTerms = sizeof(T) == 4 ? 2 : 1;
    constexpr bool kQRegs = NT * kTerms * D <= 256;               // Q's fragments stay in registers
    constexpr int ST = kStages<D>, SG = kGroups<D>;
    constexpr int NG = 2;                                         // groups whose products interleave
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ __align__(16) uint2 sm_q[kQRegs ? 1 : kWarps][kQRegs ? 1 : NT][kQRegs ? 1 : kTerms][kQRegs ? 1 : W][32];
    __shared__ __align__(8) uint64_t sm_bar[kWarps][ST];
    __shared__ int64_t sm_before[kThreads + 1];                   // the line up to each thread's sequences
    __shared__ int64_t sm_warp[kWarps];
    __shared__ int sm_len[kLens];
    __shared__ uint32_t sm_abort;
    __shared__ float sm_join[kWarps][D];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = lane >> 2, c = lane & 3;
    if (tid == 0) {
        tma_prefetch_desc(&k_map);
        tma_prefetch_desc(&v_map);
    }
    if (lane < ST) mbar_init(smem_u32(&sm_bar[warp][lane]), 1);
    mbar_fence_init();
    if (tid == 0) sm_abort = 0;
    __syncthreads();                                              // no warp polls a word or uses a barrier that is not set yet
    grid_dependency_wait();

    const int per_b = a.c.H * a.tiles;                            // units of a sequence
    // (from shared memory where they are there: a load takes microseconds while the ring's copies have the way to the SM)
    auto len_of = [&](int b) -> int { return !a.splits && b < kLens ? sm_len[b] : length_of(a, b); };
    auto steps_of = [&](int b) -> int { return steps_for(a, len_of(b)); };
    // a sequence, a unit of it and a step of that
    struct Cursor { int b, unit, s, steps; };
    Cursor f, end;                                                // what is fetched next; the last step of the run
    int me = 0, line_warps = 0;
    int64_t line_total = 0;
    if (a.splits) {
        const int unit = blockIdx.x / a.splits, parts = kWarps * a.splits, w = (blockIdx.x % a.splits) * kWarps + warp;
        f.b = unit / per_b;
        f.unit = unit % per_b;
        f.steps = steps_of(f.b);
        end = f;
        f.s = (int)((uint32_t)f.steps * w / parts);
        end.s = (int)((uint32_t)f.steps * (w + 1) / parts) - 1;
    } else {
        const int chunk = (a.c.B + kThreads - 1) / kThreads;      // sequences of a thread
        int64_t run = 0;
        for (int b = tid * chunk; b < min((tid + 1) * chunk, a.c.B); ++b) {
            const int len = length_of(a, b), steps = steps_for(a, len);
            if (steps) run += (int64_t)(steps + kUnitCost) * per_b;
            if (b < kLens) sm_len[b] = len;
        }
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int64_t o = __shfl_up_sync(0xffffffffu, run, off);
            if (lane >= off) run += o;
        }
        if (lane == 31) sm_warp[warp] = run;
        __syncthreads();
        for (int w = 0; w < warp; ++w) run += sm_warp[w];
        sm_before[tid + 1] = run;
        if (tid == 0) sm_before[0] = 0;
        __syncthreads();
        const int64_t total = sm_before[kThreads];
        const int warps = warps_of(a, total);
        me = warp * gridDim.x + blockIdx.x;
        if (me >= warps) return;
        // the lower lanes look for the run's first place, the upper ones for its last
        const int64_t place = lane < 16 ? run_begin(total, warps, me) : run_begin(total, warps, me + 1) - 1;
        int i = 0;
#pragma unroll
        for (int y = kThreads / 2; y > 0; y >>= 1)
            if (sm_before[i + y] <= place) i += y;                // the last thread whose sequences begin at or before it
        int64_t at = place - sm_before[i];
        Cursor x;
        x.b = i * chunk;
        for (;; ++x.b) {
            x.steps = steps_of(x.b);
            const int64_t cost = x.steps == 0 ? 0 : (int64_t)(x.steps + kUnitCost) * per_b;
            if (at < cost) break;
            at -= cost;
        }
        x.unit = (int)divided(at, x.steps + kUnitCost);
        x.s = (int)(at - (int64_t)x.unit * (x.steps + kUnitCost)) - kUnitCost;              // below zero: in the blank
        f = {__shfl_sync(0xffffffffu, x.b, 0), __shfl_sync(0xffffffffu, x.unit, 0), max(__shfl_sync(0xffffffffu, x.s, 0), 0),
             __shfl_sync(0xffffffffu, x.steps, 0)};
        end = {__shfl_sync(0xffffffffu, x.b, 31), __shfl_sync(0xffffffffu, x.unit, 31), __shfl_sync(0xffffffffu, x.s, 31),
               __shfl_sync(0xffffffffu, x.steps, 31)};
        line_total = total;
        line_warps = warps;
    }
    // steps of the run in the unit that x is in
    auto left_of = [&](const Cursor& x) -> int { return (x.b == end.b && x.unit == end.unit ? end.s + 1 : x.steps) - x.s; };
    int f_left = left_of(f), u_left = f_left;
    if (f_left <= 0 && !a.splits) return;                         // nothing but blanks
    Cursor u = f;                                                 // what is multiplied next
    auto next_unit = [&](Cursor& x) {                             // only where the run has more
        x.s = 0;
        if (++x.unit == per_b) {
            x.unit = 0;
            do x.steps = steps_of(++x.b); while (x.steps == 0);
        }
    };
    auto at_end = [&](const Cursor& x) { return x.b == end.b && x.unit == end.unit; };

    // ---- fetching: K's and V's rows by TMA, scales (and the mask) by cp.async ----
    const int extra = kHead + (a.p.keep_mask ? a.mask_rows * SG * 64 : 0);
    unsigned char* ring = smem + ((1024 - (smem_u32(smem) & 1023)) & 1023);
    unsigned char* heads = ring + kWarps * ST * kStepBytes<D> + warp * ST * extra;
    ring += warp * ST * kStepBytes<D>;
    const WaitCtx wc{&sm_abort, a.status};
    const int log_block = 31 - __clz(a.c.block), log_gpb = log_block - 4;
    const float* sp;                                              // of the fetched unit: k's scales for even lanes, v's for odd ones
    const int32_t* list;
    int f_live, f_h;
    bool f_q = true;                                              // the unit's queries come first, in a stage of their own
    int win, win_next, win_at;                                    // 32 entries of the list, a lane each, the next 32, and where they are
    auto list_at = [&](int i) -> int { return i < a.p.n_blocks ? list[i] : -1; };
    auto fetch_unit = [&]() {
        f_h = head_of(a, f.unit);
        const int64_t pair = (int64_t)f.b * a.c.H + f_h;
        sp = (lane & 1 ? a.c.v_scale : a.c.k_scale) + pair * a.nb;
        list = a.p.blocks ? a.p.blocks + pair * a.p.n_blocks : nullptr;
        f_live = min(len_of(f.b), a.c.S);
        f_q = true;
        if (list) {
            win_at = (f.s * SG >> log_gpb) & ~31;
            win = list_at(win_at + lane);
            win_next = list_at(win_at + 32 + lane);
        }
    };
    auto fetch_queries = [&](uint32_t body, uint32_t bar) {
        // lane: a row's place
        const int mine = tile_of(a, f.unit) * ROWS + lane, token = token_of(a, mine);
        const int64_t place = f.b * a.p.q_strides.batch + (int64_t)(f_h * a.G + mine - token * a.G) * a.p.q_strides.head +
                              (int64_t)token * a.p.q_strides.seq;
        const int rows = min(ROWS, a.R - tile_of(a, f.unit) * ROWS);
        const T* q = reinterpret_cast<const T*>(a.p.q);
        if (a.vec_q) {
            constexpr int kChunks = D * (int)sizeof(T) / 16;      // of a row
#pragma unroll
            for (int j = 0; j < ROWS * kChunks / 32; ++j) {
                const int row = (j * 32 + lane) / kChunks, chunk = (j * 32 + lane) % kChunks;
                const T* src = q + __shfl_sync(0xffffffffu, place, row) + chunk * (16 / (int)sizeof(T));
                if (row < rows) fetch<16>(body + (j * 32 + lane) * 16, src);
            }
        } else {                                                  // rows that start on any element
            T* dst = reinterpret_cast<T*>(smem + (body - smem_u32(smem)));
            for (int row = 0; row < rows; ++row) {
                const T* src = q + __shfl_sync(0xffffffffu, place, row);
#pragma unroll
                for (int d = 0; d < D; d += 32) dst[row * D + d + lane] = src[d + lane];
            }
        }
        if (lane == 0) mbar_arrive(bar);
    };
    auto fetch_step = [&](int stage) {
        if (f_left > 0 && f_q) {
            fetch_queries(smem_u32(ring + stage * kStepBytes<D>), smem_u32(&sm_bar[warp][stage]));
            f_q = false;
        } else if (f_left > 0) {
            const uint32_t head = smem_u32(heads + stage * extra), body = smem_u32(ring + stage * kStepBytes<D>);
            const uint32_t bar = smem_u32(&sm_bar[warp][stage]);
            // lanes 2g and 2g + 1: where group g is
            int pos = kNowhere, blk = -1;
            if (list) {
                const int e = (f.s * SG + min(lane >> 1, SG - 1)) >> log_gpb;
                if (__shfl_sync(0xffffffffu, e, 0) >= win_at + 32) {
                    win_at += 32;
                    win = win_next;
                    win_next = list_at(win_at + 32 + lane);
                }
                blk = __shfl_sync(0xffffffffu, win, e - win_at);
            }
            if (lane < 2 * SG) {
                const int g = f.s * SG + (lane >> 1);
                if (!list) pos = g << 4;
                else if (blk >= 0 && blk < a.nb) pos = (blk << log_block) + ((g & ((1 << log_gpb) - 1)) << 4);
                if (pos >= f_live) pos = kNowhere;
                asm volatile("st.shared.b32 [%0], %1;" ::"r"(head + (lane >> 1) * 4), "r"(pos) : "memory");
                if (pos != kNowhere) fetch<4>(head + 16 + lane * 4, sp + (pos >> log_block));
            }
            if (!list) {                                          // one copy
                if (lane == 0) {
                    mbar_arrive_expect_tx(bar, kStepBytes<D>);
                    tma_load_4d(body, &k_map, bar, 0, pos, a.strides & 2 ? f_h : 0, a.strides & 1 ? f.b : 0);
                    tma_load_4d(body + SG * Gr::kBytes, &v_map, bar, 0, pos, a.strides & 8 ? f_h : 0, a.strides & 4 ? f.b : 0);
                }
            } else {                                              // one for every `box` keys
                const bool copies = pos != kNowhere && (lane & ((a.box >> 3) - 1)) == 0;
                const uint32_t n = __popc(__ballot_sync(0xffffffffu, copies));
                if (lane == 0) mbar_arrive_expect_tx(bar, n * 2 * a.box * D);
                __syncwarp();
                if (copies) {
                    tma_load_4d(body + (lane >> 1) * Gr::kBytes, &k_map, bar, 0, pos, a.strides & 2 ? f_h : 0, a.strides & 1 ? f.b : 0);
                    tma_load_4d(body + (SG + (lane >> 1)) * Gr::kBytes, &v_map, bar, 0, pos, a.strides & 8 ? f_h : 0, a.strides & 4 ? f.b : 0);
                }
            }
            if (a.p.keep_mask) {
                const int i0 = token_of(a, tile_of(a, f.unit) * ROWS), rows = min(a.mask_rows, a.p.Sq - i0);
#pragma unroll
                for (int x = 0; x < SG / 2; ++x) {                 // 32 keys at a time
                    const int base = __shfl_sync(0xffffffffu, pos, 4 * x + 2 * (lane >> 4));
                    const int key = base == kNowhere ? a.c.S : base + (lane & 15);
                    const float* src = a.p.keep_mask + ((int64_t)f.b * a.p.Sq + i0) * a.c.S + key;
                    if (key < a.c.S)
                        for (int i = 0; i < rows; ++i)
                            fetch<4>(head + kHead + ((i * SG + 2 * x) * 16 + lane) * 4, src + (int64_t)i * a.c.S);
                }
            }
            ++f.s;
            if (--f_left == 0 && !at_end(f)) {
                next_unit(f);
                f_left = left_of(f);
                if (f_left > 0) fetch_unit();
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (f_left > 0) fetch_unit();
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) fetch_step(i);

    // ---- a unit's rows: 2c and 2c + 1 of each tile of 8 are this lane's in S^T and O^T, row r in Q ----
    float m[NT][2], inv[NT][2], e[NT][2], l[NT][2], cs[NT][2];       // inv = 2^(6 - e); cs: what a row's S is multiplied by
    // (with two terms e stays at kFixed and inv is not used)
    int lim[NT][2];                                               // keys below it are seen
    int lim_min = 0;
    float o[NT][W][4];
    uint2 qf[kQRegs ? NT : 1][kQRegs ? kTerms : 1][kQRegs ? W : 1];
    uint32_t mask_row = 0;                                        // the mask's rows of this lane's rows, a byte each
    int mask_rows = 0;                                            // that the tile's rows need
    auto clear = [&]() {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
            for (int k = 0; k < 2; ++k) { m[t][k] = kNone; e[t][k] = kTerms == 2 ? kFixed : 200.f; inv[t][k] = pow2(-100); l[t][k] = 0.f; }
#pragma unroll
            for (int i = 0; i < W; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[t][i][k] = 0.f;
        }
    };
    auto start_unit = [&](const unsigned char* rows_q) {
        const int tile = tile_of(a, u.unit), n = new_tokens(a.p.new_len, u.b, a.p.Sq);
        const int len = len_of(u.b), live = min(max(len, 0), a.c.S);
        // lane: a row
        const int mine = tile * ROWS + lane, token = token_of(a, mine);
        int my_lim = 0;
        if (lane < ROWS && mine < a.R && token < n)
            my_lim = a.p.causal ? (int)min((int64_t)live, max((int64_t)len - n + token + 1, (int64_t)0)) : live;
        lim_min = __reduce_min_sync(0xffffffffu, my_lim > 0 ? my_lim : 0x7fffffff);
        if (a.p.keep_mask) {
            const int first = __shfl_sync(0xffffffffu, token, 0), at = min(token - first, 31);
            mask_row = 0;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int k = 0; k < 2; ++k) mask_row |= (uint32_t)__shfl_sync(0xffffffffu, at, t * 8 + 2 * c + k) << (8 * (2 * t + k));
            mask_rows = min(a.mask_rows, a.p.Sq - first);
        }
        if constexpr (!kQRegs) __syncwarp();
        using Four = typename FourOf<T>::type;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const bool there = __shfl_sync(0xffffffffu, my_lim, t * 8 + r) > 0;
            Four x[W];
            uint32_t most = 0;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                x[w] = *reinterpret_cast<const Four*>(reinterpret_cast<const T*>(rows_q) + (t * 8 + r) * D + Gr::k_dim(c, w));
                x[w].largest(most);
            }
            if (__any_sync(0xffffffffu, there && most >= 0x7f800000u)) {             // infinities and NaN do not count
                most = 0;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    float y[4];
                    x[w].get(y);
#pragma unroll
                    for (int k = 0; k < 4; ++k) most = max(most, finite_abs_bits(y[k]));
                }
            }
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const int ex = min(max((int)(most >> 23) - 127, -100), 120);
            const float down = pow2(-ex), up = a.p.scale * 1.44269504f * pow2(ex);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                float y[4];
                x[w].get(y);
#pragma unroll
                for (int k = 0; k < 4; ++k) y[k] *= down;
                uint2 hi = make_uint2(half2_bits(y[0], y[1]), half2_bits(y[2], y[3]));
                if (!there) hi = make_uint2(0, 0);
                if constexpr (kQRegs) qf[t][0][w] = hi;
                else sm_q[warp][t][0][w][lane] = hi;
                if constexpr (kTerms == 2) {
                    const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&hi.x));
                    const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&hi.y));
                    hi = make_uint2(half2_bits(y[0] - f0.x, y[1] - f0.y), half2_bits(y[2] - f1.x, y[3] - f1.y));
                    if (!there) hi = make_uint2(0, 0);
                    if constexpr (kQRegs) qf[t][kTerms - 1][w] = hi;
                    else sm_q[warp][t][kTerms - 1][w][lane] = hi;
                }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                cs[t][k] = __shfl_sync(0xffffffffu, up, (2 * c + k) * 4);
                lim[t][k] = __shfl_sync(0xffffffffu, my_lim, t * 8 + 2 * c + k);
            }
        }
        clear();
        if constexpr (!kQRegs) __syncwarp();
    };
    auto q_at = [&](int t, int x, int w) -> uint2 {
        if constexpr (kQRegs) return qf[t][x][w];
        else return sm_q[warp][t][x][w][lane];
    };
    const bool clamped = a.p.score_clamp > 0.f;
    const float clamp = a.p.score_clamp * 1.44269504f;

    // ---- a step's groups of keys, NG at a time from g0 on ----
    const int k_at = Gr::swizzled(r, D == 32 ? c * 8 : c * 16);
    const int v_at[2] = {Gr::swizzled(2 * c, r * (D / 8) & ~15) + (r * (D / 8) & 15), Gr::swizzled(2 * c + 1, r * (D / 8) & ~15) + (r * (D / 8) & 15)};
    auto step = [&](int stage, int g0) {
        const unsigned char* head = heads + stage * extra;
        int pos[NG];
        float k_scale[NG], v_scale[NG];
        bool some = false, whole = true;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            pos[g] = *reinterpret_cast<const int*>(head + (g0 + g) * 4);
            const float2 sc = *reinterpret_cast<const float2*>(head + 16 + (g0 + g) * 8);
            // a group that is not there has whatever the ring held: all of it is hidden, and its scales are not looked at
            const bool there = pos[g] != kNowhere;
            k_scale[g] = there ? sc.x : 1.f;
            v_scale[g] = there ? (kTerms == 2 ? fminf(sc.y * kValue, 1e38f) : sc.y) : 1.f;
            some |= there;
            whole &= pos[g] <= lim_min - 16;
        }
        if (!some) return;
        // The mask as words, bit = key (of the step's 32 that these groups are among): lane i has the word of its row i.  What
        // hides or shows all of a step's keys from all rows is settled here.
        uint32_t word = 0xffffffffu;
        if (a.p.keep_mask) {
            const float* mask = reinterpret_cast<const float*>(head + kHead) + g0 * 16 + lane;
            uint32_t any = 0, all = 0xffffffffu;
            for (int i = 0; i < mask_rows; ++i) {
                const uint32_t v = __ballot_sync(0xffffffffu, mask[i * SG * 16] != 0.f);
                if (lane == i) word = v;
                any |= v;
                all &= v;
            }
            uint32_t seen = 0;
#pragma unroll
            for (int g = 0; g < NG; ++g)
                if (pos[g] != kNowhere) seen |= 0xffffu << (16 * g);
            if ((any & seen) == 0) return;
            if (all != 0xffffffffu) whole = false;
        }
        const unsigned char* body = ring + stage * kStepBytes<D> + g0 * Gr::kBytes;
        float s[NG][NT][4];
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int x = 0; x < 4; ++x) s[g][t][x] = 0.f;
#pragma unroll
        for (int part = 0; part < Gr::kParts; ++part) {
            constexpr int kWords = Gr::kWords;
            uint32_t w[NG][2][kWords];
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const unsigned char* src = body + g * Gr::kBytes + x * 8 * D + (k_at ^ part * 64);
                    if constexpr (D == 32) {
                        const uint2 v = *reinterpret_cast<const uint2*>(src);
                        w[g][x][0] = v.x; w[g][x][1] = v.y;
                    } else {
                        const uint4 v = *reinterpret_cast<const uint4*>(src);
                        w[g][x][0] = v.x; w[g][x][1] = v.y; w[g][x][2] = v.z; w[g][x][3] = v.w;
                    }
                }
#pragma unroll
            for (int i = 0; i < kWords; ++i)
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    uint32_t a0, a1, a2, a3;
                    codes_to_half2(w[g][0][i], a0, a2);
                    codes_to_half2(w[g][1][i], a1, a3);
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        uint32_t b0[kTerms], b1[kTerms];
#pragma unroll
                        for (int x = 0; x < kTerms; ++x) {
                            const uint2 q = q_at(t, x, part * kWords + i);
                            b0[x] = q.x;
                            b1[x] = q.y;
                        }
                        add_product<kTerms>(s[g][t], a0, a1, a2, a3, b0, b1);
                    }
                }
        }
        // s[g][t][0], [1]: key r of the group with rows 2c, 2c + 1; [2], [3]: key r + 8.  The scores are s ck.
        float ck[NG][NT][2];
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int x = 0; x < 2; ++x) ck[g][t][x] = cs[t][x] * k_scale[g];
        if (__builtin_expect(!whole || clamped, 0)) {
            uint32_t bits[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    bits[t][x] = __shfl_sync(0xffffffffu, word, mask_row >> (8 * (2 * t + x)) & 31) >> r;
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int key = 8 * (x >> 1);
                        float y = s[g][t][x] * ck[g][t][x & 1];
                        if (clamped) y = y > clamp ? clamp : y;                   // (NaN stays)
                        const bool seen = pos[g] != kNowhere && pos[g] + r + key < lim[t][x & 1] &&
                                          (bits[t][x & 1] >> (16 * g + key) & 1);
                        s[g][t][x] = seen ? y : -INFINITY;
                    }
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int t = 0; t < NT; ++t) ck[g][t][0] = ck[g][t][1] = 1.f;
        }
        auto scale_scores = [&]() {
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) s[g][t][x] *= ck[g][t][x & 1];
                    ck[g][t][0] = ck[g][t][1] = 1.f;
                }
        };
        if constexpr (kTerms == 2) scale_scores();                // (frees registers, which these builds lack: 230 us for 208 at 74 caches of 8192 keys of 128)
        float p[NG][NT][4], w[NG][NT][4];
        auto weigh = [&]() -> bool {
            float top = 0.f;
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    float f[2] = {kWeight, kWeight};
                    if constexpr (kTerms == 1) {
                        // between bounds that no weight which counts comes near, so that 0 * f is 0 and a large p shows in w
#pragma unroll
                        for (int x = 0; x < 2; ++x) f[x] = fmaxf(fminf(v_scale[g] * inv[t][x], 1e38f), 1e-24f);
                    }
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        p[g][t][x] = exp2_fast(fmaf(s[g][t][x], ck[g][t][x & 1], -m[t][x & 1]));
                        w[g][t][x] = p[g][t][x] * f[x & 1];
                        if constexpr (kTerms == 2) p[g][t][x] = w[g][t][x];      // (l is brought down once, where it leaves)
                        top = fmaxf(top, w[g][t][x]);
                    }
                }
            return top > kLimit;
        };
        if (__builtin_expect(__any_sync(0xffffffffu, weigh()), 0)) {
            // The scores as fp32 has them, and no longer products behind which the reference lies by up to half a unit in their last
            // place: from 2^28 on that would be a weight above fp16's range.
            scale_scores();
            // `worth`: what the weight of key r, or r + 8, brings to O besides itself, in powers of two
            auto move = [&](const float (&worth)[NG][2]) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float top = -INFINITY;
#pragma unroll
                        for (int g = 0; g < NG; ++g) top = fmaxf(top, fmaxf(s[g][t][x], s[g][t][x + 2]));
#pragma unroll
                        for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                        const float m2 = fmaxf(m[t][x], ceilf(top));
                        const bool first = m[t][x] == kNone;
                        const float dm = m[t][x] - m2;
                        float y = e[t][x], fo = 1.f;
                        bool moves = m2 > kNone && m2 < INFINITY;    // the row has seen a key
                        if constexpr (kTerms == 1) {
                            y = -INFINITY;
#pragma unroll
                            for (int g = 0; g < NG; ++g) y = fmaxf(y, fmaxf(s[g][t][x] - m2 + worth[g][0], s[g][t][x + 2] - m2 + worth[g][1]));
#pragma unroll
                            for (int off = 4; off < 32; off <<= 1) y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, off));
                            y = fmaxf(first ? -INFINITY : e[t][x] + dm, ceilf(y));
                            moves = y > -1000.f && y < 1000.f;
                        }
                        if (moves) {
                            if (!first) fo = exp2_fast(kTerms == 1 ? e[t][x] + dm - y : dm);
                            l[t][x] *= first ? 1.f : exp2_fast(dm);
                            m[t][x] = m2;
                            if constexpr (kTerms == 1) { e[t][x] = y; inv[t][x] = exp2_fast(6.f - y); }
#pragma unroll
                            for (int i = 0; i < W; ++i) { o[t][i][x] *= fo; o[t][i][x + 2] *= fo; }
                        }
                    }
            };
            float worth[NG][2];
            uint32_t zero = 0;                                      // keys that have no value but zero: bit 2 g, 2 g + 1
            if constexpr (kTerms == 1) {
                // A weight brings itself times the scale of its values - unless they are all zero, when a reference by the scale
                // could push what the others bring out of fp16.  Keys with four zeros are looked at whole.
                bool some_zero = false;
#pragma unroll
                for (int g = 0; g < NG; ++g)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        worth[g][x] = fmaxf(log2f(v_scale[g]), -110.f);
                        some_zero |= (*reinterpret_cast<const uint32_t*>(body + (SG + g) * Gr::kBytes + x * 8 * D + k_at) & 0x7f7f7f7fu) == 0;
                    }
                if (__builtin_expect(__any_sync(0xffffffffu, some_zero), 0)) {
#pragma unroll
                    for (int g = 0; g < NG; ++g)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            uint32_t any = 0;
#pragma unroll
                            for (int part = 0; part < Gr::kParts; ++part) {
                                const uint32_t* src = reinterpret_cast<const uint32_t*>(body + (SG + g) * Gr::kBytes + x * 8 * D + (k_at ^ part * 64));
#pragma unroll
                                for (int i = 0; i < Gr::kWords; ++i) any |= src[i] & 0x7f7f7f7fu;
                            }
                            any |= __shfl_xor_sync(0xffffffffu, any, 1);
                            any |= __shfl_xor_sync(0xffffffffu, any, 2);
                            if (any == 0) {
                                zero |= 1u << (2 * g + x);
                                worth[g][x] = -110.f;               // as the smallest value there is
                            }
                        }
                }
            }
            move(worth);
            weigh();
            if constexpr (kTerms == 1)
                if (__builtin_expect(zero != 0, 0)) {
#pragma unroll
                    for (int g = 0; g < NG; ++g)
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int x = 0; x < 4; ++x)
                                if (zero >> (2 * g + (x >> 1)) & 1) w[g][t][x] = 0.f;
                }
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            uint32_t w0[NT][kTerms], w1[NT][kTerms];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int x = 0; x < 4; ++x) l[t][x & 1] += p[g][t][x];
                const uint32_t h0 = half2_bits(w[g][t][0], w[g][t][1]), h1 = half2_bits(w[g][t][2], w[g][t][3]);
                w0[t][0] = transposed(h0); w1[t][0] = transposed(h1);
                if constexpr (kTerms == 2) {
                    const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&h0));
                    const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
                    w0[t][1] = transposed(half2_bits(w[g][t][0] - f0.x, w[g][t][1] - f0.y));
                    w1[t][1] = transposed(half2_bits(w[g][t][2] - f1.x, w[g][t][3] - f1.y));
                }
            }
            constexpr int VW = D / 32;                              // words of V per key and lane
            uint32_t v[4][VW];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const unsigned char* src = body + (SG + g) * Gr::kBytes + (x >> 1) * 8 * D + v_at[x & 1];
                if constexpr (D == 128) {
                    const uint4 y = *reinterpret_cast<const uint4*>(src);
                    v[x][0] = y.x; v[x][1] = y.y; v[x][2] = y.z; v[x][3] = y.w;
                } else if constexpr (D == 64) {
                    const uint2 y = *reinterpret_cast<const uint2*>(src);
                    v[x][0] = y.x; v[x][1] = y.y;
                } else {
                    v[x][0] = *reinterpret_cast<const uint32_t*>(src);
                }
            }
            if (__builtin_expect(!whole, 0)) {
                // NaN among the values counts for the rows that see its key and for no other: it becomes zero, and a product
                // of "is NaN" with "is seen" says whose sums it reaches.
                uint32_t nan[4][VW], any = 0;
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int i = 0; i < VW; ++i) {
                        nan[x][i] = __vcmpeq4(v[x][i] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                        any |= nan[x][i];
                    }
                if (__any_sync(0xffffffffu, any != 0)) {
                    uint32_t i0[NT], i1[NT];
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        auto is = [&](int x) { return s[g][t][x] == -INFINITY ? 0.f : 1.f; };
                        i0[t] = transposed(half2_bits(is(0), is(1)));
                        i1[t] = transposed(half2_bits(is(2), is(3)));
                    }
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        // code 0x38 is 1
                        auto pick = [&](int x, int half) {
                            return e4m3x2_to_half2(__byte_perm(nan[x][i >> 1], nan[x + 1][i >> 1],
                                                               (i & 1) ? (half ? 0x73 : 0x62) : (half ? 0x51 : 0x40)) & 0x3838u);
                        };
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            float hit[4] = {0.f, 0.f, 0.f, 0.f};
                            mma(hit, pick(0, 0), pick(0, 1), pick(2, 0), pick(2, 1), i0[t], i1[t]);
#pragma unroll
                            for (int x = 0; x < 4; ++x)
                                if (hit[x] > 0.f) o[t][i][x] = __int_as_float(0x7fc00000);
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 4; ++x)
#pragma unroll
                        for (int i = 0; i < VW; ++i) v[x][i] &= ~nan[x][i];
                }
            }
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const uint32_t sel = (i & 1) ? 0x7362 : 0x5140;
                uint32_t a0, a1, a2, a3;
                codes_to_half2(__byte_perm(v[0][i >> 1], v[1][i >> 1], sel), a0, a1);
                codes_to_half2(__byte_perm(v[2][i >> 1], v[3][i >> 1], sel), a2, a3);
#pragma unroll
                for (int t = 0; t < NT; ++t) add_product<kTerms>(o[t][i], a0, a1, a2, a3, w0[t], w1[t], v_scale[g]);
            }
        }
    };

    // ---- a unit's sums leave: finished where this warp has seen all of it, else to scratch ----
    auto end_unit = [&](bool mine, float* slot) {
        // lane: a row's place
        const int h = head_of(a, u.unit), my_row = tile_of(a, u.unit) * ROWS + lane, token = token_of(a, my_row);
        const int head = h * a.G + my_row - token * a.G, rows = min(ROWS, a.R - tile_of(a, u.unit) * ROWS);
        const int64_t place = u.b * a.p.o_strides.batch + head * a.p.o_strides.head + token * a.p.o_strides.seq;
        const int64_t lse_place = ((int64_t)u.b * a.p.Hq + head) * a.p.Sq + token;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float sum = l[t][x];
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                if constexpr (kTerms == 2) sum *= 1.f / kWeight;
                const int row = t * 8 + 2 * c + x;
                if (mine) {
                    T* out = reinterpret_cast<T*>(a.p.o) + __shfl_sync(0xffffffffu, place, row) + r * (D / 8);
                    const int64_t at = __shfl_sync(0xffffffffu, lse_place, row);
                    const bool dead = lim[t][x] == 0 || sum == 0.f;
                    const float by = pow2((int)e[t][x] - 6) / sum;
                    if (row < rows) {
#pragma unroll
                        for (int i = 0; i < W; i += 2) {
                            const float y[4] = {dead ? 0.f : o[t][i][x] * by, dead ? 0.f : o[t][i][x + 2] * by,
                                                dead ? 0.f : o[t][i + 1][x] * by, dead ? 0.f : o[t][i + 1][x + 2] * by};
                            store4(out + 2 * i, a.vec_o != 0, y);
                        }
                        if (r == 0 && a.p.lse) a.p.lse[at] = dead ? -INFINITY : (m[t][x] == kNone ? 0.f : m[t][x] * 0.693147181f) + logf(sum);
                    }
                } else if (row < rows) {
                    float* dst = slot + row * (D + 4);
                    if (r == 0) *reinterpret_cast<float4*>(dst) = make_float4(m[t][x], e[t][x], sum, 0.f);
#pragma unroll
                    for (int i = 0; i < W; i += 2)
                        *reinterpret_cast<float4*>(dst + 4 + r * (D / 8) + 2 * i) =
                            make_float4(o[t][i][x], o[t][i][x + 2], o[t][i + 1][x], o[t][i + 1][x + 2]);
                }
            }
    };

    int stage = 0;
    uint32_t parity = 0;
    bool from_start = u.s == 0, u_q = true;
    if (u_left <= 0) clear();
    while (u_left > 0) {
        fetch_step(stage == 0 ? ST - 1 : stage - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(ST - 1) : "memory");
        if (!mbar_wait_warp(smem_u32(&sm_bar[warp][stage]), parity, wc, 0x81)) {
            // given up: what else this warp has on its way gets a last, short while
            for (int i = 0; i < ST; ++i)
                for (int x = 0; x < 4096 && !mbar_try_wait(smem_u32(&sm_bar[warp][i]), i < stage ? parity ^ 1 : parity); ++x) {}
            break;
        }
        __syncwarp();                                               // the step's head and mask are read by all lanes
        if (u_q) {
            start_unit(ring + stage * kStepBytes<D>);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // TMA writes next where these rows lay
        } else {
#pragma unroll 1
            for (int g = 0; g < SG; g += NG) step(stage, g);
        }
        __syncwarp();
        if (++stage == ST) { stage = 0; parity ^= 1; }
        if (u_q) {
            u_q = false;
            continue;
        }
        ++u.s;
        if (--u_left > 0 || a.splits) continue;
        const bool to_end = u.s == u.steps;
        if (from_start && lane == 0) {
            // the run ends in this unit, whose last step is as many places on as it has steps left
            const int64_t last = run_begin(line_total, line_warps, me + 1) - 1 + (u.steps - u.s);
            a.shares[(int64_t)u.b * per_b + u.unit] = make_int2(me, to_end ? 0 : warp_at(line_total, line_warps, last) - me);
        }
        end_unit(from_start && to_end, a.partial + (int64_t)(2 * me + (to_end ? 0 : from_start ? 1 : 0)) * a.rows * (D + 4));
        if (at_end(u)) break;
        next_unit(u);
        u_left = left_of(u);
        if (u_left <= 0) break;
        from_start = u_q = true;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    grid_launch_dependents();                                     // the join's CTAs may come as these leave
    if (!a.splits) return;

    // ---- the cluster's shares, over the rings; its CTAs take the rows in turn ----
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    float* share = reinterpret_cast<float*>(ring - warp * ST * kStepBytes<D>);
    __syncthreads();
    end_unit(false, share + warp * a.rows * (D + 4));
    if (a.splits > 1) cluster.sync();
    else __syncthreads();
    const int tile = tile_of(a, u.unit), h = head_of(a, u.unit), rank = blockIdx.x % a.splits;
    const int n = new_tokens(a.p.new_len, u.b, a.p.Sq), len = length_of(a, u.b);
    for (int row = rank; row < ROWS && tile * ROWS + row < a.R; row += a.splits) {
        const int gr = tile * ROWS + row, i = token_of(a, gr);
        T* out = reinterpret_cast<T*>(a.p.o) + u.b * a.p.o_strides.batch + (int64_t)(h * a.G + gr - token_of(a, gr) * a.G) * a.p.o_strides.head +
                 (int64_t)i * a.p.o_strides.seq;
        float* lse = a.p.lse ? a.p.lse + ((int64_t)u.b * a.p.Hq + h * a.G + gr - token_of(a, gr) * a.G) * a.p.Sq + i : nullptr;
        if (len <= 0 || i >= n || (a.p.causal && (int64_t)len - n + i + 1 <= 0)) {
            if (tid < D) st_value(out + tid, 0.f);
            if (tid == 0 && lse) *lse = -INFINITY;
            continue;
        }
        join_row<T, D, true>(kWarps * a.splits, [&](int k) -> const float* {
            const float* mine = share + ((k & (kWarps - 1)) * a.rows + row) * (D + 4);
            return a.splits > 1 ? cluster.map_shared_rank(mine, k / kWarps) : mine;
        }, sm_join, out, lse);
        __syncthreads();
    }
    if (a.splits > 1) cluster.sync();                               // until nobody reads this CTA's shared memory
}

// The warps' shares of a unit's rows joined; what no warp or a single one has seen is zeros, or finished already.  A warp takes a
// row; where units have many shares (kWide) a CTA does, whose threads first weigh the shares side by side.
constexpr int kWideThreads = 512;
template <typename T, int D, bool kWide>
__global__ void __launch_bounds__(kWide ? kWideThreads : kThreads) kv8_decode_join_kernel(const __grid_constant__ DecodeArgs a, int tile_rows) {
    constexpr int kTeam = kWide ? kWideThreads : 32, E = D / 32;
    __shared__ float sm_o[kWide ? kWideThreads / 32 : 1][D], sm_w[kWide ? kWideThreads : 1], sm_x[3][kWideThreads / 32];
    grid_dependency_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, first = kWide ? tid : lane;
    const uint32_t per_b = a.c.H * a.tiles, at = kWide ? blockIdx.x : blockIdx.x * kWarps + warp;      // rows of all units
    const uint32_t place = a.rows == 1 ? at : at / (uint32_t)a.rows;
    const int row = (int)(at - place * a.rows), b = (int)(place / per_b), unit = (int)(place - b * per_b);
    const int tile = tile_of(a, unit), h = head_of(a, unit), gr = tile * tile_rows + row;
    if (b >= a.c.B || gr >= a.R) return;
    const int2 who = a.shares[place];
    const int len = length_of(a, b), steps = steps_for(a, len), i = token_of(a, gr);
    T* out = reinterpret_cast<T*>(a.p.o) + b * a.p.o_strides.batch + (int64_t)(h * a.G + gr - i * a.G) * a.p.o_strides.head +
             (int64_t)i * a.p.o_strides.seq;
    float* lse = a.p.lse ? a.p.lse + ((int64_t)b * a.p.Hq + h * a.G + gr - i * a.G) * a.p.Sq + i : nullptr;
    const int n = new_tokens(a.p.new_len, b, a.p.Sq);
    if (steps == 0 || i >= n || (a.p.causal && (int64_t)len - n + i + 1 <= 0)) {
        for (int d = first; d < D; d += kTeam) st_value(out + d, 0.f);
        if (first == 0 && lse) *lse = -INFINITY;
        return;
    }
    if (!shares_are_there(who.x, who.y, a.warps)) {               // a warp gave up: the row is unknown
        for (int d = first; d < D; d += kTeam) st_value(out + d, __int_as_float(0x7fc00000));
        if (first == 0 && lse) *lse = __int_as_float(0x7fc00000);
        return;
    }
    if (who.y == 0) return;
    // the first share is the last thing that its warp did, the others the first
    const int parts = who.y + 1;
    auto part = [&](int k) -> const float* { return a.partial + ((int64_t)(2 * (who.x + k) + (k == 0 ? 1 : 0)) * a.rows + row) * (D + 4); };
    if constexpr (!kWide) {
        join_row<T, D, false>(parts, part, sm_o, out, lse);
    } else {
        float4 mine = make_float4(kNone, 0.f, 0.f, 0.f);
        if (tid < parts) mine = *reinterpret_cast<const float4*>(part(tid));
        float M = mine.x, L = 0.f, top = -INFINITY;
        for (int k = tid + kTeam; k < parts; k += kTeam) M = fmaxf(M, part(k)[0]);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
        if (lane == 0) sm_x[0][warp] = M;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kTeam / 32; ++w) M = fmaxf(M, sm_x[0][w]);
        for (int k = tid; k < parts; k += kTeam) {
            const float4 x = k < kTeam ? mine : *reinterpret_cast<const float4*>(part(k));
            L += x.z * exp2_fast(x.x - M);
            top = fmaxf(top, (x.x - M) + x.y);
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
            L += __shfl_xor_sync(0xffffffffu, L, off);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        }
        if (lane == 0) { sm_x[1][warp] = L; sm_x[2][warp] = top; }
        __syncthreads();
        L = 0.f;
#pragma unroll
        for (int w = 0; w < kTeam / 32; ++w) { L += sm_x[1][w]; top = fmaxf(top, sm_x[2][w]); }
        float sum[E];
#pragma unroll
        for (int x = 0; x < E; ++x) sum[x] = 0.f;
        for (int k0 = 0; k0 < parts; k0 += kTeam) {
            if (k0) {
                if (k0 + tid < parts) mine = *reinterpret_cast<const float4*>(part(k0 + tid));
                __syncthreads();
            }
            sm_w[tid] = exp2_fast((mine.x - M) + mine.y - top);
            __syncthreads();
            const int m = min(parts - k0, kTeam);
#pragma unroll 4
            for (int k = warp; k < m; k += kTeam / 32) {
                const float* src = part(k0 + k) + 4 + lane;
#pragma unroll
                for (int x = 0; x < E; ++x) sum[x] = fmaf(src[32 * x], sm_w[k], sum[x]);
            }
        }
#pragma unroll
        for (int x = 0; x < E; ++x) sm_o[warp][lane + 32 * x] = sum[x];
        __syncthreads();
        if (tid < D) {
            float y = 0.f;
#pragma unroll
            for (int w = 0; w < kTeam / 32; ++w) y += sm_o[w][tid];
            st_value(out + tid, L == 0.f ? 0.f : y * (pow2((int)top - 6) / L));
        }
        if (tid == 0 && lse) *lse = L == 0.f ? -INFINITY : (M == kNone ? 0.f : M * 0.693147181f) + logf(L);
    }
}

// How a call is cut up; a function of the problem alone, so that the size query and the launch agree.
struct Plan { int nt, tiles, rows, warps, splits; };
Plan plan_of(const ltca_kv8_cache* c, const ltca_kv8_decode_params* p) {
    const int R = p->Hq / c->H * p->Sq;
    Plan s;
    // (four tiles a warp leave the registers no room for two groups at once: 40 rows of 4000 keys of 128 85 us, in two passes 56)
    s.nt = R <= 8 ? 1 : 2;
    s.tiles = (R + 8 * s.nt - 1) / (8 * s.nt);
    s.rows = R < 8 * s.nt ? R : 8 * s.nt;
    const int64_t units = (int64_t)c->B * c->H * s.tiles;
    int64_t keys = c->S;
    if (p->blocks) keys = (int64_t)(p->n_blocks > 1 ? p->n_blocks : 1) * c->block;
    const int sg = step_groups(c->D);
    const int64_t steps = (keys + 16 * sg - 1) / (16 * sg), full = (int64_t)kPlanSms * ctas_per_sm(c->D, s.nt);
    // One cluster a unit where all of them are on the SMs at once and no warp gets more than a few steps.
    s.splits = 0;
    s.warps = 0;
    if (units <= full) {
        int n = (int)(full / units);
        if (n > kMaxCluster) n = kMaxCluster;
        if (n > (steps + kWarps - 1) / kWarps) n = (int)((steps + kWarps - 1) / kWarps);
        // Sizes between the powers of two only where a tenth of the SMs' places stays free: clusters of them leave gaps, and one
        // that comes late costs as much again (64 units in sixes 19.3 us, in fours 21.9; 144 in threes 15.9, in twos 11.6).
        const int between = n == 6 || n == 7 ? 6 : n == 3 ? 3 : 0;
        if (between && units * between * 10 <= full * 9) n = between;
        else
            while (n & (n - 1)) n &= n - 1;
        if (steps <= (int64_t)kClusterSteps * kWarps * n) {
            s.splits = n;
            return s;
        }
    }
    const int64_t want = (units * (steps + kUnitCost) + kMinCost - 1) / kMinCost;
    s.warps = (int)(want < full * kWarps ? want : full * kWarps);
    return s;
}
size_t partial_bytes(const ltca_kv8_cache* c, const Plan& s) {
    return align_up((size_t)2 * s.warps * s.rows * (c->D + 4) * sizeof(float), 256);
}
size_t shares_bytes(const ltca_kv8_cache* c, const Plan& s) {
    return s.splits ? 0 : align_up((size_t)c->B * c->H * s.tiles * sizeof(int2), 256);
}

// Keys or values as TMA sees them: [B, H, S, D] bytes, `box` keys a copy.
int make_map(ltca_ctx* ctx, CUtensorMap* map, const void* base, const ltca_strides& st, const DecodeArgs& a, int own) {
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return fail(ctx, LTCA_ERR_CUDA, "cuTensorMapEncodeTiled entry point not available");
    const int64_t limit = (int64_t)1 << 40;
    if (st.seq < 0 || st.head < 0 || st.batch < 0 || st.seq >= limit || st.head >= limit || st.batch >= limit || (st.seq == 0 && a.c.S > 1))
        return fail(ctx, LTCA_ERR_UNSUPPORTED, "decode needs a cache whose strides are between 0 (tokens: 16) and 2^40 bytes");
    // a stride that moves nothing is not told: its extent is one, and the coordinate stays 0
    const cuuint64_t dims[4] = {(cuuint64_t)a.c.D, (cuuint64_t)a.c.S, (cuuint64_t)(own & 2 ? a.c.H : 1), (cuuint64_t)(own & 1 ? a.c.B : 1)};
    const cuuint64_t strides[3] = {(cuuint64_t)(a.c.S > 1 ? st.seq : 16), (cuuint64_t)(own & 2 ? st.head : 16), (cuuint64_t)(own & 1 ? st.batch : 16)};
    const cuuint32_t box[4] = {(cuuint32_t)a.c.D, (cuuint32_t)a.box, 1, 1}, steps[4] = {1, 1, 1, 1};
    const CUtensorMapSwizzle swizzle = a.c.D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : a.c.D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_NONE;
    const CUresult rc = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(base), dims, strides, box, steps,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return rc == CUDA_SUCCESS ? LTCA_OK : fail(ctx, LTCA_ERR_CUDA, "cuTensorMapEncodeTiled failed with CUresult %d", (int)rc);
}

template <typename T, int D, int NT>
int launch(ltca_ctx* ctx, const DecodeArgs& a) {
    CUtensorMap k_map, v_map;
    if (int rc = make_map(ctx, &k_map, a.c.k, a.c.k_strides, a, a.strides)) return rc;
    if (int rc = make_map(ctx, &v_map, a.c.v, a.c.v_strides, a, a.strides >> 2)) return rc;
    const int extra = kHead + (a.p.keep_mask ? a.mask_rows * kGroups<D> * 64 : 0);
    constexpr int shares = kWarps * 8 * NT * (D + 4) * 4;
    const int ring = kWarps * kStages<D> * (kStepBytes<D> + extra), bytes = 1024 + (ring > shares ? ring : shares);
    constexpr int most = 1024 + kWarps * kStages<D> * (kStepBytes<D> + kHead + 8 * NT * kGroups<D> * 64);     // a mask row for every row
    static SmemOptIn once;
    LTCA_CUDA_OK(ctx, opt_in_dynamic_smem(once, ctx->device, kv8_decode_kernel<T, D, NT>, most > shares ? most : shares));
    const int64_t units = (int64_t)a.c.B * a.c.H * a.tiles;
    if (!a.splits) {
        const dim3 grid((unsigned)((a.warps + kWarps - 1) / kWarps));
        LTCA_CUDA_OK(ctx, launch_dependent(kv8_decode_kernel<T, D, NT>, grid, dim3(kThreads), bytes, ctx->stream, a, k_map, v_map));
        // a CTA for each row where a unit has many shares (8 rows of 16000 / 30000 keys of 128, 74 and more warps a unit: 19.3 / 25.0 us, with a
        // warp a row 43.0 / 65.8; 4 warps a unit 209 and 211; between 9 and 14 a CTA a row is faster for one row and for four, 23.9 against 28.4
        // and 30.8 against 32.8, and slower for eight, 106.0 against 102.8)
        const bool wide = a.warps > 16 * units;
        auto join = wide ? kv8_decode_join_kernel<T, D, true> : kv8_decode_join_kernel<T, D, false>;
        const int64_t rows = units * a.rows;
        const dim3 joins((unsigned)(wide ? rows : (rows + kWarps - 1) / kWarps));
        LTCA_CUDA_OK(ctx, launch_dependent(join, dim3(joins), dim3(wide ? kWideThreads : kThreads), 0, ctx->stream, a, 8 * NT));
        return LTCA_OK;
    }
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)(units * a.splits));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)a.splits;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.splits > 1 ? 2 : 1;
    LTCA_CUDA_OK(ctx, cudaLaunchKernelEx(&cfg, kv8_decode_kernel<T, D, NT>, a, k_map, v_map));
    return LTCA_OK;
}
template <typename T, int D>
int launch_rows(ltca_ctx* ctx, const DecodeArgs& a, int nt) {
    return nt == 1 ? launch<T, D, 1>(ctx, a) : launch<T, D, 2>(ctx, a);
}
template <typename T>
int launch_width(ltca_ctx* ctx, const DecodeArgs& a, int nt) {
    return a.c.D == 32 ? launch_rows<T, 32>(ctx, a, nt) : a.c.D == 64 ? launch_rows<T, 64>(ctx, a, nt) : launch_rows<T, 128>(ctx, a, nt);
}

}  // namespace

size_t kv8_decode_workspace(const ltca_kv8_cache* c, const ltca_kv8_decode_params* p) {
    const Plan s = plan_of(c, p);
    return partial_bytes(c, s) + shares_bytes(c, s);
}

int launch_kv8_decode(ltca_ctx* ctx, const ltca_kv8_cache* c, const ltca_kv8_decode_params* p) {
    const Plan s = plan_of(c, p);
    if ((int64_t)c->B * c->H * s.tiles * s.rows > 0x7fffffff) return fail(ctx, LTCA_ERR_INVALID, "too many rows of queries for one call");
    if (p->blocks && (int64_t)p->n_blocks * c->block > (1 << 30))
        return fail(ctx, LTCA_ERR_UNSUPPORTED, "the listed blocks hold more than 2^30 tokens");
    DecodeArgs a;
    memset(&a, 0, sizeof(a));
    a.c = *c; a.p = *p;
    a.nb = (c->S + c->block - 1) / c->block;
    a.G = p->Hq / c->H;
    a.R = a.G * p->Sq;
    a.tiles = s.tiles; a.rows = s.rows; a.warps = s.warps; a.splits = s.splits;
    const int es = elem_size(p->dtype);
    auto on = [&](const void* ptr, const ltca_strides& st, int to) {
        return !((reinterpret_cast<uintptr_t>(ptr) | (uintptr_t)(st.batch * es) | (uintptr_t)(st.head * es) | (uintptr_t)(st.seq * es)) & (to - 1));
    };
    a.vec_q = on(p->q, p->q_strides, 16);
    a.vec_o = on(p->o, p->o_strides, 4 * es);
    // new tokens that 8 NT rows in a line reach
    const int span = (8 * s.nt - 1 + a.G - 1) / a.G + 1;
    a.mask_rows = span < p->Sq ? span : p->Sq;
    a.box = 16 * step_groups(c->D);
    if (p->blocks && c->block < a.box) a.box = c->block;
    a.strides = (c->B > 1 && c->k_strides.batch ? 1 : 0) | (c->H > 1 && c->k_strides.head ? 2 : 0) |
                (c->B > 1 && c->v_strides.batch ? 4 : 0) | (c->H > 1 && c->v_strides.head ? 8 : 0);
    a.status = ctx->d_status;
    const size_t need = partial_bytes(c, s) + shares_bytes(c, s);
    if (need && (!p->workspace || p->workspace_bytes < need)) return fail(ctx, LTCA_ERR_WORKSPACE, "decode needs %zu bytes of workspace", need);
    a.partial = reinterpret_cast<float*>(p->workspace);
    a.shares = reinterpret_cast<int2*>(static_cast<char*>(p->workspace) + partial_bytes(c, s));
    return p->dtype == LTCA_BF16 ? launch_width<__nv_bfloat16>(ctx, a, s.nt) : launch_width<float>(ctx, a, s.nt);
}

}  // namespace ltca
