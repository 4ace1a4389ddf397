// Attention of the newest tokens over an 8-bit cache: see ltca_kv8_decode in include/ltc_attn.h.
//
// The work is one pass over the codes, 2 D bytes a key for the rows (new tokens x heads of queries that share the head of
// keys) of a pair (sequence, head of keys): bound by memory as long as a byte costs the SM little.  On the FMA pipe it costs
// a multiplication per row and the conversions; so the products run on the tensor pipe, transposed, with the rows as the
// narrow side of the tile:
//     S^T [16 keys x 8 rows] = K [16 x D] Q^T [D x 8],      O^T [D x 8] += V^T [D x 16] W^T [16 x 8]
// (m16n8k16, fp16 operands, fp32 accumulators in registers).  e4m3 codes are exact in fp16, so that K and V come from the
// cache with one conversion per two codes and no scale; Q is brought to [1, 2) by a power of two per row and rounded to fp16,
// which keeps bf16's 8 bits; fp32 rows travel in two fp16 terms (22 bits), and so do their weights.
//
// The order of the contracted index is free as long as both operands agree.  A lane therefore takes whole pieces of rows: of
// K, 4 D/16 consecutive-by-16 bytes of two keys; of V, D/8 bytes of four keys, whose bytes a permutation brings side by side.
// What a lane fetches (cp.async into slots of its own) is what it multiplies: the ring needs no barrier but the wait.
//
// Softmax.  With t the score in powers of two, a row keeps a reference m and e (whole numbers) and
//     l = sum 2^(t - m),      O = sum 2^(t - m) (v_scale 2^(6 - e)) code.
// e makes room for values of any size in fp16's range: weights lie around 2^6 where they matter, are as fine as 2^-24, and may
// rise to 2^14 before m and e have to move.  So the usual step asks one vote of the warp instead of a reduction of maxima and
// a multiplication of O, and every factor that ever touches O is a power of two.
#include <cooperative_groups.h>

#include "kv8.cuh"

namespace ltca {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStages = 3;                  // steps of a warp's keys in shared memory, all but one of them in flight
constexpr int kMaxCluster = 16;             // CTAs of one pair that merge through shared memory
constexpr int kStepBytes = 4096;            // keys and values of a warp's step: KG groups of 16 keys
constexpr int kHead = 64;                   // a step's scales and positions
constexpr float kNone = -3.402823466e38f;   // the reference of a row that has seen no key
constexpr float kLimit = 16384.f;           // largest weight before the references move

struct DecodeArgs {
    ltca_kv8_cache c;
    ltca_kv8_decode_params p;
    int nb, G, R;               // blocks of tokens; heads of queries per head of keys; rows of a pair
    int tiles;                  // of 8 NT rows
    int nsplit, cluster;        // CTAs of a tile; whether they are a cluster
    float* partial;             // [pairs * tiles][nsplit][8 NT][D + 3] where they are not
};

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
template <int N>
__device__ __forceinline__ void fetch(uint32_t dst, const void* src) {
    if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}

// How a warp's step of KG groups of 16 keys lies in its ring, for a lane (r, c) = (lane / 4, lane % 4).
template <int D>
struct Step {
    static constexpr int KG = 128 / D;
    static constexpr int kParts = D == 128 ? 2 : 1;               // pieces of a key's row of K
    static constexpr int kPart = D == 32 ? 8 : 16;                // their bytes
    static constexpr int kVPart = D / 8;                          // bytes of a key's row of V
    static constexpr int kWords = D / 16;                         // words of K per key and lane: one per product
    static constexpr int kGroupLane = 2 * D / 16 * 8;             // bytes of a group per lane: D / 2 of K, D / 2 of V
    // K: bytes of the row that words 4 part .. hold
    static __device__ __forceinline__ int k_offset(int c, int part) { return part * 64 + c * kPart; }
    static __device__ __forceinline__ int k_dim(int c, int word) {
        return D == 32 ? c * 8 + 4 * word : (word >> 2) * 64 + c * 16 + 4 * (word & 3);
    }
};

// m, e, l of rows merge like this, and their O with the factor that comes back (o = O * 2^(E - 6) / L at the end).
struct Merged { float M, E, L; };

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 4 : NT == 2 ? 3 : 2) kv8_decode_kernel(const __grid_constant__ DecodeArgs a) {
    using St = Step<D>;
    constexpr int KG = St::KG, MTD = D / 16, ROWS = 8 * NT;
    constexpr int kTerms = sizeof(T) == 4 ? 2 : 1;
    constexpr bool kQRegs = NT * kTerms * D <= 256;               // Q's fragments stay in registers
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ __align__(16) uint2 sm_q[NT][kTerms][MTD][32];     // Q's fragments: b0, b1 of each product
    __shared__ float sm_c[ROWS];                                  // what a row's S is multiplied by (times the key's scale)
    __shared__ int sm_lim[ROWS], sm_i[ROWS];                      // keys below it are seen; which of the new tokens
    __shared__ float sm_m[kWarps][ROWS], sm_e[kWarps][ROWS], sm_l[kWarps][ROWS];
    __shared__ Merged sm_row[ROWS];
    namespace cg = cooperative_groups;
    grid_dependency_wait();

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
    const int unit = blockIdx.x, tile = unit % a.tiles, split = blockIdx.y;
    const int64_t pair = unit / a.tiles;
    const int b = (int)(pair / a.c.H), h = (int)(pair % a.c.H);
    const int n = new_tokens(a.p.new_len, b, a.p.Sq);
    const int len = a.p.kv_len ? a.p.kv_len[b] : a.c.S;
    const int live = min(max(len, 0), a.c.S);

    // rows: new token first, then the heads that share
    int lim = 0;
    {
        const int row = tile * ROWS + lane, i = row / a.G;
        if (lane < ROWS && row < a.R && i < n) {
            lim = live;
            if (a.p.causal) lim = (int)min((int64_t)lim, max((int64_t)len - n + i + 1, (int64_t)0));
        }
        if (warp == 0 && lane < ROWS) { sm_lim[lane] = lim; sm_i[lane] = i; }
    }
    const int lim_max = __reduce_max_sync(0xffffffffu, lim);
    const int lim_min = __reduce_min_sync(0xffffffffu, lim > 0 ? lim : 0x7fffffff);

    const uint8_t* kp = reinterpret_cast<const uint8_t*>(a.c.k) + b * a.c.k_strides.batch + h * a.c.k_strides.head;
    const uint8_t* vp = reinterpret_cast<const uint8_t*>(a.c.v) + b * a.c.v_strides.batch + h * a.c.v_strides.head;
    const float *ks = a.c.k_scale + pair * a.nb, *vs = a.c.v_scale + pair * a.nb;
    const int32_t* list = a.p.blocks ? a.p.blocks + pair * a.p.n_blocks : nullptr;
    const int log_block = 31 - __clz(a.c.block), log_gpb = log_block - 4;
    const int64_t groups = lim_max == 0 ? 0 : list ? (int64_t)a.p.n_blocks << log_gpb : (lim_max + 15) >> 4;
    const int64_t steps = (groups + kWarps * KG - 1) / (kWarps * KG);

    const uint32_t ring = smem_u32(smem) + warp * kStages * (kStepBytes + kHead);
    const unsigned char* ring_p = smem + warp * kStages * (kStepBytes + kHead);
    // first key of group u of this warp's part of step s; 2^31 - 1: nothing there
    auto place = [&](int64_t s, int u) -> int {
        const int64_t g = (s * kWarps + warp) * KG + u;
        if (g >= groups) return 0x7fffffff;
        if (!list) return (int)(g << 4);
        const int blk = list[g >> log_gpb];
        if (blk < 0 || blk >= a.nb) return 0x7fffffff;
        return (blk << log_block) + ((int)(g & ((1 << log_gpb) - 1)) << 4);
    };
    auto fetch_step = [&](int64_t s, int stage) {
        if (s < steps) {
            const uint32_t head = ring + stage * (kStepBytes + kHead), body = head + kHead + lane * 16;
#pragma unroll
            for (int u = 0; u < KG; ++u) {
                const int pos = place(s, u);
                if (lane == 0) asm volatile("st.shared.b32 [%0], %1;" ::"r"(head + 32 + u * 4), "r"(pos) : "memory");
                if (pos >= lim_max) continue;
                if (lane < 2) fetch<4>(head + u * 8 + lane * 4, (lane ? vs : ks) + (pos >> log_block));
                const uint32_t at = body + u * (St::kGroupLane / 16) * 512;
#pragma unroll
                for (int x = 0; x < 2; ++x) {                      // keys r, r + 8
                    const uint8_t* row = kp + (int64_t)min(pos + r + 8 * x, lim_max - 1) * a.c.k_strides.seq;
#pragma unroll
                    for (int part = 0; part < St::kParts; ++part)
                        fetch<St::kPart>(at + (x * St::kParts + part) * St::kPart / 16 * 512 + (D == 32 ? x * 8 : 0),
                                         row + St::k_offset(c, part));
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) {                      // keys 2c, 2c + 1, 2c + 8, 2c + 9
                    const uint8_t* row = vp + (int64_t)min(pos + 2 * c + (x & 1) + 8 * (x >> 1), lim_max - 1) * a.c.v_strides.seq;
                    const int byte = x * St::kVPart;
                    fetch<St::kVPart>(at + D / 32 * 512 + byte / 16 * 512 + byte % 16, row + r * St::kVPart);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch_step(split + (int64_t)i * a.nsplit, i);

    // Q: a power of two per row, then fp16 fragments for every warp
    for (int row = warp; row < ROWS; row += kWarps) {
        const int gr = tile * ROWS + row;
        const bool there = gr < a.R && gr / a.G < n;
        const T* q = reinterpret_cast<const T*>(a.p.q) + b * a.p.q_strides.batch +
                     (int64_t)(h * a.G + gr % a.G) * a.p.q_strides.head + (int64_t)(gr / a.G) * a.p.q_strides.seq;
        float x[D / 32];
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            x[i] = there ? ld_value(q + lane + 32 * i) : 0.f;
            most = max(most, finite_abs_bits(x[i]));
        }
        most = __reduce_max_sync(0xffffffffu, most);
        const int e = min(max((int)(most >> 23) - 127, -100), 120);
        const float down = pow2(-e);
        if (lane == 0) sm_c[row] = a.p.scale * 1.44269504f * pow2(e);
        // the place of channel d in the fragments: lane (row % 8, c), product `word`, halves 0 .. 3
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const int d = lane + 32 * i;
            const int cc = D == 32 ? d >> 3 : (d & 63) >> 4;
            const int word = D == 32 ? (d & 7) >> 2 : (d >> 6) * 4 + ((d & 15) >> 2);
            const float y = x[i] * down;
            const __half hi = __float2half_rn(y);
            __half* dst = reinterpret_cast<__half*>(&sm_q[row >> 3][0][word][(row & 7) * 4 + cc]) + (d & 3);
            *dst = hi;
            if (kTerms == 2)
                *(reinterpret_cast<__half*>(&sm_q[row >> 3][kTerms - 1][word][(row & 7) * 4 + cc]) + (d & 3)) =
                    __float2half_rn(y - __half2float(hi));
        }
    }
    __syncthreads();
    uint2 qf[kQRegs ? NT : 1][kQRegs ? kTerms : 1][kQRegs ? MTD : 1];
    if constexpr (kQRegs) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int x = 0; x < kTerms; ++x)
#pragma unroll
                for (int w = 0; w < MTD; ++w) qf[t][x][w] = sm_q[t][x][w][lane];
    }
    auto q_at = [&](int t, int x, int w) -> uint2 {
        if constexpr (kQRegs) return qf[t][x][w];
        else return sm_q[t][x][w][lane];
    };

    // of rows 2c and 2c + 1 of each tile of 8
    float m[NT][2], inv[NT][2], e[NT][2], l[NT][2], cs[NT][2];       // inv = 2^(6 - e)
    float o[NT][MTD][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            m[t][x] = kNone; e[t][x] = 200.f; inv[t][x] = pow2(-100); l[t][x] = 0.f;
            cs[t][x] = sm_c[t * 8 + 2 * c + x];
        }
#pragma unroll
        for (int i = 0; i < MTD; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[t][i][x] = 0.f;
    }
    const bool clamped = a.p.score_clamp > 0.f;
    const float clamp = a.p.score_clamp * 1.44269504f;
    const float* mask = a.p.keep_mask ? a.p.keep_mask + (int64_t)b * a.p.Sq * a.c.S : nullptr;

    auto group = [&](const unsigned char* body, int pos, float k_scale, float v_scale) {
        // S^T
        float s[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int x = 0; x < 4; ++x) s[t][x] = 0.f;
        {
            uint32_t w[2][St::kWords];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if constexpr (D == 32) {
                    const uint2 u = *reinterpret_cast<const uint2*>(body + x * 8);
                    w[x][0] = u.x; w[x][1] = u.y;
                } else {
#pragma unroll
                    for (int part = 0; part < St::kParts; ++part) {
                        const uint4 u = *reinterpret_cast<const uint4*>(body + (x * St::kParts + part) * 512);
                        w[x][4 * part] = u.x; w[x][4 * part + 1] = u.y; w[x][4 * part + 2] = u.z; w[x][4 * part + 3] = u.w;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < St::kWords; ++i) {
                const uint32_t a0 = e4m3x2_to_half2(w[0][i] & 0xffffu), a2 = e4m3x2_to_half2(w[0][i] >> 16);
                const uint32_t a1 = e4m3x2_to_half2(w[1][i] & 0xffffu), a3 = e4m3x2_to_half2(w[1][i] >> 16);
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int x = 0; x < kTerms; ++x) {
                        const uint2 q = q_at(t, x, i);
                        mma(s[t], a0, a1, a2, a3, q.x, q.y);
                    }
            }
        }
        // scores in powers of two; s[t][0], [1]: key r with rows 2c, 2c + 1; [2], [3]: key r + 8
        const bool whole = pos + 16 <= lim_min && !mask;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                s[t][x] *= cs[t][x & 1] * k_scale;
                if (clamped) s[t][x] = s[t][x] < clamp ? s[t][x] : (s[t][x] == s[t][x] ? clamp : s[t][x]);
            }
        if (!whole) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int row = t * 8 + 2 * c + (x & 1), j = pos + r + 8 * (x >> 1);
                    bool seen = j < sm_lim[row];
                    if (mask && seen) seen = mask[(int64_t)sm_i[row] * a.c.S + j] != 0.f;
                    if (!seen) s[t][x] = -INFINITY;
                }
        }
        float p[NT][4], f[NT][2];
        bool high = false;
        auto weigh = [&]() {
#pragma unroll
            for (int t = 0; t < NT; ++t) {
#pragma unroll
                for (int x = 0; x < 2; ++x) f[t][x] = fminf(v_scale * inv[t][x], 1e38f);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    p[t][x] = exp2_fast(s[t][x] - m[t][x & 1]);
                    high |= p[t][x] > kLimit || p[t][x] * f[t][x & 1] > kLimit;
                }
            }
        };
        weigh();
        if (__any_sync(0xffffffffu, high)) {
            const float lv = fmaxf(log2f(v_scale), -110.f);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    float top = fmaxf(s[t][x], s[t][x + 2]);
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                    const float m2 = fmaxf(m[t][x], ceilf(top));
                    const float before = m[t][x] == kNone ? -INFINITY : e[t][x] + (m[t][x] - m2);
                    const float y = fmaxf(before, ceilf(top - m2 + lv));
                    if (y > -1000.f && y < 1000.f) {              // a row that has seen a key
                        const float fo = before == -INFINITY ? 1.f : exp2_fast(before - y);
                        l[t][x] *= m[t][x] == kNone ? 1.f : exp2_fast(m[t][x] - m2);
                        m[t][x] = m2;
                        e[t][x] = y;
                        inv[t][x] = exp2_fast(6.f - y);
#pragma unroll
                        for (int i = 0; i < MTD; ++i) { o[t][i][x] *= fo; o[t][i][x + 2] *= fo; }
                    }
                }
            weigh();
        }
        // W^T
        uint32_t w0[NT][kTerms], w1[NT][kTerms];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            float w[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                l[t][x & 1] += p[t][x];
                w[x] = p[t][x] * f[t][x & 1];
            }
            const uint32_t h0 = half2_bits(w[0], w[1]), h1 = half2_bits(w[2], w[3]);
            w0[t][0] = transposed(h0); w1[t][0] = transposed(h1);
            if constexpr (kTerms == 2) {
                const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&h0));
                const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
                w0[t][1] = transposed(half2_bits(w[0] - f0.x, w[1] - f0.y));
                w1[t][1] = transposed(half2_bits(w[2] - f1.x, w[3] - f1.y));
            }
        }
        // O^T
        constexpr int VW = D / 32;                                  // words of V per key and lane
        uint32_t v[4][VW];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int byte = x * St::kVPart;
            const unsigned char* src = body + D / 32 * 512 + byte / 16 * 512 + byte % 16;
            if constexpr (D == 128) {
                const uint4 u = *reinterpret_cast<const uint4*>(src);
                v[x][0] = u.x; v[x][1] = u.y; v[x][2] = u.z; v[x][3] = u.w;
            } else if constexpr (D == 64) {
                const uint2 u = *reinterpret_cast<const uint2*>(src);
                v[x][0] = u.x; v[x][1] = u.y;
            } else {
                v[x][0] = *reinterpret_cast<const uint32_t*>(src);
            }
        }
        if (!whole) {
            // NaN among the values counts for the rows that see its key and for no other: it becomes zero, and a product of
            // "is NaN" with "is seen" says whose sums it reaches.
            uint32_t nan[4][VW];
            uint32_t some = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int i = 0; i < VW; ++i) {
                    nan[x][i] = __vcmpeq4(v[x][i] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                    some |= nan[x][i];
                }
            if (__any_sync(0xffffffffu, some != 0)) {
                uint32_t i0[NT], i1[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    auto is = [&](int x) { return s[t][x] == -INFINITY ? 0.f : 1.f; };
                    i0[t] = transposed(half2_bits(is(0), is(1)));
                    i1[t] = transposed(half2_bits(is(2), is(3)));
                }
#pragma unroll
                for (int i = 0; i < MTD; ++i) {
                    // code 0x38 is 1
                    auto pick = [&](int x, int half) {
                        return e4m3x2_to_half2(__byte_perm(nan[x][i >> 1], nan[x + 1][i >> 1], (i & 1) ? (half ? 0x73 : 0x62)
                                                                                                       : (half ? 0x51 : 0x40)) & 0x3838u);
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
        for (int i = 0; i < MTD; ++i) {
            const uint32_t sel = (i & 1) ? 0x7362 : 0x5140;
            const uint32_t x0 = __byte_perm(v[0][i >> 1], v[1][i >> 1], sel), x1 = __byte_perm(v[2][i >> 1], v[3][i >> 1], sel);
            const uint32_t a0 = e4m3x2_to_half2(x0 & 0xffffu), a1 = e4m3x2_to_half2(x0 >> 16);
            const uint32_t a2 = e4m3x2_to_half2(x1 & 0xffffu), a3 = e4m3x2_to_half2(x1 >> 16);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int x = 0; x < kTerms; ++x) mma(o[t][i], a0, a1, a2, a3, w0[t][x], w1[t][x]);
        }
    };

    int stage = 0;
    for (int64_t s = split; s < steps; s += a.nsplit) {
        fetch_step(s + (int64_t)(kStages - 1) * a.nsplit, (stage + kStages - 1) % kStages);
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        __syncwarp();                                               // the step's head is read by all lanes
        const unsigned char* head = ring_p + stage * (kStepBytes + kHead);
#pragma unroll
        for (int u = 0; u < KG; ++u) {
            const int pos = *reinterpret_cast<const int*>(head + 32 + u * 4);
            if (pos >= lim_max) continue;
            const float2 sc = *reinterpret_cast<const float2*>(head + u * 8);
            group(head + kHead + lane * 16 + u * (St::kGroupLane / 16) * 512, pos, sc.x, sc.y);
        }
        __syncwarp();
        stage = (stage + 1) % kStages;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    grid_launch_dependents();

    // ---- the warps' sums, tile by tile, then the CTAs' ----
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) l[t][x] += __shfl_xor_sync(0xffffffffu, l[t][x], off);
            if (r == 0) {
                const int row = t * 8 + 2 * c + x;
                sm_m[warp][row] = m[t][x]; sm_e[warp][row] = e[t][x]; sm_l[warp][row] = l[t][x];
            }
        }
    float* sm_o = reinterpret_cast<float*>(smem);                   // [kWarps][8][D], over the ring
    float* sm_part = sm_o + kWarps * 8 * D;                         // [ROWS][D]
    const bool alone = a.nsplit == 1;
    const int64_t slot = (int64_t)unit * a.nsplit + split;
    auto finish = [&](int row, int d, float sum, const Merged& g) {
        const int gr = tile * ROWS + row;
        if (gr >= a.R) return;
        const bool dead = sm_lim[row] == 0 || g.L == 0.f;
        T* out = reinterpret_cast<T*>(a.p.o) + b * a.p.o_strides.batch + (int64_t)(h * a.G + gr % a.G) * a.p.o_strides.head +
                 (int64_t)(gr / a.G) * a.p.o_strides.seq;
        st_value(out + d, dead ? 0.f : sum * (pow2((int)g.E - 6) / g.L));
        if (d == 0 && a.p.lse)
            a.p.lse[((int64_t)b * a.p.Hq + h * a.G + gr % a.G) * a.p.Sq + gr / a.G] =
                dead ? -INFINITY : (g.M == kNone ? 0.f : g.M * 0.693147181f) + logf(g.L);
    };
    // the references of n parts together; get(i) gives part i's
    auto merge = [&](int parts, auto get) {
        Merged g{kNone, -INFINITY, 0.f};
        for (int i = 0; i < parts; ++i) g.M = fmaxf(g.M, get(i).M);
        for (int i = 0; i < parts; ++i) {
            const Merged x = get(i);
            g.L += x.L * exp2_fast(x.M - g.M);
            g.E = fmaxf(g.E, (x.M - g.M) + x.E);
        }
        return g;
    };
    __syncthreads();
    if (threadIdx.x < ROWS) {
        const int row = threadIdx.x;
        sm_row[row] = merge(kWarps, [&](int i) { return Merged{sm_m[i][row], sm_e[i][row], sm_l[i][row]}; });
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if (t) __syncthreads();
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < MTD; ++i)
                *reinterpret_cast<float2*>(sm_o + (warp * 8 + 2 * c + x) * D + r * (D / 8) + 2 * i) = make_float2(o[t][i][x], o[t][i][x + 2]);
        __syncthreads();
        for (int i = threadIdx.x; i < 8 * D; i += kThreads) {
            const int row = t * 8 + i / D, d = i % D;
            const Merged g = sm_row[row];
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
                sum += sm_o[w * 8 * D + i] * exp2_fast((sm_m[w][row] - g.M) + sm_e[w][row] - g.E);
            if (alone) finish(row, d, sum, g);
            else if (a.cluster) sm_part[row * D + d] = sum;
            else a.partial[(slot * ROWS + row) * (D + 3) + 3 + d] = sum;
        }
    }
    if (alone) return;
    if (!a.cluster) {
        if (threadIdx.x < ROWS) {
            float* part = a.partial + (slot * ROWS + threadIdx.x) * (D + 3);
            const Merged g = sm_row[threadIdx.x];
            part[0] = g.M; part[1] = g.E; part[2] = g.L;
        }
        return;
    }
    // every CTA of the cluster finishes a share of the rows' values
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int i = split * kThreads + threadIdx.x; i < ROWS * D; i += a.nsplit * kThreads) {
        const int row = i / D;
        const Merged g = merge(a.nsplit, [&](int k) { return *cluster.map_shared_rank(&sm_row[row], k); });
        float sum = 0.f;
        for (int k = 0; k < a.nsplit; ++k) {
            const Merged x = *cluster.map_shared_rank(&sm_row[row], k);
            sum += *cluster.map_shared_rank(sm_part + i, k) * exp2_fast((x.M - g.M) + x.E - g.E);
        }
        finish(row, i % D, sum, g);
    }
    cluster.sync();                                                 // until nobody reads this CTA's shared memory
}

// One CTA per row of a tile: the CTAs' shares from scratch.
template <typename T>
__global__ void __launch_bounds__(128) kv8_decode_merge_kernel(const __grid_constant__ DecodeArgs a, int rows) {
    grid_dependency_wait();
    const int D = a.c.D, d = threadIdx.x, row = blockIdx.y, unit = blockIdx.x, tile = unit % a.tiles, gr = tile * rows + row;
    if (gr >= a.R || d >= D) return;
    const int64_t pair = unit / a.tiles;
    const int b = (int)(pair / a.c.H), h = (int)(pair % a.c.H);
    const float* part = a.partial + ((int64_t)unit * a.nsplit * rows + row) * (D + 3);
    const int64_t next = (int64_t)rows * (D + 3);
    float M = kNone, E = -INFINITY, L = 0.f, sum = 0.f;
    for (int i = 0; i < a.nsplit; ++i) M = fmaxf(M, part[i * next]);
    for (int i = 0; i < a.nsplit; ++i) E = fmaxf(E, (part[i * next] - M) + part[i * next + 1]);
    for (int i = 0; i < a.nsplit; ++i) {
        const float* x = part + i * next;
        L += x[2] * exp2_fast(x[0] - M);
        sum += x[3 + d] * exp2_fast((x[0] - M) + x[1] - E);
    }
    // rows that are not there, or see nothing, have been given no sums that count
    const int i = gr / a.G, n = new_tokens(a.p.new_len, b, a.p.Sq), len = a.p.kv_len ? a.p.kv_len[b] : a.c.S;
    const bool dead = i >= n || (a.p.causal && (int64_t)len - n + i + 1 <= 0) || len <= 0 || L == 0.f;
    T* out = reinterpret_cast<T*>(a.p.o) + b * a.p.o_strides.batch + (int64_t)(h * a.G + gr % a.G) * a.p.o_strides.head +
             (int64_t)i * a.p.o_strides.seq;
    st_value(out + d, dead ? 0.f : sum * (pow2((int)E - 6) / L));
    if (d == 0 && a.p.lse)
        a.p.lse[((int64_t)b * a.p.Hq + h * a.G + gr % a.G) * a.p.Sq + i] = dead ? -INFINITY : (M == kNone ? 0.f : M * 0.693147181f) + logf(L);
}

// How a call is cut up; a function of the problem alone, so that the size query and the launch agree.
struct Plan { int nt, tiles, nsplit; bool cluster; };
Plan plan_of(const ltca_kv8_cache* c, const ltca_kv8_decode_params* p) {
    const int R = p->Hq / c->H * p->Sq;
    Plan s;
    s.nt = R <= 8 ? 1 : R <= 16 ? 2 : 4;
    s.tiles = (R + 8 * s.nt - 1) / (8 * s.nt);
    s.nsplit = 1;
    s.cluster = false;
    const int64_t units = (int64_t)c->B * c->H * s.tiles;
    int64_t keys = c->S;
    if (p->blocks && (int64_t)p->n_blocks * c->block < keys) keys = (int64_t)p->n_blocks * c->block;
    const int64_t steps = (keys + 16 * kWarps * 128 / c->D - 1) / (16 * kWarps * 128 / c->D);
    // four CTAs per SM, each with at least two steps; more of them where the sequences may differ in length
    const int64_t full = 4 * (int64_t)kPlanSms;
    const int64_t want = (full + units - 1) / units, cap = (steps + 1) / 2;
    int64_t n = want < cap ? want : cap;
    if (units * n >= full && steps / n >= 32) n *= 4;
    if (n > kMaxCluster && units * kMaxCluster < full) {
        s.nsplit = (int)(n < 128 ? n : 128);
        return s;
    }
    while (s.nsplit * 2 <= n && s.nsplit < kMaxCluster) s.nsplit *= 2;
    s.cluster = s.nsplit > 1;
    return s;
}

template <typename T, int D, int NT>
int launch(ltca_ctx* ctx, const DecodeArgs& a) {
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)((int64_t)a.c.B * a.c.H * a.tiles), a.nsplit);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kWarps * kStages * (kStepBytes + kHead);
    static_assert(kWarps * 8 * 128 * 4 + 32 * 128 * 4 <= kWarps * kStages * (kStepBytes + kHead), "the merge lies over the ring");
    cfg.stream = ctx->stream;
    static SmemOptIn once;
    LTCA_CUDA_OK(ctx, opt_in_dynamic_smem(once, ctx->device, kv8_decode_kernel<T, D, NT>, (int)cfg.dynamicSmemBytes));
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = (unsigned)a.nsplit;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.cluster ? 2 : 1;
    if (a.cluster && a.nsplit > 8) {
        static SmemOptIn wide;      // clusters of more than eight CTAs are an opt-in of a kernel on one device
        const uint64_t bit = (ctx->device >= 0 && ctx->device < 64) ? (1ull << ctx->device) : 0ull;
        if (!bit || !(wide.done.load(std::memory_order_acquire) & bit)) {
            LTCA_CUDA_OK(ctx, cudaFuncSetAttribute(kv8_decode_kernel<T, D, NT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
            wide.done.fetch_or(bit, std::memory_order_release);
        }
    }
    LTCA_CUDA_OK(ctx, cudaLaunchKernelEx(&cfg, kv8_decode_kernel<T, D, NT>, a));
    return LTCA_OK;
}
template <typename T, int D>
int launch_rows(ltca_ctx* ctx, const DecodeArgs& a, int nt) {
    return nt == 1 ? launch<T, D, 1>(ctx, a) : nt == 2 ? launch<T, D, 2>(ctx, a) : launch<T, D, 4>(ctx, a);
}
template <typename T>
int launch_width(ltca_ctx* ctx, const DecodeArgs& a, const Plan& s) {
    int rc = a.c.D == 32 ? launch_rows<T, 32>(ctx, a, s.nt) : a.c.D == 64 ? launch_rows<T, 64>(ctx, a, s.nt) : launch_rows<T, 128>(ctx, a, s.nt);
    if (rc || a.cluster || a.nsplit == 1) return rc;
    const dim3 grid((unsigned)((int64_t)a.c.B * a.c.H * a.tiles), 8 * s.nt);
    LTCA_CUDA_OK(ctx, launch_dependent(kv8_decode_merge_kernel<T>, grid, dim3(128), 0, ctx->stream, a, 8 * s.nt));
    return LTCA_OK;
}

size_t partial_bytes(const ltca_kv8_cache* c, const Plan& s) {
    if (s.nsplit == 1 || s.cluster) return 0;
    return align_up((size_t)c->B * c->H * s.tiles * s.nsplit * 8 * s.nt * (c->D + 3) * sizeof(float), 256);
}

}  // namespace

size_t kv8_decode_workspace(const ltca_kv8_cache* c, const ltca_kv8_decode_params* p) { return partial_bytes(c, plan_of(c, p)); }

int launch_kv8_decode(ltca_ctx* ctx, const ltca_kv8_cache* c, const ltca_kv8_decode_params* p) {
    const Plan s = plan_of(c, p);
    if ((int64_t)c->B * c->H * s.tiles > 0x7fffffff) return fail(ctx, LTCA_ERR_INVALID, "too many rows of queries for one call");
    DecodeArgs a{*c, *p, (c->S + c->block - 1) / c->block, p->Hq / c->H, p->Hq / c->H * p->Sq, s.tiles, s.nsplit, s.cluster, nullptr};
    if (const size_t need = partial_bytes(c, s)) {
        if (!p->workspace || p->workspace_bytes < need) return fail(ctx, LTCA_ERR_WORKSPACE, "decode needs %zu bytes of workspace", need);
        a.partial = reinterpret_cast<float*>(p->workspace);
    }
    return p->dtype == LTCA_BF16 ? launch_width<__nv_bfloat16>(ctx, a, s) : launch_width<float>(ctx, a, s);
}

}  // namespace ltca
