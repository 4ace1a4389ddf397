// Writing keys and values into the 8-bit cache and reading them back: see ltca_kv8_cache in include/ltc_attn.h.
// Both are bound by memory: each value is read once and written once.  Read: 8 sequences of up to 32768 keys of 128 to bf16
// 205 us = 6.56 TB/s.  Append: prompts of up to 8000 tokens, 8 sequences of 8 heads of 128 with bounds 43 us = 4.56 TB/s, held
// up by instructions (16 a value, 70 % of the issue slots); a token of each of 256 sequences 2.6 us, a launch.
#include "kv8.cuh"

namespace ltca {

namespace {

// ---- append ------------------------------------------------------------------------------------
// Of a block of tokens x_td with older codes c and scale s:  need = 2^ceil(log2(max |x| / 448)),  s' = max(s, need) (need
// alone where the block is new),  code = rn(x / s'),  and where s' > s the older codes become rn(c * s / s').
//
// A team of threads takes one block of one head of one tensor and holds all its new values in registers between the maximum
// and the rounding, in pieces of eight channels.  Calls of a few tokens give each block to a warp: nothing but latency, and
// a CTA per block would be mostly idle threads (256 sequences, 8 heads of 64, one token each: 6.8 us for 2.6).
struct AppendArgs {
    ltca_kv8_cache c;
    ltca_kv8_append_params p;
    int nb, spans;              // blocks of a sequence; of them at most this many are touched
    int vec;                    // rows of k and v start on 16-byte boundaries
    uint32_t items;             // tensors, heads and sequences
};

// The bounds' two ends of eight codes (as four pairs of fp16), NaN at both.
__device__ __forceinline__ void widen(__half2 (&lo)[4], __half2 (&hi)[4], const uint2& codes) {
    const uint32_t w[2] = {codes.x, codes.y};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t nan = __vcmpeq4(w[i] & 0x7f7f7f7fu, 0x7f7f7f7fu);
        const uint32_t low = (w[i] & ~nan) | (nan & 0xfefefefeu), high = (w[i] & ~nan) | (nan & 0x7e7e7e7eu);   // -448, 448
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint32_t a = e4m3x2_to_half2(x ? low >> 16 : low & 0xffffu), b = e4m3x2_to_half2(x ? high >> 16 : high & 0xffffu);
            lo[2 * i + x] = __hmin2(lo[2 * i + x], *reinterpret_cast<const __half2*>(&a));
            hi[2 * i + x] = __hmax2(hi[2 * i + x], *reinterpret_cast<const __half2*>(&b));
        }
    }
}

// Eight channels of a row, and their codes at 1 / scale.
struct Piece8f { float v[8]; };
__device__ __forceinline__ Piece8f load_piece(const float* x, bool vec) {
    Piece8f r;
    if (vec) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(x)), b = __ldg(reinterpret_cast<const float4*>(x) + 1);
        r = {{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) r.v[i] = x[i];
    }
    return r;
}
struct Piece8b { uint32_t v[4]; };
__device__ __forceinline__ Piece8b load_piece(const __nv_bfloat16* x, bool vec) {
    Piece8b r;
    if (vec) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(x));
        r = {{a.x, a.y, a.z, a.w}};
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            r.v[i] = (uint32_t)__bfloat16_as_ushort(x[2 * i]) | (uint32_t)__bfloat16_as_ushort(x[2 * i + 1]) << 16;
    }
    return r;
}
// The largest magnitude as bits; an infinity or NaN shows as 0x7f800000 or more.
__device__ __forceinline__ void largest(const Piece8f& p, uint32_t& m) {
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(p.v[i]) & 0x7fffffffu);
}
__device__ __forceinline__ void largest(const Piece8b& p, uint32_t& m) {
    uint32_t t = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) t = __vmaxu2(t, p.v[i] & 0x7fff7fffu);
    m = max(m, max(t << 16, t & 0xffff0000u));
}
// The smallest and the largest of each channel so far.
struct Ends8f {
    float lo[8], hi[8];
    __device__ __forceinline__ Ends8f() {
#pragma unroll
        for (int i = 0; i < 8; ++i) { lo[i] = INFINITY; hi[i] = -INFINITY; }
    }
    __device__ __forceinline__ void add(const Piece8f& p) {
#pragma unroll
        for (int i = 0; i < 8; ++i) { lo[i] = fminf(lo[i], p.v[i]); hi[i] = fmaxf(hi[i], p.v[i]); }
    }
    __device__ __forceinline__ float low(int i) const { return lo[i]; }
    __device__ __forceinline__ float high(int i) const { return hi[i]; }
};
struct Ends8b {
    __nv_bfloat162 lo[4], hi[4];
    __device__ __forceinline__ Ends8b() {
#pragma unroll
        for (int i = 0; i < 4; ++i) { lo[i] = __float2bfloat162_rn(INFINITY); hi[i] = __float2bfloat162_rn(-INFINITY); }
    }
    __device__ __forceinline__ void add(const Piece8b& p) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 x = *reinterpret_cast<const __nv_bfloat162*>(&p.v[i]);
            lo[i] = __hmin2(lo[i], x);
            hi[i] = __hmax2(hi[i], x);
        }
    }
    __device__ __forceinline__ float low(int i) const { return i & 1 ? __high2float(lo[i >> 1]) : __low2float(lo[i >> 1]); }
    __device__ __forceinline__ float high(int i) const { return i & 1 ? __high2float(hi[i >> 1]) : __low2float(hi[i >> 1]); }
};
__device__ __forceinline__ float value_of(const Piece8f& p, int i) { return p.v[i]; }
__device__ __forceinline__ float value_of(const Piece8b& p, int i) {
    return __uint_as_float(i & 1 ? p.v[i >> 1] & 0xffff0000u : p.v[i >> 1] << 16);
}
template <typename T> struct PieceOf { using type = Piece8f; using ends = Ends8f; };
template <> struct PieceOf<__nv_bfloat16> { using type = Piece8b; using ends = Ends8b; };

// P pieces per thread of a team of TEAM hold a block's new rows.
template <typename T, int TEAM, int P>
__global__ void __launch_bounds__(TEAM == 32 ? 128 : TEAM) kv8_append_kernel(const __grid_constant__ AppendArgs a) {
    constexpr int kTeamWarps = TEAM / 32;
    __shared__ uint32_t sm_max[2][kTeamWarps];
    __shared__ __half2 sm_lo[kTeamWarps][64], sm_hi[kTeamWarps][64];        // by pairs of channels
    grid_dependency_wait();
    const int tid = TEAM == 32 ? threadIdx.x & 31 : threadIdx.x, lane = threadIdx.x & 31, warp = TEAM == 32 ? 0 : threadIdx.x >> 5;
    // x: the two tensors side by side, then the heads, then the sequences; y: a sequence's blocks
    const uint32_t item = TEAM == 32 ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (item >= a.items) return;
    const bool is_v = item & 1;
    const uint32_t pair = item >> 1;
    const int b = (int)(pair / (uint32_t)a.c.H), h = (int)(pair - (uint32_t)b * a.c.H), D = a.c.D;
    const int log_chunks = 31 - __clz(D) - 3, chunks = 1 << log_chunks, log_block = 31 - __clz(a.c.block);       // pieces of a row
    const int n = new_tokens(a.p.new_len, b, a.p.n);
    const int64_t end = a.p.kv_len[b], first = end - n;
    const int64_t lo_pos = first > 0 ? first : 0, hi_pos = end < a.c.S ? end : a.c.S;       // positions that are written
    const int64_t j = (lo_pos >> log_block) + blockIdx.y, row0 = j << log_block;
    if (lo_pos >= hi_pos || row0 >= hi_pos) return;
    const int from = (int)(lo_pos > row0 ? lo_pos - row0 : 0), to = (int)(hi_pos - row0 < a.c.block ? hi_pos - row0 : a.c.block);

    const ltca_strides xs = is_v ? a.p.v_strides : a.p.k_strides, cs = is_v ? a.c.v_strides : a.c.k_strides;
    const int chunk = tid & (chunks - 1);
    // token of the block's row r: row0 + r - first
    const T* x = reinterpret_cast<const T*>(is_v ? a.p.v : a.p.k) + b * xs.batch + h * xs.head + (row0 - first) * xs.seq + chunk * 8;
    uint8_t* code = reinterpret_cast<uint8_t*>(is_v ? a.c.v : a.c.k) + b * cs.batch + h * cs.head + row0 * cs.seq + chunk * 8;
    const int64_t at = (int64_t)pair * a.nb + j;
    float* scale = (is_v ? a.c.v_scale : a.c.k_scale) + at;
    const float old = from > 0 ? *scale : 0.f;
    const bool bounded = a.c.bounds && !is_v;
    int8_t* bounds = a.c.bounds + at * 2 * D;

    typename PieceOf<T>::type piece[P];
    uint32_t most = 0;
    // a thread's rows: row0, and every (TEAM / chunks)th from there
    const int my_row = from + (tid >> log_chunks), rows = TEAM >> log_chunks;
    const int64_t x_step = rows * xs.seq, c_step = rows * cs.seq;
    x += my_row * xs.seq;
    code += my_row * cs.seq;
#pragma unroll
    for (int i = 0; i < P; ++i)
        if (my_row + i * rows < to) piece[i] = load_piece(x + i * x_step, a.vec != 0);
    typename PieceOf<T>::ends ends;
#pragma unroll
    for (int i = 0; i < P; ++i)
        if (my_row + i * rows < to) {
            largest(piece[i], most);
            if (bounded) ends.add(piece[i]);
        }
    auto of_team = [&](uint32_t x, int turn) {
        x = __reduce_max_sync(0xffffffffu, x);
        if constexpr (TEAM > 32) {
            if (lane == 0) sm_max[turn][warp] = x;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kTeamWarps; ++i) x = max(x, sm_max[turn][i]);
        }
        return x;
    };
    most = of_team(most, 0);
    const bool special = most >= 0x7f800000u;                     // infinities and NaN do not count
    if (special) {
        most = 0;
#pragma unroll
        for (int i = 0; i < P; ++i)
            if (my_row + i * rows < to) {
#pragma unroll
                for (int y = 0; y < 8; ++y) most = max(most, finite_abs_bits(value_of(piece[i], y)));
            }
        most = of_team(most, 1);
    }
    const int e = e4m3_exponent(most);
    const float need = pow2(e), now = fmaxf(old, need);
    const bool grown = from > 0 && now > old;
    const float up = now == need ? pow2(-e) : 1.f / now;                     // exact, as now is a power of two
    __half2 lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { lo[i] = __float2half2_rn(448.f); hi[i] = __float2half2_rn(-448.f); }
#pragma unroll
    for (int i = 0; i < P; ++i) {
        if (my_row + i * rows < to) {
            uint32_t w[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) w[y] = to_e4m3x2(value_of(piece[i], 2 * y) * up, value_of(piece[i], 2 * y + 1) * up);
            const uint2 c = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
            *reinterpret_cast<uint2*>(code + i * c_step) = c;
            if (bounded && special) widen(lo, hi, c);
        }
    }
    if (bounded && !special && my_row < to) {
        // rounding keeps the order: the ends of the codes are the codes of the ends
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t l = e4m3x2_to_half2(to_e4m3x2(ends.low(2 * i) * up, ends.low(2 * i + 1) * up));
            const uint32_t h = e4m3x2_to_half2(to_e4m3x2(ends.high(2 * i) * up, ends.high(2 * i + 1) * up));
            lo[i] = *reinterpret_cast<const __half2*>(&l);
            hi[i] = *reinterpret_cast<const __half2*>(&h);
        }
    }
    // The older rows: rounded again where the scale has grown, and looked at for the bounds, which thereby are those of the live
    // keys whatever became of earlier ones (tokens that were taken back, say).
    if (grown || (bounded && from > 0)) {
        const float by = old / now;
        code -= from * cs.seq;                                    // rows from the block's first on
#pragma unroll 4
        for (int i = 0; i * rows + (tid >> log_chunks) < from; ++i) {
            uint2* dst = reinterpret_cast<uint2*>(code + i * c_step);
            uint2 c = *dst;
            if (grown) {
                uint32_t w[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const float2 f = e4m3x2_to_float2(((y < 2 ? c.x : c.y) >> (y & 1) * 16) & 0xffffu);
                    w[y] = to_e4m3x2(f.x * by, f.y * by);
                }
                c = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
                *dst = c;
            }
            if (bounded) widen(lo, hi, c);
        }
    }
    if (tid == 0) *scale = now;
    if (!bounded) return;
    // the lanes, then the warps, that hold the same channels
#pragma unroll
    for (int off = 4; off < 32; off <<= 1)
        if (off >= chunks) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                lo[i] = __hmin2(lo[i], __shfl_xor_sync(0xffffffffu, lo[i], off));
                hi[i] = __hmax2(hi[i], __shfl_xor_sync(0xffffffffu, hi[i], off));
            }
        }
    if (lane < chunks) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (TEAM > 32) { sm_lo[warp][chunk * 4 + i] = lo[i]; sm_hi[warp][chunk * 4 + i] = hi[i]; }
        }
    }
    if constexpr (TEAM > 32) {
        __syncthreads();
        if (tid >= chunks) return;
#pragma unroll
        for (int w = 0; w < kTeamWarps; ++w)
#pragma unroll
            for (int i = 0; i < 4; ++i) { lo[i] = __hmin2(lo[i], sm_lo[w][tid * 4 + i]); hi[i] = __hmax2(hi[i], sm_hi[w][tid * 4 + i]); }
    } else {
        if (lane >= chunks) return;
    }
    uint32_t l[2], u[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] = u[i] = 0;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            const __half2 pl = lo[2 * i + (y >> 1)], ph = hi[2 * i + (y >> 1)];
            const float fl = y & 1 ? __high2float(pl) : __low2float(pl), fh = y & 1 ? __high2float(ph) : __low2float(ph);
            l[i] |= ((uint32_t)(int)floorf(fl * 0.25f) & 0xffu) << (8 * y);
            u[i] |= ((uint32_t)(int)ceilf(fh * 0.25f) & 0xffu) << (8 * y);
        }
    }
    *reinterpret_cast<uint2*>(bounds + chunk * 8) = make_uint2(l[0], l[1]);
    *reinterpret_cast<uint2*>(bounds + D + chunk * 8) = make_uint2(u[0], u[1]);
}

// ---- read --------------------------------------------------------------------------------------
struct ReadArgs {
    ltca_kv8_cache c;
    ltca_kv8_read_params p;
    int nb;
    int vec;                    // rows of the results start on 16-byte boundaries
    int slabs;                  // CTAs of a (sequence, head)'s rows
};

__device__ __forceinline__ uint2 ld_codes(const uint2* p) { return __ldg(p); }
__device__ __forceinline__ uint32_t ld_codes(const uint32_t* p) { return __ldg(p); }

// A thread writes 16 bytes at a time, so that a warp's stores are one run; all its codes are on their way before the first.
constexpr int kReadPieces = 4;
template <typename T>
__global__ void __launch_bounds__(256) kv8_read_kernel(const __grid_constant__ ReadArgs a) {
    constexpr int E = 16 / (int)sizeof(T);                                    // codes of a piece
    grid_dependency_wait();
    const bool is_v = blockIdx.y != 0;
    const int slab = (int)(blockIdx.x % a.slabs);
    const int64_t pair = blockIdx.x / a.slabs;
    const int b = (int)(pair / a.c.H), h = (int)(pair % a.c.H), D = a.c.D;
    const int log_chunks = 31 - __clz(D / E), log_block = 31 - __clz(a.c.block);
    const int live = a.p.kv_len ? min(max(a.p.kv_len[b], 0), a.c.S) : a.c.S;
    const ltca_strides os = is_v ? a.p.v_strides : a.p.k_strides, cs = is_v ? a.c.v_strides : a.c.k_strides;
    T* out = reinterpret_cast<T*>(is_v ? a.p.v : a.p.k) + b * os.batch + h * os.head;
    const uint8_t* code = reinterpret_cast<const uint8_t*>(is_v ? a.c.v : a.c.k) + b * cs.batch + h * cs.head;
    const float* scale = (is_v ? a.c.v_scale : a.c.k_scale) + pair * a.nb;
    using Codes = typename std::conditional<E == 8, uint2, uint32_t>::type;
    Codes w[kReadPieces];
    float sc[kReadPieces];
    const int64_t i0 = (int64_t)slab * kReadPieces * 256 + threadIdx.x;
    const int chunk = (int)(i0 & ((1 << log_chunks) - 1));
#pragma unroll
    for (int i = 0; i < kReadPieces; ++i) {
        const int64_t row = (i0 + i * 256) >> log_chunks, s = a.p.start + row;
        if (row < a.p.n && s < live) {
            w[i] = ld_codes(reinterpret_cast<const Codes*>(code + s * cs.seq + chunk * E));
            sc[i] = __ldg(scale + (s >> log_block));
        } else {
            w[i] = Codes{};
            sc[i] = 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < kReadPieces; ++i) {
        const int64_t row = (i0 + i * 256) >> log_chunks;
        if (row >= a.p.n) break;
        T* dst = out + row * os.seq + chunk * E;
        const uint32_t* cw = reinterpret_cast<const uint32_t*>(&w[i]);
        float v[E];
#pragma unroll
        for (int y = 0; y < E / 2; ++y) {
            const float2 f = e4m3x2_to_float2((cw[y >> 1] >> (y & 1) * 16) & 0xffffu);
            v[2 * y] = f.x * sc[i]; v[2 * y + 1] = f.y * sc[i];
        }
        if (!a.vec) {
#pragma unroll
            for (int y = 0; y < E; ++y) st_value(dst + y, v[y]);
        } else if constexpr (E == 4) {
            *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            uint32_t u[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * y], v[2 * y + 1]);
                u[y] = *reinterpret_cast<const uint32_t*>(&t);
            }
            *reinterpret_cast<uint4*>(dst) = make_uint4(u[0], u[1], u[2], u[3]);
        }
    }
}

bool rows_on_16(const void* p, const ltca_strides& s, int es) {
    return !((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(s.batch * es) | (uintptr_t)(s.head * es) | (uintptr_t)(s.seq * es)) & 15);
}

template <typename T, int TEAM, int P>
int launch_team(ltca_ctx* ctx, const AppendArgs& a) {
    const dim3 grid(TEAM == 32 ? (a.items + 3) / 4 : a.items, (unsigned)a.spans);
    LTCA_CUDA_OK(ctx, launch_dependent(kv8_append_kernel<T, TEAM, P>, grid, dim3(TEAM == 32 ? 128 : TEAM), 0, ctx->stream, a));
    return LTCA_OK;
}
template <typename T>
int launch_append(ltca_ctx* ctx, const AppendArgs& a) {
    // up to eight tokens: at most 128 pieces, four for each lane of a warp
    if (a.p.n <= 8) return a.p.n <= 2 ? launch_team<T, 32, 1>(ctx, a) : launch_team<T, 32, 4>(ctx, a);
    switch (a.c.block * a.c.D / 8) {
        case 64: return launch_team<T, 64, 1>(ctx, a);
        case 128: return launch_team<T, 64, 2>(ctx, a);
        case 256: return launch_team<T, 64, 4>(ctx, a);
        case 512: return launch_team<T, 128, 4>(ctx, a);
        case 1024: return launch_team<T, 128, 8>(ctx, a);
        default: return launch_team<T, 256, 8>(ctx, a);                       // 2048: 128 tokens of 128 channels
    }
}

}  // namespace

int launch_kv8_append(ltca_ctx* ctx, const ltca_kv8_cache* c, const ltca_kv8_append_params* p) {
    const int es = elem_size(p->dtype), nb = (c->S + c->block - 1) / c->block;
    // a run of n tokens touches at most this many blocks
    const int64_t spans = ((int64_t)p->n + c->block - 2) / c->block + 1;
    AppendArgs a{*c, *p, nb, (int)(spans < nb ? spans : nb), 0, 0};
    a.vec = rows_on_16(p->k, p->k_strides, es) && rows_on_16(p->v, p->v_strides, es);
    if (a.spans > 65535) return fail(ctx, LTCA_ERR_UNSUPPORTED, "append: %d tokens in blocks of %d are too many for one call", p->n, c->block);
    a.items = (uint32_t)c->B * (uint32_t)c->H * 2u;
    return p->dtype == LTCA_BF16 ? launch_append<__nv_bfloat16>(ctx, a) : launch_append<float>(ctx, a);
}

int launch_kv8_read(ltca_ctx* ctx, const ltca_kv8_cache* c, const ltca_kv8_read_params* p) {
    const int es = elem_size(p->dtype);
    ReadArgs a{*c, *p, (c->S + c->block - 1) / c->block, 0, 0};
    a.vec = rows_on_16(p->k, p->k_strides, es) && rows_on_16(p->v, p->v_strides, es);
    const int64_t pieces = (int64_t)p->n * c->D * es / 16, slabs = (pieces + kReadPieces * 256 - 1) / (kReadPieces * 256);
    if ((int64_t)c->B * c->H * slabs > 0x7fffffff) return fail(ctx, LTCA_ERR_INVALID, "read: too many positions for one call");
    a.slabs = (int)slabs;
    const dim3 grid((unsigned)((int64_t)c->B * c->H * slabs), 2);
    auto kern = p->dtype == LTCA_BF16 ? kv8_read_kernel<__nv_bfloat16> : kv8_read_kernel<float>;
    LTCA_CUDA_OK(ctx, launch_dependent(kern, grid, dim3(256), 0, ctx->stream, a));
    return LTCA_OK;
}

}  // namespace ltca
