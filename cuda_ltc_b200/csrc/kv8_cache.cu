// Writing keys and values into the 8-bit cache and reading them back: see ltca_kv8_cache in include/ltc_attn.h.
#include "kv8.cuh"

namespace ltca {

namespace {

// ---- append ------------------------------------------------------------------------------------
// Of a block of tokens x_td with older codes c and scale s:  need = 2^ceil(log2(max |x| / 448)),  s' = max(s, need) (need
// alone where the block is new),  code = rn(x / s'),  and where s' > s the older codes become rn(c * s / s').
struct AppendArgs {
    ltca_kv8_cache c;
    ltca_kv8_append_params p;
    int nb;
};

// One CTA per block of tokens, head and tensor.
template <typename T>
__global__ void __launch_bounds__(128) kv8_append_kernel(const AppendArgs a) {
    __shared__ uint32_t sm_max;
    __shared__ float sm_lo[128], sm_hi[128];
    grid_dependency_wait();
    const int b = blockIdx.x / a.c.H, h = blockIdx.x % a.c.H, D = a.c.D;
    const bool is_v = blockIdx.z != 0;
    const int n = new_tokens(a.p.new_len, b, a.p.n);
    const int64_t end = a.p.kv_len[b], first = end - n;
    const int64_t lo = first > 0 ? first : 0, hi = end < a.c.S ? end : a.c.S;       // positions that are written
    const int64_t j = lo / a.c.block + blockIdx.y;
    if (lo >= hi || j * a.c.block >= hi) return;
    const int64_t row0 = j * a.c.block;
    const int from = (int)(lo > row0 ? lo - row0 : 0), to = (int)(hi - row0 < a.c.block ? hi - row0 : a.c.block);

    const ltca_strides xs = is_v ? a.p.v_strides : a.p.k_strides, cs = is_v ? a.c.v_strides : a.c.k_strides;
    // token of the block's row r: row0 + r - first
    const T* x = reinterpret_cast<const T*>(is_v ? a.p.v : a.p.k) + b * xs.batch + h * xs.head;
    const int64_t t0 = row0 - first;
    uint8_t* code = reinterpret_cast<uint8_t*>(is_v ? a.c.v : a.c.k) + b * cs.batch + h * cs.head + row0 * cs.seq;
    const int64_t at = ((int64_t)b * a.c.H + h) * a.nb + j;
    float* scale = (is_v ? a.c.v_scale : a.c.k_scale) + at;

    if (threadIdx.x == 0) sm_max = 0;
    __syncthreads();
    uint32_t most = 0;
    for (int i = threadIdx.x; i < (to - from) * D; i += blockDim.x)
        most = max(most, finite_abs_bits(ld_value(x + (t0 + from + i / D) * xs.seq + i % D)));
    atomicMax(&sm_max, most);
    __syncthreads();
    const float need = pow2(e4m3_exponent(sm_max)), old = from > 0 ? *scale : need;
    const float now = fmaxf(old, need);
    const bool grown = from > 0 && now > old;
    for (int i = threadIdx.x; i < (to - from) * D; i += blockDim.x) {
        const int r = from + i / D, d = i % D;
        code[r * cs.seq + d] = (uint8_t)to_e4m3x2(ld_value(x + (t0 + r) * xs.seq + d) / now, 0.f);
    }
    if (grown)
        for (int i = threadIdx.x; i < from * D; i += blockDim.x) {
            uint8_t* c = code + (i / D) * cs.seq + i % D;
            *c = (uint8_t)to_e4m3x2(e4m3x2_to_float2(*c).x * (old / now), 0.f);
        }
    __syncthreads();
    if (threadIdx.x == 0) *scale = now;
    if (!a.c.bounds || is_v) return;
    for (int d = threadIdx.x; d < D; d += blockDim.x) {
        float mn = INFINITY, mx = -INFINITY;
        for (int r = 0; r < to; ++r) {
            const float v = e4m3x2_to_float2(code[r * cs.seq + d]).x;
            const bool nan = v != v;
            mn = fminf(mn, nan ? -448.f : v);
            mx = fmaxf(mx, nan ? 448.f : v);
        }
        int8_t* bd = a.c.bounds + at * 2 * D;
        bd[d] = (int8_t)floorf(mn * 0.25f);
        bd[D + d] = (int8_t)ceilf(mx * 0.25f);
    }
}

// ---- read --------------------------------------------------------------------------------------
struct ReadArgs {
    ltca_kv8_cache c;
    ltca_kv8_read_params p;
    int nb;
};

template <typename T>
__global__ void __launch_bounds__(256) kv8_read_kernel(const ReadArgs a) {
    grid_dependency_wait();
    const int b = blockIdx.x / a.c.H, h = blockIdx.x % a.c.H, D = a.c.D;
    const bool is_v = blockIdx.z != 0;
    const int64_t live = a.p.kv_len ? min(max(a.p.kv_len[b], 0), a.c.S) : a.c.S;
    const ltca_strides os = is_v ? a.p.v_strides : a.p.k_strides, cs = is_v ? a.c.v_strides : a.c.k_strides;
    T* out = reinterpret_cast<T*>(is_v ? a.p.v : a.p.k) + b * os.batch + h * os.head;
    const uint8_t* code = reinterpret_cast<const uint8_t*>(is_v ? a.c.v : a.c.k) + b * cs.batch + h * cs.head;
    const float* scale = (is_v ? a.c.v_scale : a.c.k_scale) + ((int64_t)b * a.c.H + h) * a.nb;
    const int64_t total = (int64_t)a.p.n * D;
    for (int64_t i = (int64_t)blockIdx.y * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.y * 256) {
        const int64_t r = i / D, s = a.p.start + r;
        const int d = (int)(i % D);
        float v = 0.f;
        if (s < live) v = e4m3x2_to_float2(code[s * cs.seq + d]).x * scale[s / a.c.block];
        st_value(out + r * os.seq + d, v);
    }
}

}  // namespace

int launch_kv8_append(ltca_ctx* ctx, const ltca_kv8_cache* c, const ltca_kv8_append_params* p) {
    AppendArgs a{*c, *p, (c->S + c->block - 1) / c->block};
    // a run of n tokens touches at most this many blocks
    const int64_t spans = ((int64_t)p->n + c->block - 2) / c->block + 1;
    const int64_t most = spans < a.nb ? spans : a.nb;
    if (most > 65535) return fail(ctx, LTCA_ERR_INVALID, "append: %d tokens in blocks of %d are too many for one call", p->n, c->block);
    const dim3 grid((unsigned)(c->B * c->H), (unsigned)most, 2);
    auto kern = p->dtype == LTCA_BF16 ? kv8_append_kernel<__nv_bfloat16> : kv8_append_kernel<float>;
    LTCA_CUDA_OK(ctx, launch_dependent(kern, grid, dim3(128), 0, ctx->stream, a));
    return LTCA_OK;
}

int launch_kv8_read(ltca_ctx* ctx, const ltca_kv8_cache* c, const ltca_kv8_read_params* p) {
    ReadArgs a{*c, *p, (c->S + c->block - 1) / c->block};
    const int64_t want = ((int64_t)p->n * c->D + 256 * 8 - 1) / (256 * 8);
    const dim3 grid((unsigned)(c->B * c->H), (unsigned)(want < 65535 ? want : 65535), 2);
    auto kern = p->dtype == LTCA_BF16 ? kv8_read_kernel<__nv_bfloat16> : kv8_read_kernel<float>;
    LTCA_CUDA_OK(ctx, launch_dependent(kern, grid, dim3(256), 0, ctx->stream, a));
    return LTCA_OK;
}

}  // namespace ltca
