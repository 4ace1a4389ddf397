// Which blocks of an 8-bit cache the newest tokens should read: see ltca_kv8_select in include/ltc_attn.h.
#include "kv8.cuh"

namespace ltca {

namespace {

struct SelectArgs {
    ltca_kv8_cache c;
    ltca_kv8_select_params p;
    int nb, rows;
};

// Numbers in the order of the scores; 0 is below every score's, the largest above.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = __float_as_uint(x);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

constexpr int kThreads = 256;

// One CTA per sequence and head of keys; the scores' order stays in shared memory, and a block's rank is counted.
template <typename T>
__global__ void __launch_bounds__(kThreads) kv8_select_kernel(const SelectArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    uint32_t* key = reinterpret_cast<uint32_t*>(smem);
    __shared__ int8_t qi[128];
    __shared__ uint32_t sm_max;
    __shared__ int sm_base[kThreads / 32 + 1];
    grid_dependency_wait();
    const int b = blockIdx.x / a.c.H, h = blockIdx.x % a.c.H, D = a.c.D, G = a.p.Hq / a.c.H, tid = threadIdx.x;
    const int live = a.p.kv_len ? min(max(a.p.kv_len[b], 0), a.c.S) : a.c.S;
    const int blocks = (live + a.c.block - 1) / a.c.block;
    const int n = new_tokens(a.p.new_len, b, a.p.Sq);
    const int64_t pair = (int64_t)b * a.c.H + h;
    const int8_t* bounds = a.c.bounds + pair * a.nb * 2 * D;
    const float* scale = a.c.k_scale + pair * a.nb;
    int32_t* out = a.p.blocks + pair * a.p.count;
    for (int j = tid; j < blocks; j += kThreads) key[j] = order_of(-INFINITY);
    for (int r = 0; r < G * n; ++r) {
        const T* q = reinterpret_cast<const T*>(a.p.q) + b * a.p.q_strides.batch + (h * G + r / n) * a.p.q_strides.head +
                     (r % n) * a.p.q_strides.seq;
        if (tid == 0) sm_max = 0;
        __syncthreads();
        if (tid < D) atomicMax(&sm_max, finite_abs_bits(ld_value(q + tid)));
        __syncthreads();
        const float step = pow2(int8_exponent(sm_max));
        if (tid < D) {
            const float x = ld_value(q + tid) / step;
            qi[tid] = x == x ? (int8_t)rintf(fminf(fmaxf(x, -127.f), 127.f)) : (int8_t)0;
        }
        __syncthreads();
        for (int j = tid; j < blocks; j += kThreads) {
            int sum = 0;
            for (int d = 0; d < D; ++d) sum += max(qi[d] * bounds[j * 2 * D + d], qi[d] * bounds[j * 2 * D + D + d]);
            const float s = (float)sum * scale[j] * step;
            if (s == s) key[j] = max(key[j], order_of(s));
        }
        __syncthreads();
    }
    for (int j = tid; j < blocks; j += kThreads)
        if (j < a.p.first || j >= blocks - a.p.last) key[j] = 0xffffffffu;
    __syncthreads();
    int done = 0;
    for (int j0 = 0; j0 < blocks; j0 += kThreads) {
        const int j = j0 + tid;
        bool take = false;
        if (j < blocks) {
            int rank = 0;
            const uint32_t mine = key[j];
            for (int i = 0; i < blocks; ++i) rank += key[i] > mine || (key[i] == mine && i < j);
            take = rank < a.p.count;
        }
        const uint32_t vote = __ballot_sync(0xffffffffu, take);
        if ((tid & 31) == 0) sm_base[tid >> 5] = __popc(vote);
        __syncthreads();
        int at = done;
        for (int w = 0; w < (tid >> 5); ++w) at += sm_base[w];
        if (take) out[at + __popc(vote & ((1u << (tid & 31)) - 1))] = j;
        for (int w = 0; w < kThreads / 32; ++w) done += sm_base[w];
        __syncthreads();
    }
    for (int i = done + tid; i < a.p.count; i += kThreads) out[i] = -1;
}

}  // namespace

int launch_kv8_select(ltca_ctx* ctx, const ltca_kv8_cache* c, const ltca_kv8_select_params* p) {
    SelectArgs a{*c, *p, (c->S + c->block - 1) / c->block, p->Hq / c->H * p->Sq};
    const int bytes = a.nb * 4;
    if (bytes > 200 * 1024) return fail(ctx, LTCA_ERR_UNSUPPORTED, "select: %d blocks of tokens are too many", a.nb);
    auto kern = p->dtype == LTCA_BF16 ? kv8_select_kernel<__nv_bfloat16> : kv8_select_kernel<float>;
    static SmemOptIn once[2];
    LTCA_CUDA_OK(ctx, opt_in_dynamic_smem(once[p->dtype == LTCA_BF16], ctx->device, kern, 200 * 1024));
    const dim3 grid((unsigned)(c->B * c->H));
    LTCA_CUDA_OK(ctx, launch_dependent(kern, grid, dim3(kThreads), bytes, ctx->stream, a));
    return LTCA_OK;
}

}  // namespace ltca
