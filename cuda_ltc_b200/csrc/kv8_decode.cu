// Attention of the newest tokens over an 8-bit cache: see ltca_kv8_decode in include/ltc_attn.h.
#include "kv8.cuh"

namespace ltca {

namespace {

struct DecodeArgs {
    ltca_kv8_cache c;
    ltca_kv8_decode_params p;
    int nb;
};

// One CTA per row of Q; a warp takes a key at a time.
template <typename T>
__global__ void __launch_bounds__(128) kv8_decode_kernel(const DecodeArgs a) {
    __shared__ float sm_o[4][128], sm_m[4], sm_l[4];
    grid_dependency_wait();
    const int D = a.c.D, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int i = blockIdx.y, hq = blockIdx.x % a.p.Hq, b = blockIdx.x / a.p.Hq, h = hq / (a.p.Hq / a.c.H);
    const int n = new_tokens(a.p.new_len, b, a.p.Sq);
    const int64_t len = a.p.kv_len ? a.p.kv_len[b] : a.c.S;
    int64_t live = len < a.c.S ? len : a.c.S;
    if (a.p.causal && len - n + i + 1 < live) live = len - n + i + 1;
    if (i >= n || live < 0) live = 0;
    const T* q = reinterpret_cast<const T*>(a.p.q) + b * a.p.q_strides.batch + hq * a.p.q_strides.head + i * a.p.q_strides.seq;
    const uint8_t* k = reinterpret_cast<const uint8_t*>(a.c.k) + b * a.c.k_strides.batch + h * a.c.k_strides.head;
    const uint8_t* v = reinterpret_cast<const uint8_t*>(a.c.v) + b * a.c.v_strides.batch + h * a.c.v_strides.head;
    const int64_t pair = (int64_t)b * a.c.H + h;
    const float *ks = a.c.k_scale + pair * a.nb, *vs = a.c.v_scale + pair * a.nb;
    const float* mask = a.p.keep_mask ? a.p.keep_mask + ((int64_t)b * a.p.Sq + i) * a.c.S : nullptr;
    const int32_t* list = a.p.blocks ? a.p.blocks + pair * a.p.n_blocks : nullptr;
    const int64_t keys = list ? (int64_t)a.p.n_blocks * a.c.block : live;
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t t = warp; t < keys; t += 4) {
        int64_t j = t;
        if (list) {
            const int blk = list[t / a.c.block];
            if (blk < 0 || blk >= a.nb) continue;
            j = (int64_t)blk * a.c.block + t % a.c.block;
        }
        if (j >= live || (mask && mask[j] == 0.f)) continue;
        float s = 0.f;
        for (int d = lane; d < D; d += 32) s = fmaf(ld_value(q + d), e4m3x2_to_float2(k[j * a.c.k_strides.seq + d]).x, s);
        for (int off = 16; off; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        s *= a.p.scale * ks[j / a.c.block];
        if (a.p.score_clamp > 0.f) s = fminf(s, a.p.score_clamp);
        const float mt = fmaxf(m, s), ms = mt == -INFINITY ? 0.f : mt;
        const float corr = expf(m - ms), w = expf(s - ms);
        l = l * corr + w;
        for (int d = lane, x = 0; d < D; d += 32, ++x)
            o[x] = o[x] * corr + w * vs[j / a.c.block] * e4m3x2_to_float2(v[j * a.c.v_strides.seq + d]).x;
        m = mt;
    }
    for (int d = lane, x = 0; d < D; d += 32, ++x) sm_o[warp][d] = o[x];
    if (lane == 0) { sm_m[warp] = m; sm_l[warp] = l; }
    __syncthreads();
    if ((int)threadIdx.x >= D) return;
    float M = -INFINITY, L = 0.f, acc = 0.f;
    for (int w = 0; w < 4; ++w) M = fmaxf(M, sm_m[w]);
    const float Ms = M == -INFINITY ? 0.f : M;
    for (int w = 0; w < 4; ++w) {
        L += sm_l[w] * expf(sm_m[w] - Ms);
        acc += sm_o[w][threadIdx.x] * expf(sm_m[w] - Ms);
    }
    T* out = reinterpret_cast<T*>(a.p.o) + b * a.p.o_strides.batch + hq * a.p.o_strides.head + i * a.p.o_strides.seq;
    st_value(out + threadIdx.x, L == 0.f ? 0.f : acc / L);
    if (threadIdx.x == 0 && a.p.lse) a.p.lse[((int64_t)b * a.p.Hq + hq) * a.p.Sq + i] = L == 0.f ? -INFINITY : M + logf(L);
}

}  // namespace

size_t kv8_decode_workspace(const ltca_kv8_cache*, const ltca_kv8_decode_params*) { return 0; }

int launch_kv8_decode(ltca_ctx* ctx, const ltca_kv8_cache* c, const ltca_kv8_decode_params* p) {
    DecodeArgs a{*c, *p, (c->S + c->block - 1) / c->block};
    const dim3 grid((unsigned)(c->B * p->Hq), (unsigned)p->Sq);
    auto kern = p->dtype == LTCA_BF16 ? kv8_decode_kernel<__nv_bfloat16> : kv8_decode_kernel<float>;
    LTCA_CUDA_OK(ctx, launch_dependent(kern, grid, dim3(128), 0, ctx->stream, a));
    return LTCA_OK;
}

}  // namespace ltca
