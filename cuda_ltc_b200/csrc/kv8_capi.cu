// C-ABI entry points of the 8-bit key/value cache: argument checks in front of the kernels' launches.  Every index that a
// kernel forms from these arguments and from what it reads on the device (lengths, block lists) is cut to the cache there.
#include <initializer_list>

#include "kv8.cuh"

namespace ltca {

int launch_kv8_append(ltca_ctx* ctx, const ltca_kv8_cache* c, const ltca_kv8_append_params* p);
int launch_kv8_read(ltca_ctx* ctx, const ltca_kv8_cache* c, const ltca_kv8_read_params* p);
int launch_kv8_decode(ltca_ctx* ctx, const ltca_kv8_cache* c, const ltca_kv8_decode_params* p);
size_t kv8_decode_workspace(const ltca_kv8_cache* c, const ltca_kv8_decode_params* p);
int launch_kv8_select(ltca_ctx* ctx, const ltca_kv8_cache* c, const ltca_kv8_select_params* p);

namespace {

bool misaligned(const void* p, const ltca_strides& s, int to) {
    return reinterpret_cast<uintptr_t>(p) % to || s.batch % to || s.head % to || s.seq % to;
}
// Whether a pointer lies on a boundary of its elements: kernels read whole elements at the least.
bool off_element(const void* p, int size) { return reinterpret_cast<uintptr_t>(p) % size; }
int check_words(ltca_ctx* ctx, std::initializer_list<const void*> words) {
    for (const void* p : words)
        if (off_element(p, 4)) return fail(ctx, LTCA_ERR_INVALID, "int32 and float32 arrays must be 4-byte aligned");
    return LTCA_OK;
}
int check_elements(ltca_ctx* ctx, int dtype, std::initializer_list<const void*> tensors) {
    for (const void* p : tensors)
        if (off_element(p, elem_size(dtype))) return fail(ctx, LTCA_ERR_INVALID, "a tensor must be aligned to its elements (%d bytes)", elem_size(dtype));
    return LTCA_OK;
}
// Whether two places of a [B,H,n,...] tensor share memory through a stride of zero.
bool overlaps(const ltca_strides& s, int64_t B, int64_t H, int64_t n) {
    return (B > 1 && s.batch == 0) || (H > 1 && s.head == 0) || (n > 1 && s.seq == 0);
}

// `k`, `v`: whether the call reads or writes these.
int check_cache(ltca_ctx* ctx, const ltca_kv8_cache* c, bool k, bool v) {
    if (!c) return fail(ctx, LTCA_ERR_INVALID, "null cache");
    if (c->B < 1 || c->H < 1 || c->S < 1)
        return fail(ctx, LTCA_ERR_INVALID, "bad cache shape B=%d H=%d S=%d", c->B, c->H, c->S);
    // positions and what the kernels add to them stay in 32 bits
    if (c->S > (1 << 30)) return fail(ctx, LTCA_ERR_UNSUPPORTED, "the capacity is above 2^30 tokens");
    if ((int64_t)c->B * c->H >= 1 << 30) return fail(ctx, LTCA_ERR_INVALID, "B * H is 2^30 or more");
    if (c->D != 32 && c->D != 64 && c->D != 128)
        return fail(ctx, LTCA_ERR_UNSUPPORTED, "the 8-bit cache supports head_dim 32, 64, 128 (got %d)", c->D);
    if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128)
        return fail(ctx, LTCA_ERR_UNSUPPORTED, "a scale is shared by 16, 32, 64 or 128 tokens (got %d)", c->block);
    if ((k && (!c->k || !c->k_scale)) || (v && (!c->v || !c->v_scale)))
        return fail(ctx, LTCA_ERR_INVALID, "null tensor in the cache");
    if ((k && misaligned(c->k, c->k_strides, 16)) || (v && misaligned(c->v, c->v_strides, 16)))
        return fail(ctx, LTCA_ERR_INVALID, "the cache's rows must start on 16-byte boundaries");
    if (reinterpret_cast<uintptr_t>(c->bounds) % 16) return fail(ctx, LTCA_ERR_INVALID, "bounds must be 16-byte aligned");
    return check_words(ctx, {c->k_scale, c->v_scale});
}
int check_dtype(ltca_ctx* ctx, int dtype) {
    return dtype == LTCA_F32 || dtype == LTCA_BF16 ? LTCA_OK : fail(ctx, LTCA_ERR_INVALID, "bad dtype %d", dtype);
}
int check_queries(ltca_ctx* ctx, const ltca_kv8_cache* c, int Hq, int Sq, int dtype, const void* q) {
    if (int rc = check_dtype(ctx, dtype)) return rc;
    if (!q) return fail(ctx, LTCA_ERR_INVALID, "null tensor");
    if (Hq < 1 || Hq % c->H) return fail(ctx, LTCA_ERR_INVALID, "%d heads of queries over %d heads of keys", Hq, c->H);
    if (Sq < 1) return fail(ctx, LTCA_ERR_INVALID, "no queries (Sq = %d)", Sq);
    if ((int64_t)Hq / c->H * Sq > (1 << 20))
        return fail(ctx, LTCA_ERR_UNSUPPORTED, "%lld rows of queries per head of keys: at most 2^20", (long long)Hq / c->H * Sq);
    return LTCA_OK;
}

// The context's device for a call, the caller's behind it.
struct OnDevice {
    int before = -1;
    cudaError_t e;
    explicit OnDevice(int device) {
        e = cudaGetDevice(&before);
        if (e == cudaSuccess && before != device) e = cudaSetDevice(device);
        else before = -1;
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

}  // namespace
}  // namespace ltca

using namespace ltca;

extern "C" {

int ltca_kv8_append(ltca_ctx* ctx, const ltca_kv8_cache* c, const ltca_kv8_append_params* p) {
    if (!ctx) return LTCA_ERR_INVALID;
    if (!p) return fail(ctx, LTCA_ERR_INVALID, "null parameter block");
    if (int rc = check_cache(ctx, c, true, true)) return rc;
    if (int rc = check_dtype(ctx, p->dtype)) return rc;
    if (p->n < 0) return fail(ctx, LTCA_ERR_INVALID, "negative number of tokens %d", p->n);
    if (p->n == 0) return LTCA_OK;
    if (!p->k || !p->v || !p->kv_len) return fail(ctx, LTCA_ERR_INVALID, "append needs k, v and kv_len");
    if (int rc = check_elements(ctx, p->dtype, {p->k, p->v})) return rc;
    if (int rc = check_words(ctx, {p->kv_len, p->new_len})) return rc;
    if (overlaps(c->k_strides, c->B, c->H, c->S) || overlaps(c->v_strides, c->B, c->H, c->S))
        return fail(ctx, LTCA_ERR_INVALID, "a cache that is written must not share memory between sequences, heads or tokens");
    OnDevice on(ctx->device);
    LTCA_CUDA_OK(ctx, on.e);
    return launch_kv8_append(ctx, c, p);
}

int ltca_kv8_read(ltca_ctx* ctx, const ltca_kv8_cache* c, const ltca_kv8_read_params* p) {
    if (!ctx) return LTCA_ERR_INVALID;
    if (!p) return fail(ctx, LTCA_ERR_INVALID, "null parameter block");
    if (int rc = check_cache(ctx, c, true, true)) return rc;
    if (int rc = check_dtype(ctx, p->dtype)) return rc;
    if (p->start < 0 || p->n < 0 || (int64_t)p->start + p->n > c->S)
        return fail(ctx, LTCA_ERR_INVALID, "bad range of positions %d + %d of %d", p->start, p->n, c->S);
    if (p->n == 0) return LTCA_OK;
    if (!p->k || !p->v) return fail(ctx, LTCA_ERR_INVALID, "null tensor");
    if (int rc = check_elements(ctx, p->dtype, {p->k, p->v})) return rc;
    if (int rc = check_words(ctx, {p->kv_len})) return rc;
    if (overlaps(p->k_strides, c->B, c->H, p->n) || overlaps(p->v_strides, c->B, c->H, p->n))
        return fail(ctx, LTCA_ERR_INVALID, "a result must not share memory between sequences, heads or tokens");
    OnDevice on(ctx->device);
    LTCA_CUDA_OK(ctx, on.e);
    return launch_kv8_read(ctx, c, p);
}

int ltca_kv8_decode_workspace_bytes(const ltca_kv8_cache* c, const ltca_kv8_decode_params* p, size_t* bytes_out) {
    if (!c || !p || !bytes_out) return LTCA_ERR_INVALID;
    *bytes_out = 0;
    if (check_cache(nullptr, c, false, false) || check_queries(nullptr, c, p->Hq, p->Sq, p->dtype, c)) return LTCA_OK;   // (refused by the call)
    *bytes_out = kv8_decode_workspace(c, p);
    return LTCA_OK;
}

int ltca_kv8_decode(ltca_ctx* ctx, const ltca_kv8_cache* c, const ltca_kv8_decode_params* p) {
    if (!ctx) return LTCA_ERR_INVALID;
    if (!p) return fail(ctx, LTCA_ERR_INVALID, "null parameter block");
    if (int rc = check_cache(ctx, c, true, true)) return rc;
    if (int rc = check_queries(ctx, c, p->Hq, p->Sq, p->dtype, p->q)) return rc;
    if (!p->o) return fail(ctx, LTCA_ERR_INVALID, "null tensor");
    if (int rc = check_elements(ctx, p->dtype, {p->q, p->o})) return rc;
    if (int rc = check_words(ctx, {p->lse, p->keep_mask, p->kv_len, p->new_len, p->blocks})) return rc;
    if (!(p->scale > 0.f)) return fail(ctx, LTCA_ERR_INVALID, "scale must be positive");
    if (overlaps(p->o_strides, c->B, p->Hq, p->Sq))
        return fail(ctx, LTCA_ERR_INVALID, "a result must not share memory between sequences, heads or tokens");
    if (p->blocks && p->n_blocks < 1) return fail(ctx, LTCA_ERR_INVALID, "an empty list of blocks (n_blocks = %d)", p->n_blocks);
    if (p->workspace && (reinterpret_cast<uintptr_t>(p->workspace) & 255))
        return fail(ctx, LTCA_ERR_INVALID, "workspace must be 256-byte aligned");
    OnDevice on(ctx->device);
    LTCA_CUDA_OK(ctx, on.e);
    return launch_kv8_decode(ctx, c, p);
}

int ltca_kv8_select(ltca_ctx* ctx, const ltca_kv8_cache* c, const ltca_kv8_select_params* p) {
    if (!ctx) return LTCA_ERR_INVALID;
    if (!p) return fail(ctx, LTCA_ERR_INVALID, "null parameter block");
    if (int rc = check_cache(ctx, c, false, false)) return rc;
    if (int rc = check_queries(ctx, c, p->Hq, p->Sq, p->dtype, p->q)) return rc;
    if (!c->bounds || !c->k_scale) return fail(ctx, LTCA_ERR_INVALID, "select needs a cache that keeps bounds");
    if (!p->blocks) return fail(ctx, LTCA_ERR_INVALID, "null tensor");
    if (int rc = check_elements(ctx, p->dtype, {p->q})) return rc;
    if (int rc = check_words(ctx, {p->kv_len, p->new_len, p->blocks})) return rc;
    if (p->count < 1 || p->first < 0 || p->last < 0 || (int64_t)p->first + p->last > p->count)
        return fail(ctx, LTCA_ERR_INVALID, "%d blocks with the first %d and the last %d among them", p->count, p->first, p->last);
    OnDevice on(ctx->device);
    LTCA_CUDA_OK(ctx, on.e);
    return launch_kv8_select(ctx, c, p);
}

}  // extern "C"
