// C ABI of include/wick_rocm_lfm2.h: KV caches in pages, and sampling.  Host code only.
#include <algorithm>
#include <cmath>
#include <initializer_list>

#include "wick_rocm_ctx.h"

namespace {

constexpr uint32_t kMaxSeqs = 4096, kMaxPages = 1u << 24, kMaxRows = 1u << 30;

bool misaligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a != 0; }

// An array that a call writes is none of the others (null: not given).
bool among(const void* p, std::initializer_list<const void*> others) { return p && std::find(others.begin(), others.end(), p) != others.end(); }

// What every call asks of a pool and its table; null: nothing is wrong.
const char* pool_shape(const wick_rocm_kv_pages& p) {
    if (p.page_rows < 16u || p.page_rows > 256u || (p.page_rows & (p.page_rows - 1u)) != 0) return "kv_pages: page_rows must be 16, 32, 64, 128 or 256";
    if (p.n_seqs == 0 || p.n_seqs > kMaxSeqs) return "kv_pages: n_seqs must be 1 .. 4096";
    if (p.n_pages == 0 || p.n_pages > kMaxPages) return "kv_pages: n_pages must be 1 .. 2^24";
    if (p.max_pages == 0 || (uint64_t)p.max_pages * p.page_rows > kMaxRows || (uint64_t)p.max_pages * p.n_seqs > kMaxRows)
        return "kv_pages: max_pages must be at least 1, max_pages * page_rows and max_pages * n_seqs at most 2^30";
    return nullptr;
}
const char* heads_shape(uint32_t n_kv_heads, uint32_t head_dim, int kv_dtype) {
    if (head_dim != 32u && head_dim != 64u && head_dim != 128u && head_dim != 256u) return "kv_pages: head_dim must be 32, 64, 128 or 256";
    if (n_kv_heads == 0 || n_kv_heads > 65535u) return "kv_pages: n_kv_heads must be 1 .. 65535";
    if (kv_dtype != WICK_ROCM_KV_F32 && kv_dtype != WICK_ROCM_KV_F16) return "kv_pages: kv_dtype must be WICK_ROCM_KV_F32 or WICK_ROCM_KV_F16";
    return nullptr;
}

int check_pool(wick_rocm_ctx* ctx, const wick_rocm_kv_pages* p) {
    if (!p) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages: no pool");
    if (const char* wrong = pool_shape(*p)) return fail(ctx, WICK_ROCM_ERR_BAD_SHAPE, wrong);
    if (!p->d_table || !p->d_lens || !p->d_refs) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages: null table, lens or refs");
    if (misaligned(p->d_table, 4) || misaligned(p->d_lens, 4) || misaligned(p->d_refs, 4))
        return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages: table, lens and refs must be 4-byte aligned");
    if (among(p->d_table, {p->d_lens, p->d_refs}) || p->d_lens == p->d_refs) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages: table, lens and refs are one array");
    return WICK_ROCM_OK;
}
int check_planes(wick_rocm_ctx* ctx, const wick_rocm_kv_pages& p, const wick_rocm_kv_planes& planes) {
    if (const char* wrong = heads_shape(planes.n_kv_heads, planes.head_dim, planes.kv_dtype)) return fail(ctx, WICK_ROCM_ERR_BAD_SHAPE, wrong);
    if (!planes.d_base || misaligned(planes.d_base, 16)) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages: the planes must be there and 16-byte aligned");
    const uint64_t bytes = (uint64_t)p.page_rows * planes.n_kv_heads * planes.head_dim * (planes.kv_dtype == WICK_ROCM_KV_F16 ? 2u : 4u);
    if (planes.n_planes == 0 || planes.n_planes > 1024u) return fail(ctx, WICK_ROCM_ERR_BAD_SHAPE, "kv_pages: n_planes must be 1 .. 1024");
    if (planes.n_planes > 1 && (planes.plane_bytes < bytes * p.n_pages || planes.plane_bytes % 16u != 0))
        return fail(ctx, WICK_ROCM_ERR_BAD_SHAPE, "kv_pages: plane_bytes must cover a plane and be a multiple of 16");
    if (planes.n_planes * ((bytes + 16383u) / 16384u) > 1u << 23) return fail(ctx, WICK_ROCM_ERR_BAD_SHAPE, "kv_pages: a page of all planes is more than 2^37 bytes");
    return WICK_ROCM_OK;
}

// What both calls that put tokens into pages ask of them.
int check_tokens(wick_rocm_ctx* ctx, const wick_rocm_kv_pages& p, const float* d_k, const float* d_v, uint32_t kv_stride, const void* d_k_pages,
                 const void* d_v_pages, int kv_dtype, const uint32_t* d_start, const uint32_t* d_first, uint32_t n, uint32_t n_kv_heads, uint32_t head_dim) {
    if (const char* wrong = heads_shape(n_kv_heads, head_dim, kv_dtype)) return fail(ctx, WICK_ROCM_ERR_BAD_SHAPE, wrong);
    if (!d_k || !d_v || !d_k_pages || !d_v_pages || !d_start) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages: null keys, values, pages or start");
    if (kv_stride < (uint64_t)n_kv_heads * head_dim) return fail(ctx, WICK_ROCM_ERR_BAD_SHAPE, "kv_pages: kv_stride must cover n_kv_heads * head_dim");
    if (misaligned(d_k_pages, 16) || misaligned(d_v_pages, 16)) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages: pages must be 16-byte aligned");
    if (misaligned(d_start, 4) || misaligned(d_first, 4)) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages: start and first must be 4-byte aligned");
    if (d_k_pages == d_v_pages) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages: keys and values are one plane");
    if (!d_first && n != p.n_seqs) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages: without d_first there is one token a sequence");
    if (n > 1u << 23 || (uint64_t)n * n_kv_heads * head_dim > (uint64_t)1 << 33) return fail(ctx, WICK_ROCM_ERR_BAD_SHAPE, "kv_pages: too many tokens at once");
    return WICK_ROCM_OK;
}

}  // namespace

extern "C" {

int wick_rocm_kv_paged_append(wick_rocm_ctx* ctx, const wick_rocm_kv_pages* pages, const float* d_k, const float* d_v, uint32_t kv_stride, void* d_k_pages,
                              void* d_v_pages, int kv_dtype, const uint32_t* d_start, const uint32_t* d_first, uint32_t n, uint32_t n_kv_heads,
                              uint32_t head_dim) {
    WR_ENTER(ctx);
    if (int rc = check_pool(ctx, pages)) return rc;
    if (int rc = check_tokens(ctx, *pages, d_k, d_v, kv_stride, d_k_pages, d_v_pages, kv_dtype, d_start, d_first, n, n_kv_heads, head_dim)) return rc;
    if (kv_stride % 4u != 0 || misaligned(d_k, 16) || misaligned(d_v, 16))
        return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_paged_append: keys and values must be 16-byte aligned, kv_stride a multiple of 4");
    hipError_t e = launch_kv_paged_append(*pages, d_k, d_v, kv_stride, d_k_pages, d_v_pages, kv_dtype == WICK_ROCM_KV_F16, d_start, d_first, n, n_kv_heads,
                                          head_dim, ctx->launch());
    return e == hipSuccess ? WICK_ROCM_OK : fail_hip(ctx, e, "kv_paged_append launch");
}

int wick_rocm_qk_norm_rope_paged(wick_rocm_ctx* ctx, const wick_rocm_kv_pages* pages, float* d_q, uint32_t q_stride, float* d_k, const float* d_v,
                                 uint32_t kv_stride, const float* d_q_norm, const float* d_k_norm, void* d_k_pages, void* d_v_pages, int kv_dtype,
                                 const uint32_t* d_start, const uint32_t* d_first, uint32_t n, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim, float eps,
                                 float theta_scale) {
    WR_ENTER(ctx);
    if (int rc = check_pool(ctx, pages)) return rc;
    if (int rc = check_tokens(ctx, *pages, d_k, d_v, kv_stride, d_k_pages, d_v_pages, kv_dtype, d_start, d_first, n, n_kv_heads, head_dim)) return rc;
    if (n_heads == 0 || n_heads > 65535u || n_heads % n_kv_heads != 0)
        return fail(ctx, WICK_ROCM_ERR_BAD_SHAPE, "qk_norm_rope_paged: n_heads must be 1 .. 65535, and n_kv_heads divide it");
    if (q_stride < (uint64_t)n_heads * head_dim) return fail(ctx, WICK_ROCM_ERR_BAD_SHAPE, "qk_norm_rope_paged: q_stride must cover a token's heads");
    if (!d_q || !d_q_norm || !d_k_norm || misaligned(d_q, 4) || misaligned(d_k, 4) || misaligned(d_v, 4) || misaligned(d_q_norm, 4) || misaligned(d_k_norm, 4))
        return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "qk_norm_rope_paged: queries, keys, values and norms must be there and 4-byte aligned");
    if (d_q == d_k) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "qk_norm_rope_paged: queries and keys are one array");
    hipError_t e = launch_qk_norm_rope_paged(*pages, d_q, q_stride, d_k, d_v, kv_stride, d_q_norm, d_k_norm, d_k_pages, d_v_pages, kv_dtype == WICK_ROCM_KV_F16,
                                             d_start, d_first, n, n_heads, n_kv_heads, head_dim, eps, theta_scale, ctx->launch());
    return e == hipSuccess ? WICK_ROCM_OK : fail_hip(ctx, e, "qk_norm_rope_paged launch");
}

size_t wick_rocm_attention_paged_scratch_floats(uint32_t n_seqs, uint32_t n_heads, uint32_t n_kv_heads, uint32_t head_dim) {
    if (n_seqs == 0 || n_seqs > kMaxSeqs || heads_shape(n_kv_heads, head_dim, WICK_ROCM_KV_F32) || n_heads == 0 || n_heads % n_kv_heads != 0) return 0;
    return attention_paged_scratch_floats(n_heads, n_kv_heads, head_dim);
}

int wick_rocm_attention_decode_paged(wick_rocm_ctx* ctx, const wick_rocm_kv_pages* pages, const float* d_q, uint32_t q_stride, const void* d_k_pages,
                                     const void* d_v_pages, int kv_dtype, float* d_out, uint32_t out_stride, float* d_scratch, uint32_t n_heads,
                                     uint32_t n_kv_heads, uint32_t head_dim) {
    WR_ENTER(ctx);
    if (int rc = check_pool(ctx, pages)) return rc;
    if (const char* wrong = heads_shape(n_kv_heads, head_dim, kv_dtype)) return fail(ctx, WICK_ROCM_ERR_BAD_SHAPE, wrong);
    if (n_heads == 0 || n_heads % n_kv_heads != 0) return fail(ctx, WICK_ROCM_ERR_BAD_SHAPE, "attention_paged: n_kv_heads must divide n_heads");
    if (q_stride < (uint64_t)n_heads * head_dim || out_stride < (uint64_t)n_heads * head_dim || q_stride % 4u != 0 || out_stride % 4u != 0)
        return fail(ctx, WICK_ROCM_ERR_BAD_SHAPE, "attention_paged: strides must cover n_heads * head_dim and be multiples of 4");
    if (!attention_paged_fits(*pages, n_heads, n_kv_heads)) return fail(ctx, WICK_ROCM_ERR_BAD_SHAPE, "attention_paged: too many rows and heads in all");
    if (!d_q || !d_k_pages || !d_v_pages || !d_out || !d_scratch) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "attention_paged: null device pointer");
    if (misaligned(d_q, 16) || misaligned(d_k_pages, 16) || misaligned(d_v_pages, 16) || misaligned(d_out, 16) || misaligned(d_scratch, 16))
        return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "attention_paged: q, pages, output and scratch must be 16-byte aligned");
    if (d_out == d_q && out_stride != q_stride && pages->n_seqs > 1)  // (else a sequence's queries are read before its output is written)
        return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "attention_paged: an output in place of the queries needs their stride");
    if (among(d_scratch, {d_q, d_out, d_k_pages, d_v_pages}) || among(d_out, {d_k_pages, d_v_pages}))
        return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "attention_paged: output and scratch must be arrays of their own");
    const float scale = 1.0f / sqrtf((float)head_dim);  // wick/src/model/lfm2.rs:862
    hipError_t e = launch_attention_paged(*pages, d_q, q_stride, d_k_pages, d_v_pages, kv_dtype == WICK_ROCM_KV_F16, d_out, out_stride, d_scratch, n_heads,
                                          n_kv_heads, head_dim, scale, ctx->launch());
    return e == hipSuccess ? WICK_ROCM_OK : fail_hip(ctx, e, "attention_paged launch");
}

int wick_rocm_kv_pages_fork(wick_rocm_ctx* ctx, const wick_rocm_kv_pages* pages, const uint32_t* d_parents) {
    WR_ENTER(ctx);
    if (int rc = check_pool(ctx, pages)) return rc;
    if (!d_parents || misaligned(d_parents, 4)) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages_fork: the parents must be there and 4-byte aligned");
    if (among(d_parents, {pages->d_table, pages->d_lens, pages->d_refs})) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages_fork: the parents must be an array of their own");
    hipError_t e = launch_kv_pages_fork(*pages, d_parents, ctx->launch());
    return e == hipSuccess ? WICK_ROCM_OK : fail_hip(ctx, e, "kv_pages_fork launch");
}

int wick_rocm_kv_pages_free(wick_rocm_ctx* ctx, const wick_rocm_kv_pages* pages, const uint32_t* d_rows) {
    WR_ENTER(ctx);
    if (int rc = check_pool(ctx, pages)) return rc;
    if (!d_rows || misaligned(d_rows, 4)) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages_free: the rows must be there and 4-byte aligned");
    if (among(d_rows, {pages->d_table, pages->d_lens, pages->d_refs})) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages_free: the rows must be an array of their own");
    hipError_t e = launch_kv_pages_free(*pages, d_rows, ctx->launch());
    return e == hipSuccess ? WICK_ROCM_OK : fail_hip(ctx, e, "kv_pages_free launch");
}

size_t wick_rocm_kv_pages_moves_words(const wick_rocm_kv_pages* pages) { return !pages || pool_shape(*pages) ? 0 : kv_pages_moves_words(*pages); }

int wick_rocm_kv_pages_reserve(wick_rocm_ctx* ctx, const wick_rocm_kv_pages* pages, const uint32_t* d_counts, uint32_t* d_start, uint32_t* d_moves,
                               const wick_rocm_kv_planes* planes) {
    WR_ENTER(ctx);
    if (int rc = check_pool(ctx, pages)) return rc;
    if (!d_counts || !d_start || !d_moves) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages_reserve: null device pointer");
    if (misaligned(d_counts, 4) || misaligned(d_start, 4) || misaligned(d_moves, 16))
        return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages_reserve: counts and start must be 4-byte, moves 16-byte aligned");
    if (among(d_start, {d_counts, d_moves, pages->d_table, pages->d_lens, pages->d_refs})) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages_reserve: start must be an array of its own");
    if (among(d_moves, {pages->d_table, pages->d_lens, pages->d_refs})) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages_reserve: the moves must be an array of their own");
    if (planes)
        if (int rc = check_planes(ctx, *pages, *planes)) return rc;
    hipError_t e = launch_kv_pages_reserve(*pages, d_counts, d_start, d_moves, planes, ctx->launch());
    return e == hipSuccess ? WICK_ROCM_OK : fail_hip(ctx, e, "kv_pages_reserve launch");
}

int wick_rocm_kv_pages_compact(wick_rocm_ctx* ctx, const wick_rocm_kv_pages* pages, uint32_t* d_moves, const wick_rocm_kv_planes* planes) {
    WR_ENTER(ctx);
    if (int rc = check_pool(ctx, pages)) return rc;
    if (!d_moves || misaligned(d_moves, 16)) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages_compact: the moves must be there and 16-byte aligned");
    if (among(d_moves, {pages->d_table, pages->d_lens, pages->d_refs})) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages_compact: the moves must be an array of their own");
    if (planes)
        if (int rc = check_planes(ctx, *pages, *planes)) return rc;
    hipError_t e = launch_kv_pages_compact(*pages, d_moves, planes, ctx->launch());
    return e == hipSuccess ? WICK_ROCM_OK : fail_hip(ctx, e, "kv_pages_compact launch");
}

int wick_rocm_kv_pages_copy(wick_rocm_ctx* ctx, const wick_rocm_kv_pages* pages, const wick_rocm_kv_planes* planes, const uint32_t* d_moves, uint32_t max_moves) {
    WR_ENTER(ctx);
    if (int rc = check_pool(ctx, pages)) return rc;
    if (!planes || !d_moves || misaligned(d_moves, 16)) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "kv_pages_copy: planes and moves must be there, moves 16-byte aligned");
    if (int rc = check_planes(ctx, *pages, *planes)) return rc;
    hipError_t e = launch_kv_pages_copy(*pages, *planes, d_moves, max_moves, ctx->launch());
    return e == hipSuccess ? WICK_ROCM_OK : fail_hip(ctx, e, "kv_pages_copy launch");
}

size_t wick_rocm_sample_scratch_bytes(uint32_t rows, uint32_t n) {
    return rows == 0 || rows > 65535u || n == 0 || n > kSampleMaxTokens ? 0 : sample_scratch_bytes(rows, n);
}

int wick_rocm_sample(wick_rocm_ctx* ctx, const float* d_logits, uint32_t logits_stride, uint32_t rows, uint32_t n, const wick_rocm_sample_params* d_params,
                     const float* d_uniform, uint32_t* d_out, float* d_prob, void* d_scratch) {
    WR_ENTER(ctx);
    if (n == 0 || n > kSampleMaxTokens || rows > 65535u) return fail(ctx, WICK_ROCM_ERR_BAD_SHAPE, "sample: n must be 1 .. 2^19, rows at most 65535");
    if (rows > 1 && logits_stride < n) return fail(ctx, WICK_ROCM_ERR_BAD_SHAPE, "sample: logits_stride must cover a row");
    if (!d_logits || !d_params || !d_uniform || !d_out || !d_scratch) return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "sample: null device pointer");
    if (misaligned(d_logits, 4) || misaligned(d_params, 4) || misaligned(d_uniform, 4) || misaligned(d_out, 4) || misaligned(d_prob, 4) || misaligned(d_scratch, 16))
        return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "sample: arrays must be 4-byte, scratch 16-byte aligned");
    if (among(d_out, {d_logits, d_params, d_prob, d_scratch}) || among(d_prob, {d_logits, d_params, d_scratch}) || among(d_scratch, {d_logits, d_params, d_uniform}))
        return fail(ctx, WICK_ROCM_ERR_INVALID_ARG, "sample: what is written must be arrays of their own");
    hipError_t e = launch_sample(d_logits, logits_stride, rows, n, d_params, d_uniform, d_out, d_prob, d_scratch, ctx->launch());
    return e == hipSuccess ? WICK_ROCM_OK : fail_hip(ctx, e, "sample launch");
}

}  // extern "C"
