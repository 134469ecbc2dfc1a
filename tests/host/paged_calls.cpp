// Calls on KV caches in pages, and of sampling, that have to be refused, on a runtime that only pretends (fake_hip.h): each answers with its status and
// a message, nothing is enqueued, and the call with that one thing put right goes through.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <vector>

#include "../../include/wick_rocm.h"
#include "../../include/wick_rocm_lfm2.h"
#include "fake_hip.h"

namespace {

int failures = 0;

struct Call {  // every argument of the calls; a case changes one or two
    wick_rocm_kv_pages pages{4, 8, 20, 16, nullptr, nullptr, nullptr};
    wick_rocm_kv_planes planes{nullptr, 20 * 2 * 16 * 64 * 2, 3, 2, 64, WICK_ROCM_KV_F16};
    bool no_pages = false, no_planes = false;
    float *q = nullptr, *k = nullptr, *out = nullptr, *scratch = nullptr;
    const float *v = nullptr, *qn = nullptr, *kn = nullptr;
    void *k_pages = nullptr, *v_pages = nullptr;
    uint32_t *start = nullptr, *first = nullptr, *counts = nullptr, *moves = nullptr;
    uint32_t q_stride = 256, out_stride = 256, kv_stride = 128, n = 4, n_heads = 4, n_kv = 2, hd = 64, max_moves = 5;
    int type = WICK_ROCM_KV_F16;
    // sampling
    const float *logits = nullptr, *uniform = nullptr;
    const wick_rocm_sample_params* params = nullptr;
    uint32_t* token = nullptr;
    float* prob = nullptr;
    void* work = nullptr;
    uint32_t logits_stride = 1000, rows = 3, tokens = 1000;

    const wick_rocm_kv_pages* pool() const { return no_pages ? nullptr : &pages; }
    const wick_rocm_kv_planes* moved() const { return no_planes ? nullptr : &planes; }
};

int append(wick_rocm_ctx* c, const Call& a) {
    return wick_rocm_kv_paged_append(c, a.pool(), a.k, a.v, a.kv_stride, a.k_pages, a.v_pages, a.type, a.start, a.first, a.n, a.n_kv, a.hd);
}
int rope(wick_rocm_ctx* c, const Call& a) {
    return wick_rocm_qk_norm_rope_paged(c, a.pool(), a.q, a.q_stride, a.k, a.v, a.kv_stride, a.qn, a.kn, a.k_pages, a.v_pages, a.type, a.start, a.first, a.n, a.n_heads,
                                        a.n_kv, a.hd, 1e-5f, 0.8f);
}
int attention(wick_rocm_ctx* c, const Call& a) {
    return wick_rocm_attention_decode_paged(c, a.pool(), a.q, a.q_stride, a.k_pages, a.v_pages, a.type, a.out, a.out_stride, a.scratch, a.n_heads, a.n_kv, a.hd);
}
int fork(wick_rocm_ctx* c, const Call& a) { return wick_rocm_kv_pages_fork(c, a.pool(), a.counts); }
int free_rows(wick_rocm_ctx* c, const Call& a) { return wick_rocm_kv_pages_free(c, a.pool(), a.counts); }
int reserve(wick_rocm_ctx* c, const Call& a) { return wick_rocm_kv_pages_reserve(c, a.pool(), a.counts, a.start, a.moves, a.moved()); }
int compact(wick_rocm_ctx* c, const Call& a) { return wick_rocm_kv_pages_compact(c, a.pool(), a.moves, a.moved()); }
int copy(wick_rocm_ctx* c, const Call& a) { return wick_rocm_kv_pages_copy(c, a.pool(), a.moved(), a.moves, a.max_moves); }
int sample(wick_rocm_ctx* c, const Call& a) {
    return wick_rocm_sample(c, a.logits, a.logits_stride, a.rows, a.tokens, a.params, a.uniform, a.token, a.prob, a.work);
}

template <typename T>
T* off(T* p, int n) {
    return (T*)((char*)p + n);
}

}  // namespace

int main() {
    wick_rocm_ctx* ctx = nullptr;
    if (wick_rocm_ctx_create(0, &ctx) != WICK_ROCM_OK) std::abort();
    Call good;
    void* d[16];
    for (void*& p : d)
        if (wick_rocm_buffer_alloc(ctx, 1u << 20, &p) != WICK_ROCM_OK) std::abort();
    good.pages.d_table = (uint32_t*)d[0], good.pages.d_lens = (uint32_t*)d[1], good.pages.d_refs = (uint32_t*)d[2], good.planes.d_base = d[3];
    good.q = (float*)d[4], good.k = (float*)d[5], good.v = (float*)d[6], good.out = (float*)d[7], good.scratch = (float*)d[8], good.k_pages = d[9], good.v_pages = d[10];
    good.start = (uint32_t*)d[11], good.counts = (uint32_t*)d[12], good.moves = (uint32_t*)d[13], good.qn = (float*)d[14], good.kn = (float*)d[15];
    good.logits = good.q, good.uniform = good.k, good.params = (wick_rocm_sample_params*)d[6], good.token = (uint32_t*)d[7], good.prob = (float*)d[9], good.work = d[10];
    const int kShape = WICK_ROCM_ERR_BAD_SHAPE, kArg = WICK_ROCM_ERR_INVALID_ARG;
    struct Wrong {
        const char* what;
        int status;
        std::function<void(Call&)> change;
    };
    const auto each = [&](const char* name, int (*call)(wick_rocm_ctx*, const Call&), const std::vector<Wrong>& wrongs) {
        const auto launched = [&](const Call& a, int want, const char* what) {
            const long before = fake_hip::launches;
            const int rc = call(ctx, a);
            char message[256] = "";
            wick_rocm_last_error(ctx, message, sizeof message);
            const long launches = fake_hip::launches - before;
            const bool fine = rc == want && (want == WICK_ROCM_OK ? launches > 0 : launches == 0 && std::strlen(message) > 12);
            if (!fine) failures++, std::printf("%s, %s: status %d (wanted %d), %ld launches, '%s'\n", name, what, rc, want, launches, message);
        };
        launched(good, WICK_ROCM_OK, "as it should be");
        for (const Wrong& w : wrongs) {
            Call a = good;
            w.change(a);
            launched(a, w.status, w.what);
        }
        launched(good, WICK_ROCM_OK, "as it should be, again");
        if (call(nullptr, good) != kArg) failures++, std::printf("%s: no context\n", name);
    };
    typedef std::vector<Wrong> Wrongs;
    const auto with = [](Wrongs a, const Wrongs& b) {
        a.insert(a.end(), b.begin(), b.end());
        return a;
    };
    const Wrongs pool = {
        {"no pool", kArg, [](Call& a) { a.no_pages = true; }},
        {"no table", kArg, [](Call& a) { a.pages.d_table = nullptr; }},
        {"no lens", kArg, [](Call& a) { a.pages.d_lens = nullptr; }},
        {"no refs", kArg, [](Call& a) { a.pages.d_refs = nullptr; }},
        {"table off", kArg, [](Call& a) { a.pages.d_table = off(a.pages.d_table, 2); }},
        {"refs off", kArg, [](Call& a) { a.pages.d_refs = off(a.pages.d_refs, 1); }},
        {"lens in the table", kArg, [](Call& a) { a.pages.d_lens = a.pages.d_table; }},
        {"refs in the table", kArg, [](Call& a) { a.pages.d_refs = a.pages.d_table; }},
        {"refs in the lens", kArg, [](Call& a) { a.pages.d_refs = a.pages.d_lens; }},
        {"pages of 8 rows", kShape, [](Call& a) { a.pages.page_rows = 8; }},
        {"pages of 48 rows", kShape, [](Call& a) { a.pages.page_rows = 48; }},
        {"pages of 512 rows", kShape, [](Call& a) { a.pages.page_rows = 512; }},
        {"pages of no rows", kShape, [](Call& a) { a.pages.page_rows = 0; }},
        {"no sequences", kShape, [](Call& a) { a.pages.n_seqs = a.n = 0; }},
        {"too many sequences", kShape, [](Call& a) { a.pages.n_seqs = a.n = 4097; }},
        {"no pages", kShape, [](Call& a) { a.pages.n_pages = 0; }},
        {"too many pages", kShape, [](Call& a) { a.pages.n_pages = (1u << 24) + 1; }},
        {"no columns", kShape, [](Call& a) { a.pages.max_pages = 0; }},
        {"too many rows", kShape, [](Call& a) { a.pages.max_pages = (1u << 26) + 1; }},
        {"too large a table", kShape, [](Call& a) { a.pages.n_seqs = a.n = 4096, a.pages.max_pages = (1u << 18) + 1; }},
    };
    const Wrongs heads = {
        {"head_dim 0", kShape, [](Call& a) { a.hd = a.planes.head_dim = 0; }},
        {"head_dim 96", kShape, [](Call& a) { a.hd = a.planes.head_dim = 96; }},
        {"head_dim 512", kShape, [](Call& a) { a.hd = a.planes.head_dim = 512; }},
        {"no KV heads", kShape, [](Call& a) { a.n_kv = a.planes.n_kv_heads = 0; }},
        {"too many KV heads", kShape, [](Call& a) { a.n_kv = a.planes.n_kv_heads = 1u << 16; }},
        {"a type that is none", kShape, [](Call& a) { a.type = a.planes.kv_dtype = 2; }},
        {"a negative type", kShape, [](Call& a) { a.type = a.planes.kv_dtype = -1; }},
    };
    const Wrongs tokens = with(with(pool, heads), {
        {"no keys", kArg, [](Call& a) { a.k = nullptr; }},
        {"no values", kArg, [](Call& a) { a.v = nullptr; }},
        {"no pages of keys", kArg, [](Call& a) { a.k_pages = nullptr; }},
        {"no pages of values", kArg, [](Call& a) { a.v_pages = nullptr; }},
        {"no start", kArg, [](Call& a) { a.start = nullptr; }},
        {"start off", kArg, [](Call& a) { a.start = off(a.start, 2); }},
        {"first off", kArg, [](Call& a) { a.first = off(a.counts, 3); }},
        {"pages off", kArg, [](Call& a) { a.v_pages = off(a.v_pages, 8); }},
        {"one plane", kArg, [](Call& a) { a.v_pages = a.k_pages; }},
        {"short stride", kShape, [](Call& a) { a.kv_stride = 124; }},
        {"one token a sequence, but one more", kArg, [](Call& a) { a.n = 5; }},
        {"one token a sequence, but none", kArg, [](Call& a) { a.n = 0; }},
        {"too many tokens", kShape, [](Call& a) { a.first = a.counts, a.n = (1u << 23) + 1; }},
    });
    each("append", append, with(tokens, {
        {"odd stride", kArg, [](Call& a) { a.kv_stride = 130; }},
        {"keys off", kArg, [](Call& a) { a.k = off(a.k, 4); }},
        {"values off", kArg, [](Call& a) { a.v = off(a.v, 8); }},
    }));
    each("rope", rope, with(tokens, {
        {"no queries", kArg, [](Call& a) { a.q = nullptr; }},
        {"no norm of queries", kArg, [](Call& a) { a.qn = nullptr; }},
        {"no norm of keys", kArg, [](Call& a) { a.kn = nullptr; }},
        {"queries off", kArg, [](Call& a) { a.q = off(a.q, 2); }},
        {"keys off", kArg, [](Call& a) { a.k = off(a.k, 2); }},
        {"values off", kArg, [](Call& a) { a.v = off(a.v, 1); }},
        {"norm off", kArg, [](Call& a) { a.kn = off(a.kn, 2); }},
        {"queries and keys in one place", kArg, [](Call& a) { a.q = a.k; }},
        {"no heads", kShape, [](Call& a) { a.n_heads = 0; }},
        {"heads that no KV head divides", kShape, [](Call& a) { a.n_heads = 5, a.q_stride = 320; }},
        {"too many heads", kShape, [](Call& a) { a.n_heads = 1u << 16; }},
        {"short stride of queries", kShape, [](Call& a) { a.q_stride = 255; }},
    }));
    each("attention", attention, with(with(pool, heads), {
        {"no queries", kArg, [](Call& a) { a.q = nullptr; }},
        {"no pages of keys", kArg, [](Call& a) { a.k_pages = nullptr; }},
        {"no pages of values", kArg, [](Call& a) { a.v_pages = nullptr; }},
        {"no output", kArg, [](Call& a) { a.out = nullptr; }},
        {"no scratch", kArg, [](Call& a) { a.scratch = nullptr; }},
        {"queries off", kArg, [](Call& a) { a.q = off(a.q, 4); }},
        {"pages off", kArg, [](Call& a) { a.k_pages = off(a.k_pages, 2); }},
        {"output off", kArg, [](Call& a) { a.out = off(a.out, 8); }},
        {"scratch off", kArg, [](Call& a) { a.scratch = off(a.scratch, 4); }},
        {"no heads", kShape, [](Call& a) { a.n_heads = 0; }},
        {"heads that no KV head divides", kShape, [](Call& a) { a.n_heads = 5, a.q_stride = a.out_stride = 320; }},
        {"short stride of queries", kShape, [](Call& a) { a.q_stride = 252; }},
        {"odd stride of queries", kShape, [](Call& a) { a.q_stride = 258; }},
        {"short stride of the output", kShape, [](Call& a) { a.out_stride = 128; }},
        {"odd stride of the output", kShape, [](Call& a) { a.out_stride = 257; }},
        {"heads past 2^32", kShape, [](Call& a) { a.n_heads = 1u << 26; }},
        {"too many rows and heads in all", kShape, [](Call& a) { a.pages.n_seqs = 4096, a.pages.max_pages = 1u << 18, a.n_heads = a.n_kv = 64, a.q_stride = a.out_stride = 4096; }},
        {"too many heads of all sequences", kShape, [](Call& a) { a.pages.n_seqs = 4096, a.n_heads = a.n_kv = 513, a.q_stride = a.out_stride = 513 * 64; }},
        {"output in place at another stride", kArg, [](Call& a) { a.out = a.q, a.out_stride = 512; }},
        {"output in the keys", kArg, [](Call& a) { a.out = (float*)a.k_pages; }},
        {"output in the values", kArg, [](Call& a) { a.out = (float*)a.v_pages; }},
        {"scratch in the queries", kArg, [](Call& a) { a.scratch = a.q; }},
        {"scratch in the output", kArg, [](Call& a) { a.scratch = a.out; }},
        {"scratch in the keys", kArg, [](Call& a) { a.scratch = (float*)a.k_pages; }},
    }));
    const Wrongs counts = with(pool, {
        {"no numbers", kArg, [](Call& a) { a.counts = nullptr; }},
        {"numbers off", kArg, [](Call& a) { a.counts = off(a.counts, 2); }},
    });
    const Wrongs moves = with(pool, {
        {"no moves", kArg, [](Call& a) { a.moves = nullptr; }},
        {"moves off", kArg, [](Call& a) { a.moves = off(a.moves, 4); }},
    });
    const Wrongs planes = with(heads, {
        {"no base", kArg, [](Call& a) { a.planes.d_base = nullptr; }},
        {"base off", kArg, [](Call& a) { a.planes.d_base = off((char*)a.planes.d_base, 8); }},
        {"no planes", kShape, [](Call& a) { a.planes.n_planes = 0; }},
        {"too many planes", kShape, [](Call& a) { a.planes.n_planes = 1025; }},
        {"planes that overlap", kShape, [](Call& a) { a.planes.plane_bytes -= 16; }},
        {"planes off each other", kShape, [](Call& a) { a.planes.plane_bytes += 8; }},
        {"pages past any memory", kShape, [](Call& a) { a.pages.page_rows = 256, a.planes = {a.planes.d_base, (size_t)1 << 45, 1024, 65535, 256, WICK_ROCM_KV_F32}; }},
    });
    each("fork", fork, with(counts, {
        {"parents in the lengths", kArg, [](Call& a) { a.counts = a.pages.d_lens; }},
        {"parents in the table", kArg, [](Call& a) { a.counts = a.pages.d_table; }},
        {"parents in the refs", kArg, [](Call& a) { a.counts = a.pages.d_refs; }},
    }));
    each("free", free_rows, with(counts, {{"rows in the lengths", kArg, [](Call& a) { a.counts = a.pages.d_lens; }}}));
    each("free", free_rows, {{"rows in the table", kArg, [](Call& a) { a.counts = a.pages.d_table; }}, {"rows in the refs", kArg, [](Call& a) { a.counts = a.pages.d_refs; }}});
    each("reserve", reserve, with(with(with(counts, moves), planes), {
        {"no start", kArg, [](Call& a) { a.start = nullptr; }},
        {"start off", kArg, [](Call& a) { a.start = off(a.start, 1); }},
        {"start in the counts", kArg, [](Call& a) { a.start = a.counts; }},
        {"start in the lengths", kArg, [](Call& a) { a.start = a.pages.d_lens; }},
        {"start in the table", kArg, [](Call& a) { a.start = a.pages.d_table; }},
        {"start in the refs", kArg, [](Call& a) { a.start = a.pages.d_refs; }},
        {"start in the moves", kArg, [](Call& a) { a.start = a.moves; }},
        {"moves in the refs", kArg, [](Call& a) { a.moves = a.pages.d_refs; }},
    }));
    each("compact", compact, with(moves, planes));
    each("compact", compact, {{"moves in the table", kArg, [](Call& a) { a.moves = a.pages.d_table; }}, {"moves in the lengths", kArg, [](Call& a) { a.moves = a.pages.d_lens; }}});
    each("copy", copy, with(with(moves, planes), {{"no planes at all", kArg, [](Call& a) { a.no_planes = true; }}}));
    each("sample", sample, {
        {"no logits", kArg, [](Call& a) { a.logits = nullptr; }},
        {"no rules", kArg, [](Call& a) { a.params = nullptr; }},
        {"no uniform numbers", kArg, [](Call& a) { a.uniform = nullptr; }},
        {"no output", kArg, [](Call& a) { a.token = nullptr; }},
        {"no scratch", kArg, [](Call& a) { a.work = nullptr; }},
        {"logits off", kArg, [](Call& a) { a.logits = off(a.logits, 2); }},
        {"rules off", kArg, [](Call& a) { a.params = off(a.params, 2); }},
        {"uniform numbers off", kArg, [](Call& a) { a.uniform = off(a.uniform, 1); }},
        {"output off", kArg, [](Call& a) { a.token = off(a.token, 2); }},
        {"probabilities off", kArg, [](Call& a) { a.prob = off(a.prob, 2); }},
        {"scratch off", kArg, [](Call& a) { a.work = off((char*)a.work, 8); }},
        {"no tokens", kShape, [](Call& a) { a.tokens = 0; }},
        {"too many tokens", kShape, [](Call& a) { a.tokens = a.logits_stride = (1u << 19) + 1; }},
        {"too many rows", kShape, [](Call& a) { a.rows = 65536; }},
        {"short stride", kShape, [](Call& a) { a.logits_stride = 999; }},
        {"picks and probabilities in one place", kArg, [](Call& a) { a.prob = (float*)a.token; }},
        {"picks in the logits", kArg, [](Call& a) { a.token = (uint32_t*)a.logits; }},
        {"picks in the rules", kArg, [](Call& a) { a.token = (uint32_t*)a.params; }},
        {"probabilities in the logits", kArg, [](Call& a) { a.prob = (float*)a.logits; }},
        {"scratch in the logits", kArg, [](Call& a) { a.work = (void*)a.logits; }},
        {"scratch in the picks", kArg, [](Call& a) { a.work = a.token; }},
    });
    // what may be left out, or is at its limit
    const auto goes = [&](const char* what, int (*call)(wick_rocm_ctx*, const Call&), long launches, const std::function<void(Call&)>& change) {
        Call a = good;
        change(a);
        const long before = fake_hip::launches;
        const int rc = call(ctx, a);
        if (rc != WICK_ROCM_OK || fake_hip::launches - before != launches) failures++, std::printf("%s: status %d, %ld launches\n", what, rc, fake_hip::launches - before);
    };
    goes("no tokens to append", append, 0, [](Call& a) { a.first = a.counts, a.n = 0; });
    goes("no tokens to rotate", rope, 0, [](Call& a) { a.first = a.counts, a.n = 0; });
    goes("tokens at any stride and place", rope, 1, [](Call& a) { a.q = off(a.q, 4), a.k = off(a.k, 8), a.q_stride = 257, a.kv_stride = 131; });
    goes("no moves to make", copy, 0, [](Call& a) { a.max_moves = 0; });
    goes("one plane at any stride", copy, 1, [](Call& a) { a.planes.n_planes = 1, a.planes.plane_bytes = 1; });
    goes("pages reserved, copied by the caller", reserve, 1, [](Call& a) { a.no_planes = true; });
    goes("rows reserved and copied", reserve, 2, [](Call&) {});
    goes("a short table in one launch", attention, 1, [](Call&) {});
    goes("a long table in two", attention, 2, [](Call& a) { a.pages.max_pages = 1000; });
    goes("an output in place of the queries", attention, 1, [](Call& a) { a.out = a.q; });
    goes("one sequence's in place at any stride", attention, 1, [](Call& a) { a.out = a.q, a.out_stride = 512, a.pages.n_seqs = 1; });
    goes("picks in place of the uniform numbers", sample, 3, [](Call& a) { a.token = (uint32_t*)a.uniform; });
    goes("the largest pool", attention, 2, [](Call& a) { a.pages = {4096, 1u << 18, 1u << 24, 16, a.pages.d_table, a.pages.d_lens, a.pages.d_refs}, a.n_heads = a.n_kv = 1; });
    goes("no rows to pick from", sample, 0, [](Call& a) { a.rows = 0; });
    goes("one row at any stride, no probabilities", sample, 3, [](Call& a) { a.rows = 1, a.logits_stride = 0, a.prob = nullptr; });
    goes("the most tokens and rows", sample, 3, [](Call& a) { a.rows = 65535, a.tokens = a.logits_stride = 1u << 19; });
    // sizes
    if (wick_rocm_sample_scratch_bytes(0, 10) || wick_rocm_sample_scratch_bytes(65536, 10) || wick_rocm_sample_scratch_bytes(1, 0) ||
        wick_rocm_sample_scratch_bytes(1, (1u << 19) + 1) || wick_rocm_sample_scratch_bytes(65535, 1u << 19) < (size_t)65535 << 21)
        failures++, std::printf("scratch of picks\n");
    if (wick_rocm_attention_paged_scratch_floats(0, 4, 2, 64) || wick_rocm_attention_paged_scratch_floats(4097, 4, 2, 64) ||
        wick_rocm_attention_paged_scratch_floats(4, 5, 2, 64) || wick_rocm_attention_paged_scratch_floats(4, 0, 2, 64) ||
        wick_rocm_attention_paged_scratch_floats(4, 4, 2, 65) || !wick_rocm_attention_paged_scratch_floats(4096, 64, 1, 256) ||
        wick_rocm_attention_paged_scratch_floats(1, 4, 2, 64) != wick_rocm_attention_paged_scratch_floats(4096, 4, 2, 64))
        failures++, std::printf("scratch of attention\n");
    wick_rocm_kv_pages p = good.pages;
    // each of a step's copies, each of a pool's pages moved, and a word a page behind them
    if (wick_rocm_kv_pages_moves_words(nullptr) || wick_rocm_kv_pages_moves_words(&p) < 4 + 4 * 10 + 20) failures++, std::printf("words of moves\n");
    p.n_seqs = 4000;
    if (wick_rocm_kv_pages_moves_words(&p) < 4 + 4 * 4000 + 20) failures++, std::printf("words of many sequences' moves\n");
    p.page_rows = 17;
    if (wick_rocm_kv_pages_moves_words(&p)) failures++, std::printf("words of no pool\n");
    for (void* x : d) wick_rocm_buffer_free(ctx, x);
    wick_rocm_ctx_destroy(ctx);
    return failures ? 1 : 0;
}
