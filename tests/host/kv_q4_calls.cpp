// Calls on 4-bit KV caches that have to be refused, on a runtime that only pretends (fake_hip.h): each answers with its status and a message,
// nothing is enqueued, and the call with that one thing put right goes through.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <string>
#include <vector>

#include "../../include/wick_rocm.h"
#include "../../include/wick_rocm_lfm2.h"
#include "fake_hip.h"

namespace {

int failures = 0;

struct Call {  // every argument of the five calls; a case changes one or two
    const void *k = nullptr, *v = nullptr, *q = nullptr;
    void *k_cache = nullptr, *v_cache = nullptr, *out = nullptr, *weights = nullptr, *scratch = nullptr, *kept = nullptr;
    uint32_t kv_stride = 128, q_stride = 256, out_stride = 256, row = 10, n = 4, max_seq = 64, n_heads = 4, n_kv = 2, hd = 64, seq = 50, keep = 4, recent = 8, drop = 20;
};

int append(wick_rocm_ctx* c, const Call& a) {
    return wick_rocm_kv_q4_append(c, (const float*)a.k, (const float*)a.v, a.kv_stride, a.k_cache, a.v_cache, a.row, nullptr, a.n, a.max_seq, a.n_kv, a.hd);
}
int read(wick_rocm_ctx* c, const Call& a) { return wick_rocm_kv_q4_read(c, a.k_cache, (float*)a.out, a.out_stride, a.row, a.n, a.max_seq, a.n_kv, a.hd); }
int decode(wick_rocm_ctx* c, const Call& a) {
    return wick_rocm_attention_decode_q4(c, (const float*)a.q, a.k_cache, a.v_cache, (float*)a.out, (float*)a.weights, (float*)a.scratch, a.seq, nullptr, a.max_seq,
                                         a.n_heads, a.n_kv, a.hd);
}
int prefill(wick_rocm_ctx* c, const Call& a) {
    return wick_rocm_attention_prefill_q4(c, (const float*)a.q, a.q_stride, a.k_cache, a.v_cache, (float*)a.out, a.out_stride, (float*)a.weights,
                                          (float*)a.scratch, a.row, a.n, a.max_seq, a.n_heads, a.n_kv, a.hd);
}
int evict(wick_rocm_ctx* c, const Call& a) {
    return wick_rocm_kv_q4_evict(c, a.k_cache, a.v_cache, (float*)a.weights, (uint32_t*)a.kept, (float*)a.scratch, a.seq, a.keep, a.recent, a.drop, a.max_seq,
                                 a.n_kv, a.hd);
}

}  // namespace

int main() {
    wick_rocm_ctx* ctx = nullptr;
    if (wick_rocm_ctx_create(0, &ctx) != WICK_ROCM_OK) std::abort();
    Call good;
    void* d[9];
    for (void*& p : d)
        if (wick_rocm_buffer_alloc(ctx, 1u << 20, &p) != WICK_ROCM_OK) std::abort();
    good.k = d[0], good.v = d[1], good.q = d[2], good.k_cache = d[3], good.v_cache = d[4], good.out = d[5], good.weights = d[6], good.scratch = d[7], good.kept = d[8];
    const auto off = [](const void* p, int n) { return (void*)((char*)p + n); };
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
    const std::vector<Wrong> shape = {
        {"head_dim 0", kShape, [](Call& a) { a.hd = 0; }},          {"head_dim 48", kShape, [](Call& a) { a.hd = 48; }},
        {"head_dim 96", kShape, [](Call& a) { a.hd = 96; }},        {"head_dim 512", kShape, [](Call& a) { a.hd = 512; }},
        {"no KV heads", kShape, [](Call& a) { a.n_kv = 0; }},       {"too many KV heads", kShape, [](Call& a) { a.n_kv = 1u << 16; }},
        {"no rows", kShape, [](Call& a) { a.max_seq = 0; }},        {"too many rows", kShape, [](Call& a) { a.max_seq = (1u << 24) + 1; }},
    };
    const auto with = [&](std::vector<Wrong> more) {
        more.insert(more.end(), shape.begin(), shape.end());
        return more;
    };
    each("append", append, with({
        {"no keys", kArg, [](Call& a) { a.k = nullptr; }},
        {"no values", kArg, [](Call& a) { a.v = nullptr; }},
        {"no key cache", kArg, [](Call& a) { a.k_cache = nullptr; }},
        {"no value cache", kArg, [](Call& a) { a.v_cache = nullptr; }},
        {"short stride", kShape, [](Call& a) { a.kv_stride = 124; }},
        {"odd stride", kShape, [](Call& a) { a.kv_stride = 130; }},
        {"keys off", kArg, [&](Call& a) { a.k = off(a.k, 4); }},
        {"values off", kArg, [&](Call& a) { a.v = off(a.v, 8); }},
        {"cache off", kArg, [&](Call& a) { a.v_cache = off(a.v_cache, 8); }},
        {"one cache", kArg, [](Call& a) { a.v_cache = a.k_cache; }},
        {"rows past the end", kArg, [](Call& a) { a.row = 61; }},
        {"rows past 2^32", kArg, [](Call& a) { a.row = 4294967295u; }},
        {"more rows than there are", kArg, [](Call& a) { a.n = 65; }},
    }));
    each("read", read, with({
        {"no cache", kArg, [](Call& a) { a.k_cache = nullptr; }},
        {"no output", kArg, [](Call& a) { a.out = nullptr; }},
        {"short stride", kShape, [](Call& a) { a.out_stride = 124; }},
        {"odd stride", kShape, [](Call& a) { a.out_stride = 129; }},
        {"output off", kArg, [&](Call& a) { a.out = off(a.out, 4); }},
        {"rows past the end", kArg, [](Call& a) { a.row = 61; }},
        {"rows past 2^32", kArg, [](Call& a) { a.row = 4294967294u; }},
    }));
    const std::vector<Wrong> attention = with({
        {"no queries", kArg, [](Call& a) { a.q = nullptr; }},
        {"no key cache", kArg, [](Call& a) { a.k_cache = nullptr; }},
        {"no value cache", kArg, [](Call& a) { a.v_cache = nullptr; }},
        {"no output", kArg, [](Call& a) { a.out = nullptr; }},
        {"weights without scratch", kArg, [](Call& a) { a.scratch = nullptr; }},
        {"no heads", kShape, [](Call& a) { a.n_heads = 0; }},
        {"heads that no KV head divides", kShape, [](Call& a) { a.n_heads = 5, a.q_stride = a.out_stride = 320; }},
        {"queries off", kArg, [&](Call& a) { a.q = off(a.q, 4); }},
        {"output off", kArg, [&](Call& a) { a.out = off(a.out, 12); }},
        {"key cache off", kArg, [&](Call& a) { a.k_cache = off(a.k_cache, 2); }},
        {"value cache off", kArg, [&](Call& a) { a.v_cache = off(a.v_cache, 8); }},
        {"scratch off", kArg, [&](Call& a) { a.scratch = off(a.scratch, 4); }},
        {"weights off", kArg, [&](Call& a) { a.weights = off(a.weights, 2); }},
        {"weights and the output over the queries", kArg, [](Call& a) { a.q = a.out; }},
    });
    auto one = attention, many = attention;
    one.push_back({"rows past the end", kArg, [](Call& a) { a.seq = 65; }});
    one.push_back({"heads past 2^32", kShape, [](Call& a) { a.n_heads = 1u << 26; }});
    one.push_back({"nothing to write zeros to", kArg, [](Call& a) { a.seq = 0, a.out = nullptr; }});
    each("decode", decode, one);
    many.push_back({"rows past the end", kArg, [](Call& a) { a.row = 61; }});
    many.push_back({"rows past 2^32", kArg, [](Call& a) { a.row = 4294967295u; }});
    many.push_back({"short stride of queries", kShape, [](Call& a) { a.q_stride = 252; }});
    many.push_back({"odd stride of queries", kShape, [](Call& a) { a.q_stride = 258; }});
    many.push_back({"short stride of the output", kShape, [](Call& a) { a.out_stride = 128; }});
    many.push_back({"odd stride of the output", kShape, [](Call& a) { a.out_stride = 257; }});
    each("prefill", prefill, many);
    each("evict", evict, with({
        {"no key cache", kArg, [](Call& a) { a.k_cache = nullptr; }},
        {"no value cache", kArg, [](Call& a) { a.v_cache = nullptr; }},
        {"one cache", kArg, [](Call& a) { a.v_cache = a.k_cache; }},
        {"no weights", kArg, [](Call& a) { a.weights = nullptr; }},
        {"no room for the rows", kArg, [](Call& a) { a.kept = nullptr; }},
        {"nothing dropped", kArg, [](Call& a) { a.drop = 0; }},
        {"more dropped than may go", kArg, [](Call& a) { a.drop = 39; }},
        {"sums past 2^32", kArg, [](Call& a) { a.keep = 4294967290u; }},
        {"rows past the end", kArg, [](Call& a) { a.seq = 65; }},
        {"cache off", kArg, [&](Call& a) { a.k_cache = off(a.k_cache, 4); }},
        {"weights off", kArg, [&](Call& a) { a.weights = off(a.weights, 1); }},
        {"rows off", kArg, [&](Call& a) { a.kept = off(a.kept, 2); }},
        {"no scratch", kArg, [](Call& a) { a.scratch = nullptr; }},
        {"scratch off", kArg, [&](Call& a) { a.scratch = off(a.scratch, 8); }},
    }));
    // what needs no launch
    Call none = good;
    none.n = 0;
    const long before = fake_hip::launches;
    if (append(ctx, none) || read(ctx, none) || prefill(ctx, none) || fake_hip::launches != before) failures++, std::printf("no tokens\n");
    if (wick_rocm_kv_q4_bytes(100, 3, 64) != 100 * 3 * 36 || wick_rocm_kv_q4_bytes(100, 3, 48) || wick_rocm_kv_q4_bytes(0, 3, 64) ||
        wick_rocm_kv_q4_bytes(1u << 24, 8, 256) != (size_t)8 * 144 << 24 || wick_rocm_kv_q4_bytes((1u << 24) + 1, 8, 256))
        failures++, std::printf("bytes\n");
    // the scratch of many tokens serves fewer
    for (uint32_t hd : {32u, 64u, 128u, 256u})
        for (uint32_t heads : {1u, 8u, 32u})
            for (int weights : {0, 1}) {
                size_t most = 0;
                for (uint32_t n = 1; n < 5000; n = n < 100 ? n + 1 : n * 9 / 8) {
                    const size_t floats = wick_rocm_attention_q4_scratch_floats(n, 4096, 4 * heads, heads, hd, weights);
                    if (floats < most || floats > (64u << 20)) failures++, std::printf("scratch of %u tokens, %u heads of %u: %zu\n", n, heads, hd, floats);
                    most = floats;
                }
            }
    // a token's state of every head, however many
    if (wick_rocm_attention_q4_scratch_floats(1, 2, 66000, 33000, 32, 1) < (size_t)66000 * (32 + 4 + 2 + 2)) failures++, std::printf("scratch of 66000 heads\n");
    for (void* p : d) wick_rocm_buffer_free(ctx, p);
    wick_rocm_ctx_destroy(ctx);
    return failures ? 1 : 0;
}
