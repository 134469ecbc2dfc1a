// What the launches of attention over 4-bit caches leave in the scratch, by the grids that they are launched with (fake_hip.h), against what
// wick_rocm_attention_q4_scratch_floats asks for: over all head sizes, few and many heads, short and long prompts and caches.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <string>

#include "../../include/wick_rocm.h"
#include "../../include/wick_rocm_lfm2.h"
#include "fake_hip.h"

int main() {
    wick_rocm_ctx* ctx = nullptr;
    if (wick_rocm_ctx_create(0, &ctx) != WICK_ROCM_OK) std::abort();
    void* d[7];
    for (void*& p : d)
        if (wick_rocm_buffer_alloc(ctx, 4096, &p) != WICK_ROCM_OK) std::abort();
    int failures = 0;
    long most_splits = 0, split = 0, shared = 0, calls = 0;
    for (const uint32_t hd : {32u, 64u, 128u, 256u})
        for (const uint32_t n_kv : {1u, 2u, 3u, 4u, 6u, 8u, 33u, 600u})
            for (const uint32_t group : {1u, 2u, 3u, 4u, 8u, 16u, 17u, 80u})
                for (uint32_t n = 1; n <= 5000; n = n < 4 ? n + 1 : n * 13 / 8)
                    for (const uint32_t pos0 : {0u, 60u, 700u, 5000u, 40000u, 170000u})
                        for (const int weights : {0, 1}) {
                            const uint32_t n_heads = n_kv * group, max_seq = pos0 + n + 100, rows = n * group, stride = n_heads * hd;
                            fake_hip::kernels();
                            const int rc = n == 1 ? wick_rocm_attention_decode_q4(ctx, (float*)d[0], d[1], d[2], (float*)d[3], weights ? (float*)d[4] : nullptr,
                                                                                  (float*)d[5], pos0 + 1, nullptr, max_seq, n_heads, n_kv, hd)
                                                  : wick_rocm_attention_prefill_q4(ctx, (float*)d[0], stride, d[1], d[2], (float*)d[3], stride,
                                                                                   weights ? (float*)d[4] : nullptr, (float*)d[5], pos0, n, max_seq, n_heads, n_kv, hd);
                            const size_t records = wick_rocm_attention_q4_scratch_floats(n, max_seq, n_heads, n_kv, hd, 0) / (hd + 4);
                            const size_t behind = wick_rocm_attention_q4_scratch_floats(n, max_seq, n_heads, n_kv, hd, 1) - records * (hd + 4);
                            size_t splits = 0, sums = 0;
                            bool merged = false, added = false;
                            for (const std::string& k : fake_hip::kernels()) {
                                const size_t grid = std::strtoul(k.c_str() + k.rfind('(') + 1, nullptr, 10);
                                const char* const args = k.c_str() + k.find('<') + 1;
                                const auto is = [&](const char* name) { return k.find(name) != std::string::npos; };
                                if (is("attention_q4_few_kernel")) splits = grid / (n_kv * ((rows + 15) / 16));
                                if (is("attention_q4_kernel")) {
                                    const size_t wg_rows = 32 * std::strtoul(std::string(args).substr(std::string(args).find(',') + 1).c_str(), nullptr, 10);
                                    splits = grid / (n_kv * ((rows + wg_rows - 1) / wg_rows));
                                }
                                if (is("attention_q4_weights_kernel")) sums = grid * 128;
                                merged |= is("merge_kernel") || is("finish_kernel"), added |= is("add_weights_kernel");
                            }
                            calls++, split += merged, shared += added;
                            if (merged && (long)splits > most_splits) most_splits = (long)splits;
                            const bool fine = rc == WICK_ROCM_OK && splits >= 1 && (merged || splits == 1) && (!merged || (size_t)n * n_heads * splits <= records) &&
                                              (!added || 2 * (size_t)n * n_heads + sums <= behind);
                            if (!fine && failures++ < 20)
                                std::printf("%u tokens behind %u, %u heads over %u of %u, weights %d: status %d, %zu splits, %zu records, %zu sums in %zu\n", n, pos0, n_heads, n_kv,
                                            hd, weights, rc, splits, records, sums, behind);
                        }
    std::printf("%ld calls, %ld split (in %ld at the most), %ld with shares\n", calls, split, most_splits, shared);
    if (split < 1000 || shared < 1000 || most_splits < 65) failures++;
    for (void* p : d) wick_rocm_buffer_free(ctx, p);
    wick_rocm_ctx_destroy(ctx);
    return failures ? 1 : 0;
}
