// A token's attention over no row of a 4-bit cache: zeros for heads that there can be, a refusal for others, on a runtime that only pretends (fake_hip.h).
#include <cstdint>
#include <cstdio>
#include <cstdlib>

#include "../../include/wick_rocm.h"
#include "../../include/wick_rocm_lfm2.h"
#include "fake_hip.h"

int main() {
    wick_rocm_ctx* ctx = nullptr;
    if (wick_rocm_ctx_create(0, &ctx) != WICK_ROCM_OK) std::abort();
    void* d[5];
    for (void*& p : d)
        if (wick_rocm_buffer_alloc(ctx, 1u << 16, &p) != WICK_ROCM_OK) std::abort();
    int failures = 0;
    const struct {
        uint32_t heads, n_kv;
        int want;
    } cases[] = {{4, 2, WICK_ROCM_OK}, {0, 2, WICK_ROCM_ERR_BAD_SHAPE}, {5, 2, WICK_ROCM_ERR_BAD_SHAPE}, {1, 2, WICK_ROCM_ERR_BAD_SHAPE}, {8, 8, WICK_ROCM_OK}};
    for (const auto& c : cases)
        for (const uint32_t seq_len : {0u, 7u}) {
            const long before = fake_hip::launches;
            const int rc = wick_rocm_attention_decode_q4(ctx, (float*)d[0], d[1], d[2], (float*)d[3], nullptr, (float*)d[4], seq_len, nullptr, 64, c.heads, c.n_kv, 64);
            if (rc != c.want || (fake_hip::launches > before) != (c.want == WICK_ROCM_OK))
                failures++, std::printf("%u heads over %u, %u rows: status %d, %ld launches\n", c.heads, c.n_kv, seq_len, rc, fake_hip::launches - before);
        }
    for (void* p : d) wick_rocm_buffer_free(ctx, p);
    wick_rocm_ctx_destroy(ctx);
    return failures ? 1 : 0;
}
