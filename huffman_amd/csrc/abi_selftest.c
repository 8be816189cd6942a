/*
 * abi_selftest.c -- the host side of the C ABI under AddressSanitizer + UndefinedBehaviorSanitizer
 * (make -C huffman_amd/csrc sanitize-host).  It needs no GPU: it drives the entry points that are
 * host arithmetic and the argument checks every other entry point runs before its first HIP call.
 * With a GPU present hf_ctx_create succeeds and the context is destroyed again.
 */
#include <stdio.h>
#include <string.h>

#include "../../include/huffhip.h"

#define CHECK(cond)                                                          \
    do {                                                                     \
        if (!(cond)) {                                                       \
            fprintf(stderr, "abi selftest: %s failed, line %d\n", #cond, __LINE__); \
            return 1;                                                        \
        }                                                                    \
    } while (0)

int main(void) {
    CHECK(hf_abi_version() == HF_ABI_VERSION);
    for (int code = -12; code <= 1; ++code) CHECK(hf_error_string(code) != NULL);
    CHECK(hf_num_chunks(0) == 0 && hf_num_chunks(1) == 1 && hf_num_chunks(16385) == 2);
    CHECK(hf_payload_bound_words(16384) == 64ull * 129ull);

    /* TreeQualityAnalyzer and AdaptiveThreshold: host arithmetic over every width */
    uint64_t freq[256];
    uint8_t len[256];
    for (int i = 0; i < 256; ++i) {
        freq[i] = (uint64_t)(i * 2654435761u) >> 7;
        len[i] = (uint8_t)(1 + i % 16);
    }
    for (int W = 1; W <= 64; ++W) {
        uint16_t a, e, r;
        const int rc = hf_quality(NULL, freq, len, 256, W, &a, &e, &r);
        CHECK(rc == HF_OK || rc == HF_ERR_RANGE);
        hf_adaptive_config cfg;
        for (uint32_t ent = 0; ent < 0x80000u; ent += 0x3FFFu) {
            const int rc2 = hf_adaptive_threshold(ent, 256, W, &cfg);
            CHECK(rc2 == HF_OK || rc2 == HF_ERR_RANGE || (W < 2 && rc2 == HF_ERR_ARG));
        }
    }
    CHECK(hf_quality(NULL, NULL, len, 256, 32, NULL, NULL, NULL) == HF_ERR_ARG);
    CHECK(hf_adaptive_threshold(0, 256, 32, NULL) == HF_ERR_ARG);

    /* container planning: host arithmetic */
    hf_container_info info;
    for (uint64_t n = 0; n < 100000; n += 7777)
        for (int kind = 0; kind < 2; ++kind)
            for (int layout = 0; layout < 3; ++layout) {
                CHECK(hf_container_plan(n, layout, kind, n / 3, &info) == HF_OK);
                CHECK(info.total_bytes % 16 == 0 && info.off_payload % 16 == 0);
                CHECK(info.total_bytes >= info.off_payload + 16);
            }
    /* ... with a placement (wire format version 2): slotted streams carry a words array, paged
       streams with records carry no codebook section, paged streams without carry the one */
    for (uint64_t n = 0; n < 100000; n += 7777)
        for (int kind = 0; kind < 2; ++kind)
            for (int placement = 0; placement < 3; ++placement) {
                CHECK(hf_container_plan_placed(n, HF_LAYOUT_U8, kind, placement, n / 3, &info) == HF_OK);
                CHECK(info.placement == (uint32_t)placement && info.total_bytes % 16 == 0);
                CHECK((info.off_chunk_words != 0) == (placement == HF_PLACEMENT_SLOTTED));
                CHECK((info.off_codebook == 0) ==
                      (placement == HF_PLACEMENT_PAGED && kind == HF_CODEBOOK_PER_CHUNK));
            }
    CHECK(hf_container_plan_placed(1, 0, 0, 3, 1, &info) == HF_ERR_ARG);
    CHECK(hf_pages_bound_words(0) == 0 && hf_pages_bound_words(16385) == 2ull * hf_pages_bound_words(1));
    CHECK(hf_container_plan(1, 9, 0, 1, &info) == HF_ERR_ARG);
    CHECK(hf_container_plan(1, 0, 0, 1, NULL) == HF_ERR_ARG);

    /* every context-taking entry point rejects a null context before it touches HIP */
    CHECK(hf_flush(NULL) == HF_ERR_ARG && hf_sync(NULL) == HF_ERR_ARG);
    CHECK(hf_symbol_sort(NULL, freq, 256, freq, NULL) == HF_ERR_ARG);
    CHECK(hf_entropy(NULL, freq, 256, NULL, NULL) == HF_ERR_ARG);
    CHECK(hf_encode(NULL, NULL, 0, 0, NULL, NULL, NULL, 0, NULL, NULL) == HF_ERR_ARG);
    CHECK(hf_decode(NULL, NULL, 0, NULL, NULL, 0, 0, NULL, NULL, 0) == HF_ERR_ARG);
    CHECK(hf_decode_chunks_to(NULL, NULL, 0, NULL, NULL, 0, 0, NULL, NULL, NULL, 0, NULL, 0, 0) ==
          HF_ERR_ARG);
    CHECK(hf_last_hip_error(NULL) == 0);
    CHECK(hf_ctx_reserve(NULL, 0, HF_RESERVE_ALL) == HF_ERR_ARG);
    CHECK(hf_zero_dev(NULL, NULL, 0) == HF_ERR_ARG);
    CHECK(hf_symbol_stat_pages_dev(NULL, NULL, 0, 0, NULL, NULL) == HF_ERR_ARG);
    CHECK(hf_symbol_stat_allreduce(NULL, NULL, NULL) == HF_ERR_ARG);
    CHECK(hf_encode_pages(NULL, NULL, 0, 0, NULL, NULL, NULL, NULL, 0, NULL, NULL) == HF_ERR_ARG);
    CHECK(hf_encode_pages_shared(NULL, NULL, 0, 0, NULL, NULL, NULL, NULL, 0, NULL, NULL) == HF_ERR_ARG);
    CHECK(hf_decode_pages(NULL, NULL, 0, NULL, NULL, 0, 0, NULL, NULL, 0, NULL, 0, 0) == HF_ERR_ARG);
    CHECK(hf_decode_pages_shared(NULL, NULL, 0, NULL, NULL, 0, 0, NULL, NULL, NULL, 0, NULL, 0, 0) ==
          HF_ERR_ARG);
    CHECK(hf_page_codebook_download(NULL, NULL, 0, NULL, 0, NULL, NULL, NULL, NULL) == HF_ERR_ARG);
    CHECK(hf_system_codebook_chunks_static(NULL, NULL, 0, HF_MODE_HUFFMAN, 0, NULL) == HF_ERR_ARG);

    /* KV cache: the checks of every argument, strides and sizes at their ends among them (without a
       context each call ends in an error) */
    {
        static const int64_t strides[] = {0, 1, 127, 128, 1024, 1000, 1ll << 31, (1ll << 31) + 16, 1ll << 62, INT64_MAX,
                                          -1, -1024, INT64_MIN};
        static const uint32_t sizes[] = {0, 1, 7, 8, 32, 96, 256, 257, 65536, 0x7FFFFFFFu, 0x80000000u, 0xFFFFFFFFu};
        const int ns = sizeof strides / sizeof *strides, nz = sizeof sizes / sizeof *sizes;
        int32_t lists[64] = {0};
        char* const mem = (char*)(uintptr_t)4096; /* never followed */
        for (int what = 0; what < 15; ++what)
            for (int i = 0; i < (what < 6 ? ns : nz); ++i) {
                hf_kv_cache c = {mem, mem, (uint8_t*)mem, (uint8_t*)mem, 4, 16 * 1024, 1024, 128, 16, 8, 128, 128,
                                 HF_KV_FP8_E4M3, 0};
                hf_kv_batch b = {NULL, lists, lists + 8, 4, 4, 2, 2, 1};
                hf_kv_query q = {mem, mem, NULL, NULL, 4096, 128, 4096, 128, 32, 0, HF_DT_BF16, 0.1f};
                int64_t row = 1024, head = 128, path = 4;
                if (what == 0) c.page_stride = strides[i];
                if (what == 1) c.token_stride = c.head_stride = strides[i];
                if (what == 2) b.table_stride = strides[i];
                if (what == 3) q.q_row_stride = q.out_row_stride = row = strides[i];
                if (what == 4) q.q_head_stride = q.out_head_stride = head = strides[i];
                if (what == 5) path = strides[i];
                if (what == 6) c.n_pages = sizes[i];
                if (what == 7) c.page_size = sizes[i];
                if (what == 8) c.heads = sizes[i];
                if (what == 9) c.head_dim = sizes[i];
                if (what == 10) c.group = sizes[i];
                if (what == 11) c.format = sizes[i];
                if (what == 12) b.table_width = sizes[i];
                if (what == 13) {
                    b.batch = sizes[i];
                    b.d_cu_rows = lists + 16;
                }
                if (what == 14) q.q_heads = sizes[i];
                for (int dtype = -1; dtype < 4; ++dtype) {
                    CHECK(hf_kv_write(NULL, &c, &b, mem, mem, row, head, row, head, dtype) < 0);
                    CHECK(hf_kv_read(NULL, &c, &b, mem, mem, row, head, row, head, dtype) < 0);
                }
                CHECK(hf_kv_attend(NULL, &c, &b, &q, mem, 1u << 20) < 0);
                CHECK(hf_kv_attend_work_bytes(NULL, &c, &b, q.q_heads) == 0);
                CHECK(hf_kv_keep(NULL, &c, &b, lists + 32, path, 3, lists + 40, lists + 48) < 0);
            }
        CHECK(hf_kv_write(NULL, NULL, NULL, NULL, NULL, 0, 0, 0, 0, 0) == HF_ERR_ARG);
        CHECK(hf_kv_keep(NULL, NULL, NULL, NULL, 0, 0, NULL, NULL) == HF_ERR_ARG);
    }

    hf_ctx* ctx = NULL;
    const int rc = hf_ctx_create(&ctx, 0, NULL);
    if (rc == HF_OK) {
        CHECK(ctx != NULL);
        CHECK(hf_flush(ctx) == HF_OK);
        CHECK(hf_ctx_reserve(ctx, 1u << 20, HF_RESERVE_ALL) == HF_OK);
        CHECK(hf_ctx_reserve(ctx, 1, 0x80u) == HF_ERR_ARG);
        CHECK(hf_zero_dev(ctx, NULL, 0) == HF_OK);
        CHECK(hf_symbol_stat_allreduce(ctx, NULL, NULL) == HF_ERR_ARG);
        CHECK(hf_ctx_destroy(ctx) == HF_OK);
    } else {
        CHECK(rc == HF_ERR_HIP && ctx == NULL);  /* no GPU here: a clean error, no fallback */
    }
    puts("abi selftest ok");
    return 0;
}
