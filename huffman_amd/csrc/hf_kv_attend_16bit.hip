// Attention over a cache of 16-bit values (kernels: hf_kv_attend.h, hf_kv_block.h), and the choice of the kernel.
#include "hf_kv_block.h"

void hf_launch_kv_attend_fp8_e4m3(const hf_kv_attend_args&, int, int, hipStream_t);
void hf_launch_kv_attend_fp8_e5m2(const hf_kv_attend_args&, int, int, hipStream_t);
void hf_launch_kv_attend_fp4_e2m1(const hf_kv_attend_args&, int, int, hipStream_t);

// Rows of a tile: the rows a sequence has at most, so that a small call's products are not mostly
// empty, up to four wavefronts of 32.
int hf_kv_attend_tile_rows(uint32_t max_q, uint32_t per, uint32_t head_dim) {
    const uint64_t rows = (uint64_t)max_q * per;
    if (rows <= 16) return 16;
    return rows <= 32 ? 32 : rows <= 64 ? 64 : rows <= 128 || head_dim > 128 ? 128 : 256;
}

void hf_launch_kv_attend(const hf_kv_attend_args& a, int dtype, int format, int tile_rows,
                         hipStream_t st) {
    switch (format) {
        case HF_KV_BF16: kv_launch_dim<HF_DT_BF16, HF_KV_BF16>(a, tile_rows, st); break;
        case HF_KV_FP16: kv_launch_dim<HF_DT_FP16, HF_KV_FP16>(a, tile_rows, st); break;
        case HF_KV_FP8_E4M3: hf_launch_kv_attend_fp8_e4m3(a, dtype, tile_rows, st); break;
        case HF_KV_FP8_E5M2: hf_launch_kv_attend_fp8_e5m2(a, dtype, tile_rows, st); break;
        case HF_KV_FP4_E2M1: hf_launch_kv_attend_fp4_e2m1(a, dtype, tile_rows, st); break;
        default: break;
    }
}
