// Attention over a cache of fp8_e4m3 codes (kernels: hf_kv_attend.h, hf_kv_block.h).
#include "hf_kv_block.h"

void hf_launch_kv_attend_fp8_e4m3(const hf_kv_attend_args& a, int dtype, int tile_rows,
                                hipStream_t st) {
    if (dtype == HF_DT_BF16) kv_launch_dim<HF_DT_BF16, HF_KV_FP8_E4M3>(a, tile_rows, st);
    else kv_launch_dim<HF_DT_FP16, HF_KV_FP8_E4M3>(a, tile_rows, st);
}
