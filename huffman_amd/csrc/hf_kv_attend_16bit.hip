// Attention over a cache of 16-bit values (kernels: hf_kv_attend.h, hf_kv_block.h), and the choice of the kernel.
#include "hf_kv_block.h"

void hf_launch_kv_attend_fp8_e4m3(const hf_kv_attend_args&, int, int, hipStream_t);
void hf_launch_kv_attend_fp8_e5m2(const hf_kv_attend_args&, int, int, hipStream_t);
void hf_launch_kv_attend_fp4_e2m1(const hf_kv_attend_args&, int, int, hipStream_t);

// Rows of a tile, by the rows a sequence has at most.  Measured (us; 8 cache heads x 4, head_dim 128,
// fp8, contexts of about 5000) with tiles of 16 / 64 / 128 / 256: 32 sequences of 20 rows 131 / 104 /
// 135 / 313, of 64 rows 226 / 122 / 158 / 332; 16 of 68 rows 141 / 98 / 78 / 120, of 128 rows 204 /
// 115 / 94 / 145, of 160 rows 292 / 186 / 147 / 137; 64 sequences of 4 rows 155 / 201 / 271 / -.
// A padded head_dim of 256 fills the registers of the 128-row kernel, which is the fastest from 8
// rows (172 against 204 with 16) to 64 (77 against 111 with 64, 163 with 16): it has that one only.
int hf_kv_attend_tile_rows(uint32_t max_q, uint32_t per, uint32_t head_dim) {
    const uint64_t rows = (uint64_t)max_q * per;
    if (head_dim > 128) return 128;
    return rows <= 16 ? 16 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
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
