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
// rows (172 against 204 with 16) to 64 (77 against 111 with 64, 163 with 16): it has that one only.  Below
// 8 rows it is slow: single tokens of 64 sequences of up to 8001 tokens, 4 cache heads of 160 to 256 in e4m3,
// take 515 to 540 us whether 1, 2 or 4 query heads share them, a quarter of the rate of 128 (88 to 90).
// The rule goes by the longest sequence of the call: a chunk of 1000 rows beside 63 single tokens takes
// 585 us in one call, 146 + 154 in two.
int hf_kv_attend_tile_rows(uint32_t max_q, uint32_t per, uint32_t head_dim) {
    const uint64_t rows = (uint64_t)max_q * per;
    if (head_dim > 128) return 128;
    return rows <= 16 ? 16 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
}

namespace {
// The cut of a call of many sequences (see kv_find), by one workgroup: the wavefronts of the attending
// kernels would each walk all the lists.  Decode (8 heads x 4, head_dim 128, e4m3) of 256 sequences of
// up to 512 tokens: 58 us with this launch, 69 without; of 1024: 230, 463; 4096 of up to 256: 617, 4541.
// (At 128 of up to 1024 it is not needed yet: 58 without it.)
constexpr int kPlanThreads = 1024;
__global__ __launch_bounds__(kPlanThreads) void hf_k_kv_plan(const hf_kv_attend_args a, const uint32_t tile_rows) {
    __shared__ float sums[2][kPlanThreads / 64];
    __shared__ uint32_t units[kPlanThreads / 64];
    const uint32_t batch = a.s.batch, wave = threadIdx.x >> 6;
    const bool lane0 = hf_lane() == 0;
    float work = 0.0f, tiles = 0.0f;
    for (uint64_t b = threadIdx.x; b < batch; b += kPlanThreads) {
        const kv_shape s = kv_shape_of(a, tile_rows, (uint32_t)b);
        work += (float)s.tiles * (float)s.steps;
        tiles += (float)s.tiles;
    }
    work = kv_wave_sum(work);
    tiles = kv_wave_sum(tiles);
    if (lane0) {
        sums[0][wave] = work;
        sums[1][wave] = tiles;
    }
    __syncthreads();
    work = tiles = 0.0f;
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        work += sums[0][w];
        tiles += sums[1][w];
    }
    kv_steps p(a, tile_rows, work, tiles);
    uint32_t total;
    int turn = 0;
    do {
        uint32_t mine = 0;
        for (uint64_t b = threadIdx.x; b < batch; b += kPlanThreads) {
            const kv_shape s = kv_shape_of(a, tile_rows, (uint32_t)b);
            mine += s.tiles * p.ranges(s);
        }
        mine = hf_wave_sum_u32(mine);
        __syncthreads();
        if (lane0) units[wave] = mine;
        __syncthreads();
        total = 0;
        for (int w = 0; w < kPlanThreads / 64; ++w) total += units[w];
    } while (p.raise(a, total, turn++));
    uint32_t before = 0;
    bool split = false;
    for (uint64_t b0 = 0; b0 < batch; b0 += kPlanThreads) {
        const uint64_t b = b0 + threadIdx.x;
        const kv_shape s = kv_shape_of(a, tile_rows, (uint32_t)(b < batch ? b : batch));
        const uint32_t ranges = p.ranges(s), own = s.tiles * ranges, incl = kv_wave_scan(own);
        __syncthreads();
        if (hf_lane() == 63) units[wave] = incl;
        __syncthreads();
        uint32_t first = before + incl - own;
        for (uint32_t w = 0; w < kPlanThreads / 64; ++w) {
            if (w < wave) first += units[w];
            before += units[w];
        }
        if (b < batch) *(hf_u32x4*)(a.plan + 4 * (int64_t)b) = hf_u32x4{first, s.tiles, ranges, s.steps};
        split = split || (s.tiles && ranges > 1);
    }
    split = __syncthreads_or(split) != 0;
    if (threadIdx.x == 0) {
        a.plan[4 * (int64_t)batch] = split;
        a.plan[4 * (int64_t)batch + 1] = total;
    }
}
}  // namespace

void hf_launch_kv_attend(const hf_kv_attend_args& a, int dtype, int format, int tile_rows,
                         hipStream_t st) {
    if (a.s.batch > HF_KV_OWN_CUT)
        hipLaunchKernelGGL(hf_k_kv_plan, dim3(1), dim3(kPlanThreads), 0, st, a, (uint32_t)tile_rows);
    switch (format) {
        case HF_KV_BF16: kv_launch_dim<HF_DT_BF16, HF_KV_BF16>(a, tile_rows, st); break;
        case HF_KV_FP16: kv_launch_dim<HF_DT_FP16, HF_KV_FP16>(a, tile_rows, st); break;
        case HF_KV_FP8_E4M3: hf_launch_kv_attend_fp8_e4m3(a, dtype, tile_rows, st); break;
        case HF_KV_FP8_E5M2: hf_launch_kv_attend_fp8_e5m2(a, dtype, tile_rows, st); break;
        case HF_KV_FP4_E2M1: hf_launch_kv_attend_fp4_e2m1(a, dtype, tile_rows, st); break;
        default: break;
    }
}
