// Attention of a sequence's last rows over its quantised pages: the kernel, as a template over the
// type of the queries, the format of the cache and the padded head dimension DP.
//
//   o_i = sum_t p_it v_t / sum_t p_it,   p_it = exp(scale q_i . k_t - m_i),   t over what i may see
//
// One unit = 16 rows (tokens x query heads of one cache head of one sequence) against one range
// of the sequence's tokens; a workgroup of four wavefronts takes a unit, its wavefronts taking the
// unit's tokens 32 at a time in turn, each with its own running maximum and sum, and joins them
// through LDS at the end.  There is no LDS and no barrier in the loop: the products are arranged so
// that every operand is where it is needed,
//
//   S^T = K Q^T   A = 16 tokens of K, B = 16 rows of Q: a lane gets, of row lane % 16, four tokens
//   O^T = V^T P^T B = P^T needs, of row lane % 16, eight tokens in the lane: those it has from two
//                 products S^T, since the order of the tokens inside a product is free as long as A
//                 and B agree; A = V^T needs eight tokens of one d in a lane: a lane loads its
//                 DP / 16 neighbouring d of eight tokens and pairs them up with byte permutes
//
// and the d that a lane holds are free in the same way (any order that Q and K, or V and O, share).
// Codes become 16-bit operands with the conversions that apply a power-of-two scale for nothing, so
// scales may differ by token and by group of d.  The sums of S and O and the statistics are kept in
// 32 bits; p is rounded to the type of the queries for the second product, as the codes' values are
// exact in it (fp16: unless they leave its range, as reading the cache in fp16 would).  O is divided
// by the sum of the p as rounded, one more product, with ones: what rounding p does to the weights
// then cancels where few tokens carry a row (a row of one token gives that token's values exactly).
// The logarithm of the sum is taken from the p in 32 bits.
#pragma once

#include "hf_kv.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

typedef __attribute__((address_space(4))) int32_t kv_const_i32;
constexpr int kWaves = 4;
constexpr int kStep = 32;  // tokens a wavefront takes at a time

template <int QT>
struct kv_type;
template <>
struct kv_type<HF_DT_BF16> {
    // bit patterns: exponent field of both halves, its lowest bit, one
    static constexpr uint32_t expo = 0x7F807F80u, unit = 0x00800080u, one = 0x3F80u;
    static constexpr float off = 0.0f, rise = 8.0f;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
    }
    static __device__ __forceinline__ f32x4 mma(hf_u32x4 a, hf_u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <>
struct kv_type<HF_DT_FP16> {
    static constexpr uint32_t expo = 0x7C007C00u, unit = 0x04000400u, one = 0x3C00u;
    // p is held 2^7 up and may rise by 2^8 more, to 2^15: a p that fp16 flushes is below 2^-31 of
    // the largest, so even a long row of such tokens beside one large one keeps its weight
    static constexpr float off = 7.0f, rise = 8.0f;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
    }
    static __device__ __forceinline__ f32x4 mma(hf_u32x4 a, hf_u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};

// Two codes (elements 2i and 2i + 1 of the word) times the scale, as 16-bit values.
template <int QT, int FMT, int I>
__device__ __forceinline__ uint32_t kv_pair(const uint32_t w, const float s) {
    if constexpr (FMT == HF_KV_FP8_E4M3) {
        if constexpr (QT == HF_DT_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, I == 1));
        else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, I == 1));
    } else if constexpr (FMT == HF_KV_FP8_E5M2) {
        if constexpr (QT == HF_DT_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, s, I == 1));
        else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w, s, I == 1));
    } else if constexpr (FMT == HF_KV_FP4_E2M1) {
        if constexpr (QT == HF_DT_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, I));
        else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, I));
    } else {
        return w;  // two 16-bit values
    }
}

// Bytes from global memory into consecutive 32-bit words (2 bytes: the low half of one).
template <int BYTES>
struct kv_raw {
    uint32_t w[BYTES >= 4 ? BYTES / 4 : 1];
    __device__ __forceinline__ void load(const hf_g8* p) {
        if constexpr (BYTES == 2) {
            w[0] = *(__attribute__((address_space(1))) const uint16_t*)p;
        } else if constexpr (BYTES == 4) {
            w[0] = *(__attribute__((address_space(1))) const uint32_t*)p;
        } else if constexpr (BYTES == 8) {
            const hf_u32x2 a = *(const hf_gmem_u32x2*)p;
            w[0] = a.x;
            w[1] = a.y;
        } else {
#pragma unroll
            for (int i = 0; i < BYTES / 16; ++i) {
                const hf_u32x4 a = *(const hf_gmem_u32x4*)(p + 16 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) w[4 * i + j] = a[j];
            }
        }
    }
};

template <int FMT>
constexpr int kv_bits() {
    return FMT == HF_KV_FP4_E2M1 ? 4 : (FMT == HF_KV_FP8_E4M3 || FMT == HF_KV_FP8_E5M2) ? 8 : 16;
}

__device__ __forceinline__ float kv_row_max(float a) {  // over the lanes of a row: l, l ^ 16, l ^ 32, l ^ 48
    a = fmaxf(a, __shfl_xor(a, 16));
    return fmaxf(a, __shfl_xor(a, 32));
}
__device__ __forceinline__ float kv_row_sum(float a) {
    a += __shfl_xor(a, 16);
    return a + __shfl_xor(a, 32);
}

// Exponent of a weight, p = exp2(score x scale + nm).  Fused, the error of scale x maximum is the same factor
// for the whole row; where it could pass 1 / 256 of a power of two (kv_huge, of a wavefront's rows), the
// products are rounded first, as the maximum's was.  Whether a score calls for a new maximum is decided on
// this very number: from 2^25 on the two forms differ by a power of two and more, and a weight that passed
// as the one could leave fp16's range as the other.
__device__ __forceinline__ float kv_exponent(const float score, const float scale, const float nm, const bool huge) {
    return huge ? score * scale + nm : __builtin_fmaf(score, scale, nm);
}
__device__ __forceinline__ bool kv_huge(const float nm) {
    return __ballot(fabsf(nm) > 65536.0f && nm != 3.402823466e38f) != 0;
}

// Has the values' loads waited for here: left to their first use, which is in a loop that issues
// loads of its own, the wait there would be for those too, in every turn.
template <int N>
__device__ __forceinline__ void kv_arrived(hf_u32x4 (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(x[i]));
}

// ---- the cut of a call into units ---------------------------------------------------------------
// The cut is made on the device from the call's own lengths, so a captured call follows lengths that
// change between replays and a ragged batch is cut evenly.  All sequences' steps (32 tokens)
// times their row tiles are summed and divided by the units aimed at; a sequence has as many equal
// ranges as it needs for about that many steps.  Tiles of 16 rows leave little behind per unit (a
// range's partial outputs), so their units are many and small.  Larger tiles leave as much as they
// read, so there are as many units as run at once: where the tiles alone are fewer than half of
// that, the steps of a range are raised until the units do not start a second round; where they are
// not, a range may be a quarter longer before it is cut.
// Units of a sequence are numbered range by range, in it by cache head, in it by row tile, so that
// the tiles that read the same tokens are neighbours; and since consecutive workgroups go to the
// eight XCDs in turn, each with an L2 of its own, XCD x takes the x-th eighth of the units.
// Up to HF_KV_OWN_CUT sequences every wavefront makes the whole cut by itself, a sequence to a lane, and
// workgroup 0 leaves it in memory for the kernel that joins the ranges.  More sequences are cut by
// one workgroup in a launch in front (hf_k_kv_plan), and a unit is searched in what it left.
struct kv_cut {
    uint32_t unit, b, n_before;  // unit; its sequence; units of the sequences before that
    uint32_t tiles, ranges, steps_each;
};
struct kv_shape {
    uint32_t tiles, steps;
};
__device__ __forceinline__ kv_shape kv_shape_of(const hf_kv_attend_args& a, const uint32_t tile_rows, const uint32_t b) {
    kv_shape s = {0, 0};
    if (b < a.s.batch) {
        const hf_kv_seq q = hf_kv_sequence(a.s, b, a.c.page_shift);
        if (q.bad) atomicOr(a.err, HF_KERR_CORRUPT);
        s.tiles = q.n > 0 ? a.c.heads * (((uint32_t)q.n * a.per + tile_rows - 1u) / tile_rows) : 0u;
        s.steps = ((uint32_t)q.len + kStep - 1u) / kStep;
    }
    return s;
}
__device__ __forceinline__ uint32_t kv_div_up(const uint32_t x, const uint32_t y) { return (x + y - 1u) / y; }
__device__ __forceinline__ uint32_t kv_wave_scan(const uint32_t v) {  // inclusive
    uint32_t incl = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t up = __shfl_up(incl, o);
        if (hf_lane() >= o) incl += up;
    }
    return incl;
}
__device__ __forceinline__ float kv_wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
struct kv_steps {
    uint32_t each, slack;  // steps of a range, those let pass
    bool fit;              // the units are to be no more than aimed at
    // (the sums of tiles x steps and of tiles decide nothing but the cut, and all who make it have the
    // same ones: floats do)
    __device__ __forceinline__ kv_steps(const hf_kv_attend_args& a, const uint32_t tile_rows, const float work,
                                        const float tiles) {
        each = max((uint32_t)(work / (float)a.target * 1.0001f) + 1u, a.min_steps);
        fit = tile_rows > 16 && 2.0f * tiles <= (float)a.target;
        slack = tile_rows > 16 && !fit ? each / 4u : 0u;
    }
    __device__ __forceinline__ uint32_t ranges(const kv_shape& s) const {
        return s.steps <= each + slack ? 1u : kv_div_up(s.steps - slack, each);
    }
    // whether units were too many and are to be counted again
    __device__ __forceinline__ bool raise(const hf_kv_attend_args& a, const uint32_t units, const int turn) {
        if (!fit || turn == 8 || units <= a.target) return false;
        each += max(1u, each / 16u);
        return true;
    }
};
struct kv_plan_dev {
    kv_steps steps;
    uint32_t total;  // units
    kv_shape first;  // of the lane's sequence among the first 64: most calls have no more
};
__device__ __forceinline__ kv_plan_dev kv_plan_now(const hf_kv_attend_args& a, const uint32_t tile_rows) {
    const kv_shape lane = kv_shape_of(a, tile_rows, hf_lane());
    float work = (float)lane.tiles * (float)lane.steps, tiles = (float)lane.tiles;
    for (uint32_t b0 = 64; b0 < a.s.batch; b0 += 64) {
        const kv_shape s = kv_shape_of(a, tile_rows, b0 + hf_lane());
        work += (float)s.tiles * (float)s.steps;
        tiles += (float)s.tiles;
    }
    kv_plan_dev p = {kv_steps(a, tile_rows, kv_wave_sum(work), kv_wave_sum(tiles)), 0u, lane};
    int turn = 0;
    do {
        uint32_t total = p.first.tiles * p.steps.ranges(p.first);
        for (uint32_t b0 = 64; b0 < a.s.batch; b0 += 64) {
            const kv_shape s = kv_shape_of(a, tile_rows, b0 + hf_lane());
            total += s.tiles * p.steps.ranges(s);
        }
        p.total = hf_wave_sum_u32(total);
    } while (p.steps.raise(a, p.total, turn++));
    return p;
}
// Walks the sequences 64 at a time; `pick` sees a lane's sequence, its shape and ranges and the units
// before it, and says whether it is the one.
template <typename F>
__device__ __forceinline__ bool kv_walk(const hf_kv_attend_args& a, const uint32_t tile_rows, const kv_plan_dev& p,
                                        F&& pick, kv_cut& cut) {
    uint32_t before = 0;
    for (uint32_t b0 = 0; b0 < a.s.batch; b0 += 64) {
        const uint32_t b = b0 + hf_lane();
        kv_shape s = p.first;
        if (b0) s = kv_shape_of(a, tile_rows, b);
        const uint32_t ranges = p.steps.ranges(s);
        const uint32_t own = s.tiles * ranges, incl = kv_wave_scan(own);
        const unsigned long long hit = __ballot(pick(b, s, ranges, before + incl - own));
        if (hit) {
            const int l = __ffsll((unsigned long long)hit) - 1;
            cut.b = b0 + l;
            cut.n_before = before + __builtin_amdgcn_readlane(incl - own, l);
            cut.tiles = __builtin_amdgcn_readlane(s.tiles, l);
            cut.ranges = __builtin_amdgcn_readlane(ranges, l);
            const uint32_t steps = __builtin_amdgcn_readlane(s.steps, l);
            cut.steps_each = (kv_div_up(steps, cut.ranges) + kWaves - 1u) / kWaves * kWaves;
            return true;
        }
        before += __builtin_amdgcn_readlane(incl, 63);
    }
    return false;
}
// The unit of this workgroup among `total`; false: none.
__device__ __forceinline__ bool kv_unit_of(const hf_kv_attend_args& a, const uint32_t total, uint32_t& unit) {
    // (offsets that cover a row twice, which is reported, can count more units than the call has)
    const uint32_t eighth = total <= a.units ? (total + 7u) / 8u : a.units;
    if (8u * (uint64_t)eighth > a.units) {
        if (blockIdx.x == 0 && threadIdx.x == 0) atomicOr(a.err, HF_KERR_CORRUPT);
        return false;
    }
    unit = blockIdx.x % 8u * eighth + blockIdx.x / 8u;
    return blockIdx.x / 8u < eighth && unit < total;
}
// The last of `count` numbers, which ascend, that is at most `most` (the first, if none is), for a
// wavefront: 64 looked at at a time.  `number` gives the i-th.
template <typename F>
__device__ __forceinline__ uint32_t kv_last(const uint32_t count, F&& number, const uint32_t most) {
    uint32_t at = 0, among = count;
    while (among > 1) {
        const uint32_t apart = (among + 63u) / 64u, mine = apart * hf_lane();
        bool past = true;
        if (mine < among) past = number(at + mine) > most;
        const unsigned long long ends = __ballot(past);
        const uint32_t k = ends ? max((int)__ffsll(ends) - 2, 0) : 63;
        at += k * apart;
        among = min(apart, among - k * apart);
    }
    return at;
}
// The unit's sequence in the cut that hf_k_kv_plan left: the last one with no more units before it
// than the unit's number.
__device__ __forceinline__ bool kv_search(const hf_kv_attend_args& a, kv_cut& cut) {
    const uint32_t total = __builtin_amdgcn_readfirstlane(a.plan[4 * (int64_t)a.s.batch + 1]);
    if (!kv_unit_of(a, total, cut.unit)) return false;
    const uint32_t b = kv_last(a.s.batch, [&](const uint32_t i) { return a.plan[4 * (int64_t)i]; }, cut.unit);
    const hf_u32x4 p = *(const hf_u32x4*)(a.plan + 4 * (int64_t)b);
    cut.b = b;
    cut.n_before = __builtin_amdgcn_readfirstlane(p[0]);
    cut.tiles = __builtin_amdgcn_readfirstlane(p[1]);
    cut.ranges = __builtin_amdgcn_readfirstlane(p[2]);
    cut.steps_each = (kv_div_up(__builtin_amdgcn_readfirstlane(p[3]), cut.ranges) + kWaves - 1u) / kWaves * kWaves;
    return __builtin_amdgcn_readfirstlane(cut.unit) - cut.n_before < cut.tiles * cut.ranges;
}
// The cut in memory: of each sequence the units before it, tiles, ranges and steps; behind the last
// sequence whether any has more than one range, and all units.
__device__ __forceinline__ bool kv_find(const hf_kv_attend_args& a, const uint32_t tile_rows, kv_cut& cut) {
    if (a.s.batch > HF_KV_OWN_CUT) return kv_search(a, cut);
    const kv_plan_dev p = kv_plan_now(a, tile_rows);
    if (blockIdx.x == 0 && threadIdx.x < 64 && a.join) {
        bool split = false;
        kv_walk(a, tile_rows, p, [&](const uint32_t b, const kv_shape& s, const uint32_t ranges, const uint32_t first) {
            if (b < a.s.batch) *(hf_u32x4*)(a.plan + 4 * (int64_t)b) = hf_u32x4{first, s.tiles, ranges, s.steps};
            split = split || (s.tiles && ranges > 1);
            return false;
        }, cut);
        split = __ballot(split) != 0;
        if (threadIdx.x == 0) a.plan[4 * (int64_t)a.s.batch] = split;
    }
    if (!kv_unit_of(a, p.total, cut.unit)) return false;
    const uint32_t unit = cut.unit;
    return kv_walk(a, tile_rows, p, [&](uint32_t, const kv_shape& s, const uint32_t ranges, const uint32_t first) {
        return unit < first + s.tiles * ranges;
    }, cut);
}

// ---- one unit ------------------------------------------------------------------------------------
template <int QT, int FMT, int DP>
struct kv_unit {
    typedef kv_type<QT> T;
    static constexpr int bits = kv_bits<FMT>();
    // K: a lane loads pieces of DPC consecutive d of a token: four lanes take 4 DPC of them
    static constexpr int DPC = bits == 16 ? 8 : bits == 8 ? 16 : DP == 64 ? 16 : 32;
    static constexpr int KP = DP / (4 * DPC);  // pieces per token and lane
    static constexpr int KB = DPC * bits / 8;  // bytes of a piece
    static constexpr int KS = DP / 32;         // products along d
    // V: a lane loads VD consecutive d of eight tokens
    static constexpr int VD = DP / 16;
    static constexpr int VB = VD * bits / 8;

    // what a wavefront holds of 32 tokens, as loaded
    struct tile {
        kv_raw<KB> k[2][KP];
        kv_raw<VB> v[8];
        hf_u32x2 ks[bits == 16 ? 1 : KP];  // scale bytes of the lane's eight tokens, by piece
        hf_u32x2 vs;
    };
    struct pages {  // of four groups of eight tokens
        int32_t id[4];
    };

    const hf_kv_attend_args& a;
    const int lane, m, g;
    uint32_t head;
    hf_kv_seq q;
    const hf_gi32* table;
    f32x4 acc[VD];
    f32x4 div;      // sums of the rounded p (all four alike)
    float nm, sum;  // p = exp2(scale_log2 s + nm); the lane's share of the sum of p
    hf_u32x4 qr[KS];
    uint32_t bad, odd;  // a page out of range; values that were left out
    // the lane's own part of its places in the pools and in the scales
    const hf_g8 *kbase, *vbase, *ksbase, *vsbase;
    bool cuts;  // head_dim ends inside the padded one

    __device__ __forceinline__ kv_unit(const hf_kv_attend_args& args)
        : a(args), lane(hf_lane()), m(lane & 15), g(lane >> 4), bad(0), odd(0) {}

    // Lanes whose d are behind head_dim load the row's first ones instead: of K the values are
    // cleared, of V they make outputs that nobody takes.
    __device__ __forceinline__ void bases() {
        cuts = a.c.head_dim < (uint32_t)DP;
        const int dk = DPC * g < (int)a.c.head_dim ? DPC * g : 0, dv = VD * m < (int)a.c.head_dim ? VD * m : 0;
        const int64_t h = (int64_t)head * a.c.head_stride;
        kbase = (const hf_g8*)a.c.k + h + (int64_t)(m & 3) * a.c.token_stride + dk * bits / 8;
        vbase = (const hf_g8*)a.c.v + h + dv * bits / 8;
        const int64_t hs = (int64_t)head * a.c.groups << a.c.page_shift;
        ksbase = (const hf_g8*)a.c.k_scale + hs + ((int64_t)(dk >> a.c.group_shift) << a.c.page_shift);
        vsbase = (const hf_g8*)a.c.v_scale + hs + ((int64_t)(dv >> a.c.group_shift) << a.c.page_shift);
    }
    __device__ __forceinline__ int64_t place(const uint32_t at, int32_t page_id, int64_t& scale) {
        uint32_t pg = (uint32_t)page_id;
        if (pg >= a.c.n_pages) {
            bad = 1;
            pg = 0;
        }
        const uint32_t off = group_at(at) & ((1u << a.c.page_shift) - 1u);
        scale = (int64_t)((uint64_t)pg * (a.c.heads * a.c.groups << a.c.page_shift) + off);
        return (int64_t)((uint64_t)pg * (uint32_t)a.c.page_stride + (uint64_t)off * (uint32_t)a.c.token_stride);
    }

    // d of the lane's elements of product ks: first of eight
    __device__ __forceinline__ int d_of(const int ks) const {
        constexpr int per = DPC / 8;
        return 4 * DPC * (ks / per) + DPC * g + 8 * (ks % per);
    }

    __device__ __forceinline__ void load_q(const int32_t row_lo, const int32_t rows) {
        const int32_t i = row_lo + m;
        const bool on = i < rows;
        const int32_t tok = (on ? i : 0) / (int32_t)a.per, hq = (on ? i : 0) % (int32_t)a.per;
        const hf_g8* p = (const hf_g8*)a.q.p + ((int64_t)(q.row0 + tok) * a.q.row_stride +
                                                (int64_t)(head * a.per + hq) * a.q.head_stride) * 2;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int d = d_of(ks);
            hf_u32x4 x = {0, 0, 0, 0};
            if (on && d < (int)a.c.head_dim) x = *(const hf_gmem_u32x4*)(p + 2 * d);
            qr[ks] = x;
        }
        nm = 3.402823466e38f;
        sum = 0.0f;
        div = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < VD; ++c) acc[c] = f32x4{0, 0, 0, 0};
    }

    // Tokens past the end of the sequence are taken from its last group of eight (a page holds
    // whole groups, so all eight are inside it) and masked later.
    __device__ __forceinline__ uint32_t group_at(const uint32_t t) const {
        const uint32_t last = ((uint32_t)q.len - 1u) & ~7u;
        return min(t, last);
    }
    __device__ __forceinline__ int32_t page_at(const uint32_t t) {
        int32_t p = table[group_at(t) >> a.c.page_shift];
        return p;
    }
    // The pages of 32 tokens, four groups of eight: through the scalar cache, so that the wait for
    // them is not one for the vector loads in front of them.
    __device__ __forceinline__ void find(const uint32_t t, pages& p) const {
        const kv_const_i32* tab = (const kv_const_i32*)(const int32_t*)table;
#pragma unroll
        for (int i = 0; i < 4; ++i) p.id[i] = tab[__builtin_amdgcn_readfirstlane(group_at(t + 8u * i) >> a.c.page_shift)];
    }
    static __device__ __forceinline__ int32_t of_group(const pages& p, const int i) {
        const int32_t lo = i & 1 ? p.id[1] : p.id[0], hi = i & 1 ? p.id[3] : p.id[2];
        return i & 2 ? hi : lo;
    }
    __device__ __forceinline__ void load_k(const uint32_t t, const pages p, tile& x) {
        int64_t sc;
        const hf_g8* pk = kbase + place(t + 8u * (m >> 2), of_group(p, m >> 2), sc);
        const int dk = DPC * g < (int)a.c.head_dim ? DPC * g : 0;
        // (where nothing is cut, a constant offset)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int h = 0; h < KP; ++h) {
                const int d = cuts && 4 * DPC * h + DPC * g >= (int)a.c.head_dim ? 0 : 4 * DPC * h;
                x.k[b][h].load(pk + d * bits / 8);
            }
            pk += 4 * (int64_t)a.c.token_stride;
        }
        if constexpr (bits != 16) {
#pragma unroll
            for (int h = 0; h < KP; ++h) {
                const int d = cuts && 4 * DPC * h + DPC * g >= (int)a.c.head_dim ? 0 : 4 * DPC * h;
                x.ks[h] = *(const hf_gmem_u32x2*)(
                    ksbase + sc + ((((dk + d) >> a.c.group_shift) - (dk >> a.c.group_shift)) << a.c.page_shift));
            }
        }
    }
    __device__ __forceinline__ void load_v(const uint32_t t, const pages p, tile& x) {
        int64_t sc;
        const hf_g8* pv = vbase + place(t + 8u * g, of_group(p, g), sc);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x.v[j].load(pv);
            pv += a.c.token_stride;
        }
        if constexpr (bits != 16) x.vs = *(const hf_gmem_u32x2*)(vsbase + sc);
    }

    // Which of the lane's eight tokens t + 8 g + 0..7 row i (of the sequence's n rows) may see.
    __device__ __forceinline__ uint32_t seen(const int32_t row, const uint32_t t, const bool on) const {
        return seen_at(row, t + 8u * g, on);
    }
    __device__ __forceinline__ uint32_t seen_at(const int32_t row, const uint32_t t, const bool on) const {
        const int32_t j = (int32_t)t - q.past;  // draft number of the first of them
        uint32_t bits8;
        if (a.mask) {
            const int32_t w = j >> 5;
            const uint32_t* words = a.mask + (int64_t)(q.row0 + (on ? row : 0)) * a.mask_words;
            const uint32_t lo = w < 0 ? ~0u : (uint32_t)w < a.mask_words ? words[w] : 0u;
            const uint32_t hi = w + 1 < 0 ? ~0u : (uint32_t)(w + 1) < a.mask_words ? words[w + 1] : 0u;
            bits8 = __builtin_amdgcn_alignbit(hi, lo, (uint32_t)j & 31u) & 0xFFu;
        } else {
            const int32_t can = min(max(row - j + 1, 0), 8);
            bits8 = (1u << can) - 1u;
        }
        const int32_t left = min(max(q.n - j, 0), 8);  // tokens there are
        return on ? bits8 & ((1u << left) - 1u) : 0u;
    }

    // VD elements of V, as loaded, times their scale, as 16-bit pairs.
    static __device__ __forceinline__ void decode(const kv_raw<VB>& r, const float s, uint32_t (&w)[VD / 2]) {
        if constexpr (bits == 16) {
#pragma unroll
            for (int i = 0; i < VD / 2; ++i) w[i] = r.w[i];
        } else if constexpr (bits == 8) {
#pragma unroll
            for (int i = 0; i < VD / 4; ++i) {
                w[2 * i] = kv_pair<QT, FMT, 0>(r.w[i], s);
                w[2 * i + 1] = kv_pair<QT, FMT, 1>(r.w[i], s);
            }
        } else {
            w[0] = kv_pair<QT, FMT, 0>(r.w[0], s);
            w[1] = kv_pair<QT, FMT, 1>(r.w[0], s);
            if constexpr (VD >= 8) {
                w[2] = kv_pair<QT, FMT, 2>(r.w[0], s);
                w[3] = kv_pair<QT, FMT, 3>(r.w[0], s);
            }
            if constexpr (VD >= 16) {
                w[4] = kv_pair<QT, FMT, 0>(r.w[1], s);
                w[5] = kv_pair<QT, FMT, 1>(r.w[1], s);
                w[6] = kv_pair<QT, FMT, 2>(r.w[1], s);
                w[7] = kv_pair<QT, FMT, 3>(r.w[1], s);
            }
        }
    }

    // The eight tokens of the lane as operand A of the product along tokens, for each of its d.
    __device__ __forceinline__ void columns(const tile& x, const uint32_t there, hf_u32x4 (&av)[VD]) const {
        uint32_t v[8][VD / 2];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // scale byte j of vs to the exponent of a float
            const uint32_t w = j < 4 ? x.vs.x : x.vs.y;
            const uint32_t sb = ((j & 3) == 3 ? w >> 1 : w << (23 - 8 * (j & 3))) & 0x7F800000u;
            const float s = __uint_as_float(sb);
            decode(x.v[j], s, v[j]);
            if (!(there >> j & 1u)) {  // nothing is known of what the page holds behind the last token
#pragma unroll
                for (int i = 0; i < VD / 2; ++i) v[j][i] = 0;
            }
        }
#pragma unroll
        for (int i = 0; i < VD / 2; ++i)
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
                av[2 * i][jj] = __builtin_amdgcn_perm(v[2 * jj + 1][i], v[2 * jj][i], 0x05040100u);
                av[2 * i + 1][jj] = __builtin_amdgcn_perm(v[2 * jj + 1][i], v[2 * jj][i], 0x07060302u);
            }
    }

    // The values of VD elements from d of token `off` of a page (codes at p), as the products take them.
    __device__ __forceinline__ void values(const hf_g8* p, const int32_t page, const uint32_t off, const int d,
                                           float (&v)[VD]) const {
        kv_raw<VB> r;
        r.load(p);
        float s = 0.0f;
        if constexpr (bits != 16)
            s = __uint_as_float((uint32_t)((const hf_g8*)a.c.v_scale)[(((int64_t)page * a.c.heads + head) * a.c.groups
                                                                       << a.c.page_shift) + off +
                                                                      ((int64_t)(d >> a.c.group_shift) << a.c.page_shift)]
                                << 23);
        uint32_t w[VD / 2];
        decode(r, s, w);
#pragma unroll
        for (int i = 0; i < VD / 2; ++i) {
            const uint32_t x = w[i];
            if constexpr (QT == HF_DT_BF16) {
                v[2 * i] = __uint_as_float(x << 16);
                v[2 * i + 1] = __uint_as_float(x & 0xFFFF0000u);
            } else {
                const f16x2 h = __builtin_bit_cast(f16x2, x);
                v[2 * i] = (float)h.x;
                v[2 * i + 1] = (float)h.y;
            }
        }
    }

    // A step: 32 tokens from t.  FULL: every row sees all of them.
    // next_k, next_v: called where the tile's K and V are in use no more, to load the next ones there.
    template <bool FULL, typename NK, typename NV>
    __device__ __forceinline__ void step(const uint32_t t, const tile& x, const int32_t row_lo,
                                         const int32_t rows, NK&& next_k, NV&& next_v) {
        hf_u32x4 ka[2][KS];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int h = 0; h < KP; ++h) {
                float f = 0.0f;
                if constexpr (bits != 16) {
                    const uint32_t w = b ? x.ks[h].y : x.ks[h].x;
                    f = __uint_as_float(__builtin_amdgcn_ubfe(w, 8u * (m & 3), 8u) << 23);
                }
                if constexpr (bits == 16) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) ka[b][h][i] = x.k[b][h].w[i];
                } else if constexpr (bits == 8) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        ka[b][2 * h + i / 2][2 * (i % 2)] = kv_pair<QT, FMT, 0>(x.k[b][h].w[i], f);
                        ka[b][2 * h + i / 2][2 * (i % 2) + 1] = kv_pair<QT, FMT, 1>(x.k[b][h].w[i], f);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < KB / 4; ++i) {
                        constexpr int per = DPC / 8;
                        ka[b][per * h + i][0] = kv_pair<QT, FMT, 0>(x.k[b][h].w[i], f);
                        ka[b][per * h + i][1] = kv_pair<QT, FMT, 1>(x.k[b][h].w[i], f);
                        ka[b][per * h + i][2] = kv_pair<QT, FMT, 2>(x.k[b][h].w[i], f);
                        ka[b][per * h + i][3] = kv_pair<QT, FMT, 3>(x.k[b][h].w[i], f);
                    }
                }
            }
        }
        if (cuts) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
                    if (d_of(ks) >= (int)a.c.head_dim) ka[b][ks] = hf_u32x4{0, 0, 0, 0};
        }
        next_k();
        f32x4 s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            s[b] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s[b] = T::mma(ka[b][ks], qr[ks], s[b]);
        }
        if constexpr (!FULL) {
            const int32_t i = row_lo + m;
            const uint32_t see = seen((i < rows ? i : 0) / (int32_t)a.per, t, i < rows);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                s[e / 4][e % 4] = see >> e & 1u ? s[e / 4][e % 4] : -__builtin_inff();
        }
        float top = s[0][0];
#pragma unroll
        for (int e = 1; e < 8; ++e) top = fmaxf(top, s[e / 4][e % 4]);
        // seldom after the first step: sums and outputs to a new maximum
        bool huge = kv_huge(nm);
        if (__ballot(kv_exponent(top, a.scale_log2, nm, huge) > T::off + T::rise)) {
            const float was = nm;
            nm = fminf(was, T::off - kv_row_max(top) * a.scale_log2);
            const float f = __builtin_amdgcn_exp2f(nm - was);
            sum *= f;
            div *= f;
#pragma unroll
            for (int c = 0; c < VD; ++c) acc[c] *= f;
            huge = kv_huge(nm);
        }
        hf_u32x4 p;
        float e[8];
        if (huge) {
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = kv_exponent(s[i / 4][i % 4], a.scale_log2, nm, true);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = kv_exponent(s[i / 4][i % 4], a.scale_log2, nm, false);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            e[i] = __builtin_amdgcn_exp2f(e[i]);
            sum += e[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = T::pack(e[2 * i], e[2 * i + 1]);
        constexpr uint32_t two = T::one | T::one << 16;
        div = T::mma(hf_u32x4{two, two, two, two}, p, div);
        hf_u32x4 av[VD];
        uint32_t there = 0xFFu;
        if constexpr (!FULL) {
            const int32_t left = min(max(q.len - (int32_t)(t + 8u * g), 0), 8);
            there = (1u << left) - 1u;
        }
        columns(x, there, av);
        next_v();
        if constexpr (!FULL) {
            // A token that some rows may not see must not reach them as 0 x infinity or NaN: what is
            // not finite is left out here and added at the end (left_out).
#pragma unroll
            for (int c = 0; c < VD; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t hit = ((av[c][i] & T::expo) + T::unit) & 0x80008000u;
                    odd |= hit;
                    av[c][i] &= ~((hit >> 15) * 0xFFFFu);
                }
        }
#pragma unroll
        for (int c = 0; c < VD; ++c)
            acc[c] = T::mma(av[c], p, acc[c]);
    }

    // The values of tokens t .. t + 31 that are not finite, to the rows that see them.
    __device__ __forceinline__ void left_out(const uint32_t t, const int32_t row_lo, const int32_t rows) {
#pragma unroll 1
        for (uint32_t at = t; at < t + kStep && at < (uint32_t)q.len; ++at) {
            const int32_t pg = page_at(at);
            if ((uint32_t)pg >= a.c.n_pages) continue;
            const uint32_t off = at & ((1u << a.c.page_shift) - 1u);
            const hf_g8* p = (const hf_g8*)a.c.v + (int64_t)pg * a.c.page_stride + (int64_t)off * a.c.token_stride +
                             (int64_t)head * a.c.head_stride;
            const int32_t i = row_lo + m;
            const bool on = i < rows;
            const bool sees = on && (at < (uint32_t)q.past || (seen_at((on ? i : 0) / (int32_t)a.per, at, on) & 1u));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = VD * (4 * g + e);
                if (sees && d < (int)a.c.head_dim) {
                    float v[VD];
                    values(p + d * bits / 8, pg, off, d, v);
#pragma unroll
                    for (int c = 0; c < VD; ++c)
                        if (!(fabsf(v[c]) <= 3.402823466e38f)) acc[c][e] += v[c];
                }
            }
        }
    }
};

// Logarithm of the sum of exp(scale s), from the sum of exp2(scale_log2 s + nm).
__device__ __forceinline__ float kv_lse(const float nm, const float sum) {
    return sum == 0.0f ? -__builtin_inff() : 0.6931471805599453f * (__builtin_amdgcn_logf(sum) - nm);
}

// Scratch of a workgroup: what two wavefronts hand to the other two.
template <int DP>
struct kv_lds {
    f32x4 acc[2][DP / 16][64];
    float nm[2][64], sum[2][64], div[2][64];
};

// Bound by memory and the latency of its loads: 64 sequences of up to 8001 tokens, 8 heads of 128 in
// e4m3 (675 MB), in 149 us, 4.5 TB/s; 64 of 32 k at 5.1 TB/s, where a large read reaches 6.1.  The
// registers of a tile are loaded again as soon as they have been turned into operands (a second tile
// in flight costs a wavefront of two and was slower, 187 us).
template <int QT, int FMT, int DP>
__global__ __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(2)))
void hf_k_kv_attend(const hf_kv_attend_args a) {
    typedef kv_unit<QT, FMT, DP> U;
    constexpr uint32_t tile_rows = 16;
    __shared__ kv_lds<DP> lds;
    kv_cut cut;
    if (!kv_find(a, tile_rows, cut)) return;
    U u(a);
    u.q = hf_kv_sequence(a.s, cut.b, a.c.page_shift);
    const uint32_t in_seq = cut.unit - cut.n_before;
    const uint32_t row_tiles = cut.tiles / a.c.heads;
    const uint32_t range = in_seq / cut.tiles, tile = in_seq % cut.tiles;
    u.head = tile / row_tiles;
    const int32_t rows = u.q.n * (int32_t)a.per;
    const int32_t row_lo = (int32_t)(tile % row_tiles * tile_rows);
    u.table = (const hf_gi32*)(a.s.table + (int64_t)cut.b * a.s.table_stride);
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);

    // tokens of the unit, and how far every row of the tile sees all of them
    const int32_t tok_lo = row_lo / (int32_t)a.per;
    const int32_t tok_hi = (min(row_lo + (int32_t)tile_rows, rows) - 1) / (int32_t)a.per;
    const uint32_t whole = (uint32_t)(a.mask ? u.q.past : u.q.past + tok_lo + 1);
    uint32_t end = (uint32_t)(a.mask ? u.q.len : u.q.past + tok_hi + 1);
    const uint32_t t_lo = range * cut.steps_each * kStep;
    end = min(end, t_lo + cut.steps_each * kStep);

    u.load_q(row_lo, rows);
    u.bases();
    uint32_t t = t_lo + kStep * (uint32_t)wave;
    if (t < end) {
        constexpr uint32_t stride = kStep * kWaves;
        typename U::tile x;
        typename U::pages p;
        u.find(t, p);
        u.load_k(t, p, x);
        u.load_v(t, p, x);
        u.find(t + stride, p);
        kv_arrived(u.qr);
        auto one = [&](auto&& next_k, auto&& next_v) {
            if (t + kStep <= whole && t + kStep <= end) u.template step<true>(t, x, row_lo, rows, next_k, next_v);
            else u.template step<false>(t, x, row_lo, rows, next_k, next_v);
        };
        // The next tokens' bytes, and the pages of those behind them, are under way as soon as the
        // registers of the present ones are free.  (The last turn stands apart: loads under a
        // condition would make every wait one for all of them.)
#pragma unroll 1
        for (; t + stride < end; t += stride)
            one([&]() { u.load_k(t + stride, p, x); },
                [&]() {
                    u.load_v(t + stride, p, x);
                    u.find(t + 2 * stride, p);
                });
        one([]() {}, []() {});
    }
    if (__ballot(u.odd != 0)) {
        for (t = t_lo + kStep * (uint32_t)wave; t < end; t += kStep * kWaves)
            if (t + kStep > whole || t + kStep > end) u.left_out(t, row_lo, rows);
    }
    if (u.bad) atomicOr(a.err, HF_KERR_CORRUPT);

    // join the wavefronts: 2 and 3 hand to 0 and 1, then 1 to 0
    u.sum = kv_row_sum(u.sum);
#pragma unroll 1
    for (int half = 2; half >= 1; half >>= 1) {
        if (wave >= half && wave < 2 * half) {
            lds.nm[wave - half][u.lane] = u.nm;
            lds.sum[wave - half][u.lane] = u.sum;
            lds.div[wave - half][u.lane] = u.div[0];
#pragma unroll
            for (int c = 0; c < U::VD; ++c) lds.acc[wave - half][c][u.lane] = u.acc[c];
        }
        __syncthreads();
        if (wave < half) {
            const float other = lds.nm[wave][u.lane];
            const float least = fminf(u.nm, other);
            const float f = __builtin_amdgcn_exp2f(least - u.nm);
            const float h = __builtin_amdgcn_exp2f(least - other);
            u.nm = least;
            u.sum = u.sum * f + lds.sum[wave][u.lane] * h;
            u.div[0] = u.div[0] * f + lds.div[wave][u.lane] * h;
#pragma unroll
            for (int c = 0; c < U::VD; ++c) u.acc[c] = u.acc[c] * f + lds.acc[wave][c][u.lane] * h;
        }
        __syncthreads();
    }
    if (wave != 0) return;
    const int32_t i = row_lo + u.m;
    if (i >= rows) return;
    if (cut.ranges > 1) {  // to be joined with the other ranges
        const int64_t row = (int64_t)cut.unit * tile_rows + u.m;
        float* dst = a.part + row * DP;
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int c = 0; c < U::VD; c += 4)
                *(f32x4*)(dst + U::VD * (4 * u.g + e) + c) =
                    f32x4{u.acc[c][e], u.acc[c + 1][e], u.acc[c + 2][e], u.acc[c + 3][e]};
        if (u.g == 0) *(f32x4*)(a.part_ml + 4 * row) = f32x4{u.nm, u.sum, u.div[0], 0.0f};
    } else {
        const int32_t tok = i / (int32_t)a.per, hq = i % (int32_t)a.per;
        const uint32_t out_head = u.head * a.per + hq;
        const float f = u.div[0] == 0.0f ? 0.0f : 1.0f / u.div[0];  // no token seen: zeros
        hf_g8* dst = (hf_g8*)a.out.p + ((int64_t)(u.q.row0 + tok) * a.out.row_stride +
                                        (int64_t)out_head * a.out.head_stride) * 2;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int d = U::VD * (4 * u.g + e);
            if (d < (int)a.c.head_dim) {
#pragma unroll
                for (int c = 0; c < U::VD; c += 4)
                    *(hf_gmem_u32x2*)(dst + 2 * (d + c)) =
                        hf_u32x2{U::T::pack(u.acc[c][e] * f, u.acc[c + 1][e] * f),
                                 U::T::pack(u.acc[c + 2][e] * f, u.acc[c + 3][e] * f)};
            }
        }
        if (a.lse && u.g == 0)
            a.lse[(int64_t)(u.q.row0 + tok) * a.c.heads * a.per + out_head] = kv_lse(u.nm, u.sum);
    }
}

// Joins the ranges of rows that have several: a wavefront takes a row of a head at a time, DP / 4
// lanes along it and the ranges dealt to the groups of lanes that are left.  4 us for one
// token, 11 for eight trees of up to 63 tokens x 32 heads in four ranges.  A row's sequence is searched
// (the whole call for 4096 sequences of 3 rows, one of them long: 876 us; with the offsets walked 1420).
template <int QT, int DP>
__global__ __launch_bounds__(256) void hf_k_kv_join(const hf_kv_attend_args a, const uint32_t tile_rows) {
    typedef kv_type<QT> T;
    constexpr uint32_t cols = DP / 4, deal = 64 / cols;
    if (a.plan[4 * (int64_t)a.s.batch] == 0) return;
    const uint32_t q_heads = a.c.heads * a.per, all = a.s.rows * q_heads;
    const uint32_t first_id = blockIdx.x * 4u + (uint32_t)__builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    for (uint32_t id = first_id; id < all; id += gridDim.x * 4u) {
        const int32_t row = (int32_t)(id / q_heads);
        const uint32_t out_head = id % q_heads;
        uint32_t b = (uint32_t)row;
        if (a.s.cu) {
            b = kv_last(a.s.batch, [&](const uint32_t i) { return (uint32_t)a.s.cu[i]; }, b);
            if (row < a.s.cu[b] || row >= a.s.cu[b + 1]) continue;  // of no sequence
        }
        const hf_u32x4 plan = *(const hf_u32x4*)(a.plan + 4 * (int64_t)b);
        const uint32_t before = plan[0], tiles = plan[1], ranges = plan[2];
        if (tiles == 0 || ranges < 2) continue;
        const hf_kv_seq q = hf_kv_sequence(a.s, b, a.c.page_shift);
        const uint32_t i = (uint32_t)(row - q.row0) * a.per + out_head % a.per;
        const uint32_t tile = out_head / a.per * (tiles / a.c.heads) + i / tile_rows;
        // (offsets that cover a row twice, which the attending kernel reports, can count more units
        // than there are)
        if ((uint64_t)before + (uint64_t)tiles * ranges > a.units) continue;
        const int64_t first = (int64_t)(before + tile) * tile_rows + i % tile_rows;
        const int64_t jump = (int64_t)tiles * tile_rows;
        const uint32_t col = (uint32_t)hf_lane() % cols, part = (uint32_t)hf_lane() / cols;
        float least = 3.402823466e38f;
        for (uint32_t s = hf_lane(); s < ranges; s += 64) least = fminf(least, a.part_ml[4 * (first + s * jump)]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) least = fminf(least, __shfl_xor(least, o));
        f32x4 acc = {0, 0, 0, 0};
        float sum = 0.0f, div = 0.0f;
#pragma unroll 4
        for (uint32_t s = part; s < ranges; s += deal) {
            const int64_t at = first + s * jump;
            const f32x4 ml = *(const f32x4*)(a.part_ml + 4 * at);
            const float w = __builtin_amdgcn_exp2f(least - ml[0]);
            sum += w * ml[1];
            div += w * ml[2];
            acc += w * *(const f32x4*)(a.part + at * DP + 4 * col);
        }
#pragma unroll
        for (int o = cols; o < 64; o <<= 1) {
            sum += __shfl_xor(sum, o);
            div += __shfl_xor(div, o);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], o);
        }
        const float f = div == 0.0f ? 0.0f : 1.0f / div;
        if (part == 0 && 4 * col < a.c.head_dim) {
            hf_g8* dst = (hf_g8*)a.out.p + ((int64_t)row * a.out.row_stride + (int64_t)out_head * a.out.head_stride) * 2;
            *(hf_gmem_u32x2*)(dst + 8 * col) =
                hf_u32x2{T::pack(acc[0] * f, acc[1] * f), T::pack(acc[2] * f, acc[3] * f)};
        }
        if (a.lse && hf_lane() == 0)
            a.lse[(int64_t)row * q_heads + out_head] = kv_lse(least, sum);
    }
}

}  // namespace
