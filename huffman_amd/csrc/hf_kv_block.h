// Attention of many rows (a drafted tree, a chunk of a prompt) over quantised pages: like
// hf_k_kv_attend, but the WR wavefronts of a workgroup have 32 rows each and share what they read.
//
// The workgroup takes TT tokens at a time: its wavefronts load the codes, turn them into 16-bit
// operands once (a conversion that applies the scale, and byte permutes for V) and put them into LDS,
// K as [token][d], V transposed as [d][token]; then every wavefront multiplies its own rows with
// them.  The codes of the next tokens are loaded into registers while the present ones are in use.
//   S^T = K Q^T    32 tokens x 32 rows: a lane has, of row lane % 32, sixteen tokens
//   O^T = V^T P^T  needs eight tokens of the lane's row as operand B, in registers, as it has them: K's
//                  tokens are read in an order (bits 2 and 3 of a token's number swapped) that makes
//                  them eight neighbours, sixteen bytes of a row of V^T
// 16-byte pieces of a row are stored at their number XOR a number of the row, such that sixteen lanes
// that read or write the same column of sixteen rows meet sixteen different places of the banks.
#pragma once

#include "hf_kv_attend.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int QT>
__device__ __forceinline__ f32x16 kv_mma32(hf_u32x4 a, hf_u32x4 b, f32x16 c) {
    if constexpr (QT == HF_DT_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// a + the sum of a pair of 16-bit values
template <int QT>
__device__ __forceinline__ float kv_add_pair(const uint32_t pair, const float a) {
    constexpr uint32_t two = kv_type<QT>::one | kv_type<QT>::one << 16;
    if constexpr (QT == HF_DT_BF16) {
        typedef short s16x2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), __builtin_bit_cast(bf16x2, two), a, false);
    } else {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pair), __builtin_bit_cast(f16x2, two), a, false);
    }
}

template <int DP, int TT>
struct kv_share {
    hf_u32x4 k[TT][DP / 8];
    hf_u32x4 v[DP][TT / 8];
    uint32_t odd[TT / 32];  // values that are not finite, per 32 tokens
};

template <int QT, int FMT, int DP, int WR>
struct kv_block {
    typedef kv_type<QT> T;
    typedef kv_unit<QT, FMT, DP, 1> U;
    static constexpr int TT = WR == 1 ? 32 : 64;
    static constexpr int bits = kv_bits<FMT>();
    static constexpr int VD = DP / 16, KS = DP / 16, NB = DP / 32, NT = TT / 32;
    static constexpr int CH = TT / 8;  // 16-byte pieces of a row of V^T
    // a wavefront stages K or V of 32 tokens: parts of all of them, and of one
    static constexpr int parts = 2 * NT, own = parts / WR;
    static_assert(own >= 1 && own * WR == parts, "staging is dealt evenly");

};

// A part as loaded: K of 32 tokens (two tokens of the lane, KP pieces each) or V (eight tokens), and
// their scale bytes, in the same registers.
template <int QT, int FMT, int DP>
struct kv_part {
    typedef kv_unit<QT, FMT, DP, 1> U;
    static constexpr int kw = U::KB / 4, vw = U::VB >= 4 ? U::VB / 4 : 1;
    static constexpr int words = 2 * U::KP * kw > 8 * vw ? 2 * U::KP * kw : 8 * vw;
    uint32_t w[words];
    hf_u32x2 s[U::bits == 16 ? 1 : 2 * U::KP];
};

// Loads of a wavefront's K part: tokens t + 16 b + m of 32, d in pieces as in kv_unit.
template <int QT, int FMT, int DP>
__device__ __forceinline__ void kv_load_k(const kv_unit<QT, FMT, DP, 1>& u, const hf_kv_attend_args& a, const uint32_t t,
                                          const int32_t (&pages)[2], kv_part<QT, FMT, DP>& x, uint32_t& bad) {
    typedef kv_unit<QT, FMT, DP, 1> U;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        int32_t page = pages[b];
        if ((uint32_t)page >= a.c.n_pages) { bad = 1; page = 0; }
        const uint32_t off = u.group_at(t + 16u * b + 8u * (u.m >> 3)) & ((1u << a.c.page_shift) - 1u);
        const hf_g8* p = (const hf_g8*)a.c.k + (int64_t)page * a.c.page_stride +
                         (int64_t)(off + (u.m & 7)) * a.c.token_stride + (int64_t)u.head * a.c.head_stride;
        const int64_t sc = (((int64_t)page * a.c.heads + u.head) * a.c.groups << a.c.page_shift) + off;
#pragma unroll
        for (int h = 0; h < U::KP; ++h) {
            const int d = 4 * U::DPC * h + U::DPC * u.g;
            kv_raw<U::KB> r;
            if (d < (int)a.c.head_dim) r.load(p + d * U::bits / 8);
            else r.clear();
#pragma unroll
            for (int i = 0; i < U::KB / 4; ++i) x.w[(b * U::KP + h) * (U::KB / 4) + i] = r.w[i];
            if constexpr (U::bits != 16) {
                x.s[2 * h + b] = hf_u32x2{0, 0};
                if (d < (int)a.c.head_dim)
                    x.s[2 * h + b] = *(const hf_gmem_u32x2*)((const hf_g8*)a.c.k_scale + sc +
                                                        ((int64_t)(d >> a.c.group_shift) << a.c.page_shift));
            }
        }
    }
}
template <int QT, int FMT, int DP>
__device__ __forceinline__ void kv_load_v(const kv_unit<QT, FMT, DP, 1>& u, const hf_kv_attend_args& a, const uint32_t t,
                                          int32_t page, kv_part<QT, FMT, DP>& x, uint32_t& bad) {
    typedef kv_unit<QT, FMT, DP, 1> U;
    if ((uint32_t)page >= a.c.n_pages) { bad = 1; page = 0; }
    const uint32_t off = u.group_at(t + 8u * u.g) & ((1u << a.c.page_shift) - 1u);
    const hf_g8* p = (const hf_g8*)a.c.v + (int64_t)page * a.c.page_stride + (int64_t)off * a.c.token_stride +
                     (int64_t)u.head * a.c.head_stride + U::VB * u.m;
    const bool on = U::VD * u.m < (int)a.c.head_dim;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        kv_raw<U::VB> r;
        if (on) r.load(p);
        else r.clear();
#pragma unroll
        for (int i = 0; i < kv_part<QT, FMT, DP>::vw; ++i) x.w[j * kv_part<QT, FMT, DP>::vw + i] = r.w[i];
        p += a.c.token_stride;
    }
    if constexpr (U::bits != 16) {
        x.s[0] = hf_u32x2{0, 0};
        if (on)
            x.s[0] = *(const hf_gmem_u32x2*)((const hf_g8*)a.c.v_scale +
                                          (((int64_t)page * a.c.heads + u.head) * a.c.groups << a.c.page_shift) + off +
                                          ((int64_t)((U::VD * u.m) >> a.c.group_shift) << a.c.page_shift));
    }
}

// A K part into LDS: piece c of token row at c ^ (row % 16).
template <int QT, int FMT, int DP, int TT>
__device__ __forceinline__ void kv_store_k(const kv_unit<QT, FMT, DP, 1>& u, const int at,
                                           const kv_part<QT, FMT, DP>& x, kv_share<DP, TT>& lds) {
    typedef kv_unit<QT, FMT, DP, 1> U;
    constexpr int per = U::DPC / 8;  // 16-byte pieces that a loaded piece becomes
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int row = at + 16 * b + u.m;
#pragma unroll
        for (int h = 0; h < U::KP; ++h) {
            float f = 0.0f;
            if constexpr (U::bits != 16) {
                const uint32_t w = u.m & 4 ? x.s[2 * h + b].y : x.s[2 * h + b].x;
                f = __uint_as_float(__builtin_amdgcn_ubfe(w, 8u * (u.m & 3), 8u) << 23);
            }
            const uint32_t* kw = x.w + (b * U::KP + h) * (U::KB / 4);
#pragma unroll
            for (int i = 0; i < per; ++i) {
                hf_u32x4 o;
                if constexpr (U::bits == 16) {
                    o = hf_u32x4{kw[0], kw[1], kw[2], kw[3]};
                } else if constexpr (U::bits == 8) {
                    o[0] = kv_pair<QT, FMT, 0>(kw[2 * i], f);
                    o[1] = kv_pair<QT, FMT, 1>(kw[2 * i], f);
                    o[2] = kv_pair<QT, FMT, 0>(kw[2 * i + 1], f);
                    o[3] = kv_pair<QT, FMT, 1>(kw[2 * i + 1], f);
                } else {
                    o[0] = kv_pair<QT, FMT, 0>(kw[i], f);
                    o[1] = kv_pair<QT, FMT, 1>(kw[i], f);
                    o[2] = kv_pair<QT, FMT, 2>(kw[i], f);
                    o[3] = kv_pair<QT, FMT, 3>(kw[i], f);
                }
                const int c = (4 * U::DPC * h + U::DPC * u.g) / 8 + i;
                lds.k[row][(c ^ (row & 15)) & (DP / 8 - 1)] = o;
            }
        }
    }
}

template <int QT, int FMT, int DP, int WR>
__global__ __launch_bounds__(64 * WR) __attribute__((amdgpu_waves_per_eu(DP > 128 ? 1 : 2)))
void hf_k_kv_attend_block(const hf_kv_attend_args a) {
    typedef kv_block<QT, FMT, DP, WR> B;
    typedef kv_unit<QT, FMT, DP, 1> U;
    typedef kv_type<QT> T;
    constexpr int TT = B::TT, KS = B::KS, NB = B::NB, NT = B::NT, CH = B::CH;
    constexpr uint32_t tile_rows = 32 * WR;
    __shared__ kv_share<DP, TT> lds;
    kv_cut cut;
    if (!kv_find(a, tile_rows, blockIdx.x, cut)) return;
    U u(a);
    u.q = hf_kv_sequence(a.s, cut.b, a.c.page_shift);
    const uint32_t in_seq = blockIdx.x - cut.n_before;
    const uint32_t row_tiles = cut.tiles / a.c.heads;
    const uint32_t range = in_seq / cut.tiles, tile = in_seq % cut.tiles;
    u.head = tile / row_tiles;
    const int32_t rows = u.q.n * (int32_t)a.per;
    const int32_t row_lo = (int32_t)(tile % row_tiles * tile_rows);
    u.table = (const hf_gi32*)(a.s.table + (int64_t)cut.b * a.s.table_stride);
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int n = u.lane & 31, kg = u.lane >> 5;

    // the wavefront's row of this lane, and how far the wavefront's rows see everything, or anything
    const int32_t w_lo = row_lo + 32 * wave, i_row = w_lo + n;
    const bool on = i_row < rows;
    const int32_t tok = (on ? i_row : 0) / (int32_t)a.per, hq = (on ? i_row : 0) % (int32_t)a.per;
    const int32_t last = (min(w_lo + 32, rows) - 1) / (int32_t)a.per;
    const uint32_t len = (uint32_t)u.q.len;
    const uint32_t whole = (uint32_t)(a.mask ? u.q.past : u.q.past + w_lo / (int32_t)a.per + 1);
    const uint32_t some = w_lo >= rows ? 0u : a.mask ? len : (uint32_t)(u.q.past + last + 1);
    const int32_t tile_last = (min(row_lo + (int32_t)tile_rows, rows) - 1) / (int32_t)a.per;
    const uint32_t t_lo = range * cut.steps_each * kStep;
    const uint32_t end = min(t_lo + cut.steps_each * kStep, a.mask ? len : (uint32_t)(u.q.past + tile_last + 1));

    hf_u32x4 qr[KS];
    {
        const hf_g8* p = (const hf_g8*)a.q.p + ((int64_t)(u.q.row0 + tok) * a.q.row_stride +
                                                (int64_t)(u.head * a.per + hq) * a.q.head_stride) * 2;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int d = 16 * ks + 8 * kg;
            qr[ks] = hf_u32x4{0, 0, 0, 0};
            if (on && d < (int)a.c.head_dim) qr[ks] = *(const hf_gmem_u32x4*)(p + 2 * d);
        }
    }
    f32x16 acc[NB];
#pragma unroll
    for (int q = 0; q < NB; ++q)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[q][i] = 0.0f;
    float nm = 3.402823466e38f, sum = 0.0f, div = 0.0f;  // p = exp2(scale_log2 s + nm)
    uint32_t bad = 0;

    // the wavefront's parts of the staging: K halves first, then V halves
    constexpr int own = B::own;
    kv_part<QT, FMT, DP> part[own];
    const bool does_k = own > 1 || wave < WR / 2;  // one part each: half of the wavefronts K, half V
    const bool does_v = own > 1 || !does_k;
    auto part_at = [&](const int i) { return own > 1 ? wave * (own / 2) + i : wave % NT; };
    int32_t kpage[own > 1 ? own / 2 : 1][2], vpage[own > 1 ? own / 2 : 1];
    auto find_pages = [&](const uint32_t t) {
#pragma unroll
        for (int i = 0; i < (own > 1 ? own / 2 : 1); ++i) {
            const uint32_t at = t + 32u * part_at(i);
            if (does_k) {
                kpage[i][0] = u.page_at(at + 8u * (u.m >> 3));
                kpage[i][1] = u.page_at(at + 16u + 8u * (u.m >> 3));
            }
            if (does_v) vpage[i] = u.page_at(at + 8u * u.g);
        }
    };
    auto load = [&](const uint32_t t) {
#pragma unroll
        for (int i = 0; i < (own > 1 ? own / 2 : 1); ++i) {
            const uint32_t at = t + 32u * part_at(i);
            if (does_k) kv_load_k<QT, FMT, DP>(u, a, at, kpage[i], part[i], bad);
            if (does_v) kv_load_v<QT, FMT, DP>(u, a, at, vpage[i], part[own - 1 - i], bad);
        }
    };
    const int swz = n & ~12, krow = swz | (n & 4) << 1 | (n & 8) >> 1;  // bits 2 and 3 swapped
    const int vf = (n / (16 / CH)) % CH;

    if (t_lo < end) {
        find_pages(t_lo);
        load(t_lo);
        find_pages(t_lo + TT);
    }
    for (uint32_t t = t_lo; t < end; t += TT) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < (own > 1 ? own / 2 : 1); ++i) {
            const int at = 32 * part_at(i);
            if (does_k) kv_store_k<QT, FMT, DP, TT>(u, at, part[i], lds);
            if (does_v) {
                hf_u32x4 av[B::VD];
                const int32_t left = min(max(u.q.len - (int32_t)(t + at + 8u * u.g), 0), 8);
                typename U::tile x;
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int e = 0; e < kv_part<QT, FMT, DP>::vw; ++e)
                        x.v[j].w[e] = part[own - 1 - i].w[j * kv_part<QT, FMT, DP>::vw + e];
                x.vs = part[own - 1 - i].s[0];
                u.columns(x, (1u << left) - 1u, av);
                uint32_t odd = 0;
#pragma unroll
                for (int c = 0; c < B::VD; ++c) {
                    const int row = 16 * c + u.m;
                    lds.v[row][(at / 8 + u.g) ^ ((row / (16 / CH)) % CH)] = av[c];
                }
                if (t + TT > (uint32_t)u.q.past) {  // (only where rows see different tokens)
#pragma unroll
                    for (int c = 0; c < B::VD; ++c)
#pragma unroll
                        for (int e = 0; e < 4; ++e) odd |= ((av[c][e] & T::expo) + T::unit) & 0x80008000u;
                }
                const bool any = __ballot(odd != 0) != 0;
                if (u.lane == 0) lds.odd[at / 32] = any;
            }
        }
        if (t + TT < end) {
            load(t + TT);
            find_pages(t + 2 * TT);
        }
        __syncthreads();
        if (t >= some) continue;
        // 32 tokens after the other: half the scores and weights in registers at a time
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            const uint32_t tb = t + 32 * b;
            const bool full = tb + 32 <= whole && tb + 32 <= end;
            f32x16 s;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                s = kv_mma32<QT>(lds.k[32 * b + krow][((2 * ks + kg) ^ (krow & 15)) & (DP / 8 - 1)], qr[ks], s);
            if (!full) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t see = u.seen_at(tok, tb + 16 * h + 8 * kg, on);
#pragma unroll
                    for (int j = 0; j < 8; ++j) s[8 * h + j] = see >> j & 1u ? s[8 * h + j] : -__builtin_inff();
                }
            }
            float top = s[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
            if (__ballot(__builtin_fmaf(top, a.scale_log2, nm) > T::off + T::rise)) {
                top = fmaxf(top, __shfl_xor(top, 32));
                const float was = nm;
                nm = fminf(was, T::off - top * a.scale_log2);
                const float f = __builtin_amdgcn_exp2f(nm - was);
                sum *= f;
                div *= f;
#pragma unroll
                for (int q = 0; q < NB; ++q) acc[q] *= f;
            }
            // (fused: the error of scale x maximum is the same factor for the whole row; where it
            // could pass 1 / 256 of a power of two, the products are rounded first, as the maximum's was)
            if (__ballot(fabsf(nm) > 65536.0f && nm != 3.402823466e38f)) {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = s[i] * a.scale_log2 + nm;
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = __builtin_fmaf(s[i], a.scale_log2, nm);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(s[i]);
            if (a.lse) {
#pragma unroll
                for (int i = 0; i < 16; ++i) sum += s[i];
            }
            hf_u32x4 p[2];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i / 4][i % 4] = T::pack(s[2 * i], s[2 * i + 1]);
                div = kv_add_pair<QT>(p[i / 4][i % 4], div);
            }
            if (full || lds.odd[b] == 0) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int q = 0; q < NB; ++q)
                        acc[q] = kv_mma32<QT>(lds.v[32 * q + n][(4 * b + 2 * h + kg) ^ vf], p[h], acc[q]);
            } else {
                // infinities and NaN of tokens that some rows may not see (kv_unit::not_finite)
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {
                    const hf_u32x4 ph = h ? p[1] : p[0];
                    const uint32_t see = u.seen_at(tok, tb + 16 * h + 8 * kg, on);
                    hf_u32x4 ones;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        ones[i] = (see >> (2 * i) & 1u ? T::one : 0u) | (see >> (2 * i + 1) & 1u ? T::one << 16 : 0u);
#pragma unroll
                    for (int q = 0; q < NB; ++q) {
                        hf_u32x4 av = lds.v[32 * q + n][(4 * b + 2 * h + kg) ^ vf];
#pragma unroll 1
                        for (int kind = 0; kind < 3; ++kind) {
                            const uint32_t want = kind == 1 ? T::inf : T::inf | 0x8000u;
                            hf_u32x4 is;
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t lo = av[i] & 0xFFFFu, hi = av[i] >> 16;
                                const bool l = kind == 0 ? (lo & 0x7FFFu) > T::inf : lo == want;
                                const bool r = kind == 0 ? (hi & 0x7FFFu) > T::inf : hi == want;
                                is[i] = (l ? T::one : 0u) | (r ? T::one << 16 : 0u);
                            }
                            f32x16 count;
#pragma unroll
                            for (int i = 0; i < 16; ++i) count[i] = 0.0f;
                            count = kv_mma32<QT>(is, ones, count);
                            const float add = kind == 0 ? __builtin_nanf("") : kind == 1 ? __builtin_inff() : -__builtin_inff();
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                if (count[i] > 0.0f) acc[q][i] += add;
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if ((av[i] & 0x7FFFu) >= T::inf) av[i] &= 0xFFFF0000u;
                            if ((av[i] >> 16 & 0x7FFFu) >= T::inf) av[i] &= 0xFFFFu;
                        }
                        acc[q] = kv_mma32<QT>(av, ph, acc[q]);
                    }
                }
            }
        }
    }
    if (bad) atomicOr(a.err, HF_KERR_CORRUPT);
    sum += __shfl_xor(sum, 32);
    div += __shfl_xor(div, 32);
    if (!on) return;
    // the lane's outputs: for each of eight m, VD neighbouring d: VD m + 2 q + i / 8
    if (cut.ranges > 1) {
        const int64_t row = (int64_t)blockIdx.x * tile_rows + 32 * wave + n;
        float* dst = a.part + row * DP;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int m = 8 * (e >> 2) + 4 * kg + (e & 3);
#pragma unroll
            for (int q = 0; q < NB; q += 2)
                *(f32x4*)(dst + B::VD * m + 2 * q) = f32x4{acc[q][e], acc[q][8 + e], acc[q + 1][e], acc[q + 1][8 + e]};
        }
        if (kg == 0) *(f32x4*)(a.part_ml + 4 * row) = f32x4{nm, sum, div, 0.0f};
    } else {
        const uint32_t out_head = u.head * a.per + hq;
        const float f = div == 0.0f ? 0.0f : 1.0f / div;
        hf_g8* dst = (hf_g8*)a.out.p + ((int64_t)(u.q.row0 + tok) * a.out.row_stride +
                                        (int64_t)out_head * a.out.head_stride) * 2;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int m = 8 * (e >> 2) + 4 * kg + (e & 3);
            if (B::VD * m < (int)a.c.head_dim) {
#pragma unroll
                for (int q = 0; q < NB; q += 2)
                    *(hf_gmem_u32x2*)(dst + 2 * (B::VD * m + 2 * q)) =
                        hf_u32x2{T::pack(acc[q][e] * f, acc[q][8 + e] * f), T::pack(acc[q + 1][e] * f, acc[q + 1][8 + e] * f)};
            }
        }
        if (a.lse && kg == 0)
            a.lse[(int64_t)(u.q.row0 + tok) * a.c.heads * a.per + out_head] = kv_lse(nm, sum);
    }
}

template <int QT, int DP>
void kv_join(const hf_kv_attend_args& a, const uint32_t tile_rows, hipStream_t st) {
    if (!a.join) return;
    const uint64_t rows = (uint64_t)a.s.rows * a.c.heads * a.per;
    hipLaunchKernelGGL((hf_k_kv_join<QT, DP>), dim3((uint32_t)((rows + 3) / 4)), dim3(256), 0, st, a, tile_rows);
}
template <int QT, int FMT, int DP>
void kv_launch_rows(const hf_kv_attend_args& a, const int tile_rows, hipStream_t st) {
    if (tile_rows == 16)
        hipLaunchKernelGGL((hf_k_kv_attend<QT, FMT, DP, 1>), dim3(a.units), dim3(64 * kWaves), 0, st, a);
    else if (tile_rows == 32)
        hipLaunchKernelGGL((hf_k_kv_attend_block<QT, FMT, DP, 1>), dim3(a.units), dim3(64), 0, st, a);
    else if (tile_rows == 64)
        hipLaunchKernelGGL((hf_k_kv_attend_block<QT, FMT, DP, 2>), dim3(a.units), dim3(128), 0, st, a);
    else
        hipLaunchKernelGGL((hf_k_kv_attend_block<QT, FMT, DP, 4>), dim3(a.units), dim3(256), 0, st, a);
    kv_join<QT, DP>(a, (uint32_t)tile_rows, st);
}
template <int QT, int FMT>
void kv_launch_dim(const hf_kv_attend_args& a, const int tile_rows, hipStream_t st) {
    if (a.c.head_dim <= 64) kv_launch_rows<QT, FMT, 64>(a, tile_rows, st);
    else if (a.c.head_dim <= 128) kv_launch_rows<QT, FMT, 128>(a, tile_rows, st);
    else kv_launch_rows<QT, FMT, 256>(a, tile_rows, st);
}

}  // namespace
