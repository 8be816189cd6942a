// Attention of many rows (a drafted tree, a chunk of a prompt) over quantised pages: like
// hf_k_kv_attend, but the wavefronts of a workgroup share what they read.
//
// WR x WS wavefronts: WR groups of 32 rows, and for each WS wavefronts that take the tokens 32 at a
// time in turn.  The workgroup takes TT tokens at a time: its wavefronts load the codes, turn them
// into 16-bit operands once (a conversion that applies the scale, and byte permutes for V) and put
// them into LDS, K as [token][d], V transposed as [d][token]; then every wavefront multiplies its own
// rows with them.  The codes of the next tokens are loaded into registers while the present ones are
// in use.
//   S^T = K Q^T    32 tokens x 32 rows: a lane has, of row lane % 32, sixteen tokens
//   O^T = V^T P^T  needs eight tokens of the lane's row as operand B, in registers, as it has them: K's
//                  tokens are read in an order (bits 2 and 3 of a token's number swapped) that makes
//                  them eight neighbours, sixteen bytes of a row of V^T
// 16-byte pieces of a row are stored at their number XOR a number of the row, such that sixteen lanes
// that read or write the same column of sixteen rows meet sixteen different places of the banks.
// Bound by the chain product - softmax - product: two chunks of 1000 rows x 32 heads on 5 k tokens in
// bf16 take 211 us, 744 TFLOP/s (a large product of the library: 1381), matrix units 38 % and vector
// units 47 % busy, 1.9 wavefronts a SIMD; eight trees of up to 63 rows on 8 k tokens in e4m3 take 70 us
// and 11 to join their ranges (30 %, 44 %, 1.8).
// Everything is meant to stay in registers: a spilled address is reloaded behind the loads under way,
// and its wait is theirs.
#pragma once

#include <type_traits>

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
    if constexpr (QT == HF_DT_BF16)
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), __builtin_bit_cast(bf16x2, two), a, false);
    else
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pair), __builtin_bit_cast(f16x2, two), a, false);
}

template <int DP, int TT>
struct kv_share {
    hf_u32x4 k[TT][DP / 8];
    hf_u32x4 v[DP][TT / 8];
};
// What WS - 1 wavefronts of a row group hand to the first.
template <int DP, int WR, int WS>
struct kv_hand {
    float acc[WS > 1 ? WS - 1 : 1][WS > 1 ? WR : 1][WS > 1 ? DP / 2 : 1][64];
    float st[WS > 1 ? WS - 1 : 1][WS > 1 ? WR : 1][3][64];
};

// A part of the staging, a wavefront's work: K of 32 tokens (two tokens of the lane, KP pieces of
// each) or V of 32 tokens (eight tokens of the lane), with their scale bytes, as loaded.
template <int QT, int FMT, int DP>
struct kv_part {
    typedef kv_unit<QT, FMT, DP> U;
    static constexpr int kw = U::KB / 4, vw = U::VB >= 4 ? U::VB / 4 : 1;
    static constexpr int words = 2 * U::KP * kw > 8 * vw ? 2 * U::KP * kw : 8 * vw;
    uint32_t w[words];
    hf_u32x2 s[U::bits == 16 ? 1 : 2 * U::KP];
};

template <int QT, int FMT, int DP, int WR, int WS, int TT>
__global__ __launch_bounds__(64 * WR * WS) __attribute__((amdgpu_waves_per_eu(DP > 128 ? 1 : 2)))
void hf_k_kv_attend_block(const hf_kv_attend_args a) {
    typedef kv_unit<QT, FMT, DP> U;
    typedef kv_part<QT, FMT, DP> P;
    typedef kv_type<QT> T;
    constexpr int bits = U::bits, VD = DP / 16, KS = DP / 16, NB = DP / 32, NT = TT / 32, CH = TT / 8;
    constexpr int waves = WR * WS, own = 2 * NT / waves;  // parts of a wavefront: all K or all V
    static_assert(own >= 1 && own * waves == 2 * NT && NT % WS == 0, "staging and tokens are dealt evenly");
    constexpr uint32_t tile_rows = 32 * WR;
    __shared__ union {
        kv_share<DP, TT> x[2];
        kv_hand<DP, WR, WS> hand;
    } lds;
    __shared__ uint32_t any_odd;
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
    const int wr = wave % WR, ws = wave / WR;
    const int n = u.lane & 31, kg = u.lane >> 5;

    // the wavefront's row of this lane, and how far the wavefront's rows see everything, or anything
    const int32_t w_lo = row_lo + 32 * wr, i_row = w_lo + n;
    const bool on = i_row < rows;
    const int32_t tok = (on ? i_row : 0) / (int32_t)a.per;
    const int32_t last = (min(w_lo + 32, rows) - 1) / (int32_t)a.per;
    const uint32_t len = (uint32_t)u.q.len, past = (uint32_t)u.q.past;
    const uint32_t whole = a.mask ? past : past + (uint32_t)(w_lo / (int32_t)a.per) + 1u;
    const uint32_t some = w_lo >= rows ? 0u : a.mask ? len : past + (uint32_t)last + 1u;
    const int32_t tile_last = (min(row_lo + (int32_t)tile_rows, rows) - 1) / (int32_t)a.per;
    const uint32_t t_lo = range * cut.steps_each * kStep;
    const uint32_t end = min(t_lo + cut.steps_each * kStep, a.mask ? len : past + (uint32_t)tile_last + 1u);

    hf_u32x4 qr[KS];
    {
        const int32_t hq = (on ? i_row : 0) % (int32_t)a.per;
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
    bool huge = false;  // kv_huge of nm

    // The staging of a wavefront: K parts for the first half of the wavefronts, V for the others.  A
    // part's place is the lane's own (fixed) plus its page and its first token's place in the page.
    // Where head_dim ends inside the padded one, the lanes behind it load other d of their token: of
    // K the values are cleared, of V they make outputs that nobody takes.
    const bool is_k = wave < waves / 2;
    const int part0 = 32 * own * (is_k ? wave : wave - waves / 2);  // its first token in the tile
    const uint32_t in_page = (1u << a.c.page_shift) - 1u;
    const uint32_t page_scales = a.c.heads * a.c.groups << a.c.page_shift;
    const int my_d = is_k ? U::DPC * u.g : VD * u.m;
    const int my_off = is_k ? u.m & 7 : 0;  // token in a group of eight
    const int my_grp = 8 * (is_k ? u.m >> 3 : u.g);
    const bool cuts = a.c.head_dim < (uint32_t)DP;
    const hf_g8* const base = (const hf_g8*)(is_k ? a.c.k : a.c.v) + (int64_t)my_off * a.c.token_stride +
                              (int64_t)u.head * a.c.head_stride + (my_d < (int)a.c.head_dim ? my_d * bits / 8 : 0);
    const hf_g8* const sbase = (const hf_g8*)(is_k ? a.c.k_scale : a.c.v_scale) +
                               ((int64_t)u.head * a.c.groups << a.c.page_shift) +
                               ((int64_t)((my_d < (int)a.c.head_dim ? my_d : 0) >> a.c.group_shift) << a.c.page_shift);
    P part[own];
    int32_t page[own][2];
    auto find_pages = [&](const uint32_t t) {
#pragma unroll
        for (int i = 0; i < own; ++i) {
            page[i][0] = u.page_at(t + part0 + 32 * i + my_grp);
            if (is_k) page[i][1] = u.page_at(t + part0 + 32 * i + 16 + my_grp);
        }
    };
    // row of codes and of scale bytes of the lane's token(s) from `at` on
    auto place = [&](const uint32_t at, const int32_t page_id, const hf_g8*& p, const hf_g8*& sp) {
        uint32_t pg = (uint32_t)page_id;
        if (pg >= a.c.n_pages) {
            bad = 1;
            pg = 0;
        }
        const uint32_t off = u.group_at(at) & in_page;
        p = base + (uint64_t)pg * (uint32_t)a.c.page_stride + (uint64_t)off * (uint32_t)a.c.token_stride;
        sp = sbase + (uint64_t)pg * page_scales + off;
    };
    auto load = [&](const uint32_t t) {
#pragma unroll
        for (int i = 0; i < own; ++i) {
            const uint32_t at = t + part0 + 32 * i + my_grp;
            const hf_g8 *p, *sp;
            if (is_k) {
                const int d0 = my_d < (int)a.c.head_dim ? my_d : 0;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    place(at + 16 * b, page[i][b], p, sp);
#pragma unroll
                    for (int h = 0; h < U::KP; ++h) {
                        // (uniform where nothing is cut: then a constant offset)
                        const int d = cuts && my_d + 4 * U::DPC * h >= (int)a.c.head_dim ? 0 : 4 * U::DPC * h;
                        kv_raw<U::KB> r;
                        r.load(p + d * bits / 8);
#pragma unroll
                        for (int e = 0; e < P::kw; ++e) part[i].w[(b * U::KP + h) * P::kw + e] = r.w[e];
                        if constexpr (bits != 16)
                            part[i].s[2 * h + b] = *(const hf_gmem_u32x2*)(
                                sp + ((((d0 + d) >> a.c.group_shift) - (d0 >> a.c.group_shift)) << a.c.page_shift));
                    }
                }
            } else {
                place(at, page[i][0], p, sp);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    kv_raw<U::VB> r;
                    r.load(p);
#pragma unroll
                    for (int e = 0; e < P::vw; ++e) part[i].w[j * P::vw + e] = r.w[e];
                    p += a.c.token_stride;
                }
                if constexpr (bits != 16) part[i].s[0] = *(const hf_gmem_u32x2*)sp;
            }
        }
    };
    // Operands of the parts into LDS.  EDGE: some of the tokens may be behind the last one, where
    // nothing is known of what a page holds, or not seen by every row: what is not finite is left out
    // here, so that it does not reach other rows as 0 x infinity, and added at the end.
    auto stage = [&](const uint32_t t, kv_share<DP, TT>& to, auto edge) {
        constexpr bool EDGE = decltype(edge)::value;
#pragma unroll
        for (int i = 0; i < own; ++i) {
            const int at = part0 + 32 * i;
            if (is_k) {
                constexpr int per = U::DPC / 8;  // 16-byte pieces that a loaded piece becomes
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const int row = at + 16 * b + u.m;
#pragma unroll
                    for (int h = 0; h < U::KP; ++h) {
                        float f = 0.0f;
                        if constexpr (bits != 16) {
                            const uint32_t w = u.m & 4 ? part[i].s[2 * h + b].y : part[i].s[2 * h + b].x;
                            f = __uint_as_float(__builtin_amdgcn_ubfe(w, 8u * (u.m & 3), 8u) << 23);
                        }
                        uint32_t kw[P::kw];
#pragma unroll
                        for (int e = 0; e < P::kw; ++e) kw[e] = part[i].w[(b * U::KP + h) * P::kw + e];
#pragma unroll
                        for (int c = 0; c < per; ++c) {
                            hf_u32x4 o;
                            if constexpr (bits == 16) {
                                o = hf_u32x4{kw[0], kw[1], kw[2], kw[3]};
                            } else if constexpr (bits == 8) {
                                o[0] = kv_pair<QT, FMT, 0>(kw[2 * c], f);
                                o[1] = kv_pair<QT, FMT, 1>(kw[2 * c], f);
                                o[2] = kv_pair<QT, FMT, 0>(kw[2 * c + 1], f);
                                o[3] = kv_pair<QT, FMT, 1>(kw[2 * c + 1], f);
                            } else {
                                o[0] = kv_pair<QT, FMT, 0>(kw[c], f);
                                o[1] = kv_pair<QT, FMT, 1>(kw[c], f);
                                o[2] = kv_pair<QT, FMT, 2>(kw[c], f);
                                o[3] = kv_pair<QT, FMT, 3>(kw[c], f);
                            }
                            const int d = 4 * U::DPC * h + U::DPC * u.g;
                            if (cuts && d >= (int)a.c.head_dim) o = hf_u32x4{0, 0, 0, 0};
                            to.k[row][((d / 8 + c) ^ (row & 15)) & (DP / 8 - 1)] = o;
                        }
                    }
                }
            } else {
                hf_u32x4 av[VD];
                typename U::tile v;
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int e = 0; e < P::vw; ++e) v.v[j].w[e] = part[i].w[j * P::vw + e];
                v.vs = part[i].s[0];
                uint32_t there = 0xFFu;
                if constexpr (EDGE) there = (1u << min(max(u.q.len - (int32_t)(t + at + 8u * u.g), 0), 8)) - 1u;
                u.columns(v, there, av);
                if constexpr (EDGE) {
                    bool odd = false;
#pragma unroll
                    for (int c = 0; c < VD; ++c)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t hit = ((av[c][e] & T::expo) + T::unit) & 0x80008000u;
                            odd = odd || hit;
                            av[c][e] &= ~((hit >> 15) * 0xFFFFu);
                        }
                    if (__ballot(odd) && u.lane == 0) any_odd = 1;
                }
#pragma unroll
                for (int c = 0; c < VD; ++c) {
                    const int row = 16 * c + u.m;
                    to.v[row][(at / 8 + u.g) ^ ((row / (16 / CH)) % CH)] = av[c];
                }
            }
        }
    };
    const int krow = (n & ~12) | (n & 4) << 1 | (n & 8) >> 1;  // bits 2 and 3 swapped
    const int vf = (n / (16 / CH)) % CH;

    // The wavefront's tokens of a tile against its rows, 32 after the other (so that half of the scores
    // and weights are in registers at a time).  FULL: every row sees all of them.
    auto multiply = [&](const uint32_t t, const kv_share<DP, TT>& x, auto is_full) {
        constexpr bool FULL = decltype(is_full)::value;
#pragma unroll 1
        for (int bi = 0; bi < NT / WS; ++bi) {
            const int b = bi * WS + ws;
            f32x16 s;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                s = kv_mma32<QT>(x.k[32 * b + krow][((2 * ks + kg) ^ (krow & 15)) & (DP / 8 - 1)], qr[ks], s);
            if constexpr (!FULL) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t see = u.seen_at(tok, t + 32 * b + 16 * h + 8 * kg, on);
#pragma unroll
                    for (int j = 0; j < 8; ++j) s[8 * h + j] = see >> j & 1u ? s[8 * h + j] : -__builtin_inff();
                }
            }
            float top = s[0];
#pragma unroll
            for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
            if (__ballot(kv_exponent(top, a.scale_log2, nm, huge) > T::off + T::rise)) {
                top = fmaxf(top, __shfl_xor(top, 32));
                const float was = nm;
                nm = fminf(was, T::off - top * a.scale_log2);
                const float f = __builtin_amdgcn_exp2f(nm - was);
                sum *= f;
                div *= f;
#pragma unroll
                for (int q = 0; q < NB; ++q) acc[q] *= f;
                huge = kv_huge(nm);
            }
            if (huge) {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = kv_exponent(s[i], a.scale_log2, nm, true);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = kv_exponent(s[i], a.scale_log2, nm, false);
            }
            hf_u32x4 p[2];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[i] = __builtin_amdgcn_exp2f(s[i]);
                sum += s[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i / 4][i % 4] = T::pack(s[2 * i], s[2 * i + 1]);
                div = kv_add_pair<QT>(p[i / 4][i % 4], div);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int q = 0; q < NB; ++q)
                    acc[q] = kv_mma32<QT>(x.v[32 * q + n][(4 * b + 2 * h + kg) ^ vf], p[h], acc[q]);
        }
    };

    if (threadIdx.x == 0) any_odd = 0;
    __syncthreads();
    kv_arrived(qr);
    auto stage_at = [&](const uint32_t t, kv_share<DP, TT>& to) {
        if (t + TT > past) stage(t, to, std::true_type{});
        else stage(t, to, std::false_type{});
        if (t + TT < end) {
            load(t + TT);
            find_pages(t + 2 * TT);
        }
    };
    if (t_lo < end) {
        find_pages(t_lo);
        load(t_lo);
        find_pages(t_lo + TT);
        stage_at(t_lo, lds.x[0]);
    }
    int buf = 0;
    for (uint32_t t = t_lo; t < end; t += TT) {
        __syncthreads();  // tile t is in its half, and nobody reads the other any more
        if (t + TT <= whole) multiply(t, lds.x[buf], std::true_type{});
        else if (t < some) multiply(t, lds.x[buf], std::false_type{});
        // (behind the products: 2 % faster than in front of them)
        if (t + TT < end) stage_at(t + TT, lds.x[buf ^ 1]);
        buf ^= 1;
    }
    __syncthreads();
    if (bad) atomicOr(a.err, HF_KERR_CORRUPT);
    if (any_odd) {
        // What was left out: of the tokens staged as EDGE, the values that are not finite.
#pragma unroll 1
        for (uint32_t t = max(t_lo, past / TT * TT); t < min(end, some); ++t) {
            if (ws != (int)(t / 32 % WS)) continue;
            const int32_t pg = u.page_at(t);
            const bool sees = on && (t < past || (u.seen_at(tok, t, on) & 1u));
            if ((uint32_t)pg >= a.c.n_pages || !sees) continue;
            const uint32_t off = t & in_page;
            const hf_g8* p = (const hf_g8*)a.c.v + (int64_t)pg * a.c.page_stride + (int64_t)off * a.c.token_stride +
                             (int64_t)u.head * a.c.head_stride;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int m = 8 * (e >> 2) + 4 * kg + (e & 3), d = VD * m;
                if (d < (int)a.c.head_dim) {
                    float v[VD];
                    u.values(p + d * bits / 8, pg, off, d, v);
#pragma unroll
                    for (int c = 0; c < VD; ++c)
                        if (!(fabsf(v[c]) <= 3.402823466e38f)) acc[c / 2][8 * (c & 1) + e] += v[c];
                }
            }
        }
    }
    sum += __shfl_xor(sum, 32);
    div += __shfl_xor(div, 32);
    if constexpr (WS > 1) {  // the wavefronts of a row group, in order
        if (ws > 0) {
            lds.hand.st[ws - 1][wr][0][u.lane] = nm;
            lds.hand.st[ws - 1][wr][1][u.lane] = sum;
            lds.hand.st[ws - 1][wr][2][u.lane] = div;
#pragma unroll
            for (int q = 0; q < NB; ++q)
#pragma unroll
                for (int i = 0; i < 16; ++i) lds.hand.acc[ws - 1][wr][16 * q + i][u.lane] = acc[q][i];
        }
        __syncthreads();
        if (ws > 0) return;
#pragma unroll 1
        for (int w = 0; w < WS - 1; ++w) {
            const float other = lds.hand.st[w][wr][0][u.lane], least = fminf(nm, other);
            const float f = __builtin_amdgcn_exp2f(least - nm), h = __builtin_amdgcn_exp2f(least - other);
            nm = least;
            sum = sum * f + lds.hand.st[w][wr][1][u.lane] * h;
            div = div * f + lds.hand.st[w][wr][2][u.lane] * h;
#pragma unroll
            for (int q = 0; q < NB; ++q)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[q][i] = acc[q][i] * f + lds.hand.acc[w][wr][16 * q + i][u.lane] * h;
        }
    }
    if (!on) return;
    // the lane's outputs: for each of eight m, VD neighbouring d: VD m + 2 q + i / 8
    if (cut.ranges > 1) {
        const int64_t row = (int64_t)cut.unit * tile_rows + 32 * wr + n;
        float* dst = a.part + row * DP;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int m = 8 * (e >> 2) + 4 * kg + (e & 3);
#pragma unroll
            for (int q = 0; q < NB; q += 2)
                *(f32x4*)(dst + VD * m + 2 * q) = f32x4{acc[q][e], acc[q][8 + e], acc[q + 1][e], acc[q + 1][8 + e]};
        }
        if (kg == 0) *(f32x4*)(a.part_ml + 4 * row) = f32x4{nm, sum, div, 0.0f};
    } else {
        const uint32_t out_head = u.head * a.per + (uint32_t)(i_row % (int32_t)a.per);
        const float f = div == 0.0f ? 0.0f : 1.0f / div;
        hf_g8* dst = (hf_g8*)a.out.p + ((int64_t)(u.q.row0 + tok) * a.out.row_stride +
                                        (int64_t)out_head * a.out.head_stride) * 2;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int m = 8 * (e >> 2) + 4 * kg + (e & 3);
            if (VD * m < (int)a.c.head_dim) {
#pragma unroll
                for (int q = 0; q < NB; q += 2)
                    *(hf_gmem_u32x2*)(dst + 2 * (VD * m + 2 * q)) =
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
    const uint64_t blocks = ((uint64_t)a.s.rows * a.c.heads * a.per + 3) / 4;
    hipLaunchKernelGGL((hf_k_kv_join<QT, DP>), dim3((uint32_t)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, st, a, tile_rows);
}
template <int QT, int FMT, int DP>
void kv_launch_rows(const hf_kv_attend_args& a, const int tile_rows, hipStream_t st) {
    if constexpr (DP <= 128) {
        if (tile_rows == 16)
            hipLaunchKernelGGL((hf_k_kv_attend<QT, FMT, DP>), dim3(a.units), dim3(64 * kWaves), 0, st, a);
        else if (tile_rows == 64)
            hipLaunchKernelGGL((hf_k_kv_attend_block<QT, FMT, DP, 2, 2, 64>), dim3(a.units), dim3(256), 0, st, a);
        else if (tile_rows == 256)
            hipLaunchKernelGGL((hf_k_kv_attend_block<QT, FMT, DP, 8, 1, 128>), dim3(a.units), dim3(512), 0, st, a);
    }
    if (tile_rows == 128)
        hipLaunchKernelGGL((hf_k_kv_attend_block<QT, FMT, DP, 4, 1, 64>), dim3(a.units), dim3(256), 0, st, a);
    kv_join<QT, DP>(a, (uint32_t)tile_rows, st);
}
template <int QT, int FMT>
void kv_launch_dim(const hf_kv_attend_args& a, const int tile_rows, hipStream_t st) {
    if (a.c.head_dim <= 64) kv_launch_rows<QT, FMT, 64>(a, tile_rows, st);
    else if (a.c.head_dim <= 128) kv_launch_rows<QT, FMT, 128>(a, tile_rows, st);
    else kv_launch_rows<QT, FMT, 256>(a, tile_rows, st);
}

}  // namespace
