// The quantised KV cache: rows into pages (write), pages into rows (read), accepted drafts to the
// front (keep).  All three only move bytes: a lane owns eight consecutive elements of a row, which
// is 16 bytes of a 16-bit row and 8 or 4 bytes of codes, and a row's group of G elements is G / 8
// neighbouring lanes, so a group's largest magnitude is found with a few lane moves and no LDS.
//
// The reference codes 8-bit symbols and names fp16, fp8 and fp4 operands (reports/spec.md:22), but
// has nothing that makes them; these kernels make the 8- and 4-bit pages its coder takes.
#include "hf_kv.h"

namespace {

template <int FMT>
struct kv_fmt;  // bits of a code; the largest value: exponent, mantissa bits as in a float, value
template <>
struct kv_fmt<HF_KV_FP8_E4M3> {
    static constexpr int bits = 8, exp = 8;
    static constexpr uint32_t mant = 0x600000u;
    static constexpr float top = 448.0f;
};
template <>
struct kv_fmt<HF_KV_FP8_E5M2> {
    static constexpr int bits = 8, exp = 15;
    static constexpr uint32_t mant = 0x600000u;
    static constexpr float top = 57344.0f;
};
template <>
struct kv_fmt<HF_KV_FP4_E2M1> {
    static constexpr int bits = 4, exp = 2;
    static constexpr uint32_t mant = 0x400000u;
    static constexpr float top = 6.0f;
};
template <>
struct kv_fmt<HF_KV_BF16> {
    static constexpr int bits = 16;
};
template <>
struct kv_fmt<HF_KV_FP16> {
    static constexpr int bits = 16;
};

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kMaxTokens = 64;  // rows of the row tensors a workgroup handles, at most
constexpr int kCuLds = 1025;    // row offsets searched in LDS (more sequences: in memory)

// Where the rows of a workgroup are in the pools.
struct kv_places {
    int64_t code[kMaxTokens];   // byte offset of the token's first code, -1: nowhere
    int64_t scale[kMaxTokens];  // offset of its byte in the scales of head 0, group 0
};

// Fills the places of rows [t0, t0 + n).  All threads of the workgroup call; ends with a barrier.
__device__ __forceinline__ void find_places(const hf_kv_pools& c, const hf_kv_seqs& s,
                                            const uint32_t t0, const uint32_t n, kv_places& p,
                                            int32_t* cu_lds, uint32_t* err) {
    const bool staged = s.cu && s.batch < (uint32_t)kCuLds;
    if (staged) {
        for (uint32_t i = threadIdx.x; i <= s.batch; i += kThreads) cu_lds[i] = s.cu[i];
        __syncthreads();
    }
    // The workgroup's other wavefronts look at every sequence of the call, a share each: offsets that fall
    // hand a sequence's rows to one behind it, and a sequence without rows is met by no search.
    if (s.cu && threadIdx.x >= (uint32_t)kMaxTokens) {
        constexpr uint32_t lookers = kThreads - kMaxTokens;
        for (uint64_t b = (uint64_t)blockIdx.x * lookers + threadIdx.x - kMaxTokens; b < s.batch;
             b += (uint64_t)gridDim.x * lookers)
            if (hf_kv_sequence(s, (uint32_t)b, c.page_shift).bad) atomicOr(err, HF_KERR_CORRUPT);
    }
    if (threadIdx.x < n) {
        const int32_t row = (int32_t)(t0 + threadIdx.x);
        uint32_t b = (uint32_t)row;
        if (s.cu) {  // the last sequence whose first row is at or before this one
            uint32_t lo = 0, hi = s.batch;
            while (lo < hi) {
                const uint32_t mid = (lo + hi) / 2;
                int32_t first;
                if (staged) first = cu_lds[mid + 1];
                else first = s.cu[mid + 1];
                if (first <= row)
                    lo = mid + 1;
                else
                    hi = mid;
            }
            b = lo;
        }
        int64_t code = -1, scale = 0;
        if (b < s.batch) {  // (rows behind the last sequence have no place)
            const hf_kv_seq q = hf_kv_sequence(s, b, c.page_shift);
            const int32_t i = row - q.row0;
            bool bad = q.bad;
            if (!bad && i >= 0 && i < q.n) {
                const uint32_t pos = (uint32_t)(q.past + i);
                const int32_t page = s.table[(int64_t)b * s.table_stride + (pos >> c.page_shift)];
                if ((uint32_t)page < c.n_pages) {
                    const uint32_t off = pos & ((1u << c.page_shift) - 1u);
                    code = (int64_t)page * c.page_stride + (int64_t)off * c.token_stride;
                    scale = (((int64_t)page * c.heads * c.groups) << c.page_shift) + off;
                } else {
                    bad = true;
                }
            }
            if (bad) atomicOr(err, HF_KERR_CORRUPT);
        }
        p.code[threadIdx.x] = code;
        p.scale[threadIdx.x] = scale;
    }
    __syncthreads();
}

// Largest value of a over the 2^k lanes of an aligned group (k >= 2), in every lane of it.
__device__ __forceinline__ uint32_t group_max(uint32_t a, const uint32_t lanes) {
    auto dpp = [](uint32_t x, auto ctrl) {
        return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, decltype(ctrl)::value, 0xF, 0xF, false);
    };
    a = max(a, dpp(a, std::integral_constant<int, 0xB1>{}));  // quad_perm [1,0,3,2]
    a = max(a, dpp(a, std::integral_constant<int, 0x4E>{}));  // quad_perm [2,3,0,1]
    if (lanes >= 8) a = max(a, dpp(a, std::integral_constant<int, 0x141>{}));   // half row mirrored
    if (lanes >= 16) a = max(a, dpp(a, std::integral_constant<int, 0x140>{}));  // row mirrored
    if (lanes >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
        a = max(r[0], r[1]);
    }
    return a;
}

// Eight consecutive elements of a row.
template <int DT>
__device__ __forceinline__ void load8(const hf_g8* p, float (&x)[8]) {
    if constexpr (DT == HF_DT_FP32) {
        const f32x4 a = *(__attribute__((address_space(1))) const f32x4*)p;
        const f32x4 b = *(__attribute__((address_space(1))) const f32x4*)(p + 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = a[i];
            x[4 + i] = b[i];
        }
    } else {
        const hf_u32x4 a = *(const hf_gmem_u32x4*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == HF_DT_BF16) {
                x[2 * i] = __uint_as_float(a[i] << 16);
                x[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
            } else {
                const uint32_t w = a[i];  // (a cast of a[i] itself reads element 0)
                const f16x2 h = __builtin_bit_cast(f16x2, w);
                x[2 * i] = (float)h.x;
                x[2 * i + 1] = (float)h.y;
            }
        }
    }
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(const float a, const float b) {  // two 16-bit values
    if constexpr (DT == HF_DT_BF16) return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
    return __builtin_bit_cast(uint32_t, f16x2{(_Float16)a, (_Float16)b});
}
template <int DT>
__device__ __forceinline__ void store8(hf_g8* p, const float (&x)[8]) {
    if constexpr (DT == HF_DT_FP32) {
        *(__attribute__((address_space(1))) f32x4*)p = f32x4{x[0], x[1], x[2], x[3]};
        *(__attribute__((address_space(1))) f32x4*)(p + 16) = f32x4{x[4], x[5], x[6], x[7]};
    } else {
        hf_u32x4 a;
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = pack2<DT>(x[2 * i], x[2 * i + 1]);
        *(hf_gmem_u32x4*)p = a;
    }
}

// Quantises a lane's eight elements with the scale of their group and stores them.
//   top = max |x| over the finite elements of the group; e = the least integer with
//   top <= largest * 2^e, at least -126; code = x * 2^-e rounded to nearest even.  Both the
//   scaling (a power of two; a subnormal product is below half of the smallest code) and the
//   comparison with the largest value are exact, so a code is the only rounding of an element.
//   An infinity takes the largest code of its sign; NaN stays NaN, in e2m1, which has none, as
//   scale byte 255.  A group of zeros has e = 0.
template <int FMT>
__device__ __forceinline__ void quantise8(float (&x)[8], const uint32_t lanes, hf_g8* code,
                                          hf_g8* scale, const bool put_code, const bool put_scale) {
    typedef kv_fmt<FMT> F;
    uint32_t top = 0;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t a = __float_as_uint(x[i]) & 0x7FFFFFFFu;
        odd |= a >= 0x7F800000u;
        top = max(top, a >= 0x7F800000u ? 0u : a);
    }
    if constexpr (FMT == HF_KV_FP4_E2M1) {
        if (odd) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (x[i] != x[i]) top = 0xFFFFFFFFu;  // outlasts every magnitude of the group
        }
    }
    top = group_max(top, lanes);
    int e = (int)(top >> 23) - 127 - F::exp + ((top & 0x7FFFFFu) > F::mant ? 1 : 0);
    e = top == 0 ? 0 : max(e, -126);
    bool nan = false;
    if constexpr (FMT == HF_KV_FP4_E2M1) {
        nan = top == 0xFFFFFFFFu;
        if (nan) e = 0;
    }
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= inv;
    if (odd) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (fabsf(x[i]) == __builtin_inff()) x[i] = copysignf(F::top, x[i]);
            if (nan && x[i] != x[i]) x[i] = 0.0f;
        }
    }
    if constexpr (FMT == HF_KV_FP4_E2M1) {
        uint32_t w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], 1.0f, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], 1.0f, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], 1.0f, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], 1.0f, 3);
        if (put_code) *(__attribute__((address_space(1))) uint32_t*)code = w;
    } else {
        int w[2] = {0, 0};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if constexpr (FMT == HF_KV_FP8_E4M3) {
                w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h], x[4 * h + 1], w[h], false);
                w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h + 2], x[4 * h + 3], w[h], true);
            } else {
                w[h] = __builtin_amdgcn_cvt_pk_bf8_f32(x[4 * h], x[4 * h + 1], w[h], false);
                w[h] = __builtin_amdgcn_cvt_pk_bf8_f32(x[4 * h + 2], x[4 * h + 3], w[h], true);
            }
        }
        if (put_code) *(hf_gmem_u32x2*)code = hf_u32x2{(uint32_t)w[0], (uint32_t)w[1]};
    }
    if (put_code && put_scale) *scale = nan ? 255 : (uint8_t)(e + 127);
}

template <int FMT>
__device__ __forceinline__ void dequantise8(const hf_g8* code, const uint32_t scale, float (&x)[8]) {
    const float f = __uint_as_float(scale << 23);  // the conversion reads the exponent: 255 is NaN
    if constexpr (FMT == HF_KV_BF16) {
        load8<HF_DT_BF16>(code, x);
    } else if constexpr (FMT == HF_KV_FP16) {
        load8<HF_DT_FP16>(code, x);
    } else if constexpr (FMT == HF_KV_FP4_E2M1) {
        const uint32_t w = *(__attribute__((address_space(1))) const uint32_t*)code;
        f32x2 r[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 0),
                      __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 1),
                      __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 2),
                      __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 3)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = r[i].x;
            x[2 * i + 1] = r[i].y;
        }
    } else {
        const hf_u32x2 w = *(const hf_gmem_u32x2*)code;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f32x2 a, b;
            if constexpr (FMT == HF_KV_FP8_E4M3) {
                a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[h], f, false);
                b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[h], f, true);
            } else {
                a = __builtin_amdgcn_cvt_scalef32_pk_f32_bf8(w[h], f, false);
                b = __builtin_amdgcn_cvt_scalef32_pk_f32_bf8(w[h], f, true);
            }
            x[4 * h] = a.x;
            x[4 * h + 1] = a.y;
            x[4 * h + 2] = b.x;
            x[4 * h + 3] = b.y;
        }
    }
}

// How the pieces of a workgroup's rows are dealt to its threads: piece p of a row is its elements
// 8p .. 8p + 7, head p / (head_dim / 8).  inv = ceil(2^21 / (head_dim / 8)): the quotient is exact
// for the up to 32768 pieces of a row (1024 heads), since inv overshoots by less than 32 / 2^21.
struct kv_deal {
    uint32_t pieces, per_head, inv, tokens;
};

// Bound by memory: 42 k rows of 8 x 128 bf16 to e4m3 (260 MB) in 57 us, 4.6 TB/s (a large copy: 4.9);
// 64 rows in 3.9 us, which is a launch and three dependent loads.
template <int FMT, int DT>
__global__ __launch_bounds__(kThreads) void hf_k_kv_write(const hf_kv_pools c, const hf_kv_seqs s,
                                                          const hf_kv_rows k, const hf_kv_rows v,
                                                          const kv_deal d, uint32_t* err) {
    __shared__ kv_places place;
    __shared__ int32_t cu_lds[kCuLds];
    constexpr int es = DT == HF_DT_FP32 ? 4 : 2;
    const uint32_t t0 = blockIdx.x * d.tokens;
    const uint32_t n = min(d.tokens, s.rows - t0);
    find_places(c, s, t0, n, place, cu_lds, err);
    const uint32_t total = n * d.pieces, lanes = 1u << (c.group_shift - 3);
    uint32_t tok = threadIdx.x / d.pieces, piece = threadIdx.x % d.pieces;
    const uint32_t dtok = kThreads / d.pieces, dpiece = kThreads % d.pieces;
    for (uint32_t i = threadIdx.x; i < total; i += kThreads) {
        const int64_t at = place.code[tok];
        const uint32_t head = (piece * d.inv) >> 21, col = (piece - head * d.per_head) * 8u;
        const int64_t row = t0 + tok;
        const hf_g8* pk = (const hf_g8*)k.p + (row * k.row_stride + (int64_t)head * k.head_stride + col) * es;
        const hf_g8* pv = (const hf_g8*)v.p + (row * v.row_stride + (int64_t)head * v.head_stride + col) * es;
        const int64_t code = at + (int64_t)head * c.head_stride + (int64_t)(col * kv_fmt<FMT>::bits / 8);
        if constexpr (kv_fmt<FMT>::bits == 16) {
            if (at >= 0) {
                if constexpr (DT == HF_DT_FP32) {
                    float x[8], y[8];
                    load8<DT>(pk, x);
                    load8<DT>(pv, y);
                    store8<FMT == HF_KV_BF16 ? HF_DT_BF16 : HF_DT_FP16>((hf_g8*)c.k + code, x);
                    store8<FMT == HF_KV_BF16 ? HF_DT_BF16 : HF_DT_FP16>((hf_g8*)c.v + code, y);
                } else {  // the same type: the bits as they are
                    const hf_u32x4 x = *(const hf_gmem_u32x4*)pk, y = *(const hf_gmem_u32x4*)pv;
                    *(hf_gmem_u32x4*)((hf_g8*)c.k + code) = x;
                    *(hf_gmem_u32x4*)((hf_g8*)c.v + code) = y;
                }
            }
        } else {
            // (the lanes of a group take this turn together: pieces of a row come in whole groups)
            const uint32_t g = col >> c.group_shift;
            const int64_t sc = place.scale[tok] + ((int64_t)(head * c.groups + g) << c.page_shift);
            const bool first = (col & ((1u << c.group_shift) - 1u)) == 0;
            float x[8], y[8];
            load8<DT>(pk, x);
            load8<DT>(pv, y);
            quantise8<FMT>(x, lanes, (hf_g8*)c.k + code, (hf_g8*)c.k_scale + sc, at >= 0, first);
            quantise8<FMT>(y, lanes, (hf_g8*)c.v + code, (hf_g8*)c.v_scale + sc, at >= 0, first);
        }
        tok += dtok;
        piece += dpiece;
        if (piece >= d.pieces) {
            piece -= d.pieces;
            ++tok;
        }
    }
}

// Bound by memory: 41 k rows of 8 x 128 e4m3 to bf16 (254 MB) in 55 us, 4.6 TB/s (into the same outputs
// call after call, which the last cache then holds, 44).
template <int FMT, int DT>
__global__ __launch_bounds__(kThreads) void hf_k_kv_read(const hf_kv_pools c, const hf_kv_seqs s,
                                                         const hf_kv_rows k, const hf_kv_rows v,
                                                         const kv_deal d, uint32_t* err) {
    __shared__ kv_places place;
    __shared__ int32_t cu_lds[kCuLds];
    constexpr int es = DT == HF_DT_FP32 ? 4 : 2;
    const uint32_t t0 = blockIdx.x * d.tokens;
    const uint32_t n = min(d.tokens, s.rows - t0);
    find_places(c, s, t0, n, place, cu_lds, err);
    const uint32_t total = n * d.pieces;
    uint32_t tok = threadIdx.x / d.pieces, piece = threadIdx.x % d.pieces;
    const uint32_t dtok = kThreads / d.pieces, dpiece = kThreads % d.pieces;
    for (uint32_t i = threadIdx.x; i < total; i += kThreads) {
        const int64_t at = place.code[tok];
        const uint32_t head = (piece * d.inv) >> 21, col = (piece - head * d.per_head) * 8u;
        if (at >= 0) {
            const int64_t row = t0 + tok;
            const int64_t code = at + (int64_t)head * c.head_stride + (int64_t)(col * kv_fmt<FMT>::bits / 8);
            uint32_t sk = 0, sv = 0;
            if constexpr (kv_fmt<FMT>::bits != 16) {
                const uint32_t g = col >> c.group_shift;
                const int64_t sc = place.scale[tok] + ((int64_t)(head * c.groups + g) << c.page_shift);
                sk = ((const hf_g8*)c.k_scale)[sc];
                sv = ((const hf_g8*)c.v_scale)[sc];
            }
            float x[8], y[8];
            dequantise8<FMT>((const hf_g8*)c.k + code, sk, x);
            dequantise8<FMT>((const hf_g8*)c.v + code, sv, y);
            store8<DT>((hf_g8*)k.p + (row * k.row_stride + (int64_t)head * k.head_stride + col) * es, x);
            store8<DT>((hf_g8*)v.p + (row * v.row_stride + (int64_t)head * v.head_stride + col) * es, y);
        }
        tok += dtok;
        piece += dpiece;
        if (piece >= d.pieces) {
            piece -= d.pieces;
            ++tok;
        }
    }
}

kv_deal deal_of(const hf_kv_pools& c, const uint32_t rows, const int num_cu) {
    kv_deal d;
    d.per_head = c.head_dim / 8u;
    d.pieces = c.heads * d.per_head;
    d.inv = ((1u << 21) + d.per_head - 1u) / d.per_head;
    // one piece per thread while that leaves the GPU room (single tokens: latency), four when
    // there is work for every compute unit eight times over
    const uint64_t threads = (uint64_t)rows * d.pieces;
    const uint32_t turns = threads >= (uint64_t)num_cu * 8u * kThreads * 4u ? 4u : 1u;
    d.tokens = kThreads * turns / d.pieces;
    if (d.tokens < 1u) d.tokens = 1u;
    if (d.tokens > (uint32_t)kMaxTokens) d.tokens = kMaxTokens;
    return d;
}

// Accepted drafts move to the first places behind the past: draft path[i] of sequence b to position
// past + i, for i < path_len[b].  A path ascends, so a row's place is never behind its source, and
// the rows of a later turn of the loop come from behind every place an earlier turn wrote; inside
// a turn all loads come before all stores.  One workgroup per sequence and head: 64 trees of up to
// 48 drafts take 5.0 us, one tree 4.1, a launch and its chain of loads.
__global__ __launch_bounds__(kThreads) void hf_k_kv_keep(const hf_kv_pools c, const hf_kv_seqs s,
                                                         const int32_t* path, const int64_t path_stride,
                                                         const uint32_t path_width, const int32_t* path_len,
                                                         int32_t* new_len, const uint32_t row_bytes,
                                                         uint32_t* err) {
    const uint32_t b = blockIdx.x, head = blockIdx.y;
    const hf_kv_seq q = hf_kv_sequence(s, b, c.page_shift);
    const int32_t m = path_len[b];
    const int32_t* p = path + (int64_t)b * path_stride;
    const int32_t* table = s.table + (int64_t)b * s.table_stride;
    bool bad = q.bad || m < 0 || m > q.n || (uint32_t)m > path_width;
    if (!bad) {
        for (int32_t i = (int32_t)threadIdx.x; i < m; i += kThreads) {
            // (the table is read for steps that can be taken only: both places are the sequence's own)
            bad = bad || !hf_kv_path_ok(p, i, q.n) ||
                  (uint32_t)table[(uint32_t)(q.past + p[i]) >> c.page_shift] >= c.n_pages ||
                  (uint32_t)table[(uint32_t)(q.past + i) >> c.page_shift] >= c.n_pages;
        }
    }
    bad = __syncthreads_or(bad) != 0;
    if (threadIdx.x == 0 && head == 0) {
        new_len[b] = bad ? s.kv_len[b] : q.past + m;
        if (bad) atomicOr(err, HF_KERR_CORRUPT);
    }
    if (bad) return;
    const uint32_t lanes = row_bytes / 16u, turn = kThreads / lanes;
    const uint32_t r = threadIdx.x / lanes, sub = threadIdx.x % lanes;
    for (uint32_t i0 = 0; i0 < (uint32_t)m; i0 += turn) {
        const uint32_t i = i0 + r;
        const bool mine = r < turn && i < (uint32_t)m;
        hf_u32x4 k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
        uint8_t sk = 0, sv = 0;
        int64_t to = 0, to_scale = 0;
        if (mine) {
            const uint32_t mask = (1u << c.page_shift) - 1u;
            const uint32_t from = (uint32_t)(q.past + p[i]), dst = (uint32_t)q.past + i;
            const int64_t fp = table[from >> c.page_shift], dp = table[dst >> c.page_shift];
            const int64_t at = fp * c.page_stride + (int64_t)(from & mask) * c.token_stride +
                               (int64_t)head * c.head_stride + 16u * sub;
            to = dp * c.page_stride + (int64_t)(dst & mask) * c.token_stride +
                 (int64_t)head * c.head_stride + 16u * sub;
            k = *(const hf_gmem_u32x4*)((const hf_g8*)c.k + at);
            v = *(const hf_gmem_u32x4*)((const hf_g8*)c.v + at);
            if (sub < c.groups) {  // (a row of 16 bytes or more per scale: a lane for every group)
                const int64_t f = ((fp * c.heads + head) * c.groups + sub) << c.page_shift;
                to_scale = (((dp * c.heads + head) * c.groups + sub) << c.page_shift) + (dst & mask);
                sk = ((const hf_g8*)c.k_scale)[f + (from & mask)];
                sv = ((const hf_g8*)c.v_scale)[f + (from & mask)];
            }
        }
        __syncthreads();
        if (mine) {
            *(hf_gmem_u32x4*)((hf_g8*)c.k + to) = k;
            *(hf_gmem_u32x4*)((hf_g8*)c.v + to) = v;
            if (sub < c.groups) {
                ((hf_g8*)c.k_scale)[to_scale] = sk;
                ((hf_g8*)c.v_scale)[to_scale] = sv;
            }
        }
        __syncthreads();
    }
}

}  // namespace

// format x element type of the rows; a 16-bit cache takes and gives its own type or fp32
#define HF_KV_CASE(KERNEL, F, T)                                                                  \
    case (F) * 4 + (T):                                                                           \
        hipLaunchKernelGGL((KERNEL<F, T>), dim3(grid), dim3(kThreads), 0, st, c, s, k, v, d, err); \
        break;
#define HF_KV_CASES(KERNEL)                    \
    switch (format * 4 + dtype) {              \
        HF_KV_CASE(KERNEL, HF_KV_BF16, HF_DT_BF16)     \
        HF_KV_CASE(KERNEL, HF_KV_BF16, HF_DT_FP32)     \
        HF_KV_CASE(KERNEL, HF_KV_FP16, HF_DT_FP16)     \
        HF_KV_CASE(KERNEL, HF_KV_FP16, HF_DT_FP32)     \
        HF_KV_CASE(KERNEL, HF_KV_FP8_E4M3, HF_DT_BF16) \
        HF_KV_CASE(KERNEL, HF_KV_FP8_E4M3, HF_DT_FP16) \
        HF_KV_CASE(KERNEL, HF_KV_FP8_E4M3, HF_DT_FP32) \
        HF_KV_CASE(KERNEL, HF_KV_FP8_E5M2, HF_DT_BF16) \
        HF_KV_CASE(KERNEL, HF_KV_FP8_E5M2, HF_DT_FP16) \
        HF_KV_CASE(KERNEL, HF_KV_FP8_E5M2, HF_DT_FP32) \
        HF_KV_CASE(KERNEL, HF_KV_FP4_E2M1, HF_DT_BF16) \
        HF_KV_CASE(KERNEL, HF_KV_FP4_E2M1, HF_DT_FP16) \
        HF_KV_CASE(KERNEL, HF_KV_FP4_E2M1, HF_DT_FP32) \
        default:                                       \
            break;                                     \
    }

void hf_launch_kv_write(const hf_kv_pools& c, const hf_kv_seqs& s, const hf_kv_rows& k,
                        const hf_kv_rows& v, int dtype, int format, uint32_t* err, int num_cu,
                        hipStream_t st) {
    const kv_deal d = deal_of(c, s.rows, num_cu);
    const uint32_t grid = (s.rows + d.tokens - 1u) / d.tokens;
    HF_KV_CASES(hf_k_kv_write)
}
void hf_launch_kv_read(const hf_kv_pools& c, const hf_kv_seqs& s, const hf_kv_rows& k,
                       const hf_kv_rows& v, int dtype, int format, uint32_t* err, int num_cu,
                       hipStream_t st) {
    const kv_deal d = deal_of(c, s.rows, num_cu);
    const uint32_t grid = (s.rows + d.tokens - 1u) / d.tokens;
    HF_KV_CASES(hf_k_kv_read)
}
void hf_launch_kv_keep(const hf_kv_pools& c, const hf_kv_seqs& s, const int32_t* path,
                       int64_t path_stride, uint32_t path_width, const int32_t* path_len,
                       int32_t* new_len, uint32_t row_bytes, uint32_t* err, hipStream_t st) {
    hipLaunchKernelGGL(hf_k_kv_keep, dim3(s.batch, c.heads), dim3(kThreads), 0, st, c, s, path,
                       path_stride, path_width, path_len, new_len, row_bytes, err);
}
