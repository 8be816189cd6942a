// Shared by the KV-cache kernels: what a launch gets, formats, places of rows in the page pools.
#pragma once

#include "hf_common.h"

// One cache as the kernels see it (hf_kv_cache, checked; strides in bytes).
struct hf_kv_pools {
    uint8_t* k;
    uint8_t* v;
    uint8_t* k_scale;  // [n_pages][heads][groups][page_size], NULL for the 16-bit formats
    uint8_t* v_scale;
    uint32_t page_stride;  // (strides stay below 2^32 and in 32 bits: scalar registers are short)
    uint32_t token_stride;
    uint32_t head_stride;
    uint32_t n_pages;
    uint32_t page_shift;  // page_size = 1 << page_shift, at least 8 tokens
    uint32_t heads;
    uint32_t head_dim;    // multiple of 32, at most 256
    uint32_t group_shift; // elements of a row that share a scale = 1 << group_shift
    uint32_t groups;      // head_dim >> group_shift (0 for the 16-bit formats)
};

// The sequences of a call: rows cu[b] .. cu[b + 1] - 1 of the row tensors are the last rows of
// sequence b, which has kv_len[b] tokens in the pages table[b][*].  cu == NULL: one row each.
struct hf_kv_seqs {
    const int32_t* cu;
    const int32_t* kv_len;
    const int32_t* table;
    uint32_t table_stride;
    uint32_t width;  // pages in a row of the table
    uint32_t batch;
    uint32_t rows;   // rows of the row tensors
    uint32_t most;   // rows a sequence has at most
};

// Row tensors [rows][heads][head_dim], strides in elements, head_dim contiguous.
struct hf_kv_rows {
    void* p;
    uint32_t row_stride;
    uint32_t head_stride;
};

// Whether rows of `dim` elements, at i row_stride + j head_stride for i < rows and j < heads, lie on one
// another.  Beside the two nested orders any layout is fine whose rows stay apart: for every distance in
// heads the rows nearest to it are looked at.
inline bool hf_kv_rows_touch(const uint64_t rows, const uint64_t heads, const uint64_t row_stride,
                             const uint64_t head_stride, const uint64_t dim) {
    if (rows == 0 || heads == 0) return false;
    if ((rows > 1 && row_stride < dim) || (heads > 1 && head_stride < dim)) return true;
    if (rows == 1 || heads == 1) return false;
    if (row_stride >= (heads - 1) * head_stride + dim || head_stride >= (rows - 1) * row_stride + dim) return false;
    for (uint64_t j = 1; j < heads; ++j) {
        const uint64_t at = j * head_stride, i = at / row_stride;
        if (i < rows && at - i * row_stride < dim) return true;
        if (i + 1 < rows && (i + 1) * row_stride - at < dim) return true;
    }
    return false;
}

// Whether two row tensors of the same strides, the second `apart` elements behind the first, have an element
// in common: for every distance in heads the two rows nearest to it are looked at.
inline bool hf_kv_rows_meet(const int64_t rows, const int64_t heads, const int64_t row_stride,
                            const int64_t head_stride, const int64_t dim, const int64_t apart) {
    if (rows == 0 || heads == 0) return false;
    const int64_t extent = (rows - 1) * row_stride + (heads - 1) * head_stride + dim;
    if (apart >= extent || apart <= -extent) return false;
    for (int64_t j = 1 - heads; j < heads; ++j) {
        const int64_t rest = apart - j * head_stride;
        int64_t i = row_stride ? rest / row_stride : 0;
        if (i * row_stride > rest) --i;  // (down, also below zero)
        for (int64_t at = i; at <= i + 1; ++at) {
            const int64_t off = rest - (at <= -rows ? 1 - rows : at >= rows ? rows - 1 : at) * row_stride;
            if (off < dim && off > -dim) return true;
        }
    }
    return false;
}

struct hf_kv_attend_args {
    hf_kv_pools c;
    hf_kv_seqs s;
    hf_kv_rows q;
    hf_kv_rows out;
    float* lse;            // [rows][q_heads], NULL: not wanted
    const uint32_t* mask;  // [rows][mask_words], NULL: causal
    uint32_t mask_words;
    uint32_t per;          // query heads per cache head
    float scale_log2;      // softmax scale x log2(e)
    float* part;           // partial outputs of the units, [units][rows of a tile][padded head_dim]
    float* part_ml;        // their maxima and two sums, [units][rows of a tile][4]
    uint32_t* plan;        // [batch + 1][4]: the cut (of few sequences: for joining only)
    uint32_t target;       // units the call is cut into, about
    uint32_t min_steps;    // tokens / 32 a unit has at least
    uint32_t units;        // workgroups of the call, and room of the partial buffers
    uint32_t join;         // units may have to be joined (the partial buffers exist)
    uint32_t* err;
};

// up to this many sequences, attention finds its units without a launch in front
constexpr uint32_t HF_KV_OWN_CUT = 128;

int hf_kv_attend_tile_rows(uint32_t max_q, uint32_t per, uint32_t head_dim);
void hf_launch_kv_write(const hf_kv_pools& c, const hf_kv_seqs& s, const hf_kv_rows& k,
                        const hf_kv_rows& v, int dtype, int format, uint32_t* d_err, int num_cu,
                        hipStream_t st);
void hf_launch_kv_read(const hf_kv_pools& c, const hf_kv_seqs& s, const hf_kv_rows& k,
                       const hf_kv_rows& v, int dtype, int format, uint32_t* d_err, int num_cu,
                       hipStream_t st);
void hf_launch_kv_keep(const hf_kv_pools& c, const hf_kv_seqs& s, const int32_t* path,
                       int64_t path_stride, uint32_t path_width, const int32_t* path_len,
                       int32_t* new_len, uint32_t row_bytes, uint32_t* d_err, hipStream_t st);
void hf_launch_kv_attend(const hf_kv_attend_args& a, int dtype, int format, int tile_rows,
                         hipStream_t st);

#ifdef __HIPCC__
typedef __attribute__((address_space(1))) uint8_t hf_g8;
typedef __attribute__((address_space(1))) const int32_t hf_gi32;

// Sequence b of a call, from the device's own lists.  Lists that do not describe rows of the call
// (offsets that fall or leave the row tensors, more rows than tokens, more tokens than the table
// holds or than 2^31 - 65536, so that the numbers of tokens a little behind the last stay positive)
// give n = 0 and bad = true: nothing of such a sequence is read or written.
struct hf_kv_seq {
    int32_t row0, n, past, len;
    bool bad;
};
__host__ __device__ __forceinline__ hf_kv_seq hf_kv_sequence(const hf_kv_seqs& s, const uint32_t b,
                                                             const uint32_t page_shift) {
    hf_kv_seq q;
    int32_t lo = (int32_t)b, hi = (int32_t)b + 1;
    if (s.cu) {
        lo = s.cu[b];
        hi = s.cu[b + 1];
    }
    q.len = s.kv_len[b];
    q.row0 = lo;
    q.n = (int32_t)((uint32_t)hi - (uint32_t)lo);  // (may wrap: such lists are bad)
    q.past = (int32_t)((uint32_t)q.len - (uint32_t)q.n);
    q.bad = lo < 0 || hi < lo || (uint32_t)hi > s.rows || (uint32_t)q.n > s.most || q.len < q.n ||
            q.len > 0x7FFF0000 || (uint64_t)(uint32_t)q.len > ((uint64_t)s.width << page_shift);
    if (q.bad) {
        q.row0 = 0;
        q.n = 0;
        q.past = 0;
        q.len = 0;
    }
    return q;
}
// Whether step i of a path, draft path[i] of a sequence's n rows to place i, can be taken: it is one of the
// rows and behind the draft of the step before.  A step is looked at for itself alone: what the steps in
// front of it hold may be anything.
__host__ __device__ __forceinline__ bool hf_kv_path_ok(const int32_t* path, const int32_t i, const int32_t n) {
    const int32_t j = path[i];
    return j >= 0 && j < n && (i == 0 || path[i - 1] < j);
}
#endif
