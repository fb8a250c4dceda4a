// kv_cache.hpp -- the E4M3 KV cache as the kernels see it: where a token's
// codes lie, a page's scale, and which tokens a call works on.
//
// A (page, head) block is T * D bytes, T tokens in blocks of 16, in the order
// in which attention's matrix instructions take their operands:
//   K: [D / 16][16 tokens][16]       a lane's 16 bytes are 16 elements of one
//                                    token (the reduction of q k^T)
//   V: [4 groups of 4 tokens][D][4]  a lane's word is four tokens of one
//                                    column (the reduction of p v)
// so a wavefront's 16-byte loads are contiguous in both, and neither codes nor
// probabilities change lanes on their way into the matrix cores.
//
// Scales are powers of two: when a later token raises its page's, the codes
// that stay are encoded again without a second rounding (except where they
// fall below the smallest normal code, 2^-6), and the product of a code and
// its scale is exact in fp32 and bf16.
#pragma once

#include "lcml_device.hpp"

namespace lcml {

struct KvTokens {
    const int32_t *table;   // [seqs][table_stride]: pages of a sequence
    const int32_t *kv_len;  // [seqs]: tokens of a sequence, this call's included
    const int32_t *cu;      // [seqs + 1]: the call's rows of each sequence
    int64_t table_stride;
    int32_t table_cols, seqs, tokens, pages;
    int32_t heads, dim, tshift;  // KV heads, head size, log2 of a page's tokens
};

// a sequence's rows and the position of its first one; n <= 0: none (an
// out-of-range row range counts as none)
struct SeqRows {
    int32_t row0, n, pos0, len;
};

__device__ inline SeqRows seq_rows(const KvTokens &t, int32_t b) {
    SeqRows r;
    r.row0 = t.cu[b];
    const int32_t end = t.cu[b + 1];
    r.n = r.row0 < 0 || end > t.tokens || end < r.row0 ? 0 : end - r.row0;
    r.len = t.kv_len[b];
    if (r.len < 0) r.len = 0;
    r.pos0 = r.len - r.n;  // negative: those rows have no token
    return r;
}

// the page at place c of sequence b's table, or -1
__device__ inline int32_t page_of(const KvTokens &t, int32_t b, int32_t c) {
    if (c < 0 || c >= t.table_cols) return -1;
    const int32_t p = t.table[(int64_t)b * t.table_stride + c];
    return p >= 0 && p < t.pages ? p : -1;
}

// byte of element e (of D) of slot t in its (page, head) block
__host__ __device__ inline int64_t k_place(int32_t t, int32_t e, int32_t D) {
    return (int64_t)(t >> 4) * 16 * D + (e >> 4) * 256 + (t & 15) * 16 + (e & 15);
}
__host__ __device__ inline int64_t v_place(int32_t t, int32_t e, int32_t D) {
    return (int64_t)(t >> 2) * 4 * D + e * 4 + (t & 3);
}

// One attention call.
struct AttentionArgs {
    KvTokens t;
    const void *q;
    void *o;
    const uint8_t *k, *v;
    const float *ks, *vs;
    int64_t q_token, q_head, o_token, o_head;  // strides in elements
    int64_t max_q, max_kv, window;             // window 0: none
    int32_t q_heads, causal, q_bf16, o_bf16;
    float scale;
    uint32_t sinks;  // first positions that the window does not hide
    // groups of sequences that share their first tokens (none: groups 0)
    const int32_t *group_seq, *prefix_len;  // [groups + 1] first sequences, [groups] shared tokens
    int32_t groups;
};

// One call that plans a step (kv_plan.hip).
struct KvPlan {
    const int32_t *new_tokens, *ended, *first_own;  // [seqs]; the last two may be NULL
    const int32_t *kv_len_in, *free_in;             // [seqs], [1]
    int32_t *free_pages;                            // [pages], the first free_in[0] are free
    int32_t *table;
    int64_t table_stride;
    int32_t table_cols, seqs, pages, tshift;
    int32_t *kv_len, *cu_q, *left;  // [seqs], [seqs + 1], [1]
    int32_t *positions;             // [tokens] or NULL
    int64_t *slots;                 // [tokens] or NULL
    int64_t tokens;
    int64_t *work;  // [seqs + 2]: new columns before each sequence, all of them, two words (kv_plan.hip)
};

// the smallest power of two s >= 2^-126 with a <= 448 s, for finite a >= 0:
// 448 = 1.75 * 2^8, so s is 2^(e-8), or 2^(e-7) where a's significand passes
// 1.75
__host__ __device__ inline float page_scale(float a) {
    const uint32_t u = f32_bits(a);
    const int32_t e = (int32_t)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return bits_f32((uint32_t)(e < 1 ? 1 : e) << 23);
}

}  // namespace lcml
