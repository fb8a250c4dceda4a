// attention_shared.hip -- attention for groups of sequences that share their
// first tokens (attention_kernels.hpp, kPrefix and kOwn).
//
// What a group shares is read once, for the rows of all its sequences
// together, which then also fill the matrix instructions' columns; each
// sequence's own tokens as ever.  Both leave parts (results divided by their
// sums, and the sums' logarithms), and one join puts a row's together:
//   o = sum_p o_p 2^(L_p) / sum_p 2^(L_p),   L_p = log2 sum_(j in p) w_j
#include "attention_kernels.hpp"

namespace lcml {
namespace {

constexpr int kMostParts = kMostSplits / 2;  // of the prefix, and of the own tokens

// fewer parts where there are too many for the join
void cap_parts(Plan &p) {
    if (p.sp.splits <= kMostParts) return;
    p.groups = p.groups / p.sp.splits * kMostParts;
    p.sp.chunk = (int32_t)((((int64_t)p.sp.chunk * p.sp.splits + kMostParts - 1) / kMostParts + 63) & ~63);
    p.sp.splits = kMostParts;
}

struct SharedPlan {
    Plan prefix, own;
};
SharedPlan make_shared_plan(int64_t tokens, int64_t seqs, int64_t groups, int64_t q_heads, int64_t kv_heads, int64_t dim,
                            int64_t max_q, int64_t max_own, int64_t max_prefix) {
    SharedPlan s{};
    s.own = make_plan(seqs, q_heads, kv_heads, dim, max_q, max_own + 63, 0, 0);  // from a multiple of 64 on
    cap_parts(s.own);
    s.own.sp.parts = s.own.sp.splits;
    if (groups == 0) return s;
    // the tiles of all groups' rows, and one more for each group that ends inside a tile
    const int64_t rows = tokens * (q_heads / kv_heads);
    s.prefix = divide(few_rows(kv_heads, dim, rows, max_prefix), kv_heads, rows, max_prefix);
    cap_parts(s.prefix);
    s.prefix.sp.tiles += (int32_t)(groups - 1);
    s.prefix.groups = kv_heads * s.prefix.sp.tiles * s.prefix.sp.splits;
    s.own.sp.first = s.prefix.sp.splits;
    s.prefix.sp.parts = s.own.sp.parts = s.prefix.sp.splits + s.own.sp.splits;
    return s;
}

template <int NQ, int NP>
hipError_t launch_shared_t(const AttentionArgs &prefix, const AttentionArgs &own, const SharedPlan &p, hipStream_t s) {
    hipError_t err = p.prefix.groups ? start_attention<kPrefix, NQ, NP>(prefix, p.prefix, s) : hipSuccess;
    if (err == hipSuccess) err = start_attention<kOwn, NQ, NP>(own, p.own, s);
    return err == hipSuccess ? start_join<kOwn, NP>(own, p.own.sp, p.own.sp.parts, s) : err;
}

}  // namespace

int64_t attention_shared_workspace(int64_t tokens, int64_t seqs, int64_t groups, int64_t q_heads, int64_t kv_heads,
                                   int64_t dim, int64_t max_q, int64_t max_own, int64_t max_prefix, int64_t *workgroups) {
    const SharedPlan p = make_shared_plan(tokens, seqs, groups, q_heads, kv_heads, dim, max_q, max_own, max_prefix);
    *workgroups = p.prefix.groups > p.own.groups ? p.prefix.groups : p.own.groups;
    return tokens * q_heads * p.own.sp.parts * (dim + 1) * 4;
}

hipError_t launch_attention_shared(const AttentionArgs &own, const int32_t *prefix_table, int64_t prefix_stride,
                                   int64_t prefix_cols, int64_t max_prefix, void *work, hipStream_t s,
                                   const char **kernel) {
    AttentionArgs prefix = own;
    prefix.t.table = prefix_table, prefix.t.table_stride = prefix_stride, prefix.t.table_cols = (int32_t)prefix_cols;
    prefix.max_q = own.t.tokens, prefix.max_kv = max_prefix, prefix.causal = 0;  // all rows lie behind it
    SharedPlan p = make_shared_plan(own.t.tokens, own.t.seqs, own.groups, own.q_heads, own.t.heads, own.t.dim, own.max_q,
                                    own.max_kv, max_prefix);
    if (p.prefix.groups) set_divisors(p.prefix.sp, prefix);
    set_divisors(p.own.sp, own);
    p.prefix.sp.o = p.own.sp.o = static_cast<float *>(work);
    p.prefix.sp.lse = p.own.sp.lse = p.own.sp.o + (int64_t)own.t.tokens * own.q_heads * p.own.sp.parts * own.t.dim;
    *kernel = p.prefix.few ? (p.own.few ? "attention_few, attention_few, attention_join" : "attention_few, attention_many, attention_join")
                           : (p.own.few ? "attention_many, attention_few, attention_join" : "attention_many, attention_many, attention_join");
    if (own.q_bf16) return own.o_bf16 ? launch_shared_t<1, 1>(prefix, own, p, s) : launch_shared_t<1, 2>(prefix, own, p, s);
    return own.o_bf16 ? launch_shared_t<2, 1>(prefix, own, p, s) : launch_shared_t<2, 2>(prefix, own, p, s);
}

}  // namespace lcml
