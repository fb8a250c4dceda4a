// attention_shared.hip -- calls of attention behind shared prefixes
// (attention_shared.hpp), and its kernels for bf16 queries.
#include "attention_shared.hpp"

namespace lcml {

int64_t attention_shared_workspace(int64_t tokens, int64_t seqs, int64_t groups, int64_t q_heads, int64_t kv_heads,
                                   int64_t dim, int64_t max_q, int64_t max_own, int64_t max_prefix, int64_t *workgroups) {
    const SharedPlan p = make_shared_plan(tokens, seqs, groups, q_heads, kv_heads, dim, max_q, max_own, max_prefix);
    const int64_t joined = make_join(tokens * q_heads, p.own.sp.parts, dim).groups, both = p.prefix.groups + p.own.groups;
    *workgroups = both > joined ? both : joined;
    return tokens * q_heads * p.own.sp.parts * (dim + 1) * 4;
}

hipError_t launch_attention_shared(const AttentionArgs &own, const int32_t *prefix_table, int64_t prefix_stride,
                                   int64_t prefix_cols, int64_t max_prefix, void *work, hipStream_t s,
                                   const char **kernel) {
    return own.q_bf16 ? launch_shared<1>(own, prefix_table, prefix_stride, prefix_cols, max_prefix, work, s, kernel)
                      : launch_attention_shared_f32(own, prefix_table, prefix_stride, prefix_cols, max_prefix, work, s, kernel);
}

}  // namespace lcml
