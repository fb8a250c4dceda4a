// attention.hip -- calls of attention over the E4M3 KV cache, and their plans
// (attention_kernels.hpp).
#include "attention_kernels.hpp"

namespace lcml {

int64_t attention_workspace(int64_t tokens, int64_t seqs, int64_t q_heads, int64_t kv_heads, int64_t dim,
                            int64_t max_q, int64_t max_kv) {
    const Plan p = make_plan(seqs, q_heads, kv_heads, dim, max_q, max_kv, 0, 0);  // a window only takes parts away
    return p.sp.splits > 1 ? tokens * q_heads * p.sp.splits * (dim + 1) * 4 : 0;
}

int64_t attention_groups(int64_t seqs, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t max_q, int64_t max_kv) {
    return make_plan(seqs, q_heads, kv_heads, dim, max_q, max_kv, 0, 0).groups;
}

hipError_t launch_attention(const AttentionArgs &a, void *work, hipStream_t s, const char **kernel) {
    Plan p = make_plan(a.t.seqs, a.q_heads, a.t.heads, a.t.dim, a.max_q, a.max_kv, a.window, 0);
    return launch_form<kPlain>(a, p, work, s, kernel);
}

}  // namespace lcml
