// attention_sinks.hip -- attention through a sliding window beside which the
// first positions stay visible (attention_kernels.hpp, kSinks).
#include "attention_kernels.hpp"

namespace lcml {

hipError_t launch_attention_sinks(const AttentionArgs &a, void *work, hipStream_t s, const char **kernel) {
    Plan p = make_plan(a.t.seqs, a.q_heads, a.t.heads, a.t.dim, a.max_q, a.max_kv, a.window, a.sinks);
    return launch_form<kSinks>(a, p, work, s, kernel);
}

}  // namespace lcml
