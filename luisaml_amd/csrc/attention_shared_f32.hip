// attention_shared_f32.hip -- attention behind shared prefixes, its kernels for
// fp32 queries (attention_shared.hpp).
#include "attention_shared.hpp"

namespace lcml {

hipError_t launch_attention_shared_f32(const AttentionArgs &own, const int32_t *prefix_table, int64_t prefix_stride,
                                       int64_t prefix_cols, int64_t max_prefix, void *work, hipStream_t s,
                                       const char **kernel) {
    return launch_shared<2>(own, prefix_table, prefix_stride, prefix_cols, max_prefix, work, s, kernel);
}

}  // namespace lcml
