// Attention over Q4_0 caches (attention.hpp).
#include "attention.hpp"

namespace chm {

hipError_t launch_attention_q4_0(const Attention& a, const AttentionPlan& plan, hipStream_t stream) {
    return launch_format<kQ4_0>(a, plan, stream);
}

}  // namespace chm
