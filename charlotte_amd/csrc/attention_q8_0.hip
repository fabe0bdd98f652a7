// Attention over Q8_0 caches (attention.hpp).
#include "attention.hpp"

namespace chm {

hipError_t launch_attention_q8_0(const Attention& a, const AttentionPlan& plan, hipStream_t stream) {
    return launch_format<kQ8_0>(a, plan, stream);
}

}  // namespace chm
