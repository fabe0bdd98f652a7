// Attention over F16 caches (attention.hpp).
#include "attention.hpp"

namespace chm {

hipError_t launch_attention_f16(const Attention& a, const AttentionPlan& plan, hipStream_t stream) {
    return launch_format<kF16>(a, plan, stream);
}

}  // namespace chm
