// Attention over pools of Q4_0 pages (paged.hpp).
#include "paged.hpp"

namespace chm {

hipError_t launch_paged_q4_0(const PagedAttention& a, uint32_t octets, hipStream_t stream) {
    return launch_paged<kQ4_0>(a, octets, stream);
}

}  // namespace chm
