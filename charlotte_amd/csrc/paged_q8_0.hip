// Attention over pools of Q8_0 pages (paged.hpp).
#include "paged.hpp"

namespace chm {

hipError_t launch_paged_q8_0(const PagedAttention& a, uint32_t octets, hipStream_t stream) {
    return launch_paged<kQ8_0>(a, octets, stream);
}

}  // namespace chm
