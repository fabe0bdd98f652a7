// Attention over pools of F16 pages (paged.hpp).
#include "paged.hpp"

namespace chm {

hipError_t launch_paged_f16(const PagedAttention& a, uint32_t octets, hipStream_t stream) {
    return launch_paged<kF16>(a, octets, stream);
}

}  // namespace chm
