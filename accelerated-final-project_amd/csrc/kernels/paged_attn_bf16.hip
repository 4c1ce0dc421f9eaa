// bf16 kernels of attention over a paged cache, head_d <= 256 (paged_attn_impl.hpp).
#include "paged_attn_impl.hpp"

namespace atn {

hipError_t launch_paged_narrow_bf16(const PagedArgs& a, hipStream_t st) {
    go_narrow<uint16_t>(a, st);
    return hipGetLastError();
}

}  // namespace atn
