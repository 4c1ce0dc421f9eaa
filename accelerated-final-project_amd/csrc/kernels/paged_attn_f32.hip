// fp32 kernels of attention over a paged cache, head_d <= 256 (paged_attn_impl.hpp).
#include "paged_attn_impl.hpp"

namespace atn {

hipError_t launch_paged_narrow_f32(const PagedArgs& a, hipStream_t st) {
    go_narrow<float>(a, st);
    return hipGetLastError();
}

}  // namespace atn
