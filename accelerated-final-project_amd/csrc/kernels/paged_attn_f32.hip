// fp32 kernels of attention over a paged cache (paged_attn_impl.hpp).
#include "paged_attn_impl.hpp"

namespace atn {

hipError_t launch_paged_f32(const PagedArgs& a, hipStream_t st) {
    paged_go<float>(a, st);
    return hipGetLastError();
}

}  // namespace atn
