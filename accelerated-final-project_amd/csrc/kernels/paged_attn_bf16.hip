// bf16 kernels of attention over a paged cache (paged_attn_impl.hpp).
#include "paged_attn_impl.hpp"

namespace atn {

hipError_t launch_paged_bf16(const PagedArgs& a, hipStream_t st) {
    paged_go<uint16_t>(a, st);
    return hipGetLastError();
}

}  // namespace atn
