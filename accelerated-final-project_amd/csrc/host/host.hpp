// What the host files share: attn_api.cpp's device state and workspaces.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>

namespace atn_host {

// The first bytes of every workspace hold synchronization words of the
// attention calls; other calls leave them alone and start behind.
constexpr size_t kSyncRegion = 40960;

int fail(hipError_t e);     // records e, returns ATN_ERR_HIP
int device(int* dev);       // the current device, or ATN_ERR_NO_DEVICE
size_t workspace_cap();     // cap of the library's own workspaces
// the stream's library workspace, of at least `bytes` (ATN_ERR_CAPTURE where it
// would have to grow during a capture)
int workspace(size_t bytes, hipStream_t stream, void** ws);

}  // namespace atn_host
