// What the library's source files share on the host side.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

namespace dsv4 {

// Test switches (dsv4_debug_set_flags, dsv4_debug_set_wait), read once per call.
struct HostState {
    int flags;
    unsigned long long wait_ns;
    int drop_tile;
};
HostState host_state();

// SMs of the current device.
int device_sms();

// cuTensorMapEncodeTiled, looked up through the runtime so that the library does not link against libcuda.
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                   CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled_fn();

}  // namespace dsv4
