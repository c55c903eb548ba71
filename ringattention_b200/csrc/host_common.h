// Host helpers shared by the library's translation units (defined in ring_attention.cu).
#pragma once

#include <atomic>
#include <cstdint>
#include <mutex>

#include <cuda.h>
#include <cuda_runtime.h>

namespace ring_host {

// Stores the thread's error text (ring_last_error_string) and returns `code`.
int fail(int code, const char* fmt, ...);

#define RING_CUDA(call)                                                                              \
    do {                                                                                             \
        cudaError_t e_ = (call);                                                                     \
        if (e_ != cudaSuccess)                                                                       \
            return ring_host::fail(RING_ERR_CUDA, "%s failed: %s (%s:%d)", #call, cudaGetErrorString(e_), __FILE__, \
                                   __LINE__);                                                        \
    } while (0)

extern std::atomic<int64_t> g_launches;  // kernels launched in this process

struct DeviceState {
    int* d_status = nullptr;  // device status word written by kernels whose bounded waits ran out
    int sm_count = 0;
    bool attr_set[12] = {};  // [one-CTA | pair | pair with two threads per row][dim == 128][bf16]: shared-memory attribute set
    bool paged_attr_set[32] = {};  // the same for the paged-cache kernels
};

extern std::mutex g_dev_mutex;

// State of the current device; the first call on a device allocates its status word.
int device_state(DeviceState** out);

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int encode_fn(EncodeTiledFn* out);

}  // namespace ring_host
