// Host helpers of rdvb.cu that the library's other sources share: the error
// text and launch counter of the C ABI, the current device's limits, the
// device status word and the tensor-map encoder. Not exported.
#pragma once
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "rdvb.h"

namespace rdvb_host __attribute__((visibility("hidden"))) {

struct Device {
    int index;
    int sm_count;
    int max_smem;  // opt-in dynamic shared memory of a block
};
constexpr int kMaxDevices = 64;

int fail_text(int code, const char* text);  // records the calling thread's message, returns code
int launched(const char* what);             // the launch's error status; counts the launch
int device(Device* out);                    // refuses a device that is not sm_100
int status_word(uint32_t** out);            // device address of the status word
int allow_smem(const void* kernel, int bytes, int device);  // dynamic shared memory, set once a kernel and device
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();  // null when the driver has none

__attribute__((format(printf, 2, 3))) inline int fail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return fail_text(code, buf);
}

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace rdvb_host
