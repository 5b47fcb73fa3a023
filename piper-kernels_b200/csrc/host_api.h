// Host helpers that piper_b200.cu shares with the other translation units:
// the per-thread error message, the per-device set-up and the device status
// word.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

namespace piper {
namespace host {

// Records `msg` as the calling thread's last error and returns `code`.
int fail(int code, const std::string& msg);
int cuda_fail(cudaError_t err, const char* what);

// The calling thread's device, checked to be sm_100 and set up.  `context`
// identifies the CUDA context the set-up belongs to: what another translation
// unit sets up itself (kernel attributes) it redoes when that changes.
struct Device {
  int index = 0;
  int sms = 0;
  unsigned long long context = 0;
  uint32_t* status = nullptr;  // the status word, in device memory
};
int ensure_device(Device* device);

// A 3-D tensor map of bytes: a box of `box_mid` rows of `inner` (64 or 128)
// bytes, swizzled for that width.
int encode_rows_map(CUtensorMap* map, const void* base, uint64_t inner, uint64_t mid, uint64_t outer,
                    uint32_t box_mid);

}  // namespace host
}  // namespace piper

#define PIPER_HOST_CUDA(call)                                       \
  do {                                                              \
    cudaError_t e_ = (call);                                        \
    if (e_ != cudaSuccess) return piper::host::cuda_fail(e_, #call); \
  } while (0)
