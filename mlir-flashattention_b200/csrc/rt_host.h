// rt_host.h — what the runtime's translation units share on the host side:
// error reporting, per-device state, stream-ordered scratch and the launch
// count, all kept in attn_rt.cu.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace rt_host {

struct Device {
  int index = 0;
  int sms = 0;
  int32_t* status = nullptr;  // the runtime's status word of this device
};

// Records `message` as the calling thread's last error; returns `code`.
int fail_with(int code, const char* message);

// The current device, set up on first use.
int device_ready(Device* out);

bool on_device(const void* p);

// Scratch ordered on `s`, freed by cudaFreeAsync on the same stream.
cudaError_t scratch(void** p, size_t bytes, cudaStream_t s);

void count_launches(int n);

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled tensor_map_encoder();

}  // namespace rt_host
