// What the translation units of the library share: the per-device record, the status of the calling thread, the count of launches and
// the driver's tensor-map calls (fmha_api.cu defines them).
#pragma once
#include <cuda.h>

#pragma GCC visibility push(hidden)
namespace fmha_host {

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

struct Device {
  int index = 0, sm_count = 1;
  unsigned* status = nullptr;       // eight device status words
  unsigned* host_word = nullptr;    // device view of the host-visible failure word
};

// Stores the status of the most recent call on this host thread and returns it.
int finish(int status);
// The current device, or FMHA_I8_ERR_*; FMHA_I8_ERR_DEVICE once if a kernel launched earlier reported a failure.
int device_for_call(Device* out);
void count_launch();
EncodeTiledFn encode_tiled();

}  // namespace fmha_host
#pragma GCC visibility pop
