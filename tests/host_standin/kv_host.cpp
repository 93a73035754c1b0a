// TEST INFRASTRUCTURE, never part of the shipped library: launchers of csrc/kv.h that only count, and the HIP call of csrc/kv_api.cpp
// that fake_hip.cpp does not have.
#include "../../asystem-amem_amd/csrc/kv.h"

static int launches = 0;

extern "C" {
hipError_t hipStreamGetDevice(hipStream_t, hipDevice_t* device) {
  *device = 0;
  return hipSuccess;
}
__attribute__((visibility("default"))) int kv_host_launches(void) { return launches; }
}

namespace amem {
hipError_t launch_kv_append(const KvCache&, const KvBatch&, const KvAppend&, int, bool, bool, hipStream_t) {
  ++launches;
  return hipSuccess;
}
hipError_t launch_kv_attend(const KvCache&, const KvBatch&, const KvAttend&, int, bool, bool, hipStream_t) {
  ++launches;
  return hipSuccess;
}
uint64_t kv_attend_workspace(const KvCache&, const KvBatch&, int, int, int) { return 4096; }
}  // namespace amem
