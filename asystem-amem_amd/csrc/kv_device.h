// What the kernels on a paged key/value cache share on the device.
#ifndef AMEM_KV_DEVICE_H_
#define AMEM_KV_DEVICE_H_

#include <hip/hip_runtime.h>

#include "kv.h"

namespace amem {
namespace {

constexpr int kWave = 64;

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <bool HALF>
__device__ __forceinline__ float to_float(uint16_t x) {
  if constexpr (HALF) return (float)__builtin_bit_cast(_Float16, x);
  else return __builtin_bit_cast(float, (uint32_t)x << 16);
}

template <bool HALF>  // nearest, ties to even
__device__ __forceinline__ uint16_t from_float(float x) {
  if constexpr (HALF) return __builtin_bit_cast(uint16_t, (_Float16)x);
  else return __builtin_bit_cast(uint16_t, (__bf16)x);
}

// The sequence that unit `u` belongs to, or -1: the number of sequences whose first unit is at most u, less one.
// The wave looks at 64 of them at a time, so a batch of up to 64 costs one round of loads and not a chain of them.
__device__ __forceinline__ int find_sequence(const KvBatch& b, int u, int shift, int spare) {
  const int lane = threadIdx.x & (kWave - 1);
  int count = 0;
  for (int s0 = 0; s0 < b.sequences; s0 += kWave) {
    const int s = s0 + lane;
    const bool below = s < b.sequences && kv_unit_base(b, s, shift, spare) <= u;
    const int n = __popcll(__ballot(below));
    count += n;
    if (n < kWave) break;
  }
  return __builtin_amdgcn_readfirstlane(count) - 1;
}

}  // namespace
}  // namespace amem
#endif
