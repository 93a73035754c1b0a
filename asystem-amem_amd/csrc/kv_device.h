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
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

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

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kInf = __builtin_inff();

// Eight 16-bit operands of a matrix instruction are one vector of four words here; HALF says which type they have.
template <bool HALF>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {  // 16 x 16, 32 deep
  if constexpr (HALF) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <bool HALF>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {  // 32 x 32, 16 deep
  if constexpr (HALF) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Eight e4m3 codes as 16-bit numbers, those of the first word times `first` and of the second times `second`, powers of two. Both types hold
// every code exactly, and fp16 its product with 2^-15 to 2^7.
template <bool HALF>
__device__ __forceinline__ u32x4 widen(u32x2 x, float first = 1.0f, float second = 1.0f) {
  u32x4 y;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float f = i ? second : first;
    if constexpr (HALF) {
      y[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[i], f, false));
      y[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[i], f, true));
    } else {
      y[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], f, false));
      y[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], f, true));
    }
  }
  return y;
}

// Scales of e4m3 values meet the weights in fp16. While those that a workgroup (or a wave) meets are within 2^kNear of the largest of its first
// tile, codes are widened in multiples of 2^kNear times that one, exactly, and so are the sums. From the first tile on where one is not ("far"), codes
// are widened as they are, and each row's weights take the scales, in multiples of a power of two of the row's own: its sums are in
// multiples of 2^far_unit(h), where 2^h is at least its largest product of weight and scale so far. Those products are at most 2^15 in it,
// and a large scale costs small ones no bits unless it comes with a weight. h falls as m grows and the weights so far shrink. Parts
// leave a workgroup in multiples of kPartUnit, in which 32 bits hold sums of every scale from 2^-64 to 2^119.
constexpr int kNear = 4;
constexpr int kPartExponent = 40;
constexpr float kPartUnit = 0x1p40f;
constexpr float kNothing = -1000.0f;  // h of a row that has seen nothing

__device__ __forceinline__ int exponent_of(float x) { return (int)(__builtin_bit_cast(uint32_t, x) >> 23 & 0xff) - 127; }
__device__ __forceinline__ int far_unit(float h) { return (int)ceilf(h) - 15; }  // its exponent

template <bool HALF>  // nearest, ties to even
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  if constexpr (HALF) return __builtin_bit_cast(uint32_t, f16x2{(_Float16)lo, (_Float16)hi});
  else return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)lo, (__bf16)hi});
}

__device__ __forceinline__ float lane_value(float x, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}

// Whether any of 16 bytes of values is an infinity or NaN.
template <bool HALF, bool EIGHT>
__device__ __forceinline__ bool not_finite(u32x4 x) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (EIGHT) {
#pragma unroll
      for (int j = 0; j < 4; ++j) bad |= (x[i] >> (8 * j) & 0x7f) == 0x7f;
    } else {
      const uint32_t e = HALF ? 0x7c00 : 0x7f80;
      bad |= (x[i] & e) == e || (x[i] >> 16 & e) == e;
    }
  }
  return bad;
}

typedef __attribute__((address_space(3))) uint8_t lds_byte;

// Rows of LDS read as columns, by each 16 lanes on their own: of four rows of 16-bit numbers (lane m gives the address of
// row m / 4, columns 4 (m % 4) on) lane m gets column m; of eight rows of bytes (row m / 2, columns 8 (m % 2) on) too.
__device__ __forceinline__ u32x2 read_columns16(const uint8_t* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(lds_byte*)p));
}
__device__ __forceinline__ u32x2 read_columns8(const uint8_t* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*)(lds_byte*)p));
}

// The sequence that unit `u` belongs to, or -1: the number of sequences whose first unit is at most u, less one.
// The wave looks at 64 of them at a time, so a batch of up to 64 costs one round of loads and not a chain of them.
__device__ __forceinline__ int find_sequence(const KvBatch& b, int u, int tile, int spare, int per_row = 1) {
  const int lane = threadIdx.x & (kWave - 1);
  int count = 0;
  for (int s0 = 0; s0 < b.sequences; s0 += kWave) {
    const int s = s0 + lane;
    const bool below = s < b.sequences && kv_unit_base(b, s, tile, spare, per_row) <= u;
    const int n = __popcll(__ballot(below));
    count += n;
    if (n < kWave) break;
  }
  return __builtin_amdgcn_readfirstlane(count) - 1;
}

}  // namespace
}  // namespace amem
#endif
