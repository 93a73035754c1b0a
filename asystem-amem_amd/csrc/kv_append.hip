// Append to a paged key/value cache, with the rotation of keys and queries on the way.
//
//   (a, b) -> (a c - b s, b c + a s)   for the pairs of the rotated dims; values pass
//
// All of it moves bytes: a row is read once and written once. An item of work is 16 dims of one head of
// one row, as two vectors of eight elements that hold both members of eight pairs, so that a lane turns them
// by itself and reads eight neighbouring cosines and sines.
#include "kv_device.h"

namespace amem {
namespace {

constexpr int kThreads = 256;

// The two vectors of item `c` of a head, and its first pair (-1: not rotated).
struct Item {
  int lo, hi, pair;
};
__device__ __forceinline__ Item item_of(const KvAppend& a, int c) {
  if (c * 16 >= a.rotary) return {c * 16, c * 16 + 8, -1};
  if (a.interleaved) return {c * 16, c * 16 + 8, c * 8};
  return {c * 8, a.rotary / 2 + c * 8, c * 8};
}

// Cosines and sines of the eight pairs from `pair` on, for row `row` at position `pos`.
__device__ __forceinline__ void angles(const KvAppend& a, int row, int pos, int pair, float (&c)[8], float (&s)[8]) {
  const int half = a.rotary / 2;
  if (a.axes == 1) {
    const int t = a.positions ? a.positions[row] : pos;
    if (t < 0 || t >= a.table_rows) {
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = s[i] = __builtin_nanf("");
      return;
    }
    const f32x4* pc = (const f32x4*)(a.cos + (int64_t)t * half + pair);
    const f32x4* ps = (const f32x4*)(a.sin + (int64_t)t * half + pair);
    const f32x4 c0 = pc[0], c1 = pc[1], s0 = ps[0], s1 = ps[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) { c[i] = c0[i]; c[i + 4] = c1[i]; s[i] = s0[i]; s[i + 4] = s1[i]; }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    int axis = 0;
    while (axis < a.axes - 1 && pair + i >= a.axis_end[axis]) ++axis;
    const int t = a.positions[axis * a.positions_stride + row];
    const bool in = t >= 0 && t < a.table_rows;
    c[i] = in ? a.cos[(int64_t)t * half + pair + i] : __builtin_nanf("");
    s[i] = in ? a.sin[(int64_t)t * half + pair + i] : __builtin_nanf("");
  }
}

// Sixteen dims, [0, 8) of the first vector and [8, 16) of the second, turned. R is float, or double where an
// e4m3 code is to come of it: the products are exact then, and one rounding to the code is all there is.
template <class R>
__device__ __forceinline__ void turn(R (&x)[16], const float (&c)[8], const float (&s)[8], bool interleaved) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int ia = interleaved ? 2 * i : i, ib = interleaved ? 2 * i + 1 : i + 8;
    const R a = x[ia], b = x[ib], cc = c[i], ss = s[i];
    x[ia] = fma(a, cc, -(b * ss));
    x[ib] = fma(b, cc, a * ss);
  }
}

template <bool HALF, class R>
__device__ __forceinline__ void load_item(const uint16_t* head, const Item& it, R (&x)[16]) {
  const u16x8 lo = *(const u16x8*)(head + it.lo), hi = *(const u16x8*)(head + it.hi);
#pragma unroll
  for (int i = 0; i < 8; ++i) { x[i] = to_float<HALF>(lo[i]); x[i + 8] = to_float<HALF>(hi[i]); }
}

template <bool HALF, class R>
__device__ __forceinline__ void load_turned(const KvAppend& a, const uint16_t* head, const Item& it, int row, int pos, R (&x)[16]) {
  load_item<HALF>(head, it, x);
  if (it.pair < 0) return;
  float c[8], s[8];
  angles(a, row, pos, it.pair, c, s);
  if (a.interleaved) turn(x, c, s, true);
  else turn(x, c, s, false);
}

template <bool HALF>
__device__ __forceinline__ void store_item(uint16_t* head, const Item& it, const float (&x)[16]) {
  u16x8 lo, hi;
#pragma unroll
  for (int i = 0; i < 8; ++i) { lo[i] = from_float<HALF>(x[i]); hi[i] = from_float<HALF>(x[i + 8]); }
  *(u16x8*)(head + it.lo) = lo;
  *(u16x8*)(head + it.hi) = hi;
}

// One workgroup for a row: its query heads and, where the cache has 16 bits (KV), its key and value heads.
template <bool HALF, bool KV>
__global__ __launch_bounds__(kThreads) void append_rows(KvCache c, KvBatch b, KvAppend a, int items) {
  const int row = blockIdx.x;
  const int s = find_sequence(b, row, 0, 0);
  if (s < 0) return;
  const KvSeq q = kv_seq(b, s);
  if (row < q.row || row >= q.row + q.n) return;
  const int pos = q.context - q.n + row - q.row;
  const int heads = a.q_heads + (KV ? 2 * c.kv_heads : 0);
  int page = -1;
  if (KV && !q.bad && pos >= 0) page = kv_page(c, b, s, pos);
  for (int i = threadIdx.x; i < heads * items; i += kThreads) {
    int h = i / items;
    const Item it = item_of(a, i % items);
    float x[16];
    if (h < a.q_heads) {
      load_turned<HALF>(a, a.q + row * a.q_token + h * a.q_head, it, row, q.bad ? -1 : pos, x);
      store_item<HALF>(a.q_out + row * a.qo_token + h * a.qo_head, it, x);
    } else if (KV && page >= 0) {
      h -= a.q_heads;
      if (h < c.kv_heads) {
        load_turned<HALF>(a, a.k + row * a.k_token + h * a.k_head, it, row, pos, x);
        store_item<HALF>((uint16_t*)(c.k + kv_offset(c, page, h, pos)), it, x);
      } else {
        h -= c.kv_heads;
        load_item<HALF>(a.v + row * a.v_token + h * a.v_head, it, x);
        store_item<HALF>((uint16_t*)(c.v + kv_offset(c, page, h, pos)), it, x);
      }
    }
  }
}

// ---- 8 bits ----

// The float nearest to x on the odd side: rounding it once more to fewer bits, and comparing it with numbers of fewer
// bits, gives what x itself would.
__device__ __forceinline__ float to_odd(double x) {
  const float f = (float)x;
  const double back = f;
  if (back == x || !(fabs(x) < __builtin_inf())) return f;
  uint32_t bits = __builtin_bit_cast(uint32_t, f);
  if (fabs(back) > fabs(x)) --bits;
  return __builtin_bit_cast(float, bits | 1);
}

// The smallest scale 2^e, e in [-64, 119], with amax <= 448 * 2^e. 448 = 1.75 * 2^8.
__device__ __forceinline__ float scale_for(float amax) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, amax);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  e = amax > 0 ? (e < -64 ? -64 : e > 119 ? 119 : e) : -64;
  return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
}

// e4m3 code of x, at most 448 in size after its division by the scale; what is not finite becomes NaN.
__device__ __forceinline__ uint32_t code_of(float x) {
  if (!(fabsf(x) < __builtin_inff())) return 0x7f;
  x = fminf(fmaxf(x, -448.0f), 448.0f);
  return __builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false) & 0xff;
}
__device__ __forceinline__ float value_of(uint32_t code) { return __builtin_amdgcn_cvt_f32_fp8((int)code, 0); }

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int m = kWave / 2; m; m >>= 1) x = fmaxf(x, __shfl_xor(x, m, kWave));
  return x;
}

// One workgroup for the new tokens that one block of slots gets, of one key or value head: first the largest of their
// values, then the codes.
template <bool HALF>
__global__ __launch_bounds__(kThreads) void append_blocks(KvCache c, KvBatch b, KvAppend a, int items) {
  const int unit = blockIdx.x;
  const bool value = (int)blockIdx.y >= c.kv_heads;
  const int h = value ? blockIdx.y - c.kv_heads : blockIdx.y;
  const int s = find_sequence(b, unit, c.block_shift, 2);
  if (s < 0) return;
  const KvSeq q = kv_seq(b, s);
  const int size = 1 << c.block_shift;
  const int first = q.context - q.n > 0 ? q.context - q.n : 0;  // positions below 0 have no slot
  const int start = ((first >> c.block_shift) + unit - kv_unit_base(b, s, c.block_shift, 2)) << c.block_shift;
  if (q.bad || !q.n || start >= q.context) return;
  const int from = start > first ? start : first, to = start + size < q.context ? start + size : q.context;
  if (from >= to) return;
  const int page = kv_page(c, b, s, start);
  if (page < 0) return;
  const uint16_t* rows = value ? a.v + h * a.v_head : a.k + h * a.k_head;
  const int64_t token = value ? a.v_token : a.k_token;
  const int row0 = q.row + q.n - q.context;  // row of position 0
  uint8_t* codes = (value ? c.v : c.k) + kv_offset(c, page, h, start);
  float* scale = (value ? c.v_scale : c.k_scale) + kv_scale_offset(c, page, h, start);

  __shared__ float part[kThreads / kWave];
  float amax = 0;
  double x[16];
  auto load = [&](int i, const Item& it) {
    const int pos = from + i / items;
    if (value) load_item<HALF>(rows + (row0 + pos) * token, it, x);
    else load_turned<HALF>(a, rows + (row0 + pos) * token, it, row0 + pos, pos, x);
  };
  for (int i = threadIdx.x; i < (to - from) * items; i += kThreads) {
    load(i, item_of(a, i % items));
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float y = fabsf(to_odd(x[j]));
      if (y < __builtin_inff()) amax = fmaxf(amax, y);
    }
  }
  amax = wave_max(amax);
  if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x / kWave] = amax;
  const float held = *scale;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kThreads / kWave; ++i) amax = fmaxf(amax, part[i]);
  const float need = scale_for(amax);
  // a scale that is no positive finite number counts as the one needed
  const float old = from == start || !(held > 0 && held < __builtin_inff()) ? need : held;
  const float now = fmaxf(old, need);
  const double inverse = 1.0 / now;
  for (int i = threadIdx.x; i < (to - from) * items; i += kThreads) {
    const Item it = item_of(a, i % items);
    load(i, it);
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 16; ++j) w[j / 4] |= code_of(to_odd(x[j] * inverse)) << (j % 4 * 8);
    uint8_t* at = codes + (from - start + i / items) * c.slot_stride;
    *(u32x2*)(at + it.lo) = u32x2{w[0], w[1]};
    *(u32x2*)(at + it.hi) = u32x2{w[2], w[3]};
  }
  if (now > old) {
    const double ratio = old * inverse;
    for (int i = threadIdx.x; i < (from - start) * items; i += kThreads) {
      u32x4* at = (u32x4*)(codes + i / items * c.slot_stride + i % items * 16);
      u32x4 w = *at;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t y = 0;
#pragma unroll
        for (int l = 0; l < 4; ++l) y |= code_of(to_odd(value_of(w[j] >> (l * 8) & 0xff) * ratio)) << (l * 8);
        w[j] = y;
      }
      *at = w;
    }
  }
  if (threadIdx.x == 0) *scale = now;
}

}  // namespace

hipError_t launch_kv_append(const KvCache& c, const KvBatch& b, const KvAppend& a, int head_dim, bool half, bool eight, hipStream_t stream) {
  const int items = head_dim / 16;
  if (!eight) {
    if (half) append_rows<true, true><<<b.tokens, kThreads, 0, stream>>>(c, b, a, items);
    else append_rows<false, true><<<b.tokens, kThreads, 0, stream>>>(c, b, a, items);
    return hipGetLastError();
  }
  const dim3 blocks(kv_units(b, c.block_shift, 2), 2 * c.kv_heads);
  if (half) append_blocks<true><<<blocks, kThreads, 0, stream>>>(c, b, a, items);
  else append_blocks<false><<<blocks, kThreads, 0, stream>>>(c, b, a, items);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || !a.q_heads) return e;
  if (half) append_rows<true, false><<<b.tokens, kThreads, 0, stream>>>(c, b, a, items);
  else append_rows<false, false><<<b.tokens, kThreads, 0, stream>>>(c, b, a, items);
  return hipGetLastError();
}

}  // namespace amem
