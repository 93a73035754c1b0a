// Append to a paged key/value cache, with the rotation of keys and queries on the way.
//
//   (a, b) -> (a c - b s, b c + a s)   for the pairs of the rotated dims; values pass
//
// All of it moves bytes: a row is read once and written once, in one launch for keys, values and queries. An item of work
// is 16 dims of one head of one row, as two vectors of eight elements that hold both members of eight pairs, so that
// a lane turns them by itself and reads eight neighbouring cosines and sines, once for all the heads that it takes.
//
// Measured, where a large copy moves 4.9 TB/s: up to 2500 rows of six sequences, 32 heads over 4, 64 dims, half of them turned, fp16: 112 MB
// in 24 us, 4.7 TB/s; 2 x 8192 rows, 64 heads over 8, 128 dims, three axes, e4m3: 395 MB in 94 us, 4.2 TB/s; the single tokens of 128
// sequences, e4m3: 8 us; one row 4.5 us, about what a launch takes.
#include <algorithm>

#include "kv_device.h"

namespace amem {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

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
  // four pairs mostly have one axis
  int at[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) at[x] = x < a.axes ? a.positions[x * a.positions_stride + row] : 0;
#pragma unroll
  for (int j = 0; j < 8; j += 4) {
    int t[4];
    bool one = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t[i] = at[0];
#pragma unroll
      for (int x = 1; x < 4; ++x) t[i] = x < a.axes && pair + j + i >= a.axis_end[x - 1] ? at[x] : t[i];
      one &= t[i] == t[0];
    }
    if (one && t[0] >= 0 && t[0] < a.table_rows) {
      const f32x4 cc = *(const f32x4*)(a.cos + (int64_t)t[0] * half + pair + j), ss = *(const f32x4*)(a.sin + (int64_t)t[0] * half + pair + j);
#pragma unroll
      for (int i = 0; i < 4; ++i) { c[j + i] = cc[i]; s[j + i] = ss[i]; }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool in = t[i] >= 0 && t[i] < a.table_rows;
        c[j + i] = in ? a.cos[(int64_t)t[i] * half + pair + j + i] : __builtin_nanf("");
        s[j + i] = in ? a.sin[(int64_t)t[i] * half + pair + j + i] : __builtin_nanf("");
      }
    }
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

struct Pair {
  u16x8 lo, hi;
};
__device__ __forceinline__ Pair load_pair(const uint16_t* head, const Item& it) { return {*(const u16x8*)(head + it.lo), *(const u16x8*)(head + it.hi)}; }

template <bool HALF, class R>
__device__ __forceinline__ void widen_pair(const Pair& p, R (&x)[16]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) { x[i] = to_float<HALF>(p.lo[i]); x[i + 8] = to_float<HALF>(p.hi[i]); }
}

template <class R>
__device__ __forceinline__ void turn(const KvAppend& a, const float (&c)[8], const float (&s)[8], R (&x)[16]) {
  if (a.interleaved) turn(x, c, s, true);
  else turn(x, c, s, false);
}

// The sequence of a row, -1 if it has none.
__device__ __forceinline__ int sequence_of_row(const KvBatch& b, int row) { return b.cu_tokens ? find_sequence(b, row, 1, 0) : row / b.uniform; }

// One wave for a share of the heads of a row: query heads and, where the cache has 16 bits (KV), its key and value heads.
// A lane keeps to the same dims, so its cosines and sines are read once, and takes four heads at a time.
template <bool HALF, bool KV>
__device__ __forceinline__ void append_rows(const KvCache& c, const KvBatch& b, const KvAppend& a, int items, int shares, int index) {
  const int row = index / shares, share = index % shares, lane = threadIdx.x & (kWave - 1);
  if (row >= b.tokens) return;
  const int s = sequence_of_row(b, row);
  if (s < 0) return;
  const KvSeq q = kv_seq(b, s);
  if (row < q.row || row >= q.row + q.n) return;
  const int pos = q.bad ? -1 : q.context - q.n + row - q.row;
  const int page = KV && pos >= 0 ? kv_page(c, b, s, pos) : -1;
  const Item it = item_of(a, lane % items);
  float co[8], si[8];
  if (it.pair >= 0) angles(a, row, pos, it.pair, co, si);
  const int heads = a.q_heads + (KV ? 2 * c.kv_heads : 0), step = kWave / items;
  const int64_t at = page >= 0 ? kv_offset(c, page, 0, pos) : 0;
  constexpr int N = 4;
  for (int h0 = share * N * step + lane / items; h0 < heads; h0 += shares * N * step) {
    Pair in[N];
    uint16_t* out[N];
    bool turned[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      int h = h0 + n * step;
      out[n] = nullptr;
      turned[n] = it.pair >= 0;
      if (h >= heads) continue;
      if (h < a.q_heads) {
        in[n] = load_pair(a.q + row * a.q_token + h * a.q_head, it);
        out[n] = a.q_out + row * a.qo_token + h * a.qo_head;
      } else if (KV && page >= 0) {
        h -= a.q_heads;
        const bool value = h >= c.kv_heads;
        if (value) {
          h -= c.kv_heads;
          turned[n] = false;
        }
        in[n] = value ? load_pair(a.v + row * a.v_token + h * a.v_head, it) : load_pair(a.k + row * a.k_token + h * a.k_head, it);
        out[n] = (uint16_t*)((value ? c.v : c.k) + at + h * c.head_stride);
      }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (!out[n]) continue;
      if (turned[n]) {
        float x[16];
        widen_pair<HALF>(in[n], x);
        turn(a, co, si, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) { in[n].lo[i] = from_float<HALF>(x[i]); in[n].hi[i] = from_float<HALF>(x[i + 8]); }
      }
      *(u16x8*)(out[n] + it.lo) = in[n].lo;
      *(u16x8*)(out[n] + it.hi) = in[n].hi;
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

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int m = kWave / 2; m; m >>= 1) x = fmaxf(x, __shfl_xor(x, m, kWave));
  return x;
}

// Two codes next to each other.
__device__ __forceinline__ uint32_t two_codes(float x, float y) { return __builtin_amdgcn_cvt_pk_fp8_f32(x, y, 0, false) & 0xffff; }

// W waves for the new tokens that one block of slots gets, of one key or value head: their values, turned, stay in registers (N
// items a lane) while the largest is found, and become codes. Keys are turned in 64 bits and rounded to odd floats, whose
// codes are those of the exact values; values need no more than 32.
template <bool HALF, int W, int N>
__device__ __forceinline__ void append_blocks(const KvCache& c, const KvBatch& b, const KvAppend& a, int items, int units, int index, float* part) {
  const int lane = threadIdx.x & (kWave - 1), turn_of = threadIdx.x / kWave % W, at_lane = turn_of * kWave + lane;
  const int h = index % c.kv_heads;
  const bool value = index / c.kv_heads & 1;
  int unit = index / c.kv_heads / 2, s = -1;
  const int shift = c.block_shift, size = 1 << shift;
  if (unit < units) {
    if (b.cu_tokens) {
      s = find_sequence(b, unit, size, 2);
      unit -= s >= 0 ? kv_unit_base(b, s, size, 2) : 0;
    } else {
      const int each = ((b.uniform - 1) >> shift) + 2;
      s = unit / each;
      unit -= s * each;
    }
  }
  KvSeq q = {};
  if (s >= 0) q = kv_seq(b, s);
  const int first = q.context - q.n > 0 ? q.context - q.n : 0;  // positions below 0 have no slot
  const int start = ((first >> shift) + unit) << shift;
  const int from = start > first ? start : first, to = start + size < q.context ? start + size : q.context;
  int page = -1;
  if (s >= 0 && !q.bad && q.n && from < to) page = kv_page(c, b, s, start);
  if (W == 1 && page < 0) return;
  const int count = page >= 0 ? (to - from) * items : 0;
  const uint16_t* rows = value ? a.v + h * a.v_head : a.k + h * a.k_head;
  const int64_t token = value ? a.v_token : a.k_token;
  const int row0 = q.row + q.n - q.context;  // row of position 0
  uint8_t* codes = nullptr;
  float* scale = nullptr;
  float held = 0, amax = 0;
  bool odd = false;  // something is not finite
  if (page >= 0) {
    codes = (value ? c.v : c.k) + kv_offset(c, page, h, start);
    scale = (value ? c.v_scale : c.k_scale) + kv_scale_offset(c, page, h, start);
    held = *scale;
  }
  float x[N][16];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int i = n * W * kWave + at_lane;
    if (i >= count) continue;
    const int pos = from + i / items;
    const Item it = item_of(a, i % items);
    const Pair in = load_pair(rows + (row0 + pos) * token, it);
    if (value || it.pair < 0) {
      widen_pair<HALF>(in, x[n]);
    } else {
      float co[8], si[8];
      angles(a, row0 + pos, pos, it.pair, co, si);
      double y[16];
      widen_pair<HALF>(in, y);
      turn(a, co, si, y);
#pragma unroll
      for (int j = 0; j < 16; ++j) x[n][j] = to_odd(y[j]);
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float y = fabsf(x[n][j]);
      const bool fine = y < __builtin_inff();
      amax = fine ? fmaxf(amax, y) : amax;
      odd |= !fine;
    }
  }
  amax = wave_max(amax);
  if constexpr (W > 1) {
    if (lane == 0) part[threadIdx.x / kWave] = amax;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) amax = fmaxf(amax, part[threadIdx.x / kWave / W * W + i]);
    if (page < 0) return;
  }
  const float need = scale_for(amax);
  // a scale that is no positive finite number counts as the one needed
  const float old = from == start || !(held > 0 && held < __builtin_inff()) ? need : held;
  const float now = fmaxf(old, need);
  const float inverse = 1.0f / now;  // exact: a power of two
  odd |= amax > 448.0f * now;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int i = n * W * kWave + at_lane;
    if (i >= count) continue;
    const Item it = item_of(a, i % items);
    uint32_t w[4];
    if (!odd) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = two_codes(x[n][4 * j] * inverse, x[n][4 * j + 1] * inverse) | two_codes(x[n][4 * j + 2] * inverse, x[n][4 * j + 3] * inverse) << 16;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[j] |= code_of(x[n][4 * j + e] * inverse) << (8 * e);
      }
    }
    uint8_t* at = codes + (from - start + i / items) * c.slot_stride;
    *(u32x2*)(at + it.lo) = u32x2{w[0], w[1]};
    *(u32x2*)(at + it.hi) = u32x2{w[2], w[3]};
  }
  if (now > old) {
    const float ratio = old * inverse;  // a power of two: products are exact, NaN stays
    for (int i = at_lane; i < (from - start) * items; i += W * kWave) {
      u32x4* at = (u32x4*)(codes + i / items * c.slot_stride + i % items * 16);
      u32x4 w = *at;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[j], false) * ratio, hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[j], true) * ratio;
        w[j] = two_codes(lo[0], lo[1]) | two_codes(hi[0], hi[1]) << 16;
      }
      *at = w;
    }
  }
  if (at_lane == 0) *scale = now;
}

template <bool HALF>
__global__ __launch_bounds__(kThreads) void append16(KvCache c, KvBatch b, KvAppend a, int items, int shares) {
  append_rows<HALF, true>(c, b, a, items, shares, blockIdx.x * kWaves + threadIdx.x / kWave);
}

// The first `block_groups` workgroups take blocks of slots, the others rows of queries.
template <bool HALF, int W, int N>
__global__ __launch_bounds__(kThreads) void append8(KvCache c, KvBatch b, KvAppend a, int items, int shares, int units, int block_groups) {
  __shared__ float part[kWaves];
  const int wave = threadIdx.x / kWave;
  if ((int)blockIdx.x < block_groups) append_blocks<HALF, W, N>(c, b, a, items, units, blockIdx.x * (kWaves / W) + wave / W, part);
  else append_rows<HALF, false>(c, b, a, items, shares, (blockIdx.x - block_groups) * kWaves + wave);
}

}  // namespace

hipError_t launch_kv_append(const KvCache& c, const KvBatch& b, const KvAppend& a, int head_dim, bool half, bool eight, hipStream_t stream) {
  const int items = head_dim / 16, heads = a.q_heads + (eight ? 0 : 2 * c.kv_heads);
  // A wave takes all heads of a row where rows are many, since its angles serve them all; with fewer rows up to as many
  // waves as have four heads for each lane share them, until there are about 4096. One wave a row and that many (us; 64 heads over 8,
  // 128 dims, 16 bits): one row 7.7 and 5.2, 500 rows 10.4 and 8.0, 4000 rows 36 and 35.
  const int most = (heads * items + 4 * kWave - 1) / (4 * kWave);
  const int shares = std::max(1, std::min(most, 4096 / std::max(1, b.tokens)));
  const int row_groups = heads ? (int)(((int64_t)b.tokens * shares + kWaves - 1) / kWaves) : 0;
  if (!eight) {
    if (half) append16<true><<<row_groups, kThreads, 0, stream>>>(c, b, a, items, shares);
    else append16<false><<<row_groups, kThreads, 0, stream>>>(c, b, a, items, shares);
    return hipGetLastError();
  }
  const int units = b.cu_tokens ? kv_units(b, 1 << c.block_shift, 2) : b.sequences * (((b.uniform - 1) >> c.block_shift) + 2);
  // Items that a block gets at most: up to 64 for single tokens, to 2048 for whole blocks. As many waves as have one or two items a
  // lane, up to four: with fewer waves and more items a lane 300 rows of 128 dims, 64 in a block, take 12 us instead of 8, 8192 rows 51
  // instead of 48; single tokens of 128 sequences 8.6 with the shortest kernel and 10.6 with the one for 256 items.
  const int block_items = items * (b.cu_tokens ? 1 << c.block_shift : std::min(b.uniform, 1 << c.block_shift));
  auto run = [&](auto kernel, int waves) {
    const int groups = (int)(((int64_t)units * 2 * c.kv_heads * waves + kWaves - 1) / kWaves);
    kernel<<<groups + row_groups, kThreads, 0, stream>>>(c, b, a, items, shares, units, groups);
  };
  if (half) {
    if (block_items <= 64) run(append8<true, 1, 1>, 1);
    else if (block_items <= 128) run(append8<true, 2, 1>, 2);
    else if (block_items <= 256) run(append8<true, 2, 2>, 2);
    else if (block_items <= 512) run(append8<true, 4, 2>, 4);
    else if (block_items <= 1024) run(append8<true, 4, 4>, 4);
    else run(append8<true, 4, 8>, 4);
  } else {
    if (block_items <= 64) run(append8<false, 1, 1>, 1);
    else if (block_items <= 128) run(append8<false, 2, 1>, 2);
    else if (block_items <= 256) run(append8<false, 2, 2>, 2);
    else if (block_items <= 512) run(append8<false, 4, 2>, 4);
    else if (block_items <= 1024) run(append8<false, 4, 4>, 4);
    else run(append8<false, 4, 8>, 4);
  }
  return hipGetLastError();
}

}  // namespace amem
