// Attention over a paged key/value cache for many rows: prompts, and chunks of them.
//
//   s_p = scale q.k_p,  m = max s_p,  l = sum exp(s_p - m),  out = sum exp(s_p - m) v_p / l,  lse = m + log l
//
// Bound by the matrix unit. A workgroup takes 256 rows that share a key/value head (32 for each of its eight waves; or 128: four
// waves, or eight with 16 rows each) through the positions they see, 64 at a time: its threads load a tile of keys
// and values while the one before is worked on, and put it into LDS as 16-bit numbers, where every wave reads all of it.
// Two tiles are held there, so that one barrier a tile is enough. Products are (keys x dims)(dims x rows) and (dims x keys)(keys x rows): a lane holds scores and sums
// of one row, the weights go from the first product's result to the second's operand without leaving their lane, and
// values are read from LDS as columns.
//
// Measured, where a large product of matrices reaches 1209 TFLOP/s: a chunk of 4096 rows over 16384 positions, 32 heads over 8, 128 dims,
// e4m3: 962 GFLOP in 0.92 ms, 1050 TFLOP/s (warm 0.99; 1.23 where the scales of values are far apart); four prompts of up to 3500 rows, bf16: 428 GFLOP
// in 0.50 ms, 860; a window of 1024 over 2 x 3001 rows, 8 heads over one, 256 dims, fp16: 39 GFLOP in 92 us, 420. The matrix unit is busy 46 and
// 41 % of the cycles of the first two; the softmax's vector instructions take most of the others, and do not run beside it. 256 dims: 27 %, LDS 36 %.
#include <algorithm>
#include <type_traits>

#include "kv_parts.h"

namespace amem {
namespace {

constexpr int kTile = 64;  // positions

template <bool HALF>
__device__ __forceinline__ u32x4 times_zero(u32x4 x) {  // zeros, NaN where an element is not finite
  constexpr uint32_t e = HALF ? 0x7c00 : 0x7f80;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = ((x[i] & e) == e ? 0x7fffu : 0) | ((x[i] >> 16 & e) == e ? 0x7fff0000u : 0);
  return x;
}

// D dims, 16 bits of fp16 (HALF) or bf16, a cache of e4m3 (EIGHT).
// W waves with R rows each, 32 or 16.
template <int D, bool HALF, bool EIGHT, int W, int R>
__global__ __launch_bounds__(W * kWave, (D == 64 ? 3 : 2)) void attend_many(KvCache c, KvBatch b, KvAttend a, Parts parts) {
  constexpr int kThreads = W * kWave;
  constexpr int kElement = EIGHT ? 1 : 2;
  constexpr int kRowLanes = D * kElement / 16;    // threads that load a position's key, or value
  constexpr int kRowsAPass = kThreads / kRowLanes;
  constexpr int kPasses = kTile / kRowsAPass;
  static_assert(kRowsAPass <= kTile, "a pass is at most a tile");
  // pads: the rows that are read together are on different banks (keys of 256 dims: 674 us with 32 bytes, 773 with 16, 780 with 64, at
  // 1100 rows of 16000 positions in e4m3; of 128 dims 16 and 32 differ by 1 %)
  constexpr int kKeyPitch = D * 2 + (R == 32 ? 16 : 32), kValuePitch = D * 2 + 2 * R, kBuffer = kTile * (kKeyPitch + kValuePitch);
  constexpr bool kHalfP = EIGHT || HALF;  // weights are fp16 where the values' type allows it
  // fp16 weights are held 2^8 times larger, which keeps small ones out of the subnormal numbers
  constexpr float kLift = kHalfP ? 8.0f : 0.0f;
  constexpr float kSlack = 7.0f;  // fp16 holds 2^(kLift + kSlack)
  // Scales of keys go into the keys where 16 bits hold every product (bf16), else into the scores.
  constexpr bool kFold = EIGHT && !HALF;
  // What a lane holds of its row: scores of kScores positions of a tile, and sums of kSums dims in kBlocks results of the matrix unit.
  constexpr int kScores = R == 32 ? 32 : 16, kBlocks = D / R, kSums = R == 32 ? 16 : 4;
  using Result = std::conditional_t<R == 32, f32x16, f32x4>;
  constexpr int kSteps = R == 32 ? 16 : 32;       // depth of a matrix instruction
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * kBuffer];
  __shared__ uint64_t lds_odd[2][kPasses * W];

  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  // heads first, so that the units of a head, which read the same keys, run on one die where heads are a multiple of eight;
  // the last units, which see most, before the others
  const int group = a.q_heads / c.kv_heads;
  int kvh, unit, split;
  pair_of(c, parts, blockIdx.x, unit, kvh, split);
  KvSeq q;
  KvUnit u;
  if (!find_unit(b, a, group, W * R, unit, q, u)) return;
  const int begin = u.from + split * parts.stretch;
  if (split && (begin >= u.to || q.bad)) return;
  const int64_t cut = part_of(c, parts, unit, kvh);  // below zero: the unit's positions are not cut
  const int end = cut >= 0 && begin + parts.stretch < u.to ? begin + parts.stretch : u.to;
  const int col = lane & (R - 1), part = lane / R;
  auto position_of = [&](int j) { return R == 32 ? j / 4 * 8 + part * 4 + j % 4 : j / 4 * 16 + part * 4 + j % 4; };
  // 8 bits: a thread widens sixteen codes to two vectors of eight dims; the first ones of all of a row's threads lie together in LDS, and
  // the second ones behind them, so that neighbouring threads write to neighbouring banks (963 -> 957 us at a chunk of 4096 over 16384). What
  // dim is at a place of a row:
  auto dim_at = [](int place) { return EIGHT ? place % (D / 2) / 8 * 16 + place / (D / 2) * 8 + place % 8 : place; };
  auto dim_of = [&](int i, int e, int part) { return dim_at(R == 32 ? i * 32 + e / 4 * 8 + part * 4 + e % 4 : i * 16 + part * 4 + e); };

  // this wave's rows, and the positions that some, and all, of them see
  const int wave_first = u.first + wave * R;
  const bool active = wave * R < u.rows;
  const int wave_last = std::min(wave_first + R - 1, u.first + u.rows - 1);
  int wave_lo = 0, wave_to = 0, all_from = 0, all_to = 0, row_from = 0, row_to = 0, token = 0, head = 0;
  u32x4 qr[D / kSteps];
  if (active) {
    row_range(a, q, wave_first / group, wave_lo, all_to);
    row_range(a, q, wave_last / group, all_from, wave_to);
    const int r = std::min(wave_first + col, wave_last);
    token = r / group;
    head = kvh * group + r % group;
    row_range(a, q, token, row_from, row_to);
    const uint16_t* p = a.q + (q.row + token) * a.q_token + head * a.q_head;
#pragma unroll
    for (int t = 0; t < D / kSteps; ++t) {
      qr[t] = *(const u32x4*)(p + dim_at(t * kSteps + part * 8));
      qr[t] = a.scale == 0 ? times_zero<HALF>(qr[t]) : qr[t] ^ (a.scale < 0 ? 0x80008000u : 0u);
    }
  }
  // weights are exp2(score * factor - top), so the factor has to be above zero for the largest score to give the largest
  // product: the scale's sign, and a scale of zero, are in the queries
  const float factor = a.scale == 0 ? 1.0f : fabsf(a.scale) * kLog2e;

  float m = -kInf, l = 0;
  Result sum[kBlocks];
#pragma unroll
  for (int i = 0; i < kBlocks; ++i)
#pragma unroll
    for (int j = 0; j < kSums; ++j) sum[i][j] = 0;
  uint32_t unit_scale = 0;  // 8 bits: the sums are in multiples of it, as bits; or (far) of the row's 2^sum_unit
  float h = kNothing;
  int sum_unit = 0;

  // ---- loading: a thread's rows of a tile
  const int my_row = tid / kRowLanes, my_col = tid % kRowLanes * 16;
  const int slot_mask = (1 << c.page_shift) - 1;
  const uint8_t* const keys = c.k + (int64_t)kvh * c.head_stride;
  const uint8_t* const values = c.v + (int64_t)kvh * c.head_stride;
  u32x4 kreg[kPasses], vreg[kPasses];
  // Pages of the tile to be loaded next, as the page table has them, of the thread's rows and (8 bits) in lane g of group g of 16.
  int page[kPasses], group_page = 0;
  uint32_t missing = 0;         // rows of the tile in the registers whose page is out of range
  uint32_t ks = 0, vs = 0;      // scales of the tile in the registers, lane g has group g's; as bits, whose order is that of the numbers
  // Nothing is done with a page here: that would wait for all loads under way. Behind the last position it is that one's.
  auto look_up = [&](int base) {
#pragma unroll
    for (int i = 0; i < kPasses; ++i) page[i] = kv_table(c, b, u.s, std::min(base + i * kRowsAPass + my_row, u.to - 1));
    if constexpr (EIGHT) group_page = kv_table(c, b, u.s, std::min(base + (lane & 3) * 16, u.to - 1));
  };
  auto load = [&](int base) {
    missing = 0;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int p = base + i * kRowsAPass + my_row, where = kv_checked(c, page[i]);
      if (where < 0) missing |= 1u << i;
      // a page's rows span less than 2^31 bytes
      const int64_t at = (int64_t)(where < 0 ? 0 : where) * c.page_stride + (uint32_t)((p & slot_mask) * (int)c.slot_stride + my_col);
      kreg[i] = *(const u32x4*)(keys + at);
      vreg[i] = *(const u32x4*)(values + at);
    }
    if constexpr (EIGHT) {
      const int64_t at = kv_scale_offset(c, kv_checked(c, group_page) < 0 ? 0 : group_page, kvh, base + (lane & 3) * 16);
      ks = ((const uint32_t*)c.k_scale)[at];
      vs = ((const uint32_t*)c.v_scale)[at];
    }
  };
  auto partial = [&](int base) { return base < u.all_from || base + kTile > u.all_to; };
  // The registers' tile into LDS. Keys of a page that is out of range become NaN, which every row that sees them gets.
  // Values are stored in multiples of unit_scale, as powers of two: a difference of exponents; or as they are (far).
  float key_scale[4];  // of the tile stored last
  uint64_t far = 0;    // not zero once a scale was far; a ballot, which stays in scalar registers
  constexpr uint32_t kExponent = 0x7f800000, kOne = 0x3f800000;
  auto seen = [&](int base) {  // this lane's group: a hidden one's scale may be anything
    const int p = base + (lane & 3) * 16;
    return p < u.to && p + 15 >= u.lo;
  };
  auto store = [&](int base, int buffer) {
    uint8_t* const at = lds + buffer * kBuffer;
    uint32_t value_scale = kOne;
    if constexpr (EIGHT) {
      if constexpr (!kFold) {
#pragma unroll
        for (int g = 0; g < 4; ++g) key_scale[g] = lane_value(__builtin_bit_cast(float, ks), g);
      }
      const uint32_t scale = seen(base) ? vs : unit_scale;
      far |= __ballot(unit_scale - scale > (uint32_t)(2 * kNear) << 23);
      value_scale = far ? kOne : scale - unit_scale + kOne;
    }
    const bool edge = partial(base);
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int r = i * kRowsAPass + my_row;
      u32x4 k = kreg[i], v = vreg[i];
      if (missing && missing >> i & 1) k = u32x4{~0u, ~0u, ~0u, ~0u};
      if (edge) {
        // a weight of zero does not hide infinities and NaN: values that no row sees become zeros here, and those that
        // only some rows see are taken out of the product and added one by one
        if (base + r < u.lo || base + r >= u.to) v = u32x4{0, 0, 0, 0};
        const uint64_t lanes = __ballot(not_finite<HALF, EIGHT>(v));
        if (lane == 0) lds_odd[buffer][i * W + wave] = lanes;
        if (lanes >> (lane / kRowLanes * kRowLanes) & ((1ull << kRowLanes) - 1)) v = u32x4{0, 0, 0, 0};
      }
      if constexpr (EIGHT) {
        const float fk = kFold ? __builtin_bit_cast(float, __shfl((int)ks, r >> 4, kWave)) : 1.0f;
        const float fv = __builtin_bit_cast(float, __shfl((int)value_scale, r >> 4, kWave));
        uint8_t* ka = at + r * kKeyPitch + my_col;
        uint8_t* va = at + kTile * kKeyPitch + r * kValuePitch + my_col;
        *(u32x4*)ka = widen<HALF>(u32x2{k[0], k[1]}, fk, fk);
        *(u32x4*)(ka + D) = widen<HALF>(u32x2{k[2], k[3]}, fk, fk);
        *(u32x4*)va = widen<true>(u32x2{v[0], v[1]}, fv, fv);
        *(u32x4*)(va + D) = widen<true>(u32x2{v[2], v[3]}, fv, fv);
      } else {
        *(u32x4*)(at + r * kKeyPitch + my_col) = k;
        *(u32x4*)(at + kTile * kKeyPitch + r * kValuePitch + my_col) = v;
      }
    }
  };

  if (begin < end) {
    look_up(begin);
    load(begin);
    look_up(begin + kTile);
    if constexpr (EIGHT) {
      const uint32_t scale = seen(begin) ? vs : 0;
#pragma unroll
      for (int g = 0; g < 4; ++g) unit_scale = std::max(unit_scale, (uint32_t)__builtin_amdgcn_readlane((int)scale, g) & kExponent);
      unit_scale += kNear << 23;
    }
    store(begin, 0);
    load(begin + kTile);
    look_up(begin + 2 * kTile);
  }
  int base = begin, buffer = 0;
  // One tile; kFar: its scales, or earlier ones, are far apart.
  auto take = [&](auto is_far) {
    constexpr bool kFar = decltype(is_far)::value;
    __syncthreads();
    const bool work = active && base < wave_to && base + kTile > wave_lo;
    const uint8_t* const tile = lds + buffer * kBuffer;
    float score[kScores];
    float f[4];
    if constexpr (EIGHT && !kFold) {
#pragma unroll
      for (int g = 0; g < 4; ++g) f[g] = key_scale[g];
    }
    if (work) {
      Result s[kTile / R];
#pragma unroll
      for (int g = 0; g < kTile / R; ++g)
#pragma unroll
        for (int j = 0; j < kSums; ++j) s[g][j] = 0;
#pragma unroll
      for (int t = 0; t < D / kSteps; ++t)
#pragma unroll
        for (int g = 0; g < kTile / R; ++g) {
          const u32x4 k = *(const u32x4*)(tile + (g * R + col) * kKeyPitch + t * kSteps * 2 + part * 16);
          if constexpr (R == 32) s[g] = mfma32<HALF>(k, qr[t], s[g]);
          else s[g] = mfma16<HALF>(k, qr[t], s[g]);
        }
      // six keys' operands ahead of the products: 1 % at 128 dims, 5 % at 256
      constexpr int kAll = D / kSteps * (kTile / R), kFirst = std::min(6, kAll);
      __builtin_amdgcn_sched_group_barrier(0x100, kFirst, 0);  // LDS reads
#pragma unroll
      for (int i = 0; i < kAll - kFirst; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);     // matrix instructions
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, kFirst, 0);
#pragma unroll
      for (int j = 0; j < kScores; ++j) score[j] = s[j / kSums][j % kSums];
    }
    if (base + kTile < end) {
      store(base + kTile, buffer ^ 1);
      load(base + 2 * kTile);
      look_up(base + 3 * kTile);
    }
    if (!work) return;

    if constexpr (EIGHT && !kFold) {
#pragma unroll
      for (int j = 0; j < kScores; ++j) score[j] *= f[R == 32 ? j / 8 : j / 4];
    }
    const bool edge = base < all_from || base + kTile > all_to;
    if (edge) {
#pragma unroll
      for (int j = 0; j < kScores; ++j) {
        const int p = base + position_of(j);
        if (p < row_from || p >= row_to) score[j] = -kInf;
      }
    }
    float top = score[0];
#pragma unroll
    for (int j = 0; j < kScores; ++j) top = __builtin_elementwise_maximum(top, score[j]);  // NaN stays
    if constexpr (R == 16) top = __builtin_elementwise_maximum(top, __shfl_xor(top, 16, kWave));
    top = __builtin_elementwise_maximum(top, __shfl_xor(top, 32, kWave));
    // m follows the largest score only when it is left behind by 2^kSlack: weights above one do no harm, and the sums are rarely
    // multiplied (for a new largest score in any of a wave's rows it would be most tiles)
    top *= factor;
    if (__any(!(top <= m + kSlack))) {
      const float now = __builtin_elementwise_maximum(m, top);
      const float shrink = now == m ? 1.0f : __builtin_amdgcn_exp2f(m - now);
      l *= shrink;
#pragma unroll
      for (int i = 0; i < kBlocks; ++i)
#pragma unroll
        for (int j = 0; j < kSums; ++j) sum[i][j] *= shrink;
      if constexpr (kFar) h = fmaxf(h + (m - now), kNothing);
      m = now;
    }
    const float sub = (m == -kInf ? 0.0f : m) - kLift;
    // weights as operands: the eight of a step are the positions of eight scores in a row
    u32x4 w[kTile / kSteps];
#pragma unroll
    for (int j = 0; j < kScores; ++j) {
      score[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(score[j], factor, -sub));
      l += score[j];
    }
    if constexpr (!kFar) {
#pragma unroll
      for (int j = 0; j < kScores / 2; ++j) w[j / 4][j % 4] = pack<kHalfP>(score[2 * j], score[2 * j + 1]);
    } else {
      // the scales are read once more, which costs less than keeping them where they are not needed
      const int p = std::min(base + (lane & 3) * 16, u.to - 1), where = kv_page(c, b, u.s, p);
      const float scales = c.v_scale[kv_scale_offset(c, where < 0 ? 0 : where, kvh, p)];
      constexpr int kEach = kScores / 4;  // scores of a lane that share a scale
      int of[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float x = score[g * kEach];
#pragma unroll
        for (int j = 1; j < kEach; ++j) x = __builtin_elementwise_maximum(x, score[g * kEach + j]);
        if constexpr (R == 16) x = __builtin_elementwise_maximum(x, __shfl_xor(x, 16, kWave));
        x = __builtin_elementwise_maximum(x, __shfl_xor(x, 32, kWave));
        of[g] = exponent_of(lane_value(scales, g));
        if (x != 0) h = fmaxf(h, exponent_of(x) + 1 + of[g]);
      }
      const int before = sum_unit;
      sum_unit = far_unit(h);
#pragma unroll
      for (int j = 0; j < kScores / 2; ++j) {
        const int by = of[2 * j / kEach] - sum_unit;
        w[j / 4][j % 4] = pack<true>(__builtin_amdgcn_ldexpf(score[2 * j], by), __builtin_amdgcn_ldexpf(score[2 * j + 1], by));
      }
#pragma unroll
      for (int i = 0; i < kBlocks; ++i)
#pragma unroll
        for (int e = 0; e < kSums; ++e) sum[i][e] = __builtin_amdgcn_ldexpf(sum[i][e], before - sum_unit);
    }
    // lane m of 16 gives the address of position m / 4 of four, dims 4 (m % 4) on, of the 16 dims that these lanes take
    const uint8_t* const columns = tile + kTile * kKeyPitch + (4 * part + (lane & 15) / 4) * kValuePitch + ((R == 32 ? (lane >> 4 & 1) * 16 : 0) + (lane & 3) * 4) * 2;
#pragma unroll
    for (int t = 0; t < kTile / kSteps; ++t)
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        const uint8_t* p = columns + t * kSteps * kValuePitch + i * R * 2;
        const u32x2 lo = read_columns16(p), hi = read_columns16(p + kSteps / 2 * kValuePitch);
        const u32x4 v = u32x4{lo[0], lo[1], hi[0], hi[1]};
        if constexpr (R == 32) sum[i] = mfma32<kHalfP>(v, w[t], sum[i]);
        else sum[i] = mfma16<kHalfP>(v, w[t], sum[i]);
      }
    if (partial(base)) {  // as store() saw it: rows of this wave may all see the tile, and those of others not
#pragma unroll 1
      for (int o = 0; o < kPasses * W; ++o) {
        const uint64_t lanes = lds_odd[buffer][o];
        if (!lanes) continue;
#pragma unroll 1
        for (int n = 0; n < kWave / kRowLanes; ++n) {
          if (!(lanes >> (n * kRowLanes) & ((1ull << kRowLanes) - 1))) continue;
          const int k = o / W * kRowsAPass + o % W * (kWave / kRowLanes) + n, p = base + k;
          const int where = kv_page(c, b, u.s, p);  // seen by some row, so below u.to
          if (where < 0) continue;                  // its key is NaN already
          const uint8_t* v = c.v + kv_offset(c, where, kvh, p);
          int own = part;
          asm volatile("" : "+v"(own));  // keeps the places of all dims from being computed, and held, before the tiles
          // the weight of k, from the lane that has it
          const int index = R == 32 ? k / 8 * 4 + k % 4 : k / 16 * 4 + k % 4;
          float x = 0;
#pragma unroll
          for (int j = 0; j < kScores; ++j)
            if (j == index) x = score[j];
          x = __shfl(x, (R == 32 ? k / 4 % 2 : k / 4 % 4) * R + col, kWave);
          if (p < row_from || p >= row_to) continue;
          if constexpr (EIGHT) {
            const float scale = c.v_scale[kv_scale_offset(c, where, kvh, p)];
            x = kFar ? __builtin_amdgcn_ldexpf(x, exponent_of(scale) - sum_unit)
                     : x * (scale / __builtin_bit_cast(float, unit_scale));
          }
#pragma unroll
          for (int i = 0; i < kBlocks; ++i)
#pragma unroll
            for (int e = 0; e < kSums; ++e) {
              if constexpr (EIGHT) sum[i][e] += x * __builtin_amdgcn_cvt_f32_fp8((int)v[dim_of(i, e, own)], 0);
              else sum[i][e] += x * to_float<HALF>(((const uint16_t*)v)[dim_of(i, e, own)]);
            }
        }
      }
    }
  };
  // A loop of its own for what comes after scales far apart: as a branch of this one between exponentials and products it would keep them from
  // mixing (a chunk of 4096 over 16384, e4m3: 945 us, and 1112).
  bool sums_far = false;
  for (; base < end && !(EIGHT && far); base += kTile, buffer ^= 1) take(std::false_type());
  if constexpr (EIGHT) {
    if (base < end) {
      sums_far = true;
      sum_unit = exponent_of(__builtin_bit_cast(float, unit_scale));
      h = m == -kInf ? kNothing : sum_unit + (kLift + kSlack);  // weights were at most 2^(kLift + kSlack)
      for (; base < end; base += kTile, buffer ^= 1) take(std::true_type());
    }
  }
  if (!active) return;

  if constexpr (R == 16) l += __shfl_xor(l, 16, kWave);
  l += __shfl_xor(l, 32, kWave);
  const float back = !EIGHT ? 1.0f : sums_far ? __builtin_amdgcn_ldexpf(1.0f, sum_unit) : __builtin_bit_cast(float, unit_scale);
  const int r = wave * R + col;
  if (r >= u.rows) return;
  if (cut >= 0) {
    const int64_t row = (cut + split) * (W * R) + r;
#pragma unroll
    for (int i = 0; i < kBlocks; ++i)
#pragma unroll
      for (int e = 0; e < kSums; e += 4)
        *(f32x4*)(parts.sums + row * D + dim_of(i, e, part)) = f32x4{sum[i][e], sum[i][e + 1], sum[i][e + 2], sum[i][e + 3]} * (EIGHT ? back / kPartUnit : 1.0f);
    if (part == 0) {
      parts.stats[row * 2] = m;
      parts.stats[row * 2 + 1] = l;
    }
    return;
  }
  const float inverse = q.bad ? __builtin_nanf("") : l == 0 ? 0.0f : back / l;
  uint16_t* const out = a.out + (q.row + token) * a.out_token + head * a.out_head;
#pragma unroll
  for (int i = 0; i < kBlocks; ++i)
#pragma unroll
    for (int e = 0; e < kSums; e += 4) {
      const f32x4 x = f32x4{sum[i][e], sum[i][e + 1], sum[i][e + 2], sum[i][e + 3]} * inverse;
      *(u32x2*)(out + dim_of(i, e, part)) = u32x2{pack<HALF>(x[0], x[1]), pack<HALF>(x[2], x[3])};
    }
  if (a.lse && part == 0)
    a.lse[(int64_t)(q.row + token) * a.q_heads + head] = q.bad ? __builtin_nanf("") : l == 0 ? -kInf : ((m - kLift) + __builtin_amdgcn_logf(l)) * kLn2;
}

// Rows of a unit, and how a workgroup is made of waves. A tile's loads are shared by all of them: a chunk of 4096 rows over 16384
// positions (32 heads over 8, 128 dims, e4m3) takes 920 us with eight waves of 32 rows and 970 with four. Four where there would be
// less than two workgroups of eight for each compute unit (2048 x 2048 positions: 69 us, and 78 with eight), and for 64
// dims, where three workgroups of them fit (9000 x 9000 positions: 428 us, and 446 with eight). 256 dims leave a wave of 32 rows a
// SIMD for itself; eight of 16 rows, two a SIMD, read LDS twice as often and are faster all the same: 2 x 3001 rows, a window of
// 1024, 8 heads over one took 121 us, and 173 with four of 32.
struct Shape {
  int rows, fit;   // of a unit; workgroups that fit at once
  bool eight;      // eight waves
};
Shape shape_of(const KvCache& c, const KvBatch& b, int group, int head_dim) {
  if (head_dim == 256) return {128, 256, true};
  if (head_dim == 64) return {128, 768, false};
  if ((int64_t)units_of(b, group, 256) * c.kv_heads >= 512) return {256, 256, true};
  return {128, 512, false};
}

void plan(const KvCache& c, const KvBatch& b, int group, const Shape& shape, const KvAttend& a, Parts* parts) {
  parts->units = units_of(b, group, shape.rows);
  int64_t span = b.max_context;
  const int64_t seen = (int64_t)a.window + shape.rows / group + 1 + 64;
  if (a.causal && a.window && seen < span) span = seen;  // else a window has no far end
  // the last rows of a prompt see more than the first ones
  const bool even = !a.causal || a.window || 2 * (int64_t)a.max_tokens <= b.max_context;
  cut_pairs(cut_of_many(shape.rows, shape.fit), c, span, even, parts);
}

template <int D, int W, int R>
hipError_t launch_waves(const KvCache& c, const KvBatch& b, const KvAttend& a, bool half, bool eight, const Parts& parts, hipStream_t stream) {
  const uint32_t grid = workgroups(c, parts);
  constexpr int kThreads = W * kWave;
  if (eight) {
    if (half) attend_many<D, true, true, W, R><<<grid, kThreads, 0, stream>>>(c, b, a, parts);
    else attend_many<D, false, true, W, R><<<grid, kThreads, 0, stream>>>(c, b, a, parts);
  } else if (half) {
    attend_many<D, true, false, W, R><<<grid, kThreads, 0, stream>>>(c, b, a, parts);
  } else {
    attend_many<D, false, false, W, R><<<grid, kThreads, 0, stream>>>(c, b, a, parts);
  }
  if (hipError_t e = hipGetLastError(); e != hipSuccess || parts.splits == 1) return e;
  return launch_join(c, b, a, parts, W * R, half || eight ? 8.0f : 0.0f, eight ? kPartUnit : 1.0f, D, half, stream);
}

template <int D>
hipError_t launch(const KvCache& c, const KvBatch& b, const KvAttend& a, bool half, bool eight, const Parts& parts, const Shape& shape, hipStream_t stream) {
  if constexpr (D == 256) {
    return launch_waves<D, 8, 16>(c, b, a, half, eight, parts, stream);
  } else if constexpr (D == 64) {
    return launch_waves<D, 4, 32>(c, b, a, half, eight, parts, stream);
  } else {
    if (shape.eight) return launch_waves<D, 8, 32>(c, b, a, half, eight, parts, stream);
    return launch_waves<D, 4, 32>(c, b, a, half, eight, parts, stream);
  }
}

}  // namespace

uint64_t kv_attend_many_workspace(const KvCache& c, const KvBatch& b, int q_heads, int head_dim) {
  const int group = q_heads / c.kv_heads;
  const Shape shape = shape_of(c, b, group, head_dim);
  return parts_bytes(cut_of_many(shape.rows, shape.fit), (int64_t)units_of(b, group, shape.rows) * c.kv_heads, b.max_context, shape.rows, head_dim);
}

hipError_t launch_kv_attend_many(const KvCache& c, const KvBatch& b, const KvAttend& a, int head_dim, bool half, bool eight, hipStream_t stream) {
  const int group = a.q_heads / c.kv_heads;
  const Shape shape = shape_of(c, b, group, head_dim);
  Parts parts;
  plan(c, b, group, shape, a, &parts);
  parts.sums = (float*)a.workspace;
  parts.stats = parts.sums + (int64_t)(parts.units * c.kv_heads - parts.whole) * parts.splits * shape.rows * head_dim;
  if (head_dim == 64) return launch<64>(c, b, a, half, eight, parts, shape, stream);
  if (head_dim == 128) return launch<128>(c, b, a, half, eight, parts, shape, stream);
  return launch<256>(c, b, a, half, eight, parts, shape, stream);
}

}  // namespace amem
