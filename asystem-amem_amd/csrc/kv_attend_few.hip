// Attention over a paged key/value cache for few rows: single tokens, drafted tokens, up to 32 rows (64 of 64 dims) that share a
// key/value head (the rows of a sequence are its new tokens times the query heads of that head's group).
//
//   s_p = scale q.k_p,  m = max s_p,  l = sum exp(s_p - m),  out = sum exp(s_p - m) v_p / l,  lse = m + log l
//
// Bound by reading keys and values once; the arithmetic has to hide behind that. Four waves of a workgroup take tiles of a
// stretch of positions in turn, each with m, l and a sum of its own, and join them in LDS at the end. Longer
// contexts are cut into several stretches (workgroups), whose parts a second kernel joins.
//
// Both products run on the matrix unit as (keys x dims)(dims x rows) and (dims x keys)(keys x rows), so that a lane
// holds scores and sums of one row: the softmax needs two exchanges between lanes a tile. Keys and values are loaded as
// they lie, whole lines by one instruction, past the caches (nothing reads them twice), and pass through LDS, wave
// by wave, to become operands. A tile's registers are loaded again for the next tile as soon as LDS has them.
//
// Measured, where reading alone reaches 6.6 TB/s: 64 single tokens of 2048 to 8192 positions, 32 heads over 8, 128 dims, e4m3: 704 MB in
// 127 us, 5.6 TB/s (136 where the scales of values are far apart); four of 32768 to 131072: 683 MB in 119 us, 5.7; 32 of 1024 to 4096, 16 heads each with
// its own keys, bf16: 675 MB in 111 us, 6.1; five drafted tokens of 24 sequences, 64 heads over 8, 64 dims, fp16: 190 MB in 44 us, 4.3; one token
// of 1000 positions: 9.2 us, 3 of them in the join: latency, of the length, then page numbers, then keys.
#include <algorithm>

#include "kv_parts.h"

namespace amem {
namespace {

constexpr int kWaves = 4;

// Whether a wave has a SIMD, and all of its registers, to itself: where two would spill.
template <int D, bool EIGHT, int NB>
constexpr bool kOneWave = D == 256 && !(EIGHT && NB == 1);

// D dims, 16 bits of fp16 (HALF) or bf16, a cache of e4m3 (EIGHT), NB blocks of 16 rows, pages of at least 16 slots (WIDE).
template <int D, bool HALF, bool EIGHT, int NB, bool WIDE>
__global__ __launch_bounds__(kWaves * kWave, (kOneWave<D, EIGHT, NB> ? 1 : 2)) void attend_few(KvCache c, KvBatch b, KvAttend a, Parts few) {
  constexpr int kElement = EIGHT ? 1 : 2;
  constexpr int kTile = EIGHT && NB == 1 && D == 64 ? 64 : 32;  // positions of a tile
  constexpr int kGroups = kTile / 16;                  // of 16 positions: rows of an operand, and never over a page's end
  constexpr int kRowLanes = D * kElement / 16;         // lanes that load a position's key, or value
  constexpr int kRowsALoad = kWave / kRowLanes;
  constexpr int kRowLoads = kTile / kRowsALoad;
  // a row in LDS: its pad puts the rows that are read together on different banks
  constexpr int kPitch = D * kElement + (EIGHT ? 16 : 32);
  constexpr int kBlocks = D / 16;
  constexpr bool kHalfP = EIGHT || HALF;  // weights are fp16 where the values' type allows it
  // fp16 weights are held 2^8 times larger, which keeps small ones out of the subnormal numbers
  constexpr float kLift = kHalfP ? 8.0f : 0.0f;
  constexpr int kLds = kWaves * kTile * kPitch, kJoin = kWaves * 16 * (D + 4) * 4;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kLds > kJoin ? kLds : kJoin];
  __shared__ float lds_m[kWaves][16 * NB], lds_l[kWaves][16 * NB];

  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  // heads first: their rows of a page are neighbours
  const int group = a.q_heads / c.kv_heads;
  int kvh, unit, split;
  pair_of(c, few, blockIdx.x, unit, kvh, split);
  KvSeq q;
  KvUnit u;
  if (!find_unit(b, a, group, 16 * NB, unit, q, u)) return;
  const int begin = u.from + split * few.stretch;
  const int64_t part = part_of(c, few, unit, kvh) + split;  // below zero: the unit's positions are not cut
  if (split && (begin >= u.to || q.bad)) return;
  const int end = part >= 0 && begin + few.stretch < u.to ? begin + few.stretch : u.to;
  const int col = lane & 15, quad = lane >> 4;

  // Queries, the operand of a block of rows: dims in the order of the keys' operand. More than one block leaves no registers
  // for them; they are in LDS then, read once a tile.
  constexpr bool kQueriesInLds = NB > 1;
  constexpr int kQueryPitch = D * 2 + 16;
  __shared__ __attribute__((aligned(16))) uint8_t lds_q[kQueriesInLds ? 16 * NB * kQueryPitch : 16];
  u32x4 qr[kQueriesInLds ? 1 : D / 32];
  int row_from[NB], row_to[NB];
  auto query = [&](int r) {
    if (r >= u.rows) r = u.rows - 1;
    r += u.first;
    return a.q + (q.row + r / group) * a.q_token + (kvh * group + r % group) * a.q_head;
  };
  auto dim_of = [&](int t) { return EIGHT ? (t / 2) * 64 + quad * 16 + (t % 2) * 8 : t * 32 + quad * 8; };
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    int r = n * 16 + col;
    if (r >= u.rows) r = u.rows - 1;
    row_range(a, q, (u.first + r) / group, row_from[n], row_to[n]);
  }
  if constexpr (kQueriesInLds) {
    for (int i = threadIdx.x; i < 16 * NB * (D / 8); i += kWaves * kWave)
      *(u32x4*)(lds_q + i / (D / 8) * kQueryPitch + i % (D / 8) * 16) = *(const u32x4*)(query(i / (D / 8)) + i % (D / 8) * 8);
    __syncthreads();
  } else {
#pragma unroll
    for (int t = 0; t < D / 32; ++t) qr[t] = *(const u32x4*)(query(col) + dim_of(t));
  }

  float m[NB], l[NB];
  f32x4 sum[NB][kBlocks];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    m[n] = -kInf;
    l[n] = 0;
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) sum[n][i] = f32x4{0, 0, 0, 0};
  }
  // 8 bits: the sums are in multiples of unit_scale, or (far) of the row's 2^sum_unit
  float unit_scale = 0, h[NB];
  int sum_unit[NB];
  bool far = false;

  uint8_t* const mine = lds + wave * kTile * kPitch;
  const uint8_t* const keys = c.k + (int64_t)kvh * c.head_stride;
  const uint8_t* const values = c.v + (int64_t)kvh * c.head_stride;
  const int slot_mask = (1 << c.page_shift) - 1;
  // where this lane writes its values, and reads columns. 8 bits: a lane reads eight rows as one column, which are to be
  // the positions of its eight weights, so position r of 32 goes to row 8 ((r % 16) / 4) + 4 (r / 16) + r % 4
  const int value_row = lane / kRowLanes, value_col = lane % kRowLanes * 16;
  auto lds_row = [](int r) { return EIGHT ? (r & ~31) + 8 * ((r & 15) >> 2) + 4 * ((r & 31) >> 4) + (r & 3) : r; };
  const int write_at = lds_row(value_row) * kPitch + value_col;
  const int read_at = EIGHT ? (8 * quad + (col >> 1)) * kPitch + (col & 1) * 8 : (4 * quad + (col >> 2)) * kPitch + (col & 3) * 8;

  u32x4 kreg[kRowLoads], vreg[kRowLoads];
  int page = 0, page_next = 0, page_after = 0;  // of position base + lane of this tile (-1: out of range), the next and the one behind it
  float ks = 0, vs = 0;

  // What the page table has for position base + lane, behind the last position that one's. Nothing is done with it here: that
  // would wait for all loads under way.
  auto look_up = [&](int base) { return kv_table(c, b, u.s, std::min(base + (lane & (kTile - 1)), u.to - 1)); };
  auto row_of = [&](int page, int p) {
    return (int64_t)(page < 0 ? 0 : page) * c.page_stride + (int64_t)(p & slot_mask) * c.slot_stride;
  };
  // this lane's offset in a group that lies in one page: 32 bits, since a page's rows span less than 2^31 bytes
  const uint32_t lane_off = (uint32_t)((value_row & 15) * (int)c.slot_stride + value_col);
  // Loads are never skipped, which would make the compiler keep the registers' old contents and copy them about: behind the last
  // tile (`more` false) all of them read one line.
  auto load_rows = [&](const uint8_t* from, int base, int page, bool more, u32x4 (&to)[kRowLoads]) {
#pragma unroll
    for (int i = 0; i < kRowLoads; ++i) {
      const uint8_t* at;
      if constexpr (WIDE) {
        const int64_t row = row_of(__builtin_amdgcn_readlane(page, i * kRowsALoad & ~15), base + i * kRowsALoad);
        at = from + (more ? row : 0) + (more ? lane_off : 0);
      } else {
        const int64_t row = row_of(__shfl(page, i * kRowsALoad + value_row, kWave), base + i * kRowsALoad + value_row) + value_col;
        at = from + (more ? row : 0);
      }
      to[i] = __builtin_nontemporal_load((const u32x4*)at);
    }
  };
  auto load_scales = [&](int base, int page, float& k, float& v) {
    if constexpr (EIGHT) {
      const int64_t at = kv_scale_offset(c, page < 0 ? 0 : page, kvh, base + lane);
      k = c.k_scale[at];
      v = c.v_scale[at];
    }
  };

  int base = begin + wave * kTile;
  constexpr int kStep = kWaves * kTile;
  auto seen = [&](int from) { return from < u.to && from + 15 >= u.lo; };  // a hidden group's scale may be anything
  float inverse_unit = 0;
  if (base < end) {
    page = look_up(base);
    page_next = look_up(base + kStep);
    page = kv_checked(c, page);
    load_rows(keys, base, page, true, kreg);
    load_scales(base, page, ks, vs);
    load_rows(values, base, page, true, vreg);
  }
  for (; base < end; base += kStep) {
    const bool more = base + kStep < end;
    const bool whole = base >= u.all_from && base + kTile <= u.all_to;
#pragma unroll
    for (int i = 0; i < kRowLoads; ++i) *(u32x4*)(mine + (i * kRowsALoad + value_row) * kPitch + value_col) = kreg[i];
    __builtin_amdgcn_wave_barrier();
    // before the loads that it must not wait for
    page_after = look_up(base + 2 * kStep);
    page_next = kv_checked(c, page_next);
    load_rows(keys, base + kStep, page_next, more, kreg);
    f32x4 score[NB][kGroups];
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
#pragma unroll
      for (int n = 0; n < NB; ++n) score[n][g] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int t = 0; t < D / 32; ++t) {
      u32x4 qt[NB];
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        if constexpr (kQueriesInLds) qt[n] = *(const u32x4*)(lds_q + (n * 16 + col) * kQueryPitch + dim_of(t) * 2);
        else qt[n] = qr[t];
      }
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        const uint8_t* p = mine + (g * 16 + col) * kPitch;
        u32x4 k;
        if constexpr (EIGHT) k = widen<HALF>(*(const u32x2*)(p + t / 2 * 64 + quad * 16 + t % 2 * 8));
        else k = *(const u32x4*)(p + t * 64 + quad * 16);
#pragma unroll
        for (int n = 0; n < NB; ++n) score[n][g] = mfma16<HALF>(k, qt[n], score[n][g]);
      }
    }
    __builtin_amdgcn_wave_barrier();

    // scores in units of log 2
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      const float f = a.scale * kLog2e * (EIGHT ? lane_value(ks, g * 16) : 1.0f);
#pragma unroll
      for (int n = 0; n < NB; ++n) score[n][g] *= f;
    }
    if (!whole) {
      const uint64_t bad = __ballot(page < 0);
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = g * 16 + quad * 4 + i, p = base + k;
#pragma unroll
          for (int n = 0; n < NB; ++n) {
            if (bad >> k & 1) score[n][g][i] = __builtin_nanf("");
            if (p < row_from[n] || p >= row_to[n]) score[n][g][i] = -kInf;
          }
        }
    } else if (__any(page < 0)) {
      const uint64_t bad = __ballot(page < 0);
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int n = 0; n < NB; ++n)
            if (bad >> (g * 16 + quad * 4 + i) & 1) score[n][g][i] = __builtin_nanf("");
    }
    // values that no row sees are stored as zeros, since a weight of zero does not hide infinities and NaN
    bool odd = false;  // some positions have such values, and may be hidden from some rows
    if (whole) {
#pragma unroll
      for (int i = 0; i < kRowLoads; ++i) *(u32x4*)(mine + write_at + lds_row(i * kRowsALoad) * kPitch) = vreg[i];
    } else {
#pragma unroll
      for (int i = 0; i < kRowLoads; ++i) {
        const int p = base + i * kRowsALoad + value_row;
        u32x4 v = vreg[i];
        if (p < u.lo || p >= u.to) v = u32x4{0, 0, 0, 0};
        // those are taken out of the product and added one by one below
        const uint64_t lanes = __ballot(not_finite<HALF, EIGHT>(v));
        odd |= lanes != 0;
        if (lanes >> (value_row * kRowLanes) & ((1ull << kRowLanes) - 1)) v = u32x4{0, 0, 0, 0};
        *(u32x4*)(mine + write_at + lds_row(i * kRowsALoad) * kPitch) = v;
      }
    }
    __builtin_amdgcn_wave_barrier();
    const int page_now = page;
    page = page_next;
    page_next = page_after;
    float ks_next = 0, vs_next = 0;
    load_scales(base + kStep, page, ks_next, vs_next);
    load_rows(values, base + kStep, page, more, vreg);

    float f_scale[kGroups];  // scales of values, in multiples of unit_scale
    if constexpr (EIGHT) {
      if (unit_scale == 0) {  // the first tile that some row sees: in front of a window's beginning others may lie
#pragma unroll
        for (int g = 0; g < kGroups; ++g) unit_scale = fmaxf(unit_scale, seen(base + g * 16) ? lane_value(vs, g * 16) : 0);
        unit_scale *= 1 << kNear;
        inverse_unit = 1.0f / unit_scale;
      }
      float least = 1, most = 0;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        f_scale[g] = far ? 1.0f : seen(base + g * 16) ? lane_value(vs, g * 16) * inverse_unit : 1.0f;
        least = fminf(least, f_scale[g]);
        most = fmaxf(most, f_scale[g]);
      }
      if (!(most <= 1 && least >= 1.0f / (1 << 2 * kNear))) {
        far = true;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          sum_unit[n] = exponent_of(unit_scale);
          h[n] = m[n] == -kInf ? kNothing : sum_unit[n] + kLift;  // weights were at most 2^kLift
        }
#pragma unroll
        for (int g = 0; g < kGroups; ++g) f_scale[g] = 1.0f;
      }
    }

    // running maximum; where it grows, what has been summed shrinks
    bool grew = false;
    float shrink[NB];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      float top = score[n][0][0];
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = __builtin_elementwise_maximum(top, score[n][g][i]);  // NaN stays
      top = __builtin_elementwise_maximum(top, __shfl_xor(top, 16, kWave));
      top = __builtin_elementwise_maximum(top, __shfl_xor(top, 32, kWave));
      const float now = __builtin_elementwise_maximum(m[n], top);
      shrink[n] = now == m[n] ? 1.0f : __builtin_amdgcn_exp2f(m[n] - now);
      grew |= now != m[n];
      if (EIGHT && far) h[n] = fmaxf(h[n] + (m[n] - now), kNothing);
      m[n] = now;
    }
    if (__any(grew)) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        l[n] *= shrink[n];
#pragma unroll
        for (int i = 0; i < kBlocks; ++i) sum[n][i] *= shrink[n];
      }
    }
    u32x4 w[NB][kGroups / 2];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const float top = (m[n] == -kInf ? 0.0f : m[n]) - kLift;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = __builtin_amdgcn_exp2f(score[n][g][i] - top);
          l[n] += x[i];
          score[n][g][i] = x[i];
        }
        w[n][g / 2][g % 2 * 2] = pack<kHalfP>(x[0], x[1]);
        w[n][g / 2][g % 2 * 2 + 1] = pack<kHalfP>(x[2], x[3]);
      }
    }
    if (EIGHT && far) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        int of[kGroups];
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          float x = score[n][g][0];
#pragma unroll
          for (int i = 1; i < 4; ++i) x = __builtin_elementwise_maximum(x, score[n][g][i]);
          x = __builtin_elementwise_maximum(x, __shfl_xor(x, 16, kWave));
          x = __builtin_elementwise_maximum(x, __shfl_xor(x, 32, kWave));
          of[g] = exponent_of(lane_value(vs, g * 16));
          if (x != 0) h[n] = fmaxf(h[n], exponent_of(x) + 1 + of[g]);
        }
        const int before = sum_unit[n];
        sum_unit[n] = far_unit(h[n]);
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
          float x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_ldexpf(score[n][g][i], of[g] - sum_unit[n]);
          w[n][g / 2][g % 2 * 2] = pack<true>(x[0], x[1]);
          w[n][g / 2][g % 2 * 2 + 1] = pack<true>(x[2], x[3]);
        }
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[n][i][e] = __builtin_amdgcn_ldexpf(sum[n][i][e], before - sum_unit[n]);
      }
    }
#pragma unroll
    for (int t = 0; t < kTile / 32; ++t)
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) {
        const uint8_t* p = mine + read_at + t * 32 * kPitch + i * 16 * kElement;
        u32x4 v;
        if constexpr (EIGHT) {
          v = widen<true>(read_columns8(p), f_scale[2 * t], f_scale[2 * t + 1]);
        } else {
          const u32x2 lo = read_columns16(p), hi = read_columns16(p + 16 * kPitch);
          v = u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
#pragma unroll
        for (int n = 0; n < NB; ++n) sum[n][i] = mfma16<kHalfP>(v, w[n][t], sum[n][i]);
      }
    __builtin_amdgcn_wave_barrier();
    if (odd) {
      // one position after the other: its values through LDS, its weights from the lanes that hold them
#pragma unroll 1
      for (int k = 0; k < kTile; ++k) {
        const int p = base + k;
        if (p < u.lo || p >= u.to) continue;
        const uint8_t* at = values + row_of(__builtin_amdgcn_readlane(page_now, k), p);
        u32x4 v = {0, 0, 0, 0};
        if (lane < kRowLanes) v = *(const u32x4*)(at + lane * 16);
        if (!__any(not_finite<HALF, EIGHT>(v))) continue;
        if (lane < kRowLanes) *(u32x4*)(mine + lane * 16) = v;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          float x = 0;
#pragma unroll
          for (int g = 0; g < kGroups; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (g == k / 16 && e == k % 4) x = score[n][g][e];
          x = __shfl(x, (k % 16 / 4) * 16 + col, kWave);
          if (p < row_from[n] || p >= row_to[n]) continue;
          if constexpr (EIGHT) {
#pragma unroll
            for (int g = 0; g < kGroups; ++g)
              if (g == k / 16) x = far ? __builtin_amdgcn_ldexpf(x, exponent_of(lane_value(vs, g * 16)) - sum_unit[n]) : x * f_scale[g];
          }
#pragma unroll
          for (int d = 0; d < kBlocks; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int i = d * 16 + quad * 4 + e;
              if constexpr (EIGHT) sum[n][d][e] += x * __builtin_amdgcn_cvt_f32_fp8((int)mine[i], 0);
              else sum[n][d][e] += x * to_float<HALF>(((const uint16_t*)mine)[i]);
            }
        }
        __builtin_amdgcn_wave_barrier();
      }
    }
    ks = ks_next;
    vs = vs_next;
  }

  // the four waves' parts become one
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    l[n] += __shfl_xor(l[n], 16, kWave);
    l[n] += __shfl_xor(l[n], 32, kWave);
    if (lane < 16) {
      lds_m[wave][n * 16 + lane] = m[n];
      lds_l[wave][n * 16 + lane] = l[n];
    }
  }
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    __syncthreads();
    float top = lds_m[0][n * 16 + col];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) top = __builtin_elementwise_maximum(top, lds_m[i][n * 16 + col]);
    float f = m[n] == top ? 1.0f : __builtin_amdgcn_exp2f(m[n] - top);
    if constexpr (EIGHT) f *= far ? __builtin_amdgcn_ldexpf(1.0f, sum_unit[n] - kPartExponent) : unit_scale / kPartUnit;
    float* at = (float*)lds + (wave * 16 + col) * (D + 4) + quad * 4;
#pragma unroll
    for (int i = 0; i < kBlocks; ++i) *(f32x4*)(at + i * 16) = sum[n][i] * f;
    __syncthreads();
    constexpr int kVectors = 16 * D / 4;
#pragma unroll
    for (int v0 = 0; v0 < kVectors; v0 += kWaves * kWave) {
      const int v = v0 + threadIdx.x, r = v / (D / 4), d = v % (D / 4) * 4;
      if (kVectors % (kWaves * kWave) && v >= kVectors) break;
      if (n * 16 + r >= u.rows) continue;
      float mm = lds_m[0][n * 16 + r];
#pragma unroll
      for (int i = 1; i < kWaves; ++i) mm = __builtin_elementwise_maximum(mm, lds_m[i][n * 16 + r]);
      float ll = 0;
      f32x4 x = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < kWaves; ++i) {
        const float mi = lds_m[i][n * 16 + r];
        ll += lds_l[i][n * 16 + r] * (mi == mm ? 1.0f : __builtin_amdgcn_exp2f(mi - mm));
        x += *(const f32x4*)((const float*)lds + (i * 16 + r) * (D + 4) + d);
      }
      if (part >= 0) {
        const int64_t row = part * (16 * NB) + n * 16 + r;
        *(f32x4*)(few.sums + row * D + d) = x;
        if (d == 0) {
          few.stats[row * 2] = mm;
          few.stats[row * 2 + 1] = ll;
        }
        continue;
      }
      const int rr = u.first + n * 16 + r, token = rr / group, head = kvh * group + rr % group;
      const float inverse = q.bad ? __builtin_nanf("") : ll == 0 ? 0.0f : (EIGHT ? kPartUnit : 1.0f) / ll;
      if (ll == 0) x = f32x4{0, 0, 0, 0};
      *(u32x2*)(a.out + (q.row + token) * a.out_token + head * a.out_head + d) =
          u32x2{pack<HALF>(x[0] * inverse, x[1] * inverse), pack<HALF>(x[2] * inverse, x[3] * inverse)};
      if (a.lse && d == 0)
        a.lse[(int64_t)(q.row + token) * a.q_heads + head] = q.bad ? __builtin_nanf("") : ll == 0 ? -kInf : ((mm - kLift) + __builtin_amdgcn_logf(ll)) * kLn2;
    }
  }
}

// Blocks of 16 rows that a workgroup takes: enough for all rows of a sequence's key/value head, so that its keys and
// values are read once.
int blocks_of(int group, int max_tokens, int head_dim) {
  const int64_t rows = (int64_t)group * max_tokens;
  return rows <= 16 ? 1 : rows <= 32 || head_dim > 64 ? 2 : rows <= 48 ? 3 : 4;
}

void plan(const KvCache& c, const KvBatch& b, int group, int head_dim, bool eight, int blocks, const KvAttend& a, Parts* few) {
  int64_t span = b.max_context;
  const int64_t seen = (int64_t)a.window + (16 * blocks) / group + 1 + 64;
  if (a.causal && a.window && seen < span) span = seen;  // else a window has no far end
  few->units = units_of(b, group, 16 * blocks);
  cut_pairs(cut_of_few(head_dim, eight, blocks), c, span, true, few);
}

template <int D, bool HALF, bool EIGHT, int NB>
hipError_t launch_few(const KvCache& c, const KvBatch& b, const KvAttend& a, const Parts& few, hipStream_t stream) {
  const uint32_t grid = workgroups(c, few);
  if constexpr (!EIGHT) {
    if (c.page_shift < 4) attend_few<D, HALF, EIGHT, NB, false><<<grid, kWaves * kWave, 0, stream>>>(c, b, a, few);
    else attend_few<D, HALF, EIGHT, NB, true><<<grid, kWaves * kWave, 0, stream>>>(c, b, a, few);
  } else {
    attend_few<D, HALF, EIGHT, NB, true><<<grid, kWaves * kWave, 0, stream>>>(c, b, a, few);
  }
  if (hipError_t e = hipGetLastError(); e != hipSuccess || few.splits == 1) return e;
  return launch_join(c, b, a, few, 16 * NB, EIGHT || HALF ? 8.0f : 0.0f, EIGHT ? kPartUnit : 1.0f, D, HALF, stream);
}

template <int D, bool HALF, bool EIGHT>
hipError_t launch_blocks(const KvCache& c, const KvBatch& b, const KvAttend& a, const Parts& few, int blocks, hipStream_t stream) {
  if (blocks == 1) return launch_few<D, HALF, EIGHT, 1>(c, b, a, few, stream);
  if (blocks == 2) return launch_few<D, HALF, EIGHT, 2>(c, b, a, few, stream);
  if constexpr (D == 64) return blocks == 3 ? launch_few<D, HALF, EIGHT, 3>(c, b, a, few, stream) : launch_few<D, HALF, EIGHT, 4>(c, b, a, few, stream);
  else return launch_few<D, HALF, EIGHT, 2>(c, b, a, few, stream);
}

template <int D>
hipError_t launch_dims(const KvCache& c, const KvBatch& b, const KvAttend& a, bool half, bool eight, const Parts& few, int blocks, hipStream_t stream) {
  if (half) return eight ? launch_blocks<D, true, true>(c, b, a, few, blocks, stream) : launch_blocks<D, true, false>(c, b, a, few, blocks, stream);
  return eight ? launch_blocks<D, false, true>(c, b, a, few, blocks, stream) : launch_blocks<D, false, false>(c, b, a, few, blocks, stream);
}

}  // namespace

uint64_t kv_attend_few_workspace(const KvCache& c, const KvBatch& b, int q_heads, int max_tokens, int head_dim) {
  const int group = q_heads / c.kv_heads, blocks = blocks_of(group, max_tokens, head_dim);
  return parts_bytes(cut_of_few(head_dim, c.block_shift > 0, blocks), (int64_t)units_of(b, group, 16 * blocks) * c.kv_heads, b.max_context, 16 * blocks, head_dim);
}

hipError_t launch_kv_attend_few(const KvCache& c, const KvBatch& b, const KvAttend& a, int head_dim, bool half, bool eight, hipStream_t stream) {
  const int group = a.q_heads / c.kv_heads, blocks = blocks_of(group, a.max_tokens, head_dim);
  Parts few;
  plan(c, b, group, head_dim, eight, blocks, a, &few);
  few.sums = (float*)a.workspace;
  few.stats = few.sums + (int64_t)(few.units * c.kv_heads - few.whole) * few.splits * (16 * blocks) * head_dim;
  if (head_dim == 64) return launch_dims<64>(c, b, a, half, eight, few, blocks, stream);
  if (head_dim == 128) return launch_dims<128>(c, b, a, half, eight, few, blocks, stream);
  return launch_dims<256>(c, b, a, half, eight, few, blocks, stream);
}

}  // namespace amem
