// Attention over a paged key/value cache: which kernel takes a call, and the join of the parts of rows whose positions were
// dealt out to several workgroups.
#include <algorithm>

#include "kv_parts.h"

namespace amem {
namespace {

constexpr int kJoinWaves = 4;

// Joins the stretches of a row and query head: W waves take the stretches in turn (one wave where they are few, since then
// rows are many).
template <int D, bool HALF, int W>
__global__ __launch_bounds__(kJoinWaves * kWave) void join_stretches(KvCache c, KvBatch b, KvAttend a, Parts parts, int tile, float lift) {
  const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int index = blockIdx.x * (kJoinWaves / W) + wave / W, turn = wave % W;
  const int row = index / a.q_heads, head = index % a.q_heads, group = a.q_heads / c.kv_heads, kvh = head / group;
  constexpr int N = D / kWave;
  float m = -kInf, l = 0, x[N] = {};
  KvSeq q;
  Unit u;
  const int s = row >= b.tokens ? -1 : b.cu_tokens ? find_sequence(b, row, 1, 0) : row / b.uniform;
  bool mine = s >= 0;
  if (mine) {
    q = kv_seq(b, s);
    mine = row >= q.row && row < q.row + q.n;
  }
  int r = 0;
  int64_t first = 0;
  if (mine) {
    r = (row - q.row) * group + head % group;
    const int unit = (b.cu_tokens ? kv_unit_base(b, s, tile, 1, group) : s * ((b.uniform * group - 1) / tile + 1)) + r / tile;
    first = part_of(c, parts, unit, kvh);
    mine = first >= 0;  // else the unit's positions were not cut
  }
  if (mine) {
    unit_at(b, a, group, tile, s, r / tile, q, u);
    int count = (u.to - u.from + parts.stretch - 1) / parts.stretch;
    count = q.bad || count < 1 ? 1 : count > parts.splits ? parts.splits : count;
    // Eight parts are loaded at once, the first eight without waiting for the lengths, which say how many there are.
    constexpr int kBatch = 8;
    for (int i0 = turn; i0 < (W > 1 ? count : kBatch); i0 += W * kBatch) {
      float mi[kBatch], li[kBatch], xi[kBatch][N];
#pragma unroll
      for (int n = 0; n < kBatch; ++n) {
        const int64_t at = (first + std::min(i0 + n * W, parts.splits - 1)) * tile + r % tile;
        mi[n] = parts.stats[at * 2];
        li[n] = parts.stats[at * 2 + 1];
#pragma unroll
        for (int j = 0; j < N; ++j) xi[n][j] = parts.sums[at * D + lane * N + j];
      }
#pragma unroll
      for (int n = 0; n < kBatch; ++n) {
        const bool there = i0 + n * W < count;  // else it may hold anything
        mi[n] = there ? mi[n] : -kInf;
        const float now = __builtin_elementwise_maximum(m, mi[n]);
        const float f = m == now ? 1.0f : __builtin_amdgcn_exp2f(m - now), g = mi[n] == now ? 1.0f : __builtin_amdgcn_exp2f(mi[n] - now);
        m = now;
        l = l * f + (there ? li[n] * g : 0);
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = x[j] * f + (there ? xi[n][j] * g : 0);
      }
    }
  }
  if constexpr (W > 1) {
    __shared__ float part[W][D], stat[W][2];
#pragma unroll
    for (int j = 0; j < N; ++j) part[turn][lane * N + j] = x[j];
    if (lane == 0) { stat[turn][0] = m; stat[turn][1] = l; }
    __syncthreads();
    if (turn) return;
#pragma unroll
    for (int i = 1; i < W; ++i) {
      const float mi = stat[i][0], now = __builtin_elementwise_maximum(m, mi);
      const float f = m == now ? 1.0f : __builtin_amdgcn_exp2f(m - now), g = mi == now ? 1.0f : __builtin_amdgcn_exp2f(mi - now);
      m = now;
      l = l * f + stat[i][1] * g;
#pragma unroll
      for (int j = 0; j < N; ++j) x[j] = x[j] * f + part[i][lane * N + j] * g;
    }
  }
  if (!mine) return;
  uint16_t* at = a.out + row * a.out_token + head * a.out_head + lane * N;
#pragma unroll
  for (int j = 0; j < N; ++j) at[j] = from_float<HALF>(q.bad ? __builtin_nanf("") : l == 0 ? 0.0f : x[j] / l);
  if (a.lse && lane == 0) a.lse[(int64_t)row * a.q_heads + head] = q.bad ? __builtin_nanf("") : l == 0 ? -kInf : ((m - lift) + __builtin_amdgcn_logf(l)) * kLn2;
}

template <int D, bool HALF>
hipError_t join(const KvCache& c, const KvBatch& b, const KvAttend& a, const Parts& parts, int tile, float lift, hipStream_t stream) {
  // the units that are cut are the first ones; without cu_tokens it is known which tokens they have
  int tokens = b.tokens;
  if (!b.cu_tokens) {
    const int group = a.q_heads / c.kv_heads, each = (b.uniform * group - 1) / tile + 1, unit = parts.units - 1 - parts.whole / c.kv_heads;
    tokens = unit / each * b.uniform + (int)std::min<int64_t>(b.uniform, ((int64_t)(unit % each + 1) * tile + group - 1) / group);
  }
  const int rows = tokens * a.q_heads;
  if (parts.splits > 8) join_stretches<D, HALF, kJoinWaves><<<rows, kJoinWaves * kWave, 0, stream>>>(c, b, a, parts, tile, lift);
  else join_stretches<D, HALF, 1><<<(rows + kJoinWaves - 1) / kJoinWaves, kJoinWaves * kWave, 0, stream>>>(c, b, a, parts, tile, lift);
  return hipGetLastError();
}

// Few rows are those where the reading of the cache bounds: up to 32 that share a key/value head, 64 of 64 dims. 64 rows of
// 128 dims (8 sequences, 16 tokens, 4096 positions, e4m3) take 50 us as few and 37 as many; 64 rows of 64 dims (64 sequences, bf16) 85
// and 108.
bool few_rows(int q_heads, int kv_heads, int max_tokens, int head_dim) {
  return (int64_t)(q_heads / kv_heads) * max_tokens <= (head_dim == 64 ? 64 : 32);
}

}  // namespace

hipError_t launch_join(const KvCache& c, const KvBatch& b, const KvAttend& a, const Parts& parts, int tile, float lift, int head_dim, bool half, hipStream_t stream) {
  if (head_dim == 64) return half ? join<64, true>(c, b, a, parts, tile, lift, stream) : join<64, false>(c, b, a, parts, tile, lift, stream);
  if (head_dim == 128) return half ? join<128, true>(c, b, a, parts, tile, lift, stream) : join<128, false>(c, b, a, parts, tile, lift, stream);
  return half ? join<256, true>(c, b, a, parts, tile, lift, stream) : join<256, false>(c, b, a, parts, tile, lift, stream);
}

uint64_t kv_attend_workspace(const KvCache& c, const KvBatch& b, int q_heads, int max_tokens, int head_dim) {
  return few_rows(q_heads, c.kv_heads, max_tokens, head_dim) ? kv_attend_few_workspace(c, b, q_heads, max_tokens, head_dim)
                                                             : kv_attend_many_workspace(c, b, q_heads, head_dim);
}

hipError_t launch_kv_attend(const KvCache& c, const KvBatch& b, const KvAttend& a, int head_dim, bool half, bool eight, hipStream_t stream) {
  if (few_rows(a.q_heads, c.kv_heads, a.max_tokens, head_dim)) return launch_kv_attend_few(c, b, a, head_dim, half, eight, stream);
  return launch_kv_attend_many(c, b, a, head_dim, half, eight, stream);
}

}  // namespace amem
