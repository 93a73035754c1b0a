// Attention over a paged key/value cache: which kernel takes a call, and the join of the parts of rows whose positions were
// dealt out to several workgroups.
#include <algorithm>

#include "kv_parts.h"

namespace amem {
namespace {

constexpr int kJoinThreads = 256;

// Joins the stretches of the pairs that were cut; 4 to 7 us, mostly latency. The last workgroup of a pair to end could join its parts
// itself, but has to see what the others wrote: their releases write back a whole L2 each (decode of four long contexts 118 -> 202 us).
//
// A thread has four dims of a row, or W threads have, which take the stretches in
// turn; B parts are loaded at once, the first of them before the lengths are known, which say how many there are, where all units have
// as many rows. `rows`: those that a unit can have.
template <int D, bool HALF, int W, int B>
__global__ __launch_bounds__(kJoinThreads) void join_stretches(KvCache c, KvBatch b, KvAttend a, Parts parts, int tile, int rows, float lift, float sum_unit) {
  constexpr int kItems = kJoinThreads / W;
  const int blocks = (rows * (D / 4) + kItems - 1) / kItems, pair = blockIdx.x / blocks, turn = threadIdx.x / kItems;
  const int item = blockIdx.x % blocks * kItems + threadIdx.x % kItems, r = item / (D / 4), d = item % (D / 4) * 4;
  const int64_t first = (int64_t)pair * parts.splits;
  float m = -kInf, l = 0;
  f32x4 x = {0, 0, 0, 0}, xi[B];
  f32x2 si[B];
  auto load = [&](int i0) {
#pragma unroll
    for (int n = 0; n < B; ++n) {
      const int64_t at = (first + std::min(i0 + n * W, parts.splits - 1)) * tile + r;
      si[n] = *(const f32x2*)(parts.stats + at * 2);
      xi[n] = *(const f32x4*)(parts.sums + at * D + d);
    }
  };
  if (!b.cu_tokens) load(turn);
  const int group = a.q_heads / c.kv_heads;
  int unit, kvh, split;
  pair_of(c, parts, parts.whole + pair, unit, kvh, split);
  KvSeq q;
  KvUnit u;
  const bool mine = find_unit(b, a, group, tile, unit, q, u) && r < u.rows;
  if (mine) {
    if (b.cu_tokens) load(turn);
    int count = (u.to - u.from + parts.stretch - 1) / parts.stretch;
    count = q.bad || count < 1 ? 1 : count > parts.splits ? parts.splits : count;
    for (int i0 = turn;;) {
#pragma unroll
      for (int n = 0; n < B; ++n) {
        const bool there = i0 + n * W < count;  // else it may hold anything
        const float mi = there ? si[n][0] : -kInf, now = __builtin_elementwise_maximum(m, mi);
        const float f = m == now ? 1.0f : __builtin_amdgcn_exp2f(m - now), g = mi == now ? 1.0f : __builtin_amdgcn_exp2f(mi - now);
        m = now;
        l = l * f + (there ? si[n][1] * g : 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = x[j] * f + (there ? xi[n][j] * g : 0);
      }
      i0 += W * B;
      if (i0 >= count) break;
      load(i0);
    }
  }
  if constexpr (W > 1) {
    __shared__ f32x4 part[W][kItems];
    __shared__ f32x2 stat[W][kItems];
    part[turn][threadIdx.x % kItems] = x;
    stat[turn][threadIdx.x % kItems] = f32x2{m, l};
    __syncthreads();
    if (turn) return;
#pragma unroll
    for (int i = 1; i < W; ++i) {
      const f32x2 s = stat[i][threadIdx.x];
      const f32x4 y = part[i][threadIdx.x];
      const float now = __builtin_elementwise_maximum(m, s[0]);
      const float f = m == now ? 1.0f : __builtin_amdgcn_exp2f(m - now), g = s[0] == now ? 1.0f : __builtin_amdgcn_exp2f(s[0] - now);
      m = now;
      l = l * f + s[1] * g;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = x[j] * f + y[j] * g;
    }
  }
  if (!mine) return;
  const int token = (u.first + r) / group, head = kvh * group + (u.first + r) % group;
  if (q.bad || l == 0) {
    x = f32x4{0, 0, 0, 0};
    l = q.bad ? __builtin_nanf("") : 0;
  }
  const float inverse = l == 0 ? 0.0f : sum_unit / l;
  *(u32x2*)(a.out + (q.row + token) * a.out_token + head * a.out_head + d) =
      u32x2{pack<HALF>(x[0] * inverse, x[1] * inverse), pack<HALF>(x[2] * inverse, x[3] * inverse)};
  if (a.lse && d == 0) a.lse[(int64_t)(q.row + token) * a.q_heads + head] = l == 0 ? -kInf : ((m - lift) + __builtin_amdgcn_logf(l)) * kLn2;
}

template <int D, bool HALF>
hipError_t join(const KvCache& c, const KvBatch& b, const KvAttend& a, const Parts& parts, int tile, float lift, float sum_unit, hipStream_t stream) {
  const int pairs = parts.units * c.kv_heads - parts.whole;
  const int rows = b.cu_tokens ? tile : (int)std::min<int64_t>(tile, (int64_t)b.uniform * (a.q_heads / c.kv_heads)), items = rows * (D / 4);
  auto blocks = [&](int each) { return pairs * ((items + each - 1) / each); };
  if (parts.splits > 8) join_stretches<D, HALF, 4, 8><<<blocks(kJoinThreads / 4), kJoinThreads, 0, stream>>>(c, b, a, parts, tile, rows, lift, sum_unit);
  else if (parts.splits > 4) join_stretches<D, HALF, 1, 8><<<blocks(kJoinThreads), kJoinThreads, 0, stream>>>(c, b, a, parts, tile, rows, lift, sum_unit);
  else join_stretches<D, HALF, 1, 4><<<blocks(kJoinThreads), kJoinThreads, 0, stream>>>(c, b, a, parts, tile, rows, lift, sum_unit);
  return hipGetLastError();
}

// Few rows are those where the reading of the cache bounds: up to 32 that share a key/value head, 64 of 64 dims. 64 rows of
// 128 dims (8 sequences, 16 tokens, 4096 positions, e4m3) take 50 us as few and 37 as many; 64 rows of 64 dims (64 sequences, bf16) 85
// and 108.
bool few_rows(int q_heads, int kv_heads, int max_tokens, int head_dim) {
  return (int64_t)(q_heads / kv_heads) * max_tokens <= (head_dim == 64 ? 64 : 32);
}

}  // namespace

hipError_t launch_join(const KvCache& c, const KvBatch& b, const KvAttend& a, const Parts& parts, int tile, float lift, float sum_unit, int head_dim, bool half, hipStream_t stream) {
  if (head_dim == 64) return half ? join<64, true>(c, b, a, parts, tile, lift, sum_unit, stream) : join<64, false>(c, b, a, parts, tile, lift, sum_unit, stream);
  if (head_dim == 128) return half ? join<128, true>(c, b, a, parts, tile, lift, sum_unit, stream) : join<128, false>(c, b, a, parts, tile, lift, sum_unit, stream);
  return half ? join<256, true>(c, b, a, parts, tile, lift, sum_unit, stream) : join<256, false>(c, b, a, parts, tile, lift, sum_unit, stream);
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
