// Attention over a paged key/value cache.
//
//   s_p = scale q.k_p,  m = max s_p,  l = sum exp(s_p - m),  out = sum exp(s_p - m) v_p / l,  lse = m + log l
//
// in one pass over the keys: m, l and the sum so far are carried along, and both are multiplied by
// exp(m_old - m_new) when a tile of keys raises m.
#include "kv_device.h"

namespace amem {
namespace {

template <bool HALF, bool EIGHT>
__device__ __forceinline__ float element(const uint8_t* at, int d) {
  if constexpr (EIGHT) return __builtin_amdgcn_cvt_f32_fp8((int)at[d], 0);
  else return to_float<HALF>(((const uint16_t*)at)[d]);
}

// One wave for a row and head: a lane takes a key of each 64, then D / 64 dims of the sum.
template <int D, bool HALF, bool EIGHT>
__global__ __launch_bounds__(kWave) void attend_row(KvCache c, KvBatch b, KvAttend a) {
  const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
  const int s = find_sequence(b, row, 0, 0);
  if (s < 0) return;
  const KvSeq q = kv_seq(b, s);
  if (row < q.row || row >= q.row + q.n) return;
  const int pos = q.context - q.n + row - q.row;
  const int kvh = h / (a.q_heads / c.kv_heads);
  int from = 0, to = q.context;
  if (a.causal && pos + 1 < to) to = pos + 1;
  if (a.window && pos - a.window + 1 > 0) from = pos - a.window + 1;
  __shared__ float qs[D], ps[kWave];
  __shared__ const uint8_t* vs[kWave];
  const uint16_t* qp = a.q + row * a.q_token + h * a.q_head;
  for (int d = lane; d < D; d += kWave) qs[d] = to_float<HALF>(qp[d]);
  __syncthreads();
  float m = -__builtin_inff(), l = 0, o[D / kWave] = {};
  bool bad = q.bad;
  for (int p0 = from; p0 < to; p0 += kWave) {
    const int p = p0 + lane;
    float x = -__builtin_inff(), vscale = 1;
    const uint8_t* v = nullptr;
    int page = 0;
    if (p < to) page = kv_page(c, b, s, p);
    if (__any(page < 0)) { bad = true; break; }
    if (p < to) {
      const uint8_t* k = c.k + kv_offset(c, page, kvh, p);
      v = c.v + kv_offset(c, page, kvh, p);
      x = 0;
      for (int d = 0; d < D; ++d) x += qs[d] * element<HALF, EIGHT>(k, d);
      x *= a.scale;
      if constexpr (EIGHT) {
        const int64_t at = kv_scale_offset(c, page, kvh, p);
        x *= c.k_scale[at];
        vscale = c.v_scale[at];
      }
    }
    float top = x;
#pragma unroll
    for (int i = kWave / 2; i; i >>= 1) top = fmaxf(top, __shfl_xor(top, i, kWave));
    if (__any(x != x)) top = __builtin_nanf("");
    const float now = top > m || top != top ? top : m;
    if (now == -__builtin_inff()) continue;
    const float shrink = expf(m - now), w = expf(x - now);
    float sum = w;
#pragma unroll
    for (int i = kWave / 2; i; i >>= 1) sum += __shfl_xor(sum, i, kWave);
    l = l * shrink + sum;
    m = now;
    ps[lane] = w * vscale;
    vs[lane] = v;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < D / kWave; ++i) o[i] *= shrink;
    for (int j = 0; j < kWave && p0 + j < to; ++j)
#pragma unroll
      for (int i = 0; i < D / kWave; ++i) o[i] += ps[j] * element<HALF, EIGHT>(vs[j], lane + i * kWave);
    __syncthreads();
  }
  const float nan = __builtin_nanf("");
#pragma unroll
  for (int i = 0; i < D / kWave; ++i)
    a.out[row * a.out_token + h * a.out_head + lane + i * kWave] = from_float<HALF>(bad ? nan : l == 0 ? 0 : o[i] / l);
  if (a.lse && lane == 0) a.lse[(int64_t)row * a.q_heads + h] = bad ? nan : l == 0 ? -__builtin_inff() : m + logf(l);
}

template <int D>
hipError_t launch(const KvCache& c, const KvBatch& b, const KvAttend& a, bool half, bool eight, hipStream_t stream) {
  const dim3 grid(b.tokens, a.q_heads);
  if (half && eight) attend_row<D, true, true><<<grid, kWave, 0, stream>>>(c, b, a);
  else if (half) attend_row<D, true, false><<<grid, kWave, 0, stream>>>(c, b, a);
  else if (eight) attend_row<D, false, true><<<grid, kWave, 0, stream>>>(c, b, a);
  else attend_row<D, false, false><<<grid, kWave, 0, stream>>>(c, b, a);
  return hipGetLastError();
}

}  // namespace

static bool few_rows(int q_heads, int kv_heads, int max_tokens, int head_dim) {
  return (int64_t)(q_heads / kv_heads) * max_tokens <= (head_dim == 256 ? 32 : 64);
}

uint64_t kv_attend_workspace(const KvCache& c, const KvBatch& b, int q_heads, int max_tokens, int head_dim) {
  return few_rows(q_heads, c.kv_heads, max_tokens, head_dim) ? kv_attend_few_workspace(c, b, q_heads, max_tokens, head_dim) : 0;
}

hipError_t launch_kv_attend(const KvCache& c, const KvBatch& b, const KvAttend& a, int head_dim, bool half, bool eight, hipStream_t stream) {
  if (few_rows(a.q_heads, c.kv_heads, a.max_tokens, head_dim)) return launch_kv_attend_few(c, b, a, head_dim, half, eight, stream);
  if (head_dim == 64) return launch<64>(c, b, a, half, eight, stream);
  if (head_dim == 128) return launch<128>(c, b, a, half, eight, stream);
  return launch<256>(c, b, a, half, eight, stream);
}

}  // namespace amem
