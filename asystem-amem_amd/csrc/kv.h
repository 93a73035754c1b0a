// Host-visible declarations of the kernels on a paged key/value cache: their argument records and launchers.
#ifndef AMEM_KV_LAUNCH_H_
#define AMEM_KV_LAUNCH_H_

#include <hip/hip_runtime_api.h>
#include <stdint.h>

#include "kv_index.h"

namespace amem {

// Strides in elements of 16 bits.
struct KvAppend {
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* q;
  uint16_t* q_out;
  const float* cos;
  const float* sin;
  const int* positions;
  int64_t k_token, k_head, v_token, v_head, q_token, q_head, qo_token, qo_head, positions_stride;
  int q_heads, rotary, interleaved, table_rows, axes;
  int axis_end[4];  // the first pair behind each axis
};

struct KvAttend {
  const uint16_t* q;
  uint16_t* out;
  float* lse;
  uint8_t* workspace;
  int64_t q_token, q_head, out_token, out_head;
  float scale;
  int q_heads, causal, window, max_tokens;
};

// `half`: the 16-bit type is fp16, else bf16; `eight`: the cache holds e4m3.
hipError_t launch_kv_append(const KvCache& c, const KvBatch& b, const KvAppend& a, int head_dim, bool half, bool eight, hipStream_t stream);
hipError_t launch_kv_attend(const KvCache& c, const KvBatch& b, const KvAttend& a, int head_dim, bool half, bool eight, hipStream_t stream);
// Few rows: at most 32 that share a key/value head, or 64 of 64 dims (more are right, and slow).
hipError_t launch_kv_attend_few(const KvCache& c, const KvBatch& b, const KvAttend& a, int head_dim, bool half, bool eight, hipStream_t stream);
uint64_t kv_attend_few_workspace(const KvCache& c, const KvBatch& b, int q_heads, int max_tokens, int head_dim);
hipError_t launch_kv_attend_many(const KvCache& c, const KvBatch& b, const KvAttend& a, int head_dim, bool half, bool eight, hipStream_t stream);
uint64_t kv_attend_many_workspace(const KvCache& c, const KvBatch& b, int q_heads, int head_dim);
uint64_t kv_attend_workspace(const KvCache& c, const KvBatch& b, int q_heads, int max_tokens, int head_dim);

}  // namespace amem
#endif
