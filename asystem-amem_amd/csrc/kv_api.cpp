// The C entry points of include/amem_kv.h: what they refuse, the paused gate, and the device they launch on.
#include <hip/hip_runtime_api.h>
#include <unistd.h>

#include <algorithm>
#include <initializer_list>
#include <mutex>
#include <utility>

#include "../../include/amem.h"
#include "../../include/amem_kv.h"
#include "ctx.h"
#include "ipc.h"
#include "kv.h"
#include "log.h"
#include "vmm.h"

namespace amem {
namespace {

int refuse(const char* what, const char* why) {
  LOGGER(ERROR, "%s: refused: %s", what, why);
  return (int)hipErrorInvalidValue;
}
#define NEED(cond, why) \
  do {                  \
    if (!(cond)) return refuse(what, why); \
  } while (0)

int log2_of(int x) { return x > 0 && (x & (x - 1)) == 0 ? __builtin_ctz(x) : -1; }

bool fits(int64_t n, int64_t stride) {
  int64_t bytes;
  return !__builtin_mul_overflow(n, stride, &bytes) && bytes >= 0 && bytes < ((int64_t)1 << 58);
}

// Strides that a view of a tensor can have: whole vectors of 16 bytes, forward, below 2^40 elements.
bool stride_ok(int64_t s, int vector) { return s >= 0 && s < ((int64_t)1 << 40) && s % vector == 0; }

int check_cache(const char* what, const amem_kv_cache* c, bool addresses, KvCache* out) {
  NEED(c, "cache is NULL");
  NEED(c->type == AMEM_KV_BF16 || c->type == AMEM_KV_F16 || c->type == AMEM_KV_E4M3, "cache type");
  NEED(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, "head_dim is not 64, 128 or 256");
  NEED(c->pages >= 1 && c->kv_heads >= 1 && c->kv_heads <= 1024, "pages or kv_heads out of range");
  const int page_shift = log2_of(c->page_slots), block_shift = log2_of(c->block_slots);
  NEED(page_shift >= 0 && page_shift <= 10, "page_slots is not a power of two from 1 to 1024");
  const bool eight = c->type == AMEM_KV_E4M3;
  const int element = eight ? 1 : 2;
  if (eight) {
    NEED(block_shift >= 4 && block_shift <= 7 && block_shift <= page_shift,
         "block_slots is not a power of two from 16 to 128 and at most page_slots");
    NEED(c->scale_page_stride >= 0 && c->scale_head_stride >= 0, "scale strides");
  } else {
    NEED(c->block_slots == 0 && c->k_scale == 0 && c->v_scale == 0, "scales with a 16-bit cache");
  }
  NEED(stride_ok(c->page_stride, 16 / element) && stride_ok(c->head_stride, 16 / element) &&
           stride_ok(c->slot_stride, 16 / element),
       "cache strides are not multiples of 16 bytes");
  // offsets fit 63 bits with room to add them up
  NEED(fits(c->pages, c->page_stride) && fits(c->kv_heads, c->head_stride) && fits(c->page_slots, c->slot_stride) &&
           fits(c->pages, c->scale_page_stride) && fits(c->kv_heads, c->scale_head_stride),
       "the cache is larger than addresses");
  NEED((c->slot_stride * element) << page_shift < (int64_t)1 << 31, "the slots of a page are 2^31 bytes or more apart");
  NEED(c->reserved == 0, "cache.reserved is not 0");
  if (addresses) {
    NEED(c->k && c->v && c->k % 16 == 0 && c->v % 16 == 0, "cache addresses are not aligned to 16 bytes");
    if (eight) NEED(c->k_scale && c->v_scale && c->k_scale % 4 == 0 && c->v_scale % 4 == 0, "addresses of the scales");
  }
  *out = {(uint8_t*)(uintptr_t)c->k, (uint8_t*)(uintptr_t)c->v, (float*)(uintptr_t)c->k_scale, (float*)(uintptr_t)c->v_scale,
          c->page_stride * element, c->head_stride * element, c->slot_stride * element, c->scale_page_stride,
          c->scale_head_stride, c->pages, c->kv_heads, page_shift, eight ? block_shift : 0};
  return 0;
}

int check_batch(const char* what, const amem_kv_batch* b, const KvCache& c, bool addresses, KvBatch* out) {
  NEED(b, "batch is NULL");
  // launches stay below 2^32 threads
  NEED(b->sequences >= 0 && b->sequences <= 1 << 20 && b->tokens >= 0 && b->tokens <= 1 << 22,
       "sequences or tokens out of range");
  NEED((int64_t)(b->tokens / 16 + 2 * b->sequences) * c.kv_heads <= 1 << 22, "tokens or sequences times kv_heads out of range");
  NEED(b->max_tokens >= 0 && b->max_tokens <= b->tokens, "max_tokens is not between 0 and tokens");
  NEED(b->table_pages >= 0 && b->table_stride >= b->table_pages, "table_pages or table_stride");
  NEED(b->max_context >= 0 && b->max_context < 1 << 30 &&
           b->max_context <= (int64_t)b->table_pages << c.page_shift && fits(b->sequences, b->table_stride),
       "max_context is above what table_pages hold, or 2^30");
  NEED(b->reserved == 0, "batch.reserved is not 0");
  if (addresses && b->sequences) {
    NEED(b->context && b->context % 4 == 0 && b->cu_tokens % 4 == 0, "addresses of the lengths");
    NEED(b->table_pages == 0 || (b->page_table && b->page_table % 4 == 0), "address of the page table");
  }
  if (!b->cu_tokens)
    NEED((int64_t)b->sequences * b->max_tokens == b->tokens, "without cu_tokens there are sequences * max_tokens rows");
  *out = {(const int*)(uintptr_t)b->page_table, (const int*)(uintptr_t)b->context, (const int*)(uintptr_t)b->cu_tokens,
          b->table_stride, b->sequences, b->table_pages, b->tokens, b->max_tokens, b->max_context};
  return 0;
}

// A tensor [token][head][dim] of 16-bit elements.
int check_rows(const char* what, const char* why, uint64_t at, int64_t token, int64_t head, int tokens, int heads) {
  NEED(at && at % 16 == 0 && stride_ok(token, 8) && stride_ok(head, 8) && fits(tokens, token) && fits(heads, head), why);
  return 0;
}

// Whether the elements of a tensor that a call writes are apart: each dimension, the smaller strides first, steps over all of those
// before it. Holds for every view that slicing and permuting gives, not for one that repeats rows.
bool apart(int64_t inner, std::initializer_list<std::pair<int64_t, int64_t>> sizes_and_strides) {
  std::pair<int64_t, int64_t> dims[4];  // stride, size
  int n = 0;
  for (const auto& d : sizes_and_strides)
    if (d.first > 1) dims[n++] = {d.second, d.first};
  std::sort(dims, dims + n);
  for (int i = 0; i < n; ++i) {
    if (dims[i].first < inner) return false;
    inner += (dims[i].second - 1) * dims[i].first;
  }
  return true;
}

// What a call may touch: bytes from `at` on.
struct Span {
  uint64_t at, bytes;
};
struct Spans {  // of one call, at most 14
  Span of[16];
  int count = 0;
  void add(const Span& span) {
    if (span.bytes) of[count++] = span;
  }
};

// Of a tensor of three outer dimensions, strides in bytes, with `inner` contiguous bytes; nothing if it is empty or absent.
Span span_of(const void* at, int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t inner) {
  if (!at || n0 < 1 || n1 < 1 || n2 < 1 || inner < 1) return {0, 0};
  return {(uint64_t)(uintptr_t)at, (uint64_t)((n0 - 1) * s0 + (n1 - 1) * s1 + (n2 - 1) * s2 + inner)};
}

bool tracked(const Ctx& c, const Span& span) {
  for (const auto& table : c.allocTable) {  // regions are apart, so the last one that begins before the span's end decides
    auto it = table.lower_bound(span.at + span.bytes);
    if (it != table.begin() && (--it)->first + it->second.allocSz > span.at) return true;
  }
  return false;
}

void cache_spans(const KvCache& c, const KvBatch& b, int head_dim, bool eight, Spans* out) {
  const int64_t slots = (int64_t)1 << c.page_shift, element = eight ? 1 : 2;
  for (const uint8_t* at : {c.k, c.v}) out->add(span_of(at, c.pages, c.page_stride, c.kv_heads, c.head_stride, slots, c.slot_stride, head_dim * element));
  for (const float* at : {c.k_scale, c.v_scale})
    out->add(span_of(at, c.pages, c.scale_page_stride * 4, c.kv_heads, c.scale_head_stride * 4, 1, 0, 4 * (slots >> c.block_shift)));
  out->add(span_of(b.page_table, b.sequences, b.table_stride * 4, 1, 0, 1, 0, (int64_t)b.table_pages * 4));
  out->add(span_of(b.context, 1, 0, 1, 0, 1, 0, (int64_t)b.sequences * 4));
  out->add(span_of(b.cu_tokens, 1, 0, 1, 0, 1, 0, ((int64_t)b.sequences + 1) * 4));
}

Span rows_span(const uint16_t* at, int64_t token, int64_t head, int tokens, int heads, int head_dim) {
  return span_of(at, tokens, token * 2, heads, head * 2, 1, 0, head_dim * 2);
}

// Runs `launch` with the cache's device current, unless the process is paused and some of `spans()` lies in memory that the
// engine tracks. The registry's lock is held meanwhile: a pause takes it for its whole length and waits for the device before it
// releases anything, so what gets enqueued here has run by then, and a call made during a pause finds the process paused.
template <class MakeSpans, class Launch>
int on_device(const char* what, int device, hipStream_t stream, MakeSpans spans, Launch launch) {
  if (!gpu_present()) {
    LOGGER(ERROR, "%s: no HIP device", what);
    return (int)hipErrorNoDevice;
  }
  int current = 0;
  if (hipError_t e = CHECK_HIP(hipGetDevice(&current)); e != hipSuccess) return (int)e;
  if (stream) {
    hipDevice_t of;
    if (hipError_t e = CHECK_HIP(hipStreamGetDevice(stream, &of)); e != hipSuccess) return (int)e;
    NEED((int)of == device, "the stream is another device's than the cache");
  }
  Ctx* c = globals().disabled > 0 ? nullptr : globals().ctx;
  std::unique_lock<std::mutex> lk;
  if (c) {
    lk = std::unique_lock<std::mutex>(c->structure);
    std::lock_guard<std::mutex> lf(c->fields);
    if (c->paused) {
      const Spans s = spans();
      for (int i = 0; i < s.count; ++i)
        if (tracked(*c, s.of[i])) {
          LOGGER(WARN, "%s: groupID:%d pid:%d is paused, and the tensor at %llx lies in tracked memory: refused", what, amem_groupID_value(),
                 getpid(), (unsigned long long)s.of[i].at);
          return (int)hipErrorInvalidValue;
        }
    }
  }
  if (device != current)
    if (hipError_t e = CHECK_HIP(hipSetDevice(device)); e != hipSuccess) return (int)e;
  (void)hipGetLastError();  // what an earlier call of the caller's left behind is no error of this one
  const hipError_t e = CHECK_HIP(launch());
  if (device != current) (void)CHECK_HIP(hipSetDevice(current));
  return (int)e;
}

}  // namespace
}  // namespace amem

using namespace amem;

extern "C" {

int amem_kv_append(const amem_kv_cache* cache, const amem_kv_batch* batch, const amem_kv_append_args* a, void* stream) {
  const char* what = "amem_kv_append";
  KvCache c;
  KvBatch b;
  if (int e = check_cache(what, cache, true, &c)) return e;
  if (int e = check_batch(what, batch, c, true, &b)) return e;
  NEED(a, "args is NULL");
  NEED(a->type == AMEM_KV_BF16 || a->type == AMEM_KV_F16, "type is not 16 bits");
  const bool eight = cache->type == AMEM_KV_E4M3;
  NEED(eight || cache->type == a->type, "a 16-bit cache has another type than the rows");
  NEED(apart(cache->head_dim, {{cache->pages, cache->page_stride}, {cache->kv_heads, cache->head_stride}, {cache->page_slots, cache->slot_stride}}),
       "slots of the cache overlap");
  NEED(!eight || apart(cache->page_slots / cache->block_slots, {{cache->pages, cache->scale_page_stride}, {cache->kv_heads, cache->scale_head_stride}}),
       "scales of the cache overlap");
  if (b.tokens) {
    if (int e = check_rows(what, "address or strides of k", a->k, a->k_token_stride, a->k_head_stride, b.tokens, c.kv_heads)) return e;
    if (int e = check_rows(what, "address or strides of v", a->v, a->v_token_stride, a->v_head_stride, b.tokens, c.kv_heads)) return e;
  }
  NEED(!a->q == !a->q_out, "q and q_out go together");
  if (a->q) {
    NEED(a->q_heads >= 1 && a->q_heads <= 1024, "q_heads out of range");
    if (int e = check_rows(what, "address or strides of q", a->q, a->q_token_stride, a->q_head_stride, b.tokens, a->q_heads)) return e;
    if (int e = check_rows(what, "address or strides of q_out", a->q_out, a->q_out_token_stride, a->q_out_head_stride, b.tokens, a->q_heads)) return e;
    NEED(apart(cache->head_dim, {{b.tokens, a->q_out_token_stride}, {a->q_heads, a->q_out_head_stride}}), "rows of q_out overlap");
  }
  const int pairs = a->rotary_dim / 2;
  NEED(a->rotary_dim >= 0 && a->rotary_dim <= cache->head_dim && a->rotary_dim % 16 == 0,
       "rotary_dim is not a multiple of 16 up to head_dim");
  KvAppend p = {(const uint16_t*)(uintptr_t)a->k, (const uint16_t*)(uintptr_t)a->v, (const uint16_t*)(uintptr_t)a->q,
                (uint16_t*)(uintptr_t)a->q_out, (const float*)(uintptr_t)a->cos, (const float*)(uintptr_t)a->sin,
                (const int*)(uintptr_t)a->positions, a->k_token_stride, a->k_head_stride, a->v_token_stride,
                a->v_head_stride, a->q_token_stride, a->q_head_stride, a->q_out_token_stride, a->q_out_head_stride,
                a->positions_stride, a->q ? a->q_heads : 0, a->rotary_dim, a->interleaved != 0, a->table_rows, 1,
                {pairs, pairs, pairs, pairs}};
  if (pairs) {
    NEED(a->cos && a->sin && a->cos % 16 == 0 && a->sin % 16 == 0 && a->table_rows >= 1, "the tables of the rotation");
    NEED(a->axes >= 1 && a->axes <= AMEM_KV_MAX_AXES, "axes out of range");
    NEED(a->axes == 1 || a->positions, "several axes need positions");
    NEED(!a->positions || (a->positions % 4 == 0 && (a->axes == 1 || a->positions_stride >= b.tokens)), "positions");
    if (a->axes > 1) {
      int64_t end = 0;
      for (int i = 0; i < a->axes; ++i) {
        NEED(a->sections[i] >= 0, "sections are not the pairs of the axes");
        end += a->sections[i];
        p.axis_end[i] = (int)(end < pairs ? end : pairs);
      }
      NEED(end == pairs, "sections are not the pairs of the axes");
    }
    p.axes = a->axes;
  }
  if (!b.tokens || !b.sequences) return 0;
  auto spans = [&] {
    Spans s;
    const int dim = cache->head_dim;
    cache_spans(c, b, dim, eight, &s);
    s.add(rows_span(p.k, p.k_token, p.k_head, b.tokens, c.kv_heads, dim));
    s.add(rows_span(p.v, p.v_token, p.v_head, b.tokens, c.kv_heads, dim));
    s.add(rows_span(p.q, p.q_token, p.q_head, b.tokens, p.q_heads, dim));
    s.add(rows_span(p.q_out, p.qo_token, p.qo_head, b.tokens, p.q_heads, dim));
    if (pairs) {
      for (const float* at : {p.cos, p.sin}) s.add(span_of(at, p.table_rows, pairs * 4, 1, 0, 1, 0, pairs * 4));
      s.add(span_of(p.positions, p.axes, p.positions_stride * 4, 1, 0, 1, 0, (int64_t)b.tokens * 4));
    }
    return s;
  };
  return on_device(what, cache->device, (hipStream_t)stream, spans, [&] {
    return launch_kv_append(c, b, p, cache->head_dim, a->type == AMEM_KV_F16, eight, (hipStream_t)stream);
  });
}

int amem_kv_attention_workspace(const amem_kv_cache* cache, const amem_kv_batch* batch, int q_heads, uint64_t* bytes) {
  const char* what = "amem_kv_attention_workspace";
  KvCache c;
  KvBatch b;
  if (int e = check_cache(what, cache, false, &c)) return e;
  if (int e = check_batch(what, batch, c, false, &b)) return e;
  NEED(q_heads >= 1 && q_heads <= 1024 && q_heads % c.kv_heads == 0, "q_heads is not a multiple of kv_heads");
  NEED((int64_t)b.tokens * q_heads <= 1 << 27, "tokens * q_heads is above 2^27");
  NEED(bytes, "bytes is NULL");
  *bytes = kv_attend_workspace(c, b, q_heads, batch->max_tokens, cache->head_dim);
  return 0;
}

int amem_kv_attention(const amem_kv_cache* cache, const amem_kv_batch* batch, const amem_kv_attention_args* a, void* stream) {
  const char* what = "amem_kv_attention";
  KvCache c;
  KvBatch b;
  if (int e = check_cache(what, cache, true, &c)) return e;
  if (int e = check_batch(what, batch, c, true, &b)) return e;
  NEED(a, "args is NULL");
  NEED(a->type == AMEM_KV_BF16 || a->type == AMEM_KV_F16, "type is not 16 bits");
  const bool eight = cache->type == AMEM_KV_E4M3;
  NEED(eight || cache->type == a->type, "a 16-bit cache has another type than the rows");
  NEED(a->q_heads >= 1 && a->q_heads <= 1024 && a->q_heads % c.kv_heads == 0, "q_heads is not a multiple of kv_heads");
  if (b.tokens) {
    if (int e = check_rows(what, "address or strides of q", a->q, a->q_token_stride, a->q_head_stride, b.tokens, a->q_heads)) return e;
    if (int e = check_rows(what, "address or strides of out", a->out, a->out_token_stride, a->out_head_stride, b.tokens, a->q_heads)) return e;
    NEED(apart(cache->head_dim, {{b.tokens, a->out_token_stride}, {a->q_heads, a->out_head_stride}}), "rows of out overlap");
  }
  NEED((int64_t)b.tokens * a->q_heads <= 1 << 27, "tokens * q_heads is above 2^27");
  NEED(a->lse % 4 == 0, "address of lse");
  NEED(a->window >= 0, "window is negative");
  NEED(a->scale - a->scale == 0, "scale is not finite");
  NEED(a->reserved == 0, "args.reserved is not 0");
  const uint64_t need = kv_attend_workspace(c, b, a->q_heads, batch->max_tokens, cache->head_dim);
  NEED(!need || (a->workspace && a->workspace % 16 == 0 && a->workspace_bytes >= need), "workspace is too small or not aligned to 16 bytes");
  if (!b.tokens || !b.sequences) return 0;
  const KvAttend p = {(const uint16_t*)(uintptr_t)a->q, (uint16_t*)(uintptr_t)a->out, (float*)(uintptr_t)a->lse,
                      (uint8_t*)(uintptr_t)a->workspace, a->q_token_stride, a->q_head_stride, a->out_token_stride,
                      a->out_head_stride, a->scale, a->q_heads, a->causal != 0, a->window, batch->max_tokens};
  auto spans = [&] {
    Spans s;
    const int dim = cache->head_dim;
    cache_spans(c, b, dim, eight, &s);
    s.add(rows_span(p.q, p.q_token, p.q_head, b.tokens, p.q_heads, dim));
    s.add(rows_span(p.out, p.out_token, p.out_head, b.tokens, p.q_heads, dim));
    s.add(span_of(p.lse, 1, 0, 1, 0, 1, 0, (int64_t)b.tokens * p.q_heads * 4));
    if (need) s.add(span_of(p.workspace, 1, 0, 1, 0, 1, 0, (int64_t)need));
    return s;
  };
  return on_device(what, cache->device, (hipStream_t)stream, spans, [&] {
    return launch_kv_attend(c, b, p, cache->head_dim, a->type == AMEM_KV_F16, eight, (hipStream_t)stream);
  });
}

}  // extern "C"
