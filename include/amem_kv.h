/*
 * amem_kv.h — operators on a paged key/value cache, exported by libamem_nccl.so.1 beside the
 * pause/resume surface of amem.h. They stand next to its gather/scatter kernels: rows of new keys
 * and values go to scattered pages of device memory, and attention reads them from there. None of
 * them has a counterpart in the reference. Plain C like amem.h.
 *
 * The cache may lie in any device memory. In memory that the engine tracks (amem_vmm_alloc +
 * amem_add_alloc_info) a pause releases it and a resume brings back the same bytes at the same
 * addresses; with 8 bits there is half as much to park. While the process is paused, calls that name
 * an address in tracked memory are refused, since there may be no memory behind it; a pause waits for those
 * already enqueued. A captured graph is the caller's: one that uses tracked memory must not be replayed while paused.
 *
 * Conventions. Device addresses are uint64_t. Every call only enqueues work on `stream` (a
 * hipStream_t of the cache's device, NULL for its default stream) and may be captured; nothing is
 * allocated, copied to the host or kept, so that tensors have to live until the stream is done with them. Everything that addresses name has to lie on the cache's
 * device, which need not be the current one. Results are the same, bit for bit, from call to call. Returns
 * 0, hipErrorInvalidValue (1) for arguments that are refused (one ERROR line says which) and for tracked
 * memory while paused, or another HIP error. Two calls that may run at the same time need different workspaces,
 * and must not write the same pages or read pages that the other writes.
 *
 * What a call writes (q_out, out, the cache and its scales in append) must not overlap itself; strides that do are refused. What it only reads may.
 *
 * Lengths, positions, page numbers and rows live in device memory and cannot be refused on the host. Where they
 * are out of range nothing outside the tensors is touched: see the notes below.
 */
#ifndef AMEM_KV_H_
#define AMEM_KV_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif
#pragma GCC visibility push(default)

enum amem_kv_type { AMEM_KV_BF16 = 0, AMEM_KV_F16 = 1, AMEM_KV_E4M3 = 2 };

#define AMEM_KV_MAX_AXES 4

/* Keys and values: element [page][head][slot][dim], dims contiguous, the other strides as given (in
 * elements, multiples of 16 bytes; the same for both; the slots of a page less than 2^31 bytes apart). 8 bits: values are code * scale, codes e4m3
 * (largest 448, no infinities), one float32 scale, a power of two from 2^-64 to 2^119, for each
 * [page][head][block of `block_slots` slots], blocks contiguous. */
typedef struct amem_kv_cache {
  uint64_t k, v;                 /* 16-byte aligned */
  uint64_t k_scale, v_scale;     /* 8 bits only, else 0 */
  int64_t page_stride, head_stride, slot_stride;
  int64_t scale_page_stride, scale_head_stride; /* in floats */
  int32_t type;                  /* amem_kv_type */
  int32_t device;
  int32_t pages, kv_heads;
  int32_t page_slots;            /* a power of two, 1 to 1024 */
  int32_t block_slots;           /* 8 bits: a power of two, 16 to 128, at most page_slots; else 0 */
  int32_t head_dim;              /* 64, 128 or 256 */
  int32_t reserved;              /* 0 */
} amem_kv_cache;

/* Sequences of a call, at most 2^20 and 2^22 tokens; tokens * q_heads is at most 2^27, and
 * (tokens / 16 + 2 * sequences) * kv_heads 2^22. Sequence s has rows [cu_tokens[s], cu_tokens[s+1]) of the token tensors (its
 * new tokens, possibly none) and context[s] tokens in the cache, those included: its row j is at
 * position context[s] - n + j, in slot position % page_slots of page page_table[s][position / page_slots].
 * Rows behind the last sequence's are left alone. A sequence whose context is negative, above
 * `max_context` or above table_pages * page_slots is out of range, and so is a page number outside
 * [0, pages) that a position needs: append writes nothing there, attention gives NaN in the
 * rows that would see it. New tokens at negative positions (a context shorter than them) are not
 * appended; as queries they see what the masks leave them, which is nothing where causal. */
typedef struct amem_kv_batch {
  uint64_t page_table;           /* int32 [sequences][table_stride] */
  uint64_t context;              /* int32 [sequences] */
  uint64_t cu_tokens;            /* int32 [sequences + 1], ascending from 0; 0: every sequence has max_tokens rows */
  int64_t table_stride;
  int32_t sequences, table_pages;
  int32_t tokens;                /* rows of the token tensors */
  int32_t max_tokens;            /* most new tokens of one sequence; a guide where cu_tokens is given */
  int32_t max_context;           /* no context[s] is above it; work is dealt out by it, so that a limit far above costs few sequences time */
  int32_t reserved;              /* 0 */
} amem_kv_batch;

/* Append: the rows k and v ([token][head][dim]) go into the cache at their positions, keys rotated on
 * the way, and q, where given, is rotated into q_out (which may be q itself). Rows stay in 16 bits (`type`);
 * a 16-bit cache has the same type.
 *
 * Rotation turns the first `rotary_dim` dims (a multiple of 16, 0: none) in pairs, (i, i + rotary_dim/2)
 * or, interleaved, (2i, 2i + 1): (a, b) -> (a c - b s, b c + a s), with c and s from row t of the
 * float32 tables [table_rows][rotary_dim/2]. t is the row's position in the cache, or, with
 * `positions` (int32 [axes][positions_stride]), positions[a][row] where a is the axis that pair i
 * belongs to: the first sections[0] pairs have axis 0, and so on. A t outside the table gives NaN.
 * Products and sums have 32 bits, and one rounding follows.
 *
 * 8 bits. For the block's new tokens of this call need = the smallest 2^e, -64 <= e <= 119, with
 * |x| <= 448 * 2^e for their finite values x. A block whose first slot is among them starts anew, with scale = need;
 * otherwise scale = max(its scale, need), and where that grew its earlier codes become code * old / scale,
 * rounded. New codes are x / scale, rounded to nearest, ties to even, from the rotated key without a
 * rounding in between; what is not finite is stored as NaN. Slots behind the new tokens keep their
 * bytes. A block belongs to one sequence of a call: two that write the same page race. */
typedef struct amem_kv_append_args {
  uint64_t k, v;                 /* 16-byte aligned, strides multiples of 8 elements, dims contiguous */
  uint64_t q, q_out;             /* or 0, both */
  uint64_t cos, sin;             /* 16-byte aligned; 0 without rotation */
  uint64_t positions;            /* or 0: the cache positions */
  int64_t k_token_stride, k_head_stride, v_token_stride, v_head_stride;
  int64_t q_token_stride, q_head_stride, q_out_token_stride, q_out_head_stride;
  int64_t positions_stride;
  int32_t type;                  /* AMEM_KV_BF16 or AMEM_KV_F16: of k, v, q */
  int32_t q_heads;
  int32_t rotary_dim, interleaved;
  int32_t table_rows, axes;      /* axes: 1 to AMEM_KV_MAX_AXES */
  int32_t sections[AMEM_KV_MAX_AXES]; /* sum rotary_dim/2; read where axes > 1 */
} amem_kv_append_args;
int amem_kv_append(const amem_kv_cache* cache, const amem_kv_batch* batch, const amem_kv_append_args* args, void* stream);

/* Attention: out[row][head] = sum over the visible positions p of w_p v_p, w = softmax(scale q.k_p), with the cache's
 * key/value head head / (q_heads / kv_heads). Row at position i of a sequence with context L sees p < L, p <= i
 * if causal, and p > i - window if window > 0. lse, where given, is the natural logarithm of the sum of
 * exp(scale q.k_p). A row that sees nothing, or nothing but scores of -infinity, gives zeros and lse
 * -infinity. What is hidden from a row does not reach it, infinities and NaN included. Weights are rounded to 16 bits
 * (bf16 where the cache is bf16, else fp16) before they meet the values; sums have 32. 8 bits: where the scales of the values
 * lie further apart than 2^4 from the first ones, the products of weights and scales are rounded in place of the weights, so that only
 * products far below a row's largest lose bits. Weights below 2^-126 of the largest count as zero, which asks for scales within 2^100 of each other.
 * Sums of bf16 values stay finite while 2^7 * context * |v| does. `out` may be q itself.
 * The queries' rows have to be in the cache already: append first, then attend, on one stream. */
typedef struct amem_kv_attention_args {
  uint64_t q, out;               /* [token][head][dim], like k in append */
  uint64_t lse;                  /* float32 [token][q_heads], or 0 */
  uint64_t workspace, workspace_bytes; /* 16-byte aligned; at least amem_kv_attention_workspace() */
  int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;
  float scale;
  int32_t type;                  /* of q and out; a 16-bit cache has the same */
  int32_t q_heads;               /* a multiple of kv_heads */
  int32_t causal;
  int32_t window;                /* 0: none */
  int32_t reserved;              /* 0 */
} amem_kv_attention_args;
int amem_kv_attention(const amem_kv_cache* cache, const amem_kv_batch* batch, const amem_kv_attention_args* args, void* stream);

/* Bytes of workspace that amem_kv_attention needs for these sizes and any mask, 0 if none (no address is read, only
 * whether cu_tokens is 0). What it holds between calls does not matter. Returns 0, or hipErrorInvalidValue. */
int amem_kv_attention_workspace(const amem_kv_cache* cache, const amem_kv_batch* batch, int q_heads, uint64_t* bytes);

#pragma GCC visibility pop
#ifdef __cplusplus
} /* extern "C" */
#endif
#endif /* AMEM_KV_H_ */
