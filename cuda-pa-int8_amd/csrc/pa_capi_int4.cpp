// extern "C" entry points of the 4-bit paged cache and of the block tables (declared in
// include/pa_mi355x.h).  Host side only: argument validation and dispatch.
#include "pa_mi355x.h"

#include <cstdint>

#include "pa_internal.hpp"

namespace {

constexpr float kLog2e = 1.4426950408889634f;

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

pa_status_t check_cache(int32_t head_dim, int32_t num_kv_heads, int32_t num_blocks,
                        int32_t block_size) {
  if (block_size <= 0 || block_size % 16 != 0 || 128 % block_size != 0)
    return PA_ERR_BAD_BLOCK_SIZE;
  if (head_dim < 8 || head_dim > 256 || head_dim % 8 != 0) return PA_ERR_UNSUPPORTED;
  if (num_kv_heads < 1 || num_blocks < 1 || (int64_t)num_blocks * num_kv_heads > UINT32_MAX)
    return PA_ERR_BAD_SHAPE;
  return PA_OK;
}

pa_status_t rows_int4(bool write, void* key, void* value, int64_t kts, int64_t khs, int64_t vts,
                      int64_t vhs, const int64_t* slot_mapping, int32_t num_tokens,
                      int32_t num_kv_heads, int32_t head_dim, void* k_cache, void* v_cache,
                      void* k_scales, void* v_scales, int32_t num_blocks, int32_t block_size,
                      int32_t bf16, pa_stream_t stream) {
  const pa_status_t st = check_cache(head_dim, num_kv_heads, num_blocks, block_size);
  if (st != PA_OK) return st;
  if (num_tokens < 0) return PA_ERR_BAD_SHAPE;
  if (num_tokens == 0) return PA_OK;
  if (!key || !value || !slot_mapping || !k_cache || !v_cache || !k_scales || !v_scales)
    return PA_ERR_NULL_POINTER;
  for (int64_t s : {kts, khs, vts, vhs})      // (16-byte row loads and stores)
    if (s < 0 || s % 8 != 0) return PA_ERR_BAD_SHAPE;
  for (const void* p : {static_cast<const void*>(key), static_cast<const void*>(value),
                        static_cast<const void*>(k_cache), static_cast<const void*>(v_cache),
                        static_cast<const void*>(k_scales), static_cast<const void*>(v_scales)})
    if (!aligned(p, 16)) return PA_ERR_BAD_SHAPE;
  if (!aligned(slot_mapping, 8)) return PA_ERR_BAD_SHAPE;
  pa::Int4Rows l{key, value, kts, khs, vts, vhs, slot_mapping, num_tokens, num_kv_heads, head_dim,
                 k_cache, v_cache, k_scales, v_scales, num_blocks, block_size, bf16 != 0,
                 reinterpret_cast<hipStream_t>(stream)};
  const hipError_t e = write ? pa::launch_int4_write(l) : pa::launch_int4_gather(l);
  return e == hipSuccess ? PA_OK : PA_ERR_LAUNCH;
}

// Validates the shape of a decode call and fills the kernels' description of it.
pa_status_t decode_shape(int32_t num_seqs, int32_t num_heads, int32_t head_dim,
                         int32_t num_kv_heads, int32_t num_blocks, int32_t block_size,
                         int32_t max_blocks, float scale, pa::Int4DecodeShape* s) {
  const pa_status_t st = check_cache(head_dim, num_kv_heads, num_blocks, block_size);
  if (st != PA_OK) return st;
  if (num_seqs < 0 || num_heads < 1 || num_heads % num_kv_heads != 0 || max_blocks < 0 ||
      (int64_t)max_blocks * block_size > INT32_MAX - 128)
    return PA_ERR_BAD_SHAPE;
  // The kernel counts the 64-token tiles of every (sequence, kv head, chunk of query heads) in 31
  // bits.
  const int64_t tiles = (int64_t)max_blocks * block_size / 64 + 1;
  if (num_seqs > INT32_MAX / num_heads || (int64_t)num_seqs * num_heads > INT32_MAX / tiles)
    return PA_ERR_BAD_SHAPE;
  *s = pa::Int4DecodeShape{num_seqs, num_heads, num_kv_heads, num_heads / num_kv_heads, head_dim,
                           num_blocks, max_blocks, __builtin_ctz((unsigned)block_size),
                           scale * kLog2e};
  return PA_OK;
}

hipError_t launch_decode(const pa::Int4Decode& l) {
  switch ((l.shape.head_dim + 31) / 32) {
#define PA_CASE(N) \
  case N: return pa::launch_int4_decode_steps<N>(l);
    PA_FOR_EACH_INT4_STEPS(PA_CASE)
#undef PA_CASE
    default: return hipErrorInvalidValue;
  }
}

size_t workspace_bytes_of(const pa::Int4DecodeShape& s) {
  switch ((s.head_dim + 31) / 32) {
#define PA_CASE(N) \
  case N: return 2 * pa::kInt4Groups * pa::int4_decode_slot_bytes<N>(s.group);
    PA_FOR_EACH_INT4_STEPS(PA_CASE)
#undef PA_CASE
    default: return 0;
  }
}

pa_status_t decode_int4(
    void* out, const void* q, const void* k_cache, const void* v_cache, const void* k_scales,
    const void* v_scales, const int32_t* block_table, const int32_t* context_lens, float scale,
    int32_t block_size, int32_t num_seqs, int32_t num_heads, int32_t head_dim,
    int32_t num_kv_heads, int32_t num_blocks, int32_t max_blocks_per_seq, int32_t bf16,
    void* counters, size_t counter_bytes, void* workspace, size_t workspace_bytes,
    uint64_t* report, uint32_t tag, pa_stream_t stream) {
  pa::Int4DecodeShape s;
  const pa_status_t st = decode_shape(num_seqs, num_heads, head_dim, num_kv_heads, num_blocks,
                                      block_size, max_blocks_per_seq, scale, &s);
  if (st != PA_OK || num_seqs == 0) return st;
  if (!out || !q || !k_cache || !v_cache || !k_scales || !v_scales || !context_lens ||
      (!block_table && max_blocks_per_seq > 0))
    return PA_ERR_NULL_POINTER;
  for (const void* p : {static_cast<const void*>(out), q, k_cache, v_cache, k_scales, v_scales})
    if (!aligned(p, 16)) return PA_ERR_BAD_SHAPE;
  if (!counters || counter_bytes < pa_decode_int4_counter_bytes() || !aligned(counters, 256) ||
      !workspace || workspace_bytes < workspace_bytes_of(s) || !aligned(workspace, 256))
    return PA_ERR_WORKSPACE;
  pa::Int4Decode l{out, q, k_cache, v_cache, k_scales, v_scales, block_table, context_lens,
                   bf16 != 0, static_cast<uint32_t*>(counters), static_cast<float*>(workspace), report, tag, s,
                   reinterpret_cast<hipStream_t>(stream)};
  return launch_decode(l) == hipSuccess ? PA_OK : PA_ERR_LAUNCH;
}

// Whether any of the first `outs` ranges meets another range.
struct Range {
  const void* p;
  size_t bytes;
};
template <int N>
bool outputs_overlap(const Range (&r)[N], int outs) {
  for (int i = 0; i < outs; ++i)
    for (int j = i + 1; j < N; ++j) {
      const auto a = reinterpret_cast<uintptr_t>(r[i].p), b = reinterpret_cast<uintptr_t>(r[j].p);
      if (r[i].bytes && r[j].bytes && a < b + r[j].bytes && b < a + r[i].bytes) return true;
    }
  return false;
}

}  // namespace

extern "C" {

pa_status_t pa_reshape_and_cache_int4(const void* key, const void* value,
                                      int64_t key_token_stride, int64_t key_head_stride,
                                      int64_t value_token_stride, int64_t value_head_stride,
                                      const int64_t* slot_mapping, int32_t num_tokens,
                                      int32_t num_kv_heads, int32_t head_dim, void* k_cache,
                                      void* v_cache, void* k_scales, void* v_scales,
                                      int32_t num_blocks, int32_t block_size, int32_t bf16_input,
                                      pa_stream_t stream) {
  return rows_int4(true, const_cast<void*>(key), const_cast<void*>(value), key_token_stride,
                   key_head_stride, value_token_stride, value_head_stride, slot_mapping,
                   num_tokens, num_kv_heads, head_dim, k_cache, v_cache, k_scales, v_scales,
                   num_blocks, block_size, bf16_input, stream);
}

pa_status_t pa_gather_cache_int4(void* key, void* value, int64_t key_token_stride,
                                 int64_t key_head_stride, int64_t value_token_stride,
                                 int64_t value_head_stride, const int64_t* slot_mapping,
                                 int32_t num_tokens, int32_t num_kv_heads, int32_t head_dim,
                                 const void* k_cache, const void* v_cache, const void* k_scales,
                                 const void* v_scales, int32_t num_blocks, int32_t block_size,
                                 int32_t bf16_output, pa_stream_t stream) {
  return rows_int4(false, key, value, key_token_stride, key_head_stride, value_token_stride,
                   value_head_stride, slot_mapping, num_tokens, num_kv_heads, head_dim,
                   const_cast<void*>(k_cache), const_cast<void*>(v_cache),
                   const_cast<void*>(k_scales), const_cast<void*>(v_scales), num_blocks,
                   block_size, bf16_output, stream);
}

size_t pa_decode_int4_counter_bytes(void) { return 3 * pa::kInt4Groups * sizeof(uint32_t); }

size_t pa_decode_int4_workspace_bytes(int32_t num_seqs, int32_t num_heads, int32_t head_dim,
                                      int32_t num_kv_heads, int32_t block_size,
                                      int32_t max_blocks_per_seq) {
  pa::Int4DecodeShape s;
  if (decode_shape(num_seqs, num_heads, head_dim, num_kv_heads, 1, block_size, max_blocks_per_seq,
                   1.f, &s) != PA_OK)
    return 0;
  return workspace_bytes_of(s);
}

pa_status_t pa_paged_decode_attn_int4(
    void* out, const void* q, const void* k_cache, const void* v_cache, const void* k_scales,
    const void* v_scales, const int32_t* block_table, const int32_t* context_lens, float scale,
    int32_t block_size, int32_t num_seqs, int32_t num_heads, int32_t head_dim,
    int32_t num_kv_heads, int32_t num_blocks, int32_t max_blocks_per_seq, int32_t bf16,
    void* counters, size_t counter_bytes, void* workspace, size_t workspace_bytes,
    pa_stream_t stream) {
  return decode_int4(out, q, k_cache, v_cache, k_scales, v_scales, block_table, context_lens, scale,
                     block_size, num_seqs, num_heads, head_dim, num_kv_heads, num_blocks,
                     max_blocks_per_seq, bf16, counters, counter_bytes, workspace,
                     workspace_bytes, nullptr, 0, stream);
}

pa_status_t pa_paged_decode_attn_int4_checked(
    void* out, const void* q, const void* k_cache, const void* v_cache, const void* k_scales,
    const void* v_scales, const int32_t* block_table, const int32_t* context_lens, float scale,
    int32_t block_size, int32_t num_seqs, int32_t num_heads, int32_t head_dim,
    int32_t num_kv_heads, int32_t num_blocks, int32_t max_blocks_per_seq, int32_t bf16,
    void* counters, size_t counter_bytes, void* workspace, size_t workspace_bytes,
    uint64_t* report, uint32_t tag, pa_stream_t stream) {
  if (!report) return PA_ERR_NULL_POINTER;
  if (!aligned(report, 8)) return PA_ERR_BAD_SHAPE;
  return decode_int4(out, q, k_cache, v_cache, k_scales, v_scales, block_table, context_lens, scale,
                     block_size, num_seqs, num_heads, head_dim, num_kv_heads, num_blocks,
                     max_blocks_per_seq, bf16, counters, counter_bytes, workspace,
                     workspace_bytes, report, tag, stream);
}

pa_status_t pa_extend_block_tables(int32_t* block_table, const int32_t* context_lens,
                                   const int32_t* new_lens, const int32_t* free_blocks,
                                   const int32_t* num_free, int32_t* context_lens_out,
                                   int32_t* num_free_out, int64_t* slot_mapping,
                                   int64_t* positions, int32_t* cu_seqlens, int32_t* status,
                                   int32_t num_seqs, int32_t max_blocks_per_seq,
                                   int32_t block_size, int32_t num_rows, int32_t free_capacity,
                                   void* counters, size_t counter_bytes, pa_stream_t stream) {
  if (block_size <= 0 || (block_size & (block_size - 1)) != 0 || block_size > 128)
    return PA_ERR_BAD_BLOCK_SIZE;
  if (num_seqs < 1 || num_seqs > PA_EXTEND_MAX_SEQS || max_blocks_per_seq < 0 || num_rows < 0 ||
      free_capacity < 0 || (int64_t)max_blocks_per_seq * block_size > INT32_MAX)
    return PA_ERR_BAD_SHAPE;
  if (!context_lens || !new_lens || !num_free || !context_lens_out || !num_free_out || !status ||
      (!block_table && max_blocks_per_seq > 0) || (!free_blocks && free_capacity > 0) ||
      (!slot_mapping && num_rows > 0))
    return PA_ERR_NULL_POINTER;
  if (!counters || counter_bytes < sizeof(uint32_t) || !aligned(counters, 4))
    return PA_ERR_WORKSPACE;
  // Work-groups read the inputs while others write the outputs: only the lengths and the free
  // count may be updated in place.
  const size_t lens = 4 * (size_t)num_seqs, rows = 8 * (size_t)num_rows;
  const Range ranges[] = {
      {block_table, lens * (size_t)max_blocks_per_seq}, {slot_mapping, rows},
      {positions, positions ? rows : 0}, {cu_seqlens, cu_seqlens ? lens + 4 : 0}, {status, 4},
      {context_lens_out, lens}, {num_free_out, 4},
      {context_lens, context_lens == context_lens_out ? 0 : lens},
      {num_free, num_free == num_free_out ? 0 : (size_t)4}, {new_lens, lens},
      {free_blocks, 4 * (size_t)free_capacity}};
  if (outputs_overlap(ranges, 7)) return PA_ERR_BAD_SHAPE;
  pa::ExtendLaunch l{block_table, context_lens, new_lens, free_blocks, num_free, context_lens_out,
                     num_free_out, slot_mapping, positions, cu_seqlens, status,
                     static_cast<uint32_t*>(counters), num_seqs, max_blocks_per_seq, block_size,
                     num_rows, free_capacity, reinterpret_cast<hipStream_t>(stream)};
  return pa::launch_extend(l) == hipSuccess ? PA_OK : PA_ERR_LAUNCH;
}

}  // extern "C"

static_assert(PA_EXTEND_MAX_SEQS == pa::kExtendMaxSeqs && PA_EXTEND_NO_BLOCKS == pa::kExtendNoBlocks &&
                  PA_EXTEND_ROW_FULL == pa::kExtendRowFull && PA_EXTEND_NO_ROWS == pa::kExtendNoRows &&
                  PA_EXTEND_BAD_LENGTH == pa::kExtendBadLength,
              "the header's numbers are the kernel's");
