// Host checks and device helpers that the cache append and the attention over the cache share.
#pragma once

#include <cstdint>
#include <string>

#include "common.cuh"

namespace gw {

inline bool is_aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

inline gw_status check_cache(const gw_kv_cache* c, const char* what) {
  if (!c || !c->k_data || !c->v_data || !c->k_scales || !c->v_scales || !is_aligned16(c->k_data) || !is_aligned16(c->v_data))
    return fail(GW_INVALID_ARGUMENT, std::string(what) + " requires a cache with 16-byte aligned codes and scales");
  if (c->page_tokens != 16 && c->page_tokens != 32 && c->page_tokens != 64 && c->page_tokens != 128)
    return fail(GW_INVALID_ARGUMENT, std::string(what) + " requires pages of 16, 32, 64 or 128 tokens");
  if (c->head_dim != 128 && c->head_dim != 256 && c->head_dim != 512)
    return fail(GW_INVALID_ARGUMENT, std::string(what) + " requires a cache with a head width of 128, 256 or 512");
  if (c->pages == 0 || c->kv_heads == 0 || uint64_t(c->pages) * c->kv_heads * c->page_tokens >= (1ull << 31) || c->kv_heads > 1024)
    return fail(GW_INVALID_ARGUMENT, std::string(what) + " requires pages, at most 1024 KV heads and fewer than 2^31 slots over all heads");
  return GW_OK;
}

// Entries of a sequence's row of the page table.
inline uint32_t page_entries(const gw_sequences& b) { return b.page_table_entries != 0 ? b.page_table_entries : b.page_table_stride; }

inline gw_status check_batch(const gw_sequences* b, const char* what) {
  if (!b) return fail(GW_INVALID_ARGUMENT, std::string(what) + " requires a batch");
  if (b->rows == 0 || b->sequences == 0) return GW_OK;
  if (!b->row_offsets || !b->context_lengths || !b->page_table || b->page_table_stride == 0)
    return fail(GW_INVALID_ARGUMENT, std::string(what) + " requires row offsets, context lengths and a page table");
  if (b->page_table_entries > b->page_table_stride)
    return fail(GW_INVALID_ARGUMENT, std::string(what) + " requires page table entries within a row's stride");
  if (b->max_rows == 0 || b->max_rows > b->rows || b->rows > (1u << 24) || b->sequences > (1u << 20) || b->page_table_stride > (1u << 24))
    return fail(GW_INVALID_ARGUMENT, std::string(what) + " requires max_rows of 1 to rows, at most 2^24 rows, 2^20 sequences and 2^24 page table entries");
  return GW_OK;
}

constexpr int kMostTokens = 1 << 30;      // of a sequence

#ifdef __CUDACC__
// What a sequence brings to a step; count 0 where its offsets cannot be followed.
struct SequenceRows {
  int first, count, context;      // row i is the token at context - count + i (below 0: none)
  bool bad;
};
__device__ __forceinline__ SequenceRows sequence_rows(const gw_sequences& b, uint32_t s) {
  const int low = b.row_offsets[s], high = b.row_offsets[s + 1], context = b.context_lengths[s];
  const bool good = low >= 0 && high >= low && uint32_t(high) <= b.rows && uint32_t(high - low) <= b.max_rows && context <= kMostTokens;
  return {low, good ? high - low : 0, good && context > 0 ? context : 0, !good};
}
#endif

}  // namespace gw
