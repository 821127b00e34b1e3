// Attention over a paged cache of E4M3 keys and values with a scale for every page and head.
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale * q . k_j - m),   m the running maximum
//
// One warp per query row and head; a lane has D / 32 elements of q, of the sum and of every cached row.
#include <string>

#include "common.cuh"
#include "paged.h"

using namespace gw;

namespace {

__device__ uint32_t g_attention_error;       // first report since it was last taken

struct Attention {
  gw_kv_cache cache;
  gw_sequences batch;
  const bf16* query;
  bf16* output;
  uint64_t query_stride, output_stride;
  uint32_t heads, group, window;
  float scale;
};

template <int V>          // head width 128 * V / 4
__global__ void __launch_bounds__(128) paged_attention_kernel(Attention a) {
  constexpr int E = V;
  griddep_enter();
  const uint32_t lane = threadIdx.x % 32, width = 32 * E;
  const uint32_t task = blockIdx.x * 4 + threadIdx.x / 32, row = task / a.heads, head = task % a.heads, kv = head / a.group;
  if (row >= a.batch.rows) return;
  uint32_t low = 0, high = a.batch.sequences;
  while (low + 1 < high) {
    const uint32_t middle = (low + high) / 2;
    if (a.batch.row_offsets[middle] <= int(row)) low = middle; else high = middle;
  }
  const SequenceRows s = sequence_rows(a.batch, low);
  if (s.bad && lane == 0) atomicCAS(&g_attention_error, 0u, 0xa2000000u | (low & 0xffffffu));
  if (int(row) < s.first || int(row) >= s.first + s.count) return;
  const int position = s.context - s.count + int(row) - s.first;
  const int begin = a.window ? max(int64_t(0), int64_t(position) - a.window + 1) : 0;
  float q[E], sum[E], total = 0.F, most = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = __bfloat162float(a.query[size_t(row) * a.query_stride + head * width + lane * E + e]) * a.scale;
    sum[e] = 0.F;
  }
  for (int token = begin; token <= position; ++token) {
    const uint32_t ordinal = token / a.cache.page_tokens, slot = token % a.cache.page_tokens;
    int page = -1;
    if (ordinal < a.batch.page_table_stride) page = a.batch.page_table[size_t(low) * a.batch.page_table_stride + ordinal];
    if (page < 0 || uint32_t(page) >= a.cache.pages) {
      if (lane == 0) atomicCAS(&g_attention_error, 0u, 0xa1000000u | (low & 0xffffffu));
      continue;
    }
    const size_t at = size_t(page) * a.cache.kv_heads + kv;
    const size_t place = (at * a.cache.page_tokens + slot) * width + lane * E;
    float dot = 0.F;
#pragma unroll
    for (int e = 0; e < E; ++e) dot = fmaf(q[e], e4m3_to_float(static_cast<const uint8_t*>(a.cache.k_data)[place + e]), dot);
#pragma unroll
    for (int m = 16; m; m /= 2) dot += __shfl_xor_sync(0xffffffffu, dot, m);
    dot *= a.cache.k_scales[at];
    const float higher = fmaxf(most, dot), before = most == -INFINITY ? 0.F : expf(most - higher), p = expf(dot - higher);
    total = total * before + p;
#pragma unroll
    for (int e = 0; e < E; ++e)
      sum[e] = sum[e] * before + p * a.cache.v_scales[at] * e4m3_to_float(static_cast<const uint8_t*>(a.cache.v_data)[place + e]);
    most = higher;
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    a.output[size_t(row) * a.output_stride + head * width + lane * E + e] = __float2bfloat16_rn(total > 0.F ? sum[e] / total : 0.F);
}

}  // namespace

uint32_t gw::take_paged_attention_error() {
  uint32_t value = 0;
  if (cudaMemcpyFromSymbol(&value, g_attention_error, sizeof(value)) != cudaSuccess) return 0xFFFFFFFDu;
  const uint32_t none = 0;
  if (value != 0 && cudaMemcpyToSymbol(g_attention_error, &none, sizeof(none)) != cudaSuccess) return 0xFFFFFFFDu;
  return value;
}

extern "C" {

size_t gw_paged_attention_scratch_bytes(const gw_kv_cache*, const gw_sequences*, uint32_t) { return 256; }

gw_status gw_paged_attention_bf16(const gw_kv_cache* cache, const gw_sequences* batch, const void* query_bf16,
                                  uint64_t query_stride, uint32_t heads, float scale, uint32_t window, void* output_bf16,
                                  uint64_t output_stride, void* scratch, size_t scratch_capacity, void* stream) {
  clear_error();
  if (gw_status s = check_cache(cache, "paged attention"); s != GW_OK) return s;
  if (gw_status s = check_batch(batch, "paged attention"); s != GW_OK) return s;
  if (batch->rows == 0 || batch->sequences == 0) return GW_OK;
  const uint64_t width = uint64_t(heads) * cache->head_dim;
  if (heads == 0 || heads % cache->kv_heads != 0 || heads / cache->kv_heads > 64)
    return fail(GW_INVALID_ARGUMENT, "paged attention requires query heads that are 1 to 64 times the cache's");
  if (!query_bf16 || !output_bf16 || !is_aligned16(query_bf16) || !is_aligned16(output_bf16) || query_stride % 8 != 0 ||
      output_stride % 8 != 0 || query_stride < width || output_stride < width)
    return fail(GW_INVALID_ARGUMENT, "paged attention requires 16-byte aligned queries and outputs with row strides divisible by 8 that hold all heads");
  if (!(scale > -3.4e38F && scale < 3.4e38F)) return fail(GW_INVALID_ARGUMENT, "paged attention requires a finite scale");
  const size_t needed = gw_paged_attention_scratch_bytes(cache, batch, heads);
  if (!scratch || reinterpret_cast<uintptr_t>(scratch) % 256 != 0 || scratch_capacity < needed)
    return fail(GW_INVALID_ARGUMENT, "paged attention requires " + std::to_string(needed) + " bytes of 256-byte aligned scratch");
  const Attention a{*cache, *batch, static_cast<const bf16*>(query_bf16), static_cast<bf16*>(output_bf16), query_stride, output_stride,
                    heads, heads / cache->kv_heads, window, scale};
  const uint64_t tasks = uint64_t(batch->rows) * heads;
  GW_CUDA_CHECK(launch_pdl(cache->head_dim == 128   ? paged_attention_kernel<4>
                           : cache->head_dim == 256 ? paged_attention_kernel<8>
                                                    : paged_attention_kernel<16>,
                           uint32_t((tasks + 3) / 4), 128, as_stream(stream), a),
                "paged attention");
  return GW_OK;
}

}  // extern "C"
