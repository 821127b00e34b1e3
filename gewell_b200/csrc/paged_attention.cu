// Attention over a paged cache of E4M3 keys and values with a scale for every page and head.
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp2(c_j k_j . q - m),   c_j = scale * log2(e) * kscale_j
//
// One block takes tiles of kTokens cached tokens, N query columns (query rows times the query heads of one KV head) at a time,
// with both products on the tensor cores and the cached codes as they are: nothing of the cache is converted or transposed.
//   S^T [tokens, N]  = K [tokens, D] Q^T          A = K as it lies in its pages (a row of D codes), B = Q
//   O^T [D, N]      += V^T [D, tokens] P^T        A = V as it lies in its pages, read along the tokens, B = P^T
// Tokens lie on the tensor memory's lanes, so a lane needs one key scale and one value scale for all its columns, and
// few query rows cost few columns: the same kernel serves single tokens and prompts.
//
// E4M3 holds four significant bits.  Queries and probabilities therefore enter as two parts, x = hi + lo with hi the nearest
// code of x and lo that of the rest (eight bits, as BF16), two products over the same codes.  Block scaling (kind::mxf8f6f4, a power
// of two for every 32 elements along the sum) gives every 32 elements of a query, and every 32 tokens of a column of P -- those
// of one warp -- a range of their own, so that small probabilities are as exact as large ones, however far below the maximum.
// That also takes the running maximum out of the loop.  The reference m of a column only has to keep FP32 sums in range: it is 0
// at first, and moves to the maximum so far (with the sums rescaled) only when a probability times its value scale exceeds 2^40, or
// when a column's first tokens all lie below 2^-40.  (Value scales below 2^-64 are taken for 2^-64, so that no probability passes
// 2^104 unseen.)  What falls below the codes of a block, 2^-17 of its largest probability and less, is missing in O and not in the sum: 31
// such tokens are 2^-12 of that one, next to a result that is rounded to 2^-8.
//
//   warp 0      TMA: chunks of [128 tokens x 128 bytes] into a ring for K and one for V, page by page; the pages' scales, and what the softmax
//               warps need to know of an item
//   warps 1, 3  one thread each issues tcgen05.mma: S of the tiles, as far ahead as there is room, and O += P V.  One thread for
//               both spent half of its time in barriers, with nothing left in the tensor pipe's queue.
//   warp 2      zeroes rows of V that no query may see: a page's slots behind its last token may hold anything, NaN included, and
//               0 * NaN is NaN.  In rows that some queries see and others do not it zeroes what is NaN; the softmax warps write NaN to
//               the results of those that see it.
//   warps 4..   softmax: for every 32 lanes two warps (four at 64 columns), each with its share of the columns.  After an item's last
//               tile they bring the next item's queries to shared memory, so that its first scores are computed while they write the
//               results of the one before.
// Two groups of softmax warps with a tile each at a time were slower (16 query rows of drafts 75 -> 84 us, a windowed prompt 128 ->
// 171 us): the warps waited for instructions.  For the same reason only the producer walks over the items, and what runs once
// an item is in short loops.
//
// Work: attention_work.h.  An item that a cut between two blocks' ranges divides leaves FP32 partial sums in the scratch
// memory, which a second kernel joins in the order of the blocks (the same bits on every run).
// A thread waits on a barrier for every phase of it, or for none: with one ring for K and V the thread of S could ask for a phase
// while the one before, of V, was still open, and a parity cannot tell that from the phase being complete.
// Every wait is bounded; a role that gives up reports it, all leave, and tensor memory is released.
//
// Measured (calls back to back, join included).  24 rows on up to 32,000 tokens, 4 KV heads of 512: 264 to 276 us from one GPU to another,
// the rate of a copy from HBM.  One row on 32,749 tokens, 2 heads of 512: 27 us against 10 us of HBM, most of it the first tile's way and the
// second launch.  64 rows in windows of 1024, 16 heads of 256: 104 to 112 us against 81.  Drafts and prompts are bound by the softmax warps, 2400 cycles a tile at 32 columns, 3400 to 4100
// at 64 (about 400 instructions a warp; their chain of latencies, four warps a scheduler, does not fill the issue slots): 80 rows on up to 9000
// tokens, 8 heads of 128, 63 us; 2048 rows in windows of 1024, 8 heads of 256, 104 us; 4096 rows on 16,384 tokens, 2 heads of 512, 2240 to
// 2270 us, 850 TFLOP/s (1970 us in a few passes, before the power limit lowers the clock), where the 64 products of a tile also read 393 KB
// of shared memory, 3100 cycles.
#include <algorithm>
#include <atomic>
#include <string>

#include "attention_work.h"
#include "common.cuh"
#include "gemm_tc.cuh"
#include "paged.h"
#include "pair.cuh"
#include "ptx.cuh"

using namespace gw;

namespace {

__device__ uint32_t g_attention_error;       // first report since it was last taken
std::atomic<bool> g_attention_ran[kMaxDeviceSlots];       // on a GPU: else the word is 0, and reading it would load the module

__host__ __device__ constexpr int softmax_warps(int columns) { return columns <= 32 ? 8 : 16; }
constexpr int kFirstSoftmaxWarp = 4;
constexpr int kChunkBytes = kTokens * 128;
constexpr int kAtomBytes = 512;              // scale atom: 128 rows x 4 blocks of 32 elements
constexpr uint32_t kHighBits = (127u + 40u) << 23, kLowBits = (127u - 40u) << 23;
constexpr int kItems = 4;                    // items that the walk is ahead at most
constexpr int kNans = 30;                    // places with NaN that are kept for an item
constexpr int kScaleTiles = 16;              // tiles whose scales are kept: more than the ring and the score buffers can hold

struct Attention {
  gw_kv_cache cache;
  gw_sequences batch;
  const bf16* query;
  bf16* output;
  uint64_t query_stride, output_stride;
  uint32_t heads, group, group_inverse, per_tile, window;    // group_inverse: x / group is x * group_inverse >> 16 for columns x
  uint32_t page_shift;                                       // page_tokens = 1 << page_shift
  float scale;
  float* partial;             // [blocks][2][N][D], then [blocks][2][2][N] maxima and sums
  int4* records;              // [blocks]: {first query row, columns, KV head, last block} of the item that its last piece begins, or last -1
};

// A piece of an item, as the producer tells the other warps; tiles of -1 end them.
struct Item {
  int begin, end, tiles, first_tile;           // token tiles of the piece, of the item; where the item's begin in the sequence
  int low, high, all_low, all_high;            // the tokens that it reads, and those that all of its queries see
  int used, token_rows, first_row, position0;  // columns with a query, query rows, the first one, its position
  int head, whole;
};

struct Shared {
  uint64_t k_full[8], k_empty[8], v_full[8], v_empty[8], v_cleared[8], scales_full[kScaleTiles], items_full[kItems], items_empty[kItems];
  uint64_t scores_full[2], scores_empty[2], probs_full[2], probs_empty[2], checked, query_full, sums_full, softmax, drained, drained_sums;
  float2 scales[kScaleTiles][8];               // {key, value} of a tile's pages; a value scale below 0: no page
  Item items[kItems];
  // NaN among the values that not every query of an item sees: {token, dimension / 16 << 16 | which of the 16}
  uint2 nans[kItems][kNans];
  int nan_count[kItems];                       // all found
  uint32_t nan_rows[kItems][2];                // a bit for each query row that sees any of those that did not fit
  int move[4];                                 // of the last tiles: some warp asks for the reference to be moved
  uint32_t tensor_memory;
  // units of all blocks, the block's range of them, and the item that has the first
  uint32_t units, from, to, item;
  uint32_t rest;               // units of that item's sequence and head in front of the range
  uint32_t sequence;
  int head, tile;
};

template <int D, int N>
struct Layout {
  static constexpr int kSoftmaxWarps = softmax_warps(N);
  static constexpr int kThreads = 32 * (kFirstSoftmaxWarp + kSoftmaxWarps);
  static constexpr int kShare = N / (kSoftmaxWarps / 4);          // columns of a warp
  static constexpr int kChunks = D / 128;
  static constexpr int kQueryBytes = kChunks * N * 128;           // one part
  static constexpr int kProbBytes = 2 * kChunkBytes;              // rows of 128 bytes: the first part in one half, the second in the other
  static constexpr int kLowOffset = 64;
  static constexpr int kAtoms = 2 * kChunks + 3;        // queries (both parts), ones, P
  static constexpr int kFloats = 7 * N + 32 * kSoftmaxWarps;      // as laid out in the kernel
  static constexpr int kSmall = kAtoms * kAtomBytes + kFloats * 4 + 8 * N;
  static constexpr int kAlignment = 1024;
  static constexpr int kStatic = 4096;                            // at least what is declared in the kernel
  static constexpr int kRoom = 227 * 1024 - kStatic - kAlignment - 2 * kQueryBytes - kProbBytes - kSmall;
  static constexpr int kRings = kRoom / kChunkBytes > 16 ? 16 : kRoom / kChunkBytes;          // chunks
  static constexpr int kKeyRing = (kRings + 1) / 2, kValueRing = kRings / 2;
  static constexpr int kSmemBytes = kAlignment + 2 * kQueryBytes + kProbBytes + kRings * kChunkBytes + kSmall;
  // tensor memory columns
  static constexpr int kScores = kChunks * N;
  static constexpr int kOnes = kScores + 2 * N;
  static constexpr int kQueryScales = kOnes + 4;
  static constexpr int kProbScales = kQueryScales + 8 * kChunks;
  static constexpr int kColumns = 512;
  static_assert(kProbScales + 8 <= kColumns, "tensor memory over-subscribed");
  static_assert(kValueRing >= 2, "a chunk and the next");
  static_assert(kKeyRing / kChunks + 4 < kScaleTiles, "scales of a tile are read before those of a later one take their place");
  static_assert(kSmemBytes > 116 * 1024, "one block an SM");
  static_assert(sizeof(Shared) + 512 <= kStatic, "");
  static_assert(N % 16 == 0 && N <= 64 && D % 128 == 0 && kShare % 8 == 0, "");
};

// ---------------------------------------------------------------------------
// walking over the block's pieces
// ---------------------------------------------------------------------------
struct Walk {
  uint32_t sequence;
  int head, tile;
  uint32_t item;
  SequenceRows rows;
  SequenceWork work;
  // the piece
  int begin, end, tiles;

  __device__ __forceinline__ SequenceWork work_of(const Attention& a) const {
    return SequenceWork{rows.context - rows.count, rows.count, int32_t(a.per_tile), int32_t(a.window)};
  }
  __device__ __forceinline__ void start(const Attention& a, const Shared& s) {
    sequence = s.sequence;
    head = s.head;
    tile = s.tile;
    item = s.item;
    if (sequence < a.batch.sequences) {
      rows = sequence_rows(a.batch, sequence);
      work = work_of(a);
    }
  }
  // The next piece; false: there is none.
  __device__ __forceinline__ bool next(const Attention& a, const Shared& s) {
    while (sequence < a.batch.sequences && item < s.to) {
      if (tile < work.query_tiles()) {
        tiles = work.token_tiles(tile);
        const Piece p = piece_of(item, tiles, s.from, s.to);
        if (p.here) {
          begin = p.begin;
          end = p.end;
          return true;
        }
        advance();
      } else {
        tile = 0;
        if (rows.count != 0 && uint32_t(++head) < a.cache.kv_heads) continue;
        head = 0;
        if (++sequence < a.batch.sequences) {
          rows = sequence_rows(a.batch, sequence);
          work = work_of(a);
        }
      }
    }
    return false;
  }
  __device__ __forceinline__ void advance() {
    item += 1 + tiles;
    ++tile;
  }
};

__device__ __forceinline__ SequenceWork sequence_work(const Attention& a, uint32_t s, bool report) {
  const SequenceRows r = sequence_rows(a.batch, s);
  if (r.bad && report) atomicCAS(&g_attention_error, 0u, 0xa2000000u | (s & 0xffffffu));
  return SequenceWork{r.context - r.count, r.count, int32_t(a.per_tile), int32_t(a.window)};
}

__device__ __forceinline__ uint32_t add_up(uint32_t a, uint32_t b) { return a + b < a ? UINT32_MAX : a + b; }

// The block's range of units and the item that its first unit belongs to.
template <int THREADS>
__device__ __forceinline__ void find_start(const Attention& a, Shared& shared) {
  constexpr int WARPS = THREADS / 32;
  __shared__ uint32_t sums[WARPS];
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  uint32_t before = 0, from = 0;
  bool idle = false;
  // First the units of all sequences, then the sequence that has the block's first one; one round does both where there is a thread for
  // every sequence.
  const bool one = a.batch.sequences <= THREADS;
#pragma unroll 1
  for (uint32_t base = 0, round = 0; round < 2; ) {
    const uint32_t s = base + threadIdx.x;
    uint32_t each = 0, mine = 0;                               // 2^32 - 1: that many or more, here and in sums
    if (s < a.batch.sequences) {
      const SequenceWork w = sequence_work(a, s, round == 0 && blockIdx.x == 0);
      each = w.too_many() ? UINT32_MAX : w.units();
      mine = __umulhi(each, a.cache.kv_heads) != 0 ? UINT32_MAX : each * a.cache.kv_heads;
    }
    uint32_t sum = mine;
#pragma unroll
    for (int m = 1; m < 32; m *= 2) {
      const uint32_t other = __shfl_up_sync(0xffffffffu, sum, m);
      if (lane >= uint32_t(m)) sum = add_up(sum, other);
    }
    if (lane == 31) sums[warp] = sum;
    __syncthreads();
    uint32_t low = before + sum - mine;
#pragma unroll 1
    for (int i = 0; i < WARPS; ++i) {
      if (uint32_t(i) < warp) low += sums[i];
      before = add_up(before, sums[i]);
    }
    __syncthreads();
    base += THREADS;
    const bool end = base >= a.batch.sequences;
    if (round == 0 && end) {
      if (before > uint32_t(INT32_MAX)) {                      // nothing is computed
        if (blockIdx.x == 0 && threadIdx.x == 0) atomicCAS(&g_attention_error, 0u, 0xa2ffffffu);
        before = 0;
      }
      const uint32_t parts = min(before, gridDim.x);
      idle = blockIdx.x >= parts;
      uint32_t to = from = before;
      if (!idle) {
        const Ranges ranges(before, parts);
        from = ranges.start(blockIdx.x);
        to = ranges.start(blockIdx.x + 1);
      }
      if (threadIdx.x == 0) {
        shared.units = before;
        shared.from = from;
        shared.to = to;
        shared.tile = 0;
        if (idle) shared.sequence = a.batch.sequences;
      }
      if (idle) break;
    }
    if ((round == 1 || (one && end)) && low <= from && from - low < mine) {
      shared.sequence = s;
      shared.head = int((from - low) / each);
      shared.rest = (from - low) - shared.head * each;
      shared.item = from - shared.rest;
    }
    if (end) {
      if (one) break;
      base = before = 0;
      ++round;
    } else if (round == 1 && before > from) {
      break;
    }
  }
  __syncthreads();
  // the query tile, 32 candidates at a time
  if (warp == 0 && !idle) {
    const SequenceWork w = sequence_work(a, shared.sequence, false);
    const uint32_t rest = shared.rest;
    int lowest = 0, highest = w.query_tiles();                 // units_before(lowest) <= rest < units_before(highest)
    uint32_t at_lowest = 0;
#pragma unroll 1
    while (highest - lowest > 1) {
      const int step = (highest - lowest + 31) / 32, candidate = min(lowest + int(lane) * step, highest);
      const uint32_t units = w.units_before(candidate);
      const uint32_t below = __ballot_sync(0xffffffffu, candidate < highest && units <= rest);
      const int at = 31 - __clz(below);
      at_lowest = __shfl_sync(0xffffffffu, units, at);
      highest = min(lowest + (at + 1) * step, highest);
      lowest += at * step;
    }
    if (lane == 0) {
      shared.tile = lowest;
      shared.item += at_lowest;
    }
  }
  __syncthreads();
}

// ---------------------------------------------------------------------------
// small pieces
// ---------------------------------------------------------------------------
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Entry of the page table as it is (-1 behind its end).  Nothing is asked of the value here: a warp that looks at it waits for it.
__device__ __forceinline__ int page_entry(const Attention& a, uint32_t sequence, int token) {
  const uint32_t ordinal = uint32_t(token) >> a.page_shift;
  return ordinal < a.batch.page_table_entries ? a.batch.page_table[size_t(sequence) * a.batch.page_table_stride + ordinal] : -1;
}
__device__ __forceinline__ uint32_t pack4(uint16_t low, uint16_t high) { return uint32_t(low) | uint32_t(high) << 16; }

// hi and lo codes of two values of size below 448: hi the nearest codes, lo those of (x - hi) * SCALE
template <int SCALE>
__device__ __forceinline__ void two_parts(float a, float b, uint16_t& hi, uint16_t& lo) {
  const __half2 x = __floats2half2_rn(a, b);
  hi = __nv_cvt_halfraw2_to_fp8x2(__half2_raw(x), __NV_SATFINITE, __NV_E4M3);
  __half2 rest = __hsub2(x, __half2(__nv_cvt_fp8x2_to_halfraw2(hi, __NV_E4M3)));
  if constexpr (SCALE != 1) rest = __hmul2(rest, __float2half2_rn(float(SCALE)));
  lo = __nv_cvt_halfraw2_to_fp8x2(__half2_raw(rest), __NV_SATFINITE, __NV_E4M3);
}

// whether a token tile has tokens outside [low, high)
__device__ __forceinline__ bool has_others(int token_tile, int low, int high) {
  const int start = token_tile * kTokens;
  return low > start || high < start + kTokens;
}

// 0xff in the bytes that are NaN in E4M3
__device__ __forceinline__ uint32_t nan_bytes(uint32_t codes) {
  const uint32_t high = ((codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
  return (high >> 7) * 255u;
}
// a bit for each byte of 0xff
__device__ __forceinline__ uint32_t one_bits(uint32_t bytes) { return (bytes & 1) | (bytes >> 7 & 2) | (bytes >> 14 & 4) | (bytes >> 21 & 8); }

// the bits below `count`, of an item's at most 64 query rows
__device__ __forceinline__ uint64_t rows_below(int count) { return count <= 0 ? 0 : count >= 64 ? ~0ull : (1ull << count) - 1; }

// matrix descriptor of rows of 128 bytes, 128-byte swizzle, read across the rows: 8 rows of the sum are 1024 bytes apart
__device__ __forceinline__ uint64_t across_desc(uint32_t address) { return ptx::smem_desc_sw128(address) | uint64_t(1024 >> 4) << 16; }

// E4M3 x E4M3, UE8M0 scales of 32 elements, FP32 sums, M = 128
__host__ __device__ constexpr uint32_t idesc_mx(uint32_t n, bool across) {
  return (across ? 3u << 15 : 0u) | ((n >> 3) << 17) | (1u << 23) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void mma_mx(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t scale_a, uint32_t scale_b, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(scale_a), "r"(scale_b)
      : "memory");
}

template <int X>
__device__ __forceinline__ void tmem_load(uint32_t address, uint32_t* r) {
  if constexpr (X == 16) {
    ptx::tmem_load16(address, r);
  } else {
    static_assert(X == 8);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(address) : "memory");
  }
}
__device__ __forceinline__ void tmem_store8(uint32_t address, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"r"(address), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
// C columns from `address` on, C a multiple of 8
template <int C>
__device__ __forceinline__ void tmem_load_columns(uint32_t address, uint32_t* r) {
#pragma unroll
  for (int j = 0; j + 16 <= C; j += 16) tmem_load<16>(address + j, r + j);
  if constexpr (C % 16 != 0) tmem_load<8>(address + C - 8, r + C - 8);
}

// v[lane] for lanes below C (a multiple of 8 up to 32), by the bits of the lane's number
template <int C>
__device__ __forceinline__ uint32_t pick(const uint32_t* v, uint32_t lane) {
  uint32_t r[C / 8];
  const bool b0 = lane & 1, b1 = lane & 2, b2 = lane & 4;
#pragma unroll
  for (int i = 0; i < C / 8; ++i) {
    const uint32_t* u = v + 8 * i;
    const uint32_t a0 = b0 ? u[1] : u[0], a1 = b0 ? u[3] : u[2], a2 = b0 ? u[5] : u[4], a3 = b0 ? u[7] : u[6];
    const uint32_t c0 = b1 ? a1 : a0, c1 = b1 ? a3 : a2;
    r[i] = b2 ? c1 : c0;
  }
  uint32_t result = r[0];
#pragma unroll
  for (int i = 1; i < C / 8; ++i) result = lane >= uint32_t(8 * i) ? r[i] : result;
  return result;
}
// v[j] summed over the lanes, for C columns (a multiple of 8 up to 32): lane j gets column j's
template <int C>
__device__ __forceinline__ float lane_sums(const float (&v)[C], uint32_t lane) {
  const bool b0 = lane & 1, b1 = lane & 2, b2 = lane & 4;
  float result = 0.F;
#pragma unroll
  for (int i = 0; i < C / 8; ++i) {
    float u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      u[j] = v[8 * i + j];
      u[j] += __shfl_xor_sync(0xffffffffu, u[j], 16);
      u[j] += __shfl_xor_sync(0xffffffffu, u[j], 8);
    }
    float x[4], y[2];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = (b2 ? u[j + 4] : u[j]) + __shfl_xor_sync(0xffffffffu, b2 ? u[j] : u[j + 4], 4);
#pragma unroll
    for (int j = 0; j < 2; ++j) y[j] = (b1 ? x[j + 2] : x[j]) + __shfl_xor_sync(0xffffffffu, b1 ? x[j] : x[j + 2], 2);
    const float sum = (b0 ? y[1] : y[0]) + __shfl_xor_sync(0xffffffffu, b0 ? y[0] : y[1], 1);
    if (lane / 8 == uint32_t(i)) result = sum;
  }
  return result;
}
// order-preserving integer of a float that is no NaN
__device__ __forceinline__ int ordered(float v) {
  const int bits = __float_as_int(v);
  return bits ^ ((bits >> 31) & 0x7fffffff);
}

// ---------------------------------------------------------------------------
// the kernel
// ---------------------------------------------------------------------------
template <int D, int N>
__global__ void __launch_bounds__(Layout<D, N>::kThreads, 1) paged_attention_kernel(const __grid_constant__ CUtensorMap k_map,
                                                                      const __grid_constant__ CUtensorMap v_map,
                                                                      const __grid_constant__ Attention a) {
  using L = Layout<D, N>;
  constexpr int CH = L::kChunks, KEYS = L::kKeyRing, VALUES = L::kValueRing, C = L::kShare, kSoftmaxWarps = L::kSoftmaxWarps, kSoftmaxThreads = 32 * kSoftmaxWarps, kThreads = L::kThreads;
  extern __shared__ uint8_t raw[];
  uint8_t* const base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint8_t* const query_hi = base;
  uint8_t* const query_lo = query_hi + L::kQueryBytes;
  uint8_t* const probs = query_lo + L::kQueryBytes;
  uint8_t* const k_ring = probs + L::kProbBytes;
  uint8_t* const v_ring = k_ring + KEYS * kChunkBytes;
  uint8_t* const atoms = v_ring + VALUES * kChunkBytes;              // [2 * CH] queries (hi, lo of a chunk), [1] ones, [2] P
  uint8_t* const ones_atom = atoms + 2 * CH * kAtomBytes;
  uint8_t* const probs_atom = ones_atom + kAtomBytes;
  float* const reference = reinterpret_cast<float*>(probs_atom + 2 * kAtomBytes); // [N] m of a column
  float* const factor = reference + N;                                            // [N]
  int* const settled = reinterpret_cast<int*>(factor + N);                        // [N] tile that set the reference: some token above 2^-40
  float* const by_warp = factor + 2 * N;                                          // [4][N]
  float* const spread = by_warp + 4 * N;                                        // [softmax warps][32]
  bf16** const output_at = reinterpret_cast<bf16**>(spread + 32 * kSoftmaxWarps); // [N]
  __shared__ Shared s;
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 8; ++i) {
      ptx::mbar_init(&s.k_full[i], 1);
      ptx::mbar_init(&s.k_empty[i], 1);
      ptx::mbar_init(&s.v_full[i], 1);
      ptx::mbar_init(&s.v_cleared[i], 1);
      ptx::mbar_init(&s.v_empty[i], 2);                          // the product's thread and the warp that zeroes
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&s.scores_full[i], 1);
      ptx::mbar_init(&s.scores_empty[i], kSoftmaxWarps);
      ptx::mbar_init(&s.probs_full[i], kSoftmaxWarps);
      ptx::mbar_init(&s.probs_empty[i], 1);
    }
    ptx::mbar_init(&s.checked, kSoftmaxWarps);
    for (int i = 0; i < 4; ++i) s.move[i] = 0;
    ptx::mbar_init(&s.softmax, kSoftmaxWarps);
    ptx::mbar_init(&s.query_full, kSoftmaxWarps);
    for (int i = 0; i < kScaleTiles; ++i) ptx::mbar_init(&s.scales_full[i], 1);
    for (int i = 0; i < kItems; ++i) {
      ptx::mbar_init(&s.items_full[i], 1);
      ptx::mbar_init(&s.items_empty[i], kSoftmaxWarps + 3);      // and both products' threads and the warp that zeroes
    }
    ptx::mbar_init(&s.sums_full, 1);
    ptx::mbar_init(&s.drained, 1);
    ptx::mbar_init(&s.drained_sums, 1);
    ptx::fence_barrier_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc(&s.tensor_memory, L::kColumns);
    ptx::tmem_relinquish();
  }
  for (int i = threadIdx.x; i < kAtomBytes / 4; i += kThreads) {        // 2^0
    for (int j = 0; j < L::kAtoms; ++j) reinterpret_cast<uint32_t*>(atoms + j * kAtomBytes)[i] = 0x7f7f7f7fu;
  }
  ptx::fence_proxy_async_smem();
  ptx::tc_fence_before_sync();
  griddep_enter();
  find_start<kThreads>(a, s);                                    // ends with __syncthreads()
  ptx::tc_fence_after_sync();
  const uint32_t tmem = s.tensor_memory;
  // Waiting threads sleep: polls took the issue slots of the softmax warps (4096 rows on 16,384 tokens 2312 -> 2184 us on one GPU).
  // What a role gave up on, reported at the end.  A thread whose wait ran out waits no more, but goes on to the end; the roles of one
  // warp or thread leave at once.
  uint32_t error = 0;
  const auto wait = [&error](uint64_t* bar, uint32_t phase, uint32_t code) {
    if (error == 0 && !ptx::mbar_wait_suspended(bar, phase)) error = code;
    return error == 0;
  };

  if (warp == 0) {
    // ----- producer: lane l brings the l-th page of a tile
    const uint32_t page_tokens = a.cache.page_tokens, boxes = kTokens / page_tokens;
    const int outside = int(a.cache.pages * a.cache.kv_heads * page_tokens);        // rows from here on read as zeros
    int issued[2] = {0, 0}, tile_count = 0;                      // chunks of K and of V so far
    if (lane == 0) a.records[blockIdx.x] = make_int4(0, 0, 0, -1);
    Walk w;
    w.start(a, s);
#pragma unroll 1
    for (int n = 0;; ++n) {
      const bool more = w.next(a, s);
      wait(&s.items_empty[n % kItems], (n / kItems & 1) ^ 1, 0xb0000000u);
      error = __reduce_max_sync(0xffffffffu, error);             // the warp leaves as one
      if (error) break;
      if (lane == 0) {
        Item& m = s.items[n % kItems];
        m.tiles = -1;                                            // the end
        s.nan_count[n % kItems] = 0;
        s.nan_rows[n % kItems][0] = s.nan_rows[n % kItems][1] = 0;
        if (more) {
          m.begin = w.begin;
          m.end = w.end;
          m.tiles = w.tiles;
          m.first_tile = w.work.first_token_tile(w.tile);
          m.low = w.work.low(w.tile);
          m.high = w.work.high(w.tile);
          m.position0 = w.work.base + w.tile * int(a.per_tile);
          m.token_rows = min(int(a.per_tile), w.rows.count - w.tile * int(a.per_tile));
          m.used = m.token_rows * int(a.group);
          m.first_row = w.rows.first + w.tile * int(a.per_tile);
          m.all_low = a.window ? max(0, m.position0 + m.token_rows - int(a.window)) : 0;
          m.all_high = max(0, m.position0 + 1);
          m.head = w.head;
          m.whole = w.begin == 0 && w.end == w.tiles;
          if (w.begin == 0 && w.end < w.tiles)
            a.records[blockIdx.x] = make_int4(m.first_row, m.used, w.head, Ranges(s.units, min(s.units, gridDim.x)).with(w.item + w.tiles));
        }
        ptx::mbar_arrive(&s.items_full[n % kItems]);
      }
      __syncwarp();
      if (!more) break;
      const int first_token = w.work.first_token_tile(w.tile) * kTokens + lane * page_tokens, low = w.work.low(w.tile), high = w.work.high(w.tile);
      // entry of the page table, or -2 for a page that is not needed
      const auto entry_of = [&](int t) {
        const int token = first_token + t * kTokens;
        return lane < boxes && t < w.end && token < high && token + int(page_tokens) > low ? page_entry(a, w.sequence, token) : -2;
      };
      const auto scales_of = [&](int entry) {
        float2 v = make_float2(0.F, -1.F);
        if (uint32_t(entry) < a.cache.pages) {
          const size_t at = size_t(entry) * a.cache.kv_heads + w.head;
          v = make_float2(a.cache.k_scales[at], a.cache.v_scales[at]);
        }
        return v;
      };
      const auto bring = [&](const CUtensorMap* map, int row, int& count, uint32_t chunks, uint64_t* full, uint64_t* empty, uint8_t* ring) {
#pragma unroll 1
        for (int c = 0; c < CH; ++c, ++count) {
          const uint32_t lap = uint32_t(count) / chunks, slot = uint32_t(count) - lap * chunks;
          wait(&empty[slot], (lap & 1) ^ 1, 0xa3000000u | slot);               // empty slots: the first lap does not wait
          error = __reduce_max_sync(0xffffffffu, error);
          if (error) return;
          if (lane == 0) ptx::mbar_expect_tx(&full[slot], kChunkBytes);
          __syncwarp();
          if (lane < boxes) ptx::tma_load_2d(ring + slot * kChunkBytes + lane * page_tokens * 128, map, c * 128, row, &full[slot]);
        }
      };
      // K of a tile, then V of the one before; the pages two tiles ahead and the scales one ahead are asked for meanwhile
      int entry = entry_of(w.begin), entry_next = entry_of(w.begin + 1), row_before = 0;
      float2 scales = scales_of(entry);
#pragma unroll 1
      for (int t = w.begin; error == 0 && w.begin < w.end && t <= w.end; ++t) {
        const int entry_after = entry_of(t + 2);
        int row = outside;
        if (t < w.end) {
          if (uint32_t(entry) < a.cache.pages) row = int((uint32_t(entry) * a.cache.kv_heads + w.head) * page_tokens);
          else if (entry != -2) atomicCAS(&g_attention_error, 0u, 0xa1000000u | (w.sequence & 0xffffffu));
          bring(&k_map, row, issued[0], KEYS, s.k_full, s.k_empty, k_ring);
          // A value scale that is no finite number, or below 0, makes the scores of its page NaN: the softmax warps mask what a query does
          // not see, and 0 times the scale itself would reach the others.  Asked here, where it costs nothing (there 16 sequences of drafts
          // took 69.7 us instead of 62.8).
          if (uint32_t(entry) < a.cache.pages && !(scales.y >= 0.F && scales.y <= 3.4028234e38F))
            scales = make_float2(__int_as_float(0x7fc00000), 1.F);
          if (lane < boxes) s.scales[tile_count % kScaleTiles][lane] = scales;
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(&s.scales_full[tile_count % kScaleTiles]);
          ++tile_count;
          scales = scales_of(entry_next);
        }
        if (error == 0 && t > w.begin) bring(&v_map, row_before, issued[1], VALUES, s.v_full, s.v_empty, v_ring);
        row_before = row;
        entry = entry_next;
        entry_next = entry_after;
      }
      if (error) break;
      w.advance();
    }
    // the copies still in flight land before the block ends
#pragma unroll 1
    for (int back = 1; back <= KEYS; ++back) {
      const int keys = issued[0] - back, values = issued[1] - back;
      if (keys >= 0) ptx::mbar_wait_bounded(&s.k_full[keys % KEYS], keys / KEYS & 1, 100000000ull);
      if (values >= 0 && back <= VALUES) ptx::mbar_wait_bounded(&s.v_full[values % VALUES], values / VALUES & 1, 100000000ull);
    }
  } else if (warp == 1) {
    // ----- S, by one thread: the compiler keeps its descriptors in uniform registers only where it knows that one thread runs the code
    // (72 to 110 cycles an instruction otherwise, whatever N; 36 at N = 16, 44 at 64 here)
    if (ptx::elect_one()) {
      int slot = 0, item = 0, scored = 0;
      uint32_t parity = 0;
      const uint64_t ring_rows = ptx::smem_desc_sw128(ptx::smem_u32(k_ring));
      const uint64_t hi_rows = ptx::smem_desc_sw128(ptx::smem_u32(query_hi)), lo_rows = ptx::smem_desc_sw128(ptx::smem_u32(query_lo));
      const uint64_t atom = ptx::smem_desc_sf_atom(ptx::smem_u32(atoms));
      ptx::tc_copy_sf_atom(tmem + L::kOnes, ptx::smem_desc_sf_atom(ptx::smem_u32(ones_atom)));
#pragma unroll 1
      for (int n = 0; wait(&s.items_full[n % kItems], n / kItems & 1, 0xb1000000u); ++n) {
        const Item& m = s.items[n % kItems];
        const int begin = m.begin, end = m.end, tiles = m.tiles;
        ptx::mbar_arrive(&s.items_empty[n % kItems]);
        if (tiles < 0) break;
        if (tiles == 0) continue;
        if (!wait(&s.query_full, item++ & 1, 0xa5000000u)) break;
        ptx::tc_fence_after_sync();
#pragma unroll 1
        for (int i = 0; i < 2 * CH; ++i) ptx::tc_copy_sf_atom(tmem + L::kQueryScales + 4 * i, atom + uint64_t(i * (kAtomBytes >> 4)));
#pragma unroll 1
        for (int t = begin; t < end; ++t) {
          const int buffer = scored & 1;
          wait(&s.scores_empty[buffer], ((scored >> 1) & 1) ^ 1, 0xa6000000u | buffer);
          const uint32_t d = tmem + L::kScores + buffer * N;
          if (!wait(&s.k_full[slot], parity, 0xa4000000u | slot)) break;
#pragma unroll 1
          for (int c = 0; c < CH; ++c) {
            ptx::tc_fence_after_sync();
            const int this_slot = slot;
            const uint64_t keys = ring_rows + uint64_t(slot * (kChunkBytes >> 4)), offset = uint64_t(c * (N * 128 >> 4));
            const uint32_t scales = tmem + L::kQueryScales + 8 * c;
#pragma unroll
            for (int part = 0; part < 2; ++part)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                mma_mx(d, keys + 2 * k, (part ? lo_rows : hi_rows) + offset + 2 * k, idesc_mx(N, false) | uint32_t(k) << 4, tmem + L::kOnes,
                       scales + 4 * part, c | part | k);
            if (++slot == KEYS) {
              slot = 0;
              parity ^= 1;
            }
            // before the commit, which comes back once its products have left the queue
            if (c + 1 < CH && !wait(&s.k_full[slot], parity, 0xa4000000u | slot)) break;
            ptx::tc_commit(&s.k_empty[this_slot]);
          }
          if (error) break;
          ptx::tc_commit(&s.scores_full[buffer]);
          ++scored;
        }
        if (error) break;
      }
      // products still in flight end before tensor memory is released
      ptx::tc_commit(&s.drained);
      ptx::mbar_wait_bounded(&s.drained, 0, 100000000ull);
    }
    __syncwarp();
  } else if (warp == 3) {
    // ----- O += P V, by one thread
    if (ptx::elect_one()) {
      int slot = 0, summed = 0;
      uint32_t parity = 0;
      const uint64_t ring_across = across_desc(ptx::smem_u32(v_ring)), probs_across = across_desc(ptx::smem_u32(probs));
      const uint64_t atom = ptx::smem_desc_sf_atom(ptx::smem_u32(probs_atom));
#pragma unroll 1
      for (int n = 0; wait(&s.items_full[n % kItems], n / kItems & 1, 0xb2000000u); ++n) {
        const Item& m = s.items[n % kItems];
        const int begin = m.begin, end = m.end, tiles = m.tiles, first_tile = m.first_tile, all_low = m.all_low, all_high = m.all_high;
        ptx::mbar_arrive(&s.items_empty[n % kItems]);
        if (tiles < 0) break;
        if (tiles == 0) continue;
#pragma unroll 1
        for (int t = begin; t < end; ++t) {
          // once the chunk is there, the warp that zeroes has finished with what was in its place before
          const bool clear = has_others(first_tile + t, all_low, all_high);
          const auto ready = [&]() {
            wait(&s.v_full[slot], parity, 0xa5100000u | slot);
            return clear ? wait(&s.v_cleared[slot], parity, 0xaf000000u | slot) : error == 0;
          };
          const int buffer = summed & 1;
          wait(&s.probs_full[buffer], (summed >> 1) & 1, 0xa7000000u);
          if (!ready()) break;
          ptx::tc_fence_after_sync();
          const uint32_t scales = tmem + L::kProbScales + 4 * buffer;
          const uint64_t p = probs_across + uint64_t(buffer * (kChunkBytes >> 4));
          ptx::tc_copy_sf_atom(scales, atom + uint64_t(buffer * (kAtomBytes >> 4)));
#pragma unroll 1
          for (int c = 0; c < CH; ++c) {
            ptx::tc_fence_after_sync();
            const int this_slot = slot;
            const uint64_t values = ring_across + uint64_t(slot * (kChunkBytes >> 4));
#pragma unroll
            for (int part = 0; part < 2; ++part)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                mma_mx(tmem + c * N, values + 256 * k, p + uint64_t(part * (L::kLowOffset >> 4)) + 256 * k, idesc_mx(N, true) | uint32_t(k) << 4,
                       tmem + L::kOnes, scales, uint32_t(t > begin) | part | k);
            if (++slot == VALUES) {
              slot = 0;
              parity ^= 1;
            }
            if (c + 1 < CH && !ready()) break;
            ptx::tc_commit(&s.v_empty[this_slot]);
          }
          if (error) break;
          ptx::tc_commit(&s.probs_empty[buffer]);
          if (t == end - 1) ptx::tc_commit(&s.sums_full);
          ++summed;
        }
        if (error) break;
      }
      ptx::tc_commit(&s.drained_sums);
      ptx::mbar_wait_bounded(&s.drained_sums, 0, 100000000ull);
    }
    __syncwarp();
  } else if (warp == 2) {
    // ----- V where not every query of an item sees it: rows that none sees are zeroed, and so are NaN in the others, whose places
    // are kept for those queries that do see them.  Every chunk is waited for, so that this warp is never a lap of the ring away.
    int slot = 0;
    uint32_t parity = 0;
#pragma unroll 1
    for (int n = 0;; ++n) {
      wait(&s.items_full[n % kItems], n / kItems & 1, 0xb3000000u);
      error = __reduce_max_sync(0xffffffffu, error);
      if (error) break;
      const Item& m = s.items[n % kItems];
      const int begin = m.begin, end = m.end, tiles = m.tiles, first_tile = m.first_tile, low = m.low, high = m.high, all_low = m.all_low, all_high = m.all_high, position0 = m.position0;
      __syncwarp();
      if (tiles < 0) break;
#pragma unroll 1
      for (int i = 0; i < CH * (end - begin); ++i) {
        const int tile = first_tile + begin + i / CH, start = tile * kTokens;
        wait(&s.v_full[slot], parity, 0xa9000000u | slot);
        error = __reduce_max_sync(0xffffffffu, error);
        if (error) break;
        if (has_others(tile, all_low, all_high)) {
          // rows of the tile: none sees them up to `first` and from `last` on, all between `all_first` and `all_last`
          uint4* rows = reinterpret_cast<uint4*>(v_ring + slot * kChunkBytes);
          const int first = min(max(low - start, 0), kTokens), last = min(max(high - start, first), kTokens);
          const int all_first = min(max(all_low - start, first), last), all_last = min(max(all_high - start, all_first), last);
#pragma unroll 1
          for (int k = lane; k < first * 8; k += 32) rows[k] = make_uint4(0, 0, 0, 0);
#pragma unroll 1
          for (int k = last * 8 + lane; k < kTokens * 8; k += 32) rows[k] = make_uint4(0, 0, 0, 0);
#pragma unroll 1
          for (int k = first * 8 + lane; k < (last - (all_last - all_first)) * 8; k += 32) {
            const int unit = k < all_first * 8 ? k : k + (all_last - all_first) * 8;
            const uint4 codes = rows[unit];
            const uint4 nan = make_uint4(nan_bytes(codes.x), nan_bytes(codes.y), nan_bytes(codes.z), nan_bytes(codes.w));
            if ((nan.x | nan.y | nan.z | nan.w) != 0) {
              rows[unit] = make_uint4(codes.x & ~nan.x, codes.y & ~nan.y, codes.z & ~nan.z, codes.w & ~nan.w);
              const int at = atomicAdd_block(&s.nan_count[n % kItems], 1), place = (unit % 8) ^ (unit / 8 % 8);       // 128-byte swizzle
              if (at < kNans) {
                s.nans[n % kItems][at] = make_uint2(start + unit / 8, uint32_t(i % CH * 8 + place) << 16 | one_bits(nan.x) | one_bits(nan.y) << 4 |
                                                                   one_bits(nan.z) << 8 | one_bits(nan.w) << 12);
              } else {
                const int ahead = start + unit / 8 - position0;    // rows from here on see the token, up to a window behind it
                const uint64_t seen = rows_below(a.window ? ahead + int(a.window) : 64) & ~rows_below(ahead);
                atomicOr_block(&s.nan_rows[n % kItems][0], uint32_t(seen));
                atomicOr_block(&s.nan_rows[n % kItems][1], uint32_t(seen >> 32));
              }
            }
          }
          ptx::fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) {
          ptx::mbar_arrive(&s.v_cleared[slot]);
          ptx::mbar_arrive(&s.v_empty[slot]);
        }
        if (++slot == VALUES) {
          slot = 0;
          parity ^= 1;
        }
      }
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&s.items_empty[n % kItems]);
      if (error) break;
    }
  } else {
    // ----- softmax.  Code that runs once an item is kept in short loops: what is not in the instruction cache costs more to
    // fetch than to execute (the reference's move, unrolled, took 16000 cycles).
    const uint32_t quadrant = warp & 3, column0 = (warp - kFirstSoftmaxWarp) / 4 * C, member = threadIdx.x - 32 * kFirstSoftmaxWarp;
    const uint32_t lanes = tmem + (quadrant * 32 << 16);
    const uint32_t row = quadrant * 32 + lane;                   // the lane's token in a tile
    const uint32_t group = a.group;
    float* const my_spread = spread + 32 * (warp - kFirstSoftmaxWarp);
    int scored_items = 0, tile_count = 0;
    // a barrier of the softmax warps, bounded as all waits are
    uint32_t meetings = 0;
    const auto together = [&]() {
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&s.softmax);
      wait(&s.softmax, meetings & 1, 0xae000000u);
      __syncwarp();
      ++meetings;
    };
    // Queries of an item: a thread takes 8 elements at a time; the 32 of four neighbouring threads share a power of two.
    const auto bring_queries = [&](const Item& m) {
      const int used = m.used, first_row = m.first_row, head0 = m.head * int(group);
      const auto load = [&](int unit) {
        const uint32_t column = unit / (D / 8), e = unit % (D / 8), at = column * a.group_inverse >> 16;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (unit < N * (D / 8) && int(column) < used)
          v = *reinterpret_cast<const uint4*>(a.query + size_t(first_row + at) * a.query_stride + size_t(head0 + column - at * group) * D + e * 8);
        return v;
      };
      uint4 next = load(member);
#pragma unroll 1
      for (int unit = member; unit < N * (D / 8); unit += kSoftmaxThreads) {
        const uint4 bits = next;
        next = load(unit + kSoftmaxThreads);
        const uint32_t words[4] = {bits.x, bits.y, bits.z, bits.w};
        uint32_t largest = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) largest = max(largest, max(words[i] << 16 & 0x7fffffffu, words[i] & 0x7fff0000u));
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        const uint32_t exponent = largest >> 23;
        // values times 2^(134 - exponent) lie below 2^8; blocks of less than 2^-114 count as zeros, infinities as NaN
        const float up = exponent == 255 ? __uint_as_float(0x7fc00000u) : exponent < 13 ? 0.F : __uint_as_float((261 - exponent) << 23);
        const uint32_t scale = exponent < 13 ? 127 : exponent - 7;
        uint16_t h[4], l[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          two_parts<16>(__uint_as_float(words[i] << 16) * up, __uint_as_float(words[i] & 0xffff0000u) * up, h[i], l[i]);
        const uint32_t column = unit / (D / 8), e = unit % (D / 8), c = e / 16, byte = e % 16 * 8;
        const uint32_t place = c * N * 128 + column * 128 + (((byte >> 4) ^ (column & 7)) << 4) + (byte & 15);
        *reinterpret_cast<uint2*>(query_hi + place) = make_uint2(pack4(h[0], h[1]), pack4(h[2], h[3]));
        *reinterpret_cast<uint2*>(query_lo + place) = make_uint2(pack4(l[0], l[1]), pack4(l[2], l[3]));
        if (e % 4 == 0) {
          const uint32_t scale_at = 2 * c * kAtomBytes + (column % 32) * 16 + column / 32 * 4 + e / 4 % 4;
          atoms[scale_at] = uint8_t(scale);
          atoms[scale_at + kAtomBytes] = uint8_t(scale - 4);
        }
      }
      ptx::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&s.query_full);
    };
    float total[C];
#pragma unroll 1
    for (int n = -1;;) {
      // the next item's queries, while the last product of the one before runs: its scores are all computed
      wait(&s.items_full[(n + 1) % kItems], (n + 1) / kItems & 1, 0xb4000000u);
      error = __reduce_max_sync(0xffffffffu, error);             // a warp goes on or leaves as one
      const bool more = error == 0 && s.items[(n + 1) % kItems].tiles >= 0;
      if (more && s.items[(n + 1) % kItems].tiles > 0) bring_queries(s.items[(n + 1) % kItems]);
      if (n >= 0) {
        const Item& m = s.items[n % kItems];
        if (m.tiles > 0) {
          const int used = m.used;
          // sums of a column over the tokens
          const float sum = lane_sums(total, lane);
          if (lane < uint32_t(C)) by_warp[quadrant * N + column0 + lane] = sum;
          together();
          const bool whole = m.whole;
          const uint32_t place = 2 * blockIdx.x + (m.begin == 0 ? 1 : 0);
          if (member < N) {
            const float v = (by_warp[member] + by_warp[N + member]) + (by_warp[2 * N + member] + by_warp[3 * N + member]);
            factor[member] = v == 0.F ? 0.F : rcp_approx_ftz(v);
            if (!whole) {
              float* const totals = a.partial + size_t(gridDim.x) * 2 * N * D + size_t(place) * 2 * N;
              // The reference of a column that sees nothing of this piece is 0 and says nothing: it must not be the largest of the join,
              // before which scores far below 0 would all vanish.
              totals[member] = v == 0.F ? -INFINITY : reference[member];
              totals[N + member] = v;
            }
          }
          together();
          wait(&s.sums_full, scored_items & 1, 0xab000000u);
          ptx::tc_fence_after_sync();
          // eight columns at a time, to the output or to the block's partial sums
          float* const partial = a.partial + size_t(place) * N * D + row;
#pragma unroll 1
          for (int j = (warp - kFirstSoftmaxWarp) / 4 * 8; j < used; j += kSoftmaxWarps / 4 * 8) {
            float by[8];
            bf16* to[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              by[e] = factor[j + e];
              to[e] = output_at[j + e] + row;
            }
            const int left = used - j;
#pragma unroll 1
            for (int c = 0; c < CH; ++c) {
              float o[8];
              tmem_load<8>(lanes + c * N + j, reinterpret_cast<uint32_t*>(o));
              ptx::tmem_load_wait();
              if (whole) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  if (e < left) to[e][c * 128] = __float2bfloat16_rn(o[e] * by[e]);
              } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  if (e < left) partial[(j + e) * D + c * 128] = o[e];
              }
            }
          }
          ++scored_items;
          const int nans = s.nan_count[n % kItems];
          if (nans != 0) {                                       // to the queries that see them
            together();                                          // behind what was written above
            const int listed = min(nans, kNans);
            const uint64_t spoilt = s.nan_rows[n % kItems][0] | uint64_t(s.nan_rows[n % kItems][1]) << 32;
#pragma unroll 1
            for (int column = warp - kFirstSoftmaxWarp; column < used; column += kSoftmaxWarps) {
              const int in_tile = int(column * a.group_inverse >> 16), position = m.position0 + in_tile;
              bf16* const to = output_at[column];
              float* const to_partial = a.partial + (size_t(place) * N + column) * D;
              const auto spoil = [&](int d) {
                if (whole) to[d] = __float2bfloat16_rn(__int_as_float(0x7fc00000));
                else to_partial[d] = __int_as_float(0x7fc00000);
              };
#pragma unroll 1
              for (int i = 0; i < listed; ++i) {
                const uint2 at = s.nans[n % kItems][i];
                const bool seen = int(at.x) <= position && (a.window == 0 || position - int(at.x) < int(a.window));
                if (seen && lane < 16 && (at.y >> lane & 1)) spoil(int(at.y >> 16) * 16 + lane);
              }
              if (spoilt >> in_tile & 1)
                for (int d = lane; d < D; d += 32) spoil(d);
            }
          }
        }
        // The sums were read: the next item's first product may overwrite them once it has the probabilities that this thread
        // publishes later.  What the item had in shared memory is free.
        ptx::tc_fence_before_sync();
        together();
        if (lane == 0) ptx::mbar_arrive(&s.items_empty[n % kItems]);
      }
      if (!more) break;
      ++n;
      const Item& m = s.items[n % kItems];
      if (int(member) < N) {
        const uint32_t at = member * a.group_inverse >> 16;
        output_at[member] = a.output + size_t(m.first_row + at) * a.output_stride + size_t(m.head * group + member - at * group) * D;
        reference[member] = 0.F;
        settled[member] = int(member) >= m.used ? -1 : INT32_MAX;
      }
      together();
      if (m.tiles == 0) {                                        // rows that see nothing
#pragma unroll 1
        for (int column = warp - kFirstSoftmaxWarp; column < m.used; column += kSoftmaxWarps)
          for (int d = lane * 8; d < D; d += 256) *reinterpret_cast<uint4*>(output_at[column] + d) = make_uint4(0, 0, 0, 0);
        continue;
      }
#pragma unroll
      for (int j = 0; j < C; ++j) total[j] = 0.F;
      const int used = m.used, begin = m.begin, end = m.end, token_rows = m.token_rows;
      const float to_log2 = a.scale * 1.4426950408889634F;

#pragma unroll 1
      for (int t = begin; t < end; ++t, ++tile_count) {
        const int entry = tile_count % kScaleTiles, buffer = tile_count & 1, round = tile_count >> 1 & 1;
        const int ahead = (m.first_tile + t) * kTokens + int(row) - m.position0;       // of the lane's token, to the first query
        wait(&s.scales_full[entry], tile_count / kScaleTiles & 1, 0xac000000u);
        const float2 scales = s.scales[entry][row >> a.page_shift];
        // The columns that see the lane's token: query row i where ahead <= i < ahead + window.  Most tiles are open: seen from every
        // column with a query (the others' queries are zeros, and nobody reads what becomes of them).
        const int tile_ahead = ahead - int(row);
        const bool open = __all_sync(0xffffffffu, scales.y >= 0.F) && tile_ahead + kTokens <= 1 &&
                          (a.window == 0 || tile_ahead + int(a.window) >= token_rows);
        uint32_t seen_from = 0, seen_span = N;                   // column0 + j - from < span, unsigned
        int seen_low = 0, seen_high = N;                         // columns that may see any of the warp's tokens
        if (!open) {
          const int from = max(0, min(ahead, N)) * int(group);
          int to = a.window ? max(0, min(ahead + int(a.window), token_rows)) * int(group) : used;
          if (!(scales.y >= 0.F)) to = 0;
          seen_from = from - column0;
          seen_span = to > from ? to - from : 0;
          seen_low = __reduce_min_sync(0xffffffffu, from);
          seen_high = __reduce_max_sync(0xffffffffu, to);
        }
        const float scale = scales.x * to_log2, value_scale = fmaxf(scales.y, 5.42101086e-20F);         // 2^-64

        wait(&s.scores_full[buffer], round, 0xa8000000u);
        if (tile_count >= 2) wait(&s.probs_empty[buffer], round ^ 1, 0xaa000000u);
        ptx::tc_fence_after_sync();
        const uint32_t scores = lanes + L::kScores + buffer * N + column0;
        uint8_t* const my_probs = probs + buffer * kChunkBytes + row * 128;
        uint8_t* const my_atom = probs_atom + buffer * kAtomBytes;
        bool added = false;
        // Once, or again after the reference moved.  What a warp that asks for a move has is not added to the sums; what the others added
        // stays: a move scales what is in the sums.
#pragma unroll 1
        for (bool moved = false;; moved = true) {
          if (int(column0) < used) {
            float p[C];
            tmem_load_columns<C>(scores, reinterpret_cast<uint32_t*>(p));
            ptx::tmem_load_wait();
            uint32_t bits[C];
#pragma unroll
            for (int j = 0; j < C; ++j) {
              p[j] = exp2_approx(fmaf(p[j], scale, -reference[column0 + j]));
              if (!open) p[j] = uint32_t(j) - seen_from < seen_span ? p[j] : 0.F;
              bits[j] = __reduce_max_sync(0xffffffffu, __float_as_uint(p[j] * value_scale));          // over the warp's tokens
            }
            const uint32_t largest = pick<C>(bits, lane);          // lane j: of column j
            const uint32_t exponent = max(largest >> 23, 8u);      // below, the factor would not be finite
            bool ask = false;
            if (!moved && lane < uint32_t(C)) {
              const uint32_t column = column0 + lane;
              ask = largest > kHighBits && int(column) < used;     // NaN too
              // what other warps find in the same tile does not count: the answer is the same whoever comes first
              if (settled[column] >= tile_count && seen_low <= int(column) && int(column) < seen_high) {
                if (largest < kLowBits) ask = true;
                else settled[column] = tile_count;
              }
              if (ask) s.move[tile_count & 3] = 1;
            }
            ask = __any_sync(0xffffffffu, ask);
            if (!moved && lane == 0) ptx::mbar_arrive(&s.checked);
            // P: the warp's 32 tokens of a column share a power of two, 2^-7 of that of the largest
            my_spread[lane] = __uint_as_float((261 - exponent) << 23);
            if (lane < uint32_t(C)) {
              const uint32_t column = column0 + lane;
              my_atom[column % 32 * 16 + column / 32 * 4 + quadrant] = uint8_t(exponent - 7);
            }
            __syncwarp();
            // 16 bytes at a time where the warp has them: half the accesses to shared memory of 8
            constexpr int STEP = C % 16 == 0 ? 16 : 8;
#pragma unroll
            for (int j = 0; j < C; j += STEP) {
              uint32_t hi[STEP / 4], lo[STEP / 4];
#pragma unroll
              for (int i = 0; i < STEP; i += 4) {
                const float4 up = *reinterpret_cast<const float4*>(my_spread + j + i);
                uint16_t h0, l0, h1, l1;
                // in this order: the factor of a column that sees none of these tokens is 2^126, and 0 stays 0
                two_parts<1>(p[j + i] * value_scale * up.x, p[j + i + 1] * value_scale * up.y, h0, l0);
                two_parts<1>(p[j + i + 2] * value_scale * up.z, p[j + i + 3] * value_scale * up.w, h1, l1);
                hi[i / 4] = pack4(h0, h1);
                lo[i / 4] = pack4(l0, l1);
              }
              const uint32_t byte = column0 + j;
              uint8_t* const to_hi = my_probs + (((byte >> 4) ^ (row & 7)) << 4) + (byte & 15);
              uint8_t* const to_lo = my_probs + ((((byte >> 4) + 4) ^ (row & 7)) << 4) + (byte & 15);
              if constexpr (STEP == 16) {
                *reinterpret_cast<uint4*>(to_hi) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4*>(to_lo) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
              } else {
                *reinterpret_cast<uint2*>(to_hi) = make_uint2(hi[0], hi[1]);
                *reinterpret_cast<uint2*>(to_lo) = make_uint2(lo[0], lo[1]);
              }
            }
            if (!added && !ask) {
              added = true;
#pragma unroll
              for (int j = 0; j < C; ++j) total[j] += p[j];
            }
          } else if (!moved && lane == 0) {                      // no queries
            ptx::mbar_arrive(&s.checked);
          }
          if (moved) break;
          wait(&s.checked, tile_count & 1, 0xad000000u);
          if (member == 0) s.move[(tile_count + 2) & 3] = 0;
          if (*reinterpret_cast<volatile int*>(&s.move[tile_count & 3]) == 0) break;
          // the reference of a column moves to the largest score so far
#pragma unroll 1
          for (int j = 0; j < C; j += 8) {
            float score[8];
            tmem_load<8>(scores + j, reinterpret_cast<uint32_t*>(score));
            ptx::tmem_load_wait();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float v = score[e] * scale;
              const bool seen = uint32_t(j + e) - seen_from < seen_span && v == v;
              const int highest = __reduce_max_sync(0xffffffffu, ordered(seen ? v : -INFINITY));
              if (lane == uint32_t(e)) by_warp[quadrant * N + column0 + j + e] = __int_as_float(highest ^ ((highest >> 31) & 0x7fffffff));
            }
          }
          together();
          if (member < N) {
            const float highest = fmaxf(fmaxf(by_warp[member], by_warp[N + member]), fmaxf(by_warp[2 * N + member], by_warp[3 * N + member]));
            const float before = reference[member];
            // A column that has not settled has had no token before this tile, and one that sees none here keeps its reference.
            const bool had = settled[member] <= tile_count, has = highest != -INFINITY;
            const float now = !has ? before : had ? fmaxf(before, highest) : highest;
            reference[member] = now;
            factor[member] = !has ? 1.F : had ? exp2_approx(before - now) : 0.F;
            if (!had && has) settled[member] = tile_count;
          }
          together();
#pragma unroll
          for (int j = 0; j < C; ++j) total[j] *= factor[column0 + j];
          if (t > begin) {                                       // the sums so far, once the product before is done
            wait(&s.probs_empty[buffer ^ 1], (tile_count - 1) >> 1 & 1, 0xab100000u);
            ptx::tc_fence_after_sync();
#pragma unroll 1
            for (int i = 0; i < CH * (C / 8); ++i) {
              const int j = i % (C / 8) * 8;
              const uint32_t at = lanes + i / (C / 8) * N + column0 + j;
              float sum[8];
              tmem_load<8>(at, reinterpret_cast<uint32_t*>(sum));
              ptx::tmem_load_wait();
#pragma unroll
              for (int e = 0; e < 8; ++e) sum[e] *= factor[column0 + j + e];
              tmem_store8(at, reinterpret_cast<const uint32_t*>(sum));
            }
            ptx::tmem_store_wait();
          }
        }
        ptx::fence_proxy_async_smem();
        ptx::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive(&s.probs_full[buffer]);
          ptx::mbar_arrive(&s.scores_empty[buffer]);
        }
      }
    }
  }
  if (error != 0) atomicCAS(&g_attention_error, 0u, error | (blockIdx.x << 8));
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  if (warp == 1) ptx::tmem_dealloc(tmem, L::kColumns);
}

// Joins the pieces of the items that are divided between blocks: block x looks after the item that block x of the attention kernel
// begins and does not end.  WPC warps share a column, each with every WPC-th piece: eight where a block has few columns, so that the pieces'
// latencies overlap.  Bound by latency: 3 to 5 us, 74 pieces of 8 columns of 512 or one or two of 64.
template <int D, int WPC>
__global__ void __launch_bounds__(256) attention_join_kernel(const __grid_constant__ Attention a, uint32_t blocks, uint32_t columns) {
  constexpr int E = D / 32;
  __shared__ float shared[WPC > 1 ? 8 : 1][D + 1];
  griddep_enter();
  const int4 record = a.records[blockIdx.x];
  if (record.w < 0) return;
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, share = warp % WPC, pieces = record.w - blockIdx.x + 1;
  const float* const totals = a.partial + size_t(blocks) * 2 * columns * D;
  const auto place = [&](uint32_t piece) { return 2 * (blockIdx.x + piece) + (piece == 0 ? 1 : 0); };
  for (uint32_t column = blockIdx.y * (8 / WPC) + warp / WPC; column < uint32_t(record.y); column += gridDim.y * (8 / WPC)) {
    float highest = -INFINITY;
    for (uint32_t p = lane; p < pieces; p += 32) highest = fmaxf(highest, totals[size_t(place(p)) * 2 * columns + column]);
#pragma unroll
    for (int m = 16; m; m /= 2) highest = fmaxf(highest, __shfl_xor_sync(0xffffffffu, highest, m));
    float sum[E] = {}, total = 0.F;                          // a piece of which the column sees nothing has -infinity, and no weight
#pragma unroll 4
    for (uint32_t p = share; p < pieces; p += WPC) {
      const float* const at = totals + size_t(place(p)) * 2 * columns + column;
      const float weight = at[0] == -INFINITY ? 0.F : exp2_approx(at[0] - highest);
      total = fmaf(weight, at[columns], total);
      const float4* const from = reinterpret_cast<const float4*>(a.partial + (size_t(place(p)) * columns + column) * D) + lane;
#pragma unroll
      for (int i = 0; i < E / 4; ++i) {
        const float4 v = from[32 * i];
        sum[4 * i] = fmaf(weight, v.x, sum[4 * i]);
        sum[4 * i + 1] = fmaf(weight, v.y, sum[4 * i + 1]);
        sum[4 * i + 2] = fmaf(weight, v.z, sum[4 * i + 2]);
        sum[4 * i + 3] = fmaf(weight, v.w, sum[4 * i + 3]);
      }
    }
    if constexpr (WPC > 1) {
      static_assert(WPC == 8, "a column a block");
#pragma unroll
      for (int e = 0; e < E; ++e) shared[warp][128 * (e / 4) + lane * 4 + e % 4] = sum[e];
      if (lane == 0) shared[warp][D] = total;
      __syncthreads();
      bf16* const to = a.output + size_t(record.x + column / a.group) * a.output_stride + size_t(record.z * a.group + column % a.group) * D;
      total = 0.F;
#pragma unroll
      for (int i = 0; i < WPC; ++i) total += shared[i][D];
      for (uint32_t d = threadIdx.x; d < uint32_t(D); d += 256) {
        float v = 0.F;
#pragma unroll
        for (int i = 0; i < WPC; ++i) v += shared[i][d];
        to[d] = __float2bfloat16_rn(total == 0.F ? 0.F : v / total);
      }
      __syncthreads();
    } else {
      bf16* const to = a.output + size_t(record.x + column / a.group) * a.output_stride + size_t(record.z * a.group + column % a.group) * D;
      const float inverse = total == 0.F ? 0.F : 1.F / total;
#pragma unroll
      for (int i = 0; i < E / 4; ++i)
        *reinterpret_cast<uint2*>(to + 128 * i + lane * 4) = make_uint2(pair::pack_bf16x2(sum[4 * i] * inverse, sum[4 * i + 1] * inverse),
                                                                        pair::pack_bf16x2(sum[4 * i + 2] * inverse, sum[4 * i + 3] * inverse));
    }
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// Columns of a block: 16 or 32 where all query rows of a sequence fit, else as many as tensor memory takes next to two tiles of
// scores at D = 512 (512 columns: D / 128 * N sums, 2 N scores, up to 44 of scales).
uint32_t columns_of(uint32_t group, uint32_t max_rows) {
  const uint64_t needed = uint64_t(group) * max_rows;
  return needed <= 16 ? 16 : needed <= 32 ? 32 : 64;
}

size_t partial_floats(uint32_t blocks, uint32_t columns, uint32_t head_dim) { return size_t(blocks) * 2 * columns * (head_dim + 2); }

template <int D, int N>
cudaError_t launch_attention(const Attention& a, const CUtensorMap& k_map, const CUtensorMap& v_map, uint32_t blocks, cudaStream_t stream) {
  static bool known[kMaxDeviceSlots] = {};            // plain bools: two threads write the same
  bool& ready = known[current_device_slot()];
  if (!ready) {
    const cudaError_t status = cudaFuncSetAttribute(paged_attention_kernel<D, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D, N>::kSmemBytes);
    if (status != cudaSuccess) return status;
    ready = true;
  }
  const cudaError_t status = launch_pdl_shared(paged_attention_kernel<D, N>, blocks, Layout<D, N>::kThreads, Layout<D, N>::kSmemBytes, stream, k_map, v_map, a);
  if (status != cudaSuccess) return status;
  // Most of the join's blocks find nothing to join: half as many as columns, and a second pass where all are used (64 windows 104 -> 103 us).
  if constexpr (N <= 32) return launch_pdl(attention_join_kernel<D, 8>, dim3(blocks, N / 2), 256, stream, a, blocks, uint32_t(N));
  else return launch_pdl(attention_join_kernel<D, 1>, dim3(blocks, 4), 256, stream, a, blocks, uint32_t(N));
}

template <int D>
cudaError_t launch_columns(uint32_t columns, const Attention& a, const CUtensorMap& k_map, const CUtensorMap& v_map, uint32_t blocks, cudaStream_t stream) {
  return columns == 16   ? launch_attention<D, 16>(a, k_map, v_map, blocks, stream)
         : columns == 32 ? launch_attention<D, 32>(a, k_map, v_map, blocks, stream)
                         : launch_attention<D, 64>(a, k_map, v_map, blocks, stream);
}

}  // namespace

uint32_t gw::take_paged_attention_error() {
  if (!g_attention_ran[current_device_slot()]) return 0;
  uint32_t value = 0;
  if (cudaMemcpyFromSymbol(&value, g_attention_error, sizeof(value)) != cudaSuccess) return 0xFFFFFFFDu;
  const uint32_t none = 0;
  if (value != 0 && cudaMemcpyToSymbol(g_attention_error, &none, sizeof(none)) != cudaSuccess) return 0xFFFFFFFDu;
  return value;
}

extern "C" {

size_t gw_paged_attention_scratch_bytes(const gw_kv_cache* cache, const gw_sequences* batch, uint32_t heads) {
  if (!cache || !batch || cache->kv_heads == 0 || heads < cache->kv_heads) return 256;
  const uint32_t blocks = sm_count(), columns = columns_of(heads / cache->kv_heads, std::max(1u, batch->max_rows));
  return align_up(partial_floats(blocks, columns, cache->head_dim) * sizeof(float), 256) + align_up(blocks * sizeof(int4), 256);
}

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
  const uint32_t group = heads / cache->kv_heads, columns = columns_of(group, batch->max_rows), blocks = sm_count();
  CUtensorMap k_map, v_map;
  std::string error;
  const uint64_t rows = uint64_t(cache->pages) * cache->kv_heads * cache->page_tokens;
  if (!encode_tensor_map_2d(&k_map, cache->k_data, cache->head_dim, rows, cache->page_tokens, &error, 0) ||
      !encode_tensor_map_2d(&v_map, cache->v_data, cache->head_dim, rows, cache->page_tokens, &error, 0))
    return fail(GW_CUDA_ERROR, "paged attention: " + error);
  const size_t floats = align_up(partial_floats(blocks, columns, cache->head_dim) * sizeof(float), 256);
  gw_sequences sequences = *batch;
  sequences.page_table_entries = page_entries(*batch);
  const Attention a{*cache, sequences, static_cast<const bf16*>(query_bf16), static_cast<bf16*>(output_bf16), query_stride, output_stride,
                    heads, group, (65536 + group - 1) / group, columns / group, window > (1u << 30) ? 0 : window, uint32_t(__builtin_ctz(cache->page_tokens)), scale,
                    static_cast<float*>(scratch), reinterpret_cast<int4*>(static_cast<uint8_t*>(scratch) + floats)};
  g_attention_ran[current_device_slot()] = true;
  const cudaStream_t s = as_stream(stream);
  GW_CUDA_CHECK((cache->head_dim == 128   ? launch_columns<128>(columns, a, k_map, v_map, blocks, s)
                 : cache->head_dim == 256 ? launch_columns<256>(columns, a, k_map, v_map, blocks, s)
                                          : launch_columns<512>(columns, a, k_map, v_map, blocks, s)),
                "paged attention");
  return GW_OK;
}

}  // extern "C"
