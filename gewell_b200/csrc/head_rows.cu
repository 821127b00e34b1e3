// Heads of queries, keys and values between the Q | K | V projection and attention: RMS norm of every head, rotation by
// position, and keys and values rounded to E4M3 into the pages of a cache.
//
// A head is D values.  LPH lanes of a warp take one (D = 128: two heads a warp); a lane has 4 V values from the head's first
// half and the 4 V values that lie half a head behind them, so that with a half-split rotation of the whole head both
// elements of a pair, and with neighbouring pairs too, are in one lane's registers.  A half-split rotation of a part of the
// head fetches its partners through shared memory.
//
//   y_i = n_i cos a - n_j sin a,  y_j = n_j cos a + n_i sin a,  a = position * f,  n = x * rsqrt(mean(x^2) + eps) * w
//
// The angle in turns, position * (f / 2 pi), is formed as the sum of two FP32 numbers, exact to 2^-28 up to position 2^24 (beyond,
// of two in 64 bits), and reduced to [-1/2, 1/2], again as two numbers: in 32 bits position 250000 at f = 1 would be off by 0.01 rad.  Its
// sine and cosine are FP32-exact; the hardware's, 2^-21 off, would let a key in ten thousand fall to the next code of E4M3.  They are
// computed once for all heads that a warp or block takes.  Everything else is FP32 and is rounded once.
#include <algorithm>
#include <atomic>
#include <string>

#include "common.cuh"
#include "paged.h"
#include "pair.cuh"

using namespace gw;

namespace {

__device__ uint32_t g_head_rows_error;       // first report since it was last taken
std::atomic<bool> g_append_ran[kMaxDeviceSlots];       // on a GPU: else the word is 0, and reading it would load the module

__device__ __forceinline__ void report(uint32_t code) { atomicCAS(&g_head_rows_error, 0u, code); }

enum Rotation { kNone, kWhole, kNeighbours, kPart };

struct Rotary {
  const float* frequencies;
  uint32_t width;
  int kind;
};

struct Heads {
  const bf16* input;
  uint64_t input_stride;
  bf16* output;
  uint64_t output_stride;
  const bf16* weight;
  uint32_t heads;
  int normalize;
};

// 4 V neighbouring BF16 values
template <int V>
struct Raw {
  uint2 bits[V];
  __device__ __forceinline__ void load(const bf16* p) {
    if constexpr (V == 1) {
      bits[0] = *reinterpret_cast<const uint2*>(p);
    } else {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      bits[0] = make_uint2(v.x, v.y);
      bits[1] = make_uint2(v.z, v.w);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < V; ++j) bits[j] = make_uint2(0, 0);
  }
  __device__ __forceinline__ void unpack(float* f) const {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      f[4 * j] = __uint_as_float(bits[j].x << 16);
      f[4 * j + 1] = __uint_as_float(bits[j].x & 0xffff0000u);
      f[4 * j + 2] = __uint_as_float(bits[j].y << 16);
      f[4 * j + 3] = __uint_as_float(bits[j].y & 0xffff0000u);
    }
  }
};

// A lane's share of the rotation: the frequencies of its pairs.
template <int V, bool WHOLE>
__device__ __forceinline__ void load_frequencies(const Rotary& r, uint32_t lane_at, uint32_t half, bool active, float* f) {
  constexpr int E = 4 * V;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    // kWhole: pair (at + e, at + e + half).  kNeighbours: E / 2 pairs of the first half, then E / 2 of the second.
    const uint32_t pair = WHOLE ? lane_at + e : e < E / 2 ? lane_at / 2 + e : (half + lane_at) / 2 + (e - E / 2);
    const bool used = active && (WHOLE || (r.kind == kNeighbours && 2 * pair < r.width));
    f[e] = used ? r.frequencies[pair] : 0.F;
  }
}

constexpr double kTurn = 0.15915494309189535, kTurnRest = -9.839338337591243e-18;       // 1 / 2 pi, and what the first lacks of it
constexpr int kNear = 1 << 24;

__device__ __forceinline__ bool is_near(int position) { return uint32_t(position) + kNear <= 2u * kNear; }
// turns as the sum of two numbers
__device__ __forceinline__ float2 near_turns(float frequency, float position) {
  constexpr float high = float(kTurn), low = float(kTurn - double(high));
  const float f = frequency * high, f_rest = fmaf(frequency, low, fmaf(frequency, high, -f));        // turns per position
  const float whole = position * f, part = whole - rintf(whole), rest = fmaf(position, f_rest, fmaf(position, f, -whole));
  const float sum = part + rest, of_rest = sum - part;
  return make_float2(sum, (part - (sum - of_rest)) + (rest - of_rest));
}
__device__ __forceinline__ float2 far_turns(float frequency, int position) {
  // the angle and its turns as the sum of two numbers each: the angle has up to 55 bits, and 2^28 turns leave 25 of 53 behind the point
  const double angle = double(frequency) * double(position), angle_rest = fma(double(frequency), double(position), -angle);
  double turns = angle * kTurn;
  const double rest = fma(angle, kTurn, -turns) + fma(angle, kTurnRest, angle_rest * kTurn);
  turns -= rint(turns);
  turns += rest;
  const float sum = float(turns);
  return make_float2(sum, float(turns - double(sum)));
}
__device__ __forceinline__ void sine_cosine(float2 turns, float& s, float& c) {
  float sine, cosine;
  sincospif(2.F * turns.x, &sine, &cosine);
  const float more = turns.y * 6.283185307179586F;
  s = fmaf(more, cosine, sine);
  c = fmaf(-more, sine, cosine);
}

template <int V>
__device__ __forceinline__ void angles(const float* frequencies, int position, float* s, float* c) {
  constexpr int E = 4 * V;
  if (is_near(position)) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float2 turns = near_turns(frequencies[e], float(position));
      s[e] = turns.x;
      c[e] = turns.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float2 turns = far_turns(frequencies[e], position);
      s[e] = turns.x;
      c[e] = turns.y;
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) sine_cosine(make_float2(s[e], c[e]), s[e], c[e]);
}

__device__ __forceinline__ void turn(float& a, float& b, float s, float c) {
  const float x = a;
  a = fmaf(-b, s, x * c);
  b = fmaf(x, s, b * c);
}

// lo / hi: a lane's values of the head's halves, in place.  `stage`: half-split rotation of a part goes through 2 * half
// floats of shared memory that belong to these LPH lanes.
template <int LPH, int V, bool WHOLE>
__device__ __forceinline__ void rotate(const Rotary& r, float* lo, float* hi, const float* s, const float* c, int position, uint32_t at,
                                       uint32_t half, bool active, float* stage) {
  constexpr int E = 4 * V;
  if (WHOLE) {
#pragma unroll
    for (int e = 0; e < E; ++e) turn(lo[e], hi[e], s[e], c[e]);
  } else if (r.kind == kNeighbours) {
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {                        // 0 times an infinity behind the width would reach its neighbour
      if (at + 2 * e < r.width) turn(lo[2 * e], lo[2 * e + 1], s[e], c[e]);
      if (half + at + 2 * e < r.width) turn(hi[2 * e], hi[2 * e + 1], s[E / 2 + e], c[E / 2 + e]);
    }
  } else if (r.kind == kPart) {
    __syncwarp();
    if (active) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        stage[at + e] = lo[e];
        stage[half + at + e] = hi[e];
      }
    }
    __syncwarp();
    const uint32_t pairs = r.width / 2;
#pragma unroll 1                                           // kept short: the other kinds' registers count
    for (uint32_t pair = at / E; pair < pairs; pair += LPH) {
      float sine, cosine;
      const float f = r.frequencies[pair];
      sine_cosine(is_near(position) ? near_turns(f, float(position)) : far_turns(f, position), sine, cosine);
      turn(stage[pair], stage[pairs + pair], sine, cosine);
    }
    __syncwarp();
    if (active) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        lo[e] = stage[at + e];
        hi[e] = stage[half + at + e];
      }
    }
  }
}

template <int LPH, int E>
__device__ __forceinline__ float inverse_rms(const float* lo, const float* hi, float inverse_width, float epsilon) {
  float sum = 0.F;
#pragma unroll
  for (int e = 0; e < E; ++e) sum = fmaf(lo[e], lo[e], fmaf(hi[e], hi[e], sum));
#pragma unroll
  for (int m = LPH / 2; m; m /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, m);
  return rsqrtf(fmaf(sum, inverse_width, epsilon));
}

// ---------------------------------------------------------------------------
// queries and keys, BF16 to BF16
// ---------------------------------------------------------------------------
struct NormRotary {
  Heads query, key;                    // key.heads == 0: none
  uint32_t rows, width, per_task, tasks;       // heads of a row that a task takes, tasks of a row
  const int32_t* positions;            // or NULL: those of the batch
  gw_sequences batch;                  // sequences == 0: every row counts; else rows of no sequence are left as they are
  Rotary rotary;
  float epsilon;
};

// Position of a row in its sequence; false: no sequence has it.
__device__ __forceinline__ bool position_in_batch(const gw_sequences& b, uint32_t row, int& position) {
  uint32_t low = 0, high = b.sequences;                    // the last sequence that starts at or before the row
  // In a decode step sequence r has row r alone: asked first, as the loads of a search wait for one another.
  SequenceRows s{0, 0, 0, false};
  if (row < high) s = sequence_rows(b, row);
  if (int(row) < s.first || int(row) >= s.first + s.count) {
    while (low + 1 < high) {
      const uint32_t middle = (low + high) / 2;
      if (b.row_offsets[middle] <= int(row)) low = middle; else high = middle;
    }
    s = sequence_rows(b, low);
  }
  position = s.context - s.count + int(row) - s.first;
  return int(row) >= s.first && int(row) < s.first + s.count;
}

constexpr int kNormWarps = 4;

// A warp takes heads of one row, queries and keys in one line, the next head's values on their way meanwhile; the row's angles are
// computed once.  Bound by HBM: 4096 rows of 18 heads of 512, 151 MB, 29 us (80% of a copy's rate; 27 with the hardware's sines).
// With a task for each head, and angles in 64 bits, it took 74 us; eight rows, 2 us in a graph.  Rotation of a part in halves goes through
// shared memory, sines for each head: 1025 rows of 32 heads of 128, 9.5 us in a graph, 6.6 as neighbouring pairs.
template <int LPH, int V, bool WHOLE>
__global__ void __launch_bounds__(32 * kNormWarps, V == 1 ? 8 : 6) qk_norm_rotary_kernel(NormRotary a) {
  constexpr int E = 4 * V, kSide = 32 / LPH;
  __shared__ float stage[kNormWarps][kSide * LPH * 2 * E];
  griddep_enter();
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, group = lane / LPH, at = lane % LPH * E, half = a.width / 2;
  const uint32_t task = blockIdx.x * kNormWarps + warp;
  const uint32_t row = task / a.tasks, first = task % a.tasks * a.per_task, last = min(first + a.per_task, a.query.heads + a.key.heads);
  if (row >= a.rows) return;
  const bool inside = at < half;
  const auto load = [&](uint32_t head, Raw<V>& lo, Raw<V>& hi) {
    lo.clear();
    hi.clear();
    if (inside && head < last) {
      const bool is_key = head >= a.query.heads;
      const bf16* from = is_key ? a.key.input + size_t(row) * a.key.input_stride : a.query.input + size_t(row) * a.query.input_stride;
      from += size_t(is_key ? head - a.query.heads : head) * a.width + at;
      lo.load(from);
      hi.load(from + half);
    }
  };
  Raw<V> next_lo, next_hi;
  load(first + group, next_lo, next_hi);
  // on their way during the search, whose loads wait for one another
  float s[E], c[E];
  load_frequencies<V, WHOLE>(a.rotary, at, half, inside, c);
  const int given = a.positions != nullptr ? a.positions[row] : 0;
  int position = 0;
  if (a.batch.sequences && !position_in_batch(a.batch, row, position)) return;
  if (a.positions != nullptr) position = given;
  angles<V>(c, position, s, c);
  const float inverse_width = 1.F / float(a.width);
#pragma unroll 1
  for (uint32_t at_head = first; at_head < last; at_head += kSide) {
    const uint32_t head = at_head + group;
    const bool active = inside && head < last, is_key = head >= a.query.heads;
    float lo[E], hi[E];
    next_lo.unpack(lo);
    next_hi.unpack(hi);
    load(head + kSide, next_lo, next_hi);
    const float rms = inverse_rms<LPH, E>(lo, hi, inverse_width, a.epsilon);
    const float inverse = (is_key ? a.key.normalize : a.query.normalize) ? rms : 1.F;
    const bf16* weight = is_key ? a.key.weight : a.query.weight;
    if (weight != nullptr && inside) {
      Raw<V> raw;
      float w[E];
      raw.load(weight + at);
      raw.unpack(w);
#pragma unroll
      for (int e = 0; e < E; ++e) lo[e] = lo[e] * inverse * w[e];
      raw.load(weight + half + at);
      raw.unpack(w);
#pragma unroll
      for (int e = 0; e < E; ++e) hi[e] = hi[e] * inverse * w[e];
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        lo[e] *= inverse;
        hi[e] *= inverse;
      }
    }
    rotate<LPH, V, WHOLE>(a.rotary, lo, hi, s, c, position, at, half, active, stage[warp] + group * LPH * 2 * E);
    if (active) {
      uint32_t out_lo[2 * V], out_hi[2 * V];
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) {
        const __nv_bfloat162 l = __floats2bfloat162_rn(lo[2 * e], lo[2 * e + 1]), u = __floats2bfloat162_rn(hi[2 * e], hi[2 * e + 1]);
        out_lo[e] = *reinterpret_cast<const uint32_t*>(&l);
        out_hi[e] = *reinterpret_cast<const uint32_t*>(&u);
      }
      bf16* to = is_key ? a.key.output + size_t(row) * a.key.output_stride : a.query.output + size_t(row) * a.query.output_stride;
      to += size_t(is_key ? head - a.query.heads : head) * a.width + at;
      if constexpr (V == 1) {
        *reinterpret_cast<uint2*>(to) = make_uint2(out_lo[0], out_lo[1]);
        *reinterpret_cast<uint2*>(to + half) = make_uint2(out_hi[0], out_hi[1]);
      } else {
        *reinterpret_cast<uint4*>(to) = make_uint4(out_lo[0], out_lo[1], out_lo[2], out_lo[3]);
        *reinterpret_cast<uint4*>(to + half) = make_uint4(out_hi[0], out_hi[1], out_hi[2], out_hi[3]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// keys and values into pages
// ---------------------------------------------------------------------------
struct Append {
  gw_kv_cache cache;
  gw_sequences batch;
  Heads key, value;
  const int32_t* positions;
  Rotary rotary;
  float epsilon;
  uint32_t each;                       // items of a block: the KV heads' keys are the first items, their values the others
};

// What the call brings to one page of one sequence.
struct Segment {
  int row, count, slot, position;      // first row, rows, slot and position of the first
  int page;                            // -1: nothing to do
};

__device__ __forceinline__ uint32_t segments_of(const SequenceRows& s, uint32_t page_tokens) {
  const int first = max(0, s.context - s.count);
  return s.count == 0 || s.context <= first ? 0 : uint32_t(s.context - 1) / page_tokens - uint32_t(first) / page_tokens + 1;
}

__device__ __forceinline__ Segment segment_at(const Append& a, uint32_t sequence, const SequenceRows& s, uint32_t which) {
  const uint32_t page_tokens = a.cache.page_tokens;
  const int begin = s.context - s.count, first = max(0, begin);
  const uint32_t ordinal = uint32_t(first) / page_tokens + which;
  const int low = max(first, int(ordinal * page_tokens)), high = min(int64_t(s.context), int64_t(ordinal + 1) * page_tokens);
  Segment g{s.first + low - begin, high - low, int(uint32_t(low) % page_tokens), low, -1};
  if (ordinal < a.batch.page_table_entries) {
    const int page = a.batch.page_table[size_t(sequence) * a.batch.page_table_stride + ordinal];
    if (page >= 0 && uint32_t(page) < a.cache.pages) g.page = page;
  }
  if (g.page < 0) report(0xa1000000u | (sequence & 0xffffffu));
  return g;
}

// Segment `wanted` of all sequences, found by a scan over their counts.  The first block scans them all and reports those that cannot be
// followed: a block for the last ones need not be there.
template <int THREADS>
__device__ __forceinline__ Segment find_segment(const Append& a, uint32_t wanted) {
  constexpr int WARPS = THREADS / 32;
  __shared__ uint32_t totals[WARPS];
  __shared__ Segment found;
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const bool reports = blockIdx.x == 0 && blockIdx.y == 0;
  if (threadIdx.x == 0) found.page = -1;
  uint32_t before = 0;
  for (uint32_t base = 0; base < a.batch.sequences; base += THREADS) {
    const uint32_t s = base + threadIdx.x;
    SequenceRows rows{0, 0, 0, false};
    if (s < a.batch.sequences) {
      rows = sequence_rows(a.batch, s);
      if (rows.bad && reports) report(0xa2000000u | (s & 0xffffffu));
    }
    const uint32_t mine = segments_of(rows, a.cache.page_tokens);
    uint32_t sum = mine;
#pragma unroll
    for (int m = 1; m < 32; m *= 2) {
      const uint32_t other = __shfl_up_sync(0xffffffffu, sum, m);
      if (lane >= uint32_t(m)) sum += other;
    }
    if (lane == 31) totals[warp] = sum;
    __syncthreads();
    uint32_t low = before + sum - mine, all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (uint32_t(w) < warp) low += totals[w];
      all += totals[w];
    }
    if (wanted >= low && wanted - low < mine) found = segment_at(a, s, rows, wanted - low);
    before += all;
    __syncthreads();
    if (wanted < before && !reports) break;
  }
  return found;
}

// Smallest power of two, 2^-64 or more, with which `loudest` (finite) fits: 448 = 1.75 * 2^8 is the largest code.
__device__ __forceinline__ float page_scale(float loudest) {
  const uint32_t bits = __float_as_uint(loudest), fraction = bits & 0x7fffffu;
  const int exponent = int(bits >> 23) - 8 + (fraction > 0x600000u);
  return __uint_as_float(uint32_t(max(exponent, 127 - 64)) << 23);
}

__device__ __forceinline__ float finite_size(float v) {
  const float size = fabsf(v);
  return size <= 3.4028234e38F ? size : 0.F;         // not of infinities and NaN
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  return uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3)) |
         uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3)) << 16;
}

__device__ __forceinline__ uint32_t softer(uint32_t codes, float ratio) {
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const __half2 pair(__nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(codes >> (8 * i)), __NV_E4M3));
    const float2 f = __half22float2(pair);
    out |= uint32_t(__nv_cvt_float2_to_fp8x2(make_float2(f.x * ratio, f.y * ratio), __NV_SATFINITE, __NV_E4M3)) << (8 * i);
  }
  return out;
}

// a word of another block's shared memory
__device__ __forceinline__ void store_word(uint32_t at, uint32_t value) {
  asm volatile("st.relaxed.cluster.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(value) : "memory");
}
// The largest of `count` words (up to 32), each waited for until it is no longer 0.
__device__ __forceinline__ uint32_t largest_of(const uint32_t* words, uint32_t count, uint32_t lane) {
  uint32_t word = 0;
  if (lane < count) {
    for (uint32_t spins = 0; (word = *const_cast<const volatile uint32_t*>(words + lane)) == 0; ++spins) {
      if (spins == 1u << 26) {                             // seconds
        report(0xa3000000u);
        break;
      }
    }
  }
  return __reduce_max_sync(0xffffffffu, word);
}

constexpr int kMostItems = 16;         // of a block

// A cluster of one to eight blocks takes the call's tokens of one page, a token at a time for LPH lanes, for a few KV heads one
// after the other (items: first the heads' keys, then their values): the angles are computed once, the next item's values are on their way
// while an item is normed, and its codes are written while the next one's are.  For every item the last warp of a block sends all
// blocks the scale that the block's tokens and the page's codes want; the largest is the page's.
// Bound by issue and by that chain: 4096 rows of 4 heads of 512 in pages of 128, 50 MB, 27 us in a graph (1.9 TB/s), 5 us of it until the
// first item is loaded; one row of each of 64 sequences, 16 heads of 256, 3.5 us; 12 us for 9 sequences of up to 700 rows, 8 heads of 128.
// A block for a page, with the tokens of a page in eight rounds and everything computed twice, took 33.6 us for the first.
template <int LPH, int V, int W, bool WHOLE>
__global__ void __launch_bounds__(32 * W, (V == 1 || W == 16 ? 32 : 20) / W) kv_append_kernel(Append a) {
  constexpr int E = 4 * V, kSide = 32 / LPH;
  constexpr uint32_t width = LPH * 2 * E, half = width / 2;
  __shared__ __align__(16) float stage[W][kSide * LPH * 2 * E];
  constexpr int kMostBlocks = W == 16 ? 8 : 1;
  __shared__ uint32_t of_block[kMostItems], arrived[kMostItems];   // the scale that the block's warps want so far, and how many they are
  __shared__ uint32_t wanted[kMostItems][kMostBlocks];             // the scale that a block of the cluster wants, 0 before
  const uint32_t blocks = W == 16 ? pair::cluster_size() : 1, rank = W == 16 ? pair::cluster_rank() : 0;
  if constexpr (W > 1) {
    if (threadIdx.x < kMostItems) {
      of_block[threadIdx.x] = arrived[threadIdx.x] = 0;
      for (int i = 0; i < kMostBlocks; ++i) wanted[threadIdx.x][i] = 0;
    }
    __syncthreads();
    if (W == 16) pair::cluster_arrive();                   // the others run, and are ready, before anything is sent to them
  }
  griddep_enter();
  const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, group = lane / LPH, at = lane % LPH * E;
  const uint32_t kv_heads = a.cache.kv_heads, first = blockIdx.y * a.each, last = min(first + a.each, 2 * kv_heads);
  const bool kept_used = first < kv_heads && (WHOLE || a.rotary.kind == kNeighbours);
  float s[E], c[E];
  if (kept_used) load_frequencies<V, WHOLE>(a.rotary, at, half, true, c);
  Segment g;
  if constexpr (W == 1) {                                  // one row a sequence
    const SequenceRows s = sequence_rows(a.batch, blockIdx.x);
    if (s.bad && threadIdx.x == 0) report(0xa2000000u | (blockIdx.x & 0xffffffu));
    if (segments_of(s, a.cache.page_tokens) == 0) return;
    g = segment_at(a, blockIdx.x, s, 0);
  } else {
    g = find_segment<32 * W>(a, blockIdx.x / blocks);
  }
  __syncwarp();
  if constexpr (W == 16) pair::cluster_wait();
  if (g.page < 0) return;                                  // all blocks of a cluster alike
  const uint32_t token = (rank * W + warp) * kSide + group;
  const bool active = token < uint32_t(g.count);
  Raw<V> next_lo, next_hi;
  const auto load = [&](uint32_t item) {
    next_lo.clear();
    next_hi.clear();
    if (active && item < last) {
      const bool is_key = item < kv_heads;
      const bf16* from = is_key ? a.key.input + size_t(g.row + token) * a.key.input_stride : a.value.input + size_t(g.row + token) * a.value.input_stride;
      from += (is_key ? item : item - kv_heads) * width + at;
      next_lo.load(from);
      next_hi.load(from + half);
    }
  };
  load(first);
  const int position = !active ? 0 : a.positions != nullptr ? a.positions[g.row + token] : g.position + int(token);
  // A lane's sines and cosines wait in shared memory: 64 registers a thread are all there are.
  float4* const kept = reinterpret_cast<float4*>(stage[warp]) + lane;
  if (kept_used) {
    angles<V>(c, position, s, c);
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      kept[e * 8] = make_float4(s[e], s[e + 1], s[e + 2], s[e + 3]);
      kept[(E + e) * 8] = make_float4(c[e], c[e + 1], c[e + 2], c[e + 3]);
    }
  }

  // Between an item's scales and its codes lies the next item: what the warps send one another is on its way meanwhile.
  float done_lo[E], done_hi[E], old_scale = 0.F, asked = 0.F;
#pragma unroll 1
  for (uint32_t item = first; item <= last; ++item) {
    float lo[E], hi[E], old = 0.F, scale = 0.F;
    if (item < last) {
      const bool is_key = item < kv_heads;
      const uint32_t head = is_key ? item : item - kv_heads;
      const Heads& h = is_key ? a.key : a.value;
      next_lo.unpack(lo);
      next_hi.unpack(hi);
      load(item + 1);
      if (g.slot > 0) old = (is_key ? a.cache.k_scales : a.cache.v_scales)[size_t(g.page) * kv_heads + head];
      if (!(old > 0.F && old <= 3.4028234e38F)) old = 0.F;
      const float inverse = h.normalize ? inverse_rms<LPH, E>(lo, hi, 1.F / float(width), a.epsilon) : 1.F;
      if (h.weight != nullptr) {
        Raw<V> raw;
        float w[E];
        raw.load(h.weight + at);
        raw.unpack(w);
#pragma unroll
        for (int e = 0; e < E; ++e) lo[e] = lo[e] * inverse * w[e];
        raw.load(h.weight + half + at);
        raw.unpack(w);
#pragma unroll
        for (int e = 0; e < E; ++e) hi[e] = hi[e] * inverse * w[e];
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          lo[e] *= inverse;
          hi[e] *= inverse;
        }
      }
      if (is_key) {
        float s[E], c[E];
        if (kept_used) {
#pragma unroll
          for (int e = 0; e < E; e += 4) {
            const float4 x = kept[e * 8], y = kept[(E + e) * 8];
            s[e] = x.x, s[e + 1] = x.y, s[e + 2] = x.z, s[e + 3] = x.w;
            c[e] = y.x, c[e + 1] = y.y, c[e + 2] = y.z, c[e + 3] = y.w;
          }
        }
        rotate<LPH, V, WHOLE>(a.rotary, lo, hi, s, c, position, at, half, true, stage[warp] + group * LPH * 2 * E);
      }

      float loudest = 0.F;                                   // of what is no NaN
#pragma unroll
      for (int e = 0; e < E; ++e) loudest = fmaxf(loudest, fmaxf(fabsf(lo[e]), fabsf(hi[e])));
      if (!(loudest <= 3.4028234e38F)) {
        loudest = 0.F;
#pragma unroll
        for (int e = 0; e < E; ++e) loudest = fmaxf(loudest, fmaxf(finite_size(lo[e]), finite_size(hi[e])));
      }
      if (!active) loudest = 0.F;
      // once all warps' scales are known, all have read the old one
      scale = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(old, page_scale(loudest)))));
      if constexpr (W > 1) {
        // The last warp of the block sends what all want.  A word is its own flag: no scale is 0.
        const uint32_t i = item - first;
        uint32_t last_one = 0, most = 0;
        if (lane == 0) {
          atomicMax_block(&of_block[i], __float_as_uint(scale));
          __threadfence_block();
          if (atomicAdd_block(&arrived[i], 1) == W - 1) {
            last_one = 1;
            __threadfence_block();
            most = *const_cast<volatile uint32_t*>(&of_block[i]);
            if (blocks == 1) *const_cast<volatile uint32_t*>(&wanted[i][0]) = most;
          }
        }
        if (W == 16 && blocks > 1 && __shfl_sync(0xffffffffu, last_one, 0)) {
          most = __shfl_sync(0xffffffffu, most, 0);
          if (lane < blocks) store_word(pair::cluster_address(&wanted[i][rank], lane), most);
        }
      }
    }
    if (item > first) {
      const uint32_t before = item - 1, head = before < kv_heads ? before : before - kv_heads;
      const bool is_key = before < kv_heads;
      float final_scale = asked;
      if constexpr (W > 1)
        final_scale = __uint_as_float(largest_of(wanted[before - first], blocks, lane));
      const float inverse_scale = __frcp_rn(final_scale);
      if (rank == 0 && threadIdx.x == 0) (is_key ? a.cache.k_scales : a.cache.v_scales)[size_t(g.page) * kv_heads + head] = final_scale;

      uint8_t* const page = static_cast<uint8_t*>(is_key ? a.cache.k_data : a.cache.v_data) +
                            (size_t(g.page) * kv_heads + head) * a.cache.page_tokens * width;
      if (g.slot > 0 && final_scale > old_scale) {         // a louder token than the page had
        const float ratio = old_scale * inverse_scale;
        uint4* codes = reinterpret_cast<uint4*>(page);
#pragma unroll(W == 16 ? 1 : 4)                           // registers
        for (uint32_t i = rank * 32 * W + threadIdx.x; i < uint32_t(g.slot) * width / 16; i += blocks * 32 * W) {
          uint4 v = codes[i];
          v = make_uint4(softer(v.x, ratio), softer(v.y, ratio), softer(v.z, ratio), softer(v.w, ratio));
          codes[i] = v;
        }
      }
      if (active) {
        uint8_t* to = page + size_t(g.slot + token) * width + at;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          done_lo[e] *= inverse_scale;
          done_hi[e] *= inverse_scale;
        }
        if constexpr (V == 1) {
          *reinterpret_cast<uint32_t*>(to) = e4m3x4(done_lo[0], done_lo[1], done_lo[2], done_lo[3]);
          *reinterpret_cast<uint32_t*>(to + half) = e4m3x4(done_hi[0], done_hi[1], done_hi[2], done_hi[3]);
        } else {
          *reinterpret_cast<uint2*>(to) = make_uint2(e4m3x4(done_lo[0], done_lo[1], done_lo[2], done_lo[3]), e4m3x4(done_lo[4], done_lo[5], done_lo[6], done_lo[7]));
          *reinterpret_cast<uint2*>(to + half) = make_uint2(e4m3x4(done_hi[0], done_hi[1], done_hi[2], done_hi[3]), e4m3x4(done_hi[4], done_hi[5], done_hi[6], done_hi[7]));
        }
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      done_lo[e] = lo[e];
      done_hi[e] = hi[e];
    }
    old_scale = old;
    asked = scale;
    __syncwarp();
  }
  if constexpr (W == 16) {                                 // nobody leaves while somebody may still send to it
    pair::cluster_arrive_relaxed();
    pair::cluster_wait();
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
gw_status check_heads(const gw_head_rows* h, bool has_output, uint32_t width, const std::string& what) {
  if (!h || !h->input || h->heads == 0 || h->heads > 1024 || !is_aligned16(h->input) || (h->weight && !is_aligned16(h->weight)))
    return fail(GW_INVALID_ARGUMENT, what + " requires 1 to 1024 heads, 16-byte aligned inputs and weights");
  if (h->input_stride % 8 != 0 || h->input_stride < uint64_t(h->heads) * width)
    return fail(GW_INVALID_ARGUMENT, what + " requires row strides divisible by 8 that hold all heads");
  if (has_output && (!h->output || !is_aligned16(h->output) || h->output_stride % 8 != 0 || h->output_stride < uint64_t(h->heads) * width ||
                     (h->output == h->input && h->output_stride != h->input_stride)))
    return fail(GW_INVALID_ARGUMENT, what + " requires a 16-byte aligned output with a row stride divisible by 8 (in place: the input's)");
  return GW_OK;
}

gw_status check_rotary(const gw_rotary* r, uint32_t width, const std::string& what, Rotary* rotary) {
  *rotary = Rotary{nullptr, 0, kNone};
  if (!r || r->width == 0) return GW_OK;
  if (!r->inverse_frequencies || r->width % 2 != 0 || r->width > width)
    return fail(GW_INVALID_ARGUMENT, what + " requires inverse frequencies and an even rotated width within the head");
  *rotary = Rotary{r->inverse_frequencies, r->width, r->interleaved ? kNeighbours : r->width == width ? kWhole : kPart};
  return GW_OK;
}

Heads heads_of(const gw_head_rows& h) {
  return Heads{static_cast<const bf16*>(h.input), h.input_stride, static_cast<bf16*>(h.output), h.output_stride,
               static_cast<const bf16*>(h.weight), h.heads, h.normalize};
}

// Parts of `count` heads such that `units` times the parts are at least `wanted`, if the heads allow it; heads of a part.
uint32_t heads_each(uint32_t count, uint64_t units, uint64_t wanted) {
  const uint64_t parts = std::min<uint64_t>(count, std::max<uint64_t>(1, (wanted + units - 1) / units));
  return uint32_t((count + parts - 1) / parts);
}

cudaError_t launch_norm_rotary(NormRotary a, cudaStream_t stream) {
  const uint32_t lanes = a.width <= 64 ? 8 : a.width <= 128 ? 16 : 32, side = 32 / lanes, heads = a.query.heads + a.key.heads;
  // Warps for 24 to an SM, then more heads a warp.  4096 rows of 18 heads of 512: 28 / 29 / 32 us with one / two / four warps a row; 1025 rows
  // of 32 heads of 128: 8.7 / 7.0 / 7.3 us with three / five / seven.
  a.per_task = side * heads_each((heads + side - 1) / side, a.rows, sm_count() * 24);
  a.tasks = (heads + a.per_task - 1) / a.per_task;
  const uint64_t tasks = uint64_t(a.rows) * a.tasks;
  if (tasks > 0xffffffffull - 64) return cudaErrorInvalidValue;
  const bool whole = a.rotary.kind == kWhole;
  const auto kernel = a.width <= 64    ? (whole ? qk_norm_rotary_kernel<8, 1, true> : qk_norm_rotary_kernel<8, 1, false>)
                      : a.width <= 128 ? (whole ? qk_norm_rotary_kernel<16, 1, true> : qk_norm_rotary_kernel<16, 1, false>)
                      : a.width <= 256 ? (whole ? qk_norm_rotary_kernel<32, 1, true> : qk_norm_rotary_kernel<32, 1, false>)
                                       : (whole ? qk_norm_rotary_kernel<32, 2, true> : qk_norm_rotary_kernel<32, 2, false>);
  return launch_pdl(kernel, uint32_t((tasks + kNormWarps - 1) / kNormWarps), 32 * kNormWarps, stream, a);
}

template <int LPH, int V, bool WHOLE>
cudaError_t launch_append(Append a, cudaStream_t stream) {
  const uint32_t page = a.cache.page_tokens, most = std::min(page, a.batch.max_rows), sequences = a.batch.sequences, heads = a.cache.kv_heads;
  constexpr uint32_t kSide = 32 / LPH;
  a.each = 1;
  if (a.batch.max_rows == 1) return launch_pdl(kv_append_kernel<LPH, V, 1, WHOLE>, dim3(sequences, 2 * heads), 32, stream, a);
  // a sequence of n rows touches at most 1 + (n + page - 2) / page pages
  const uint64_t bound = std::min(uint64_t(sequences) * (1 + (a.batch.max_rows + page - 2) / page),
                                  sequences + (uint64_t(a.batch.rows) + uint64_t(sequences) * (page - 2)) / page);
  uint32_t blocks = 1;
  if (most > 8 * kSide)
    while (16 * kSide * blocks < most) blocks *= 2;
  // Few parts of the heads: what a block does before its first item takes 5 us.  4096 rows of 4 heads of 512 in pages of 128, 264 blocks of
  // 512 threads for each part: 26 / 30 / 41 us with one / two / four parts; 9 sequences of up to 700 rows, 8 heads of 128 in pages of 16,
  // 204 blocks of 256: 15 / 14 / 11 / 12 with one / two / three / six.
  a.each = std::min<uint32_t>(kMostItems, heads_each(2 * heads, bound * blocks, most > 8 * kSide ? sm_count() : sm_count() * 4));
  const dim3 grid(uint32_t(bound) * blocks, (2 * heads + a.each - 1) / a.each);
  if (most <= 4 * kSide) return launch_pdl(kv_append_kernel<LPH, V, 4, WHOLE>, grid, 128, stream, a);
  if (most <= 8 * kSide) return launch_pdl(kv_append_kernel<LPH, V, 8, WHOLE>, grid, 256, stream, a);
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(512);
  config.stream = stream;
  cudaLaunchAttribute attributes[2]{};
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim.x = blocks;
  attributes[0].val.clusterDim.y = 1;
  attributes[0].val.clusterDim.z = 1;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attributes;
  config.numAttrs = 2;
  note_launch();
  return cudaLaunchKernelEx(&config, kv_append_kernel<LPH, V, 16, WHOLE>, a);
}

}  // namespace

uint32_t gw::take_head_rows_error() {
  if (!g_append_ran[current_device_slot()]) return 0;
  uint32_t value = 0;
  if (cudaMemcpyFromSymbol(&value, g_head_rows_error, sizeof(value)) != cudaSuccess) return 0xFFFFFFFDu;
  const uint32_t none = 0;
  if (value != 0 && cudaMemcpyToSymbol(g_head_rows_error, &none, sizeof(none)) != cudaSuccess) return 0xFFFFFFFDu;
  return value;
}

extern "C" {

gw_status gw_qk_norm_rotary_bf16(const gw_head_rows* query, const gw_head_rows* key, uint32_t rows, uint32_t head_dim,
                                 const int32_t* positions, const gw_rotary* rotary, float epsilon, void* stream) {
  clear_error();
  if (rows == 0) return GW_OK;
  const std::string what = "norm and rotation of queries and keys";
  if (head_dim == 0 || head_dim > 512 || head_dim % (head_dim <= 256 ? 8 : 16) != 0 || rows > (1u << 24))
    return fail(GW_INVALID_ARGUMENT, what + " requires a head width divisible by 8 (beyond 256: by 16) of at most 512 and at most 2^24 rows");
  NormRotary a{};
  if (gw_status s = check_heads(query, true, head_dim, what); s != GW_OK) return s;
  a.query = heads_of(*query);
  if (key) {
    if (gw_status s = check_heads(key, true, head_dim, what); s != GW_OK) return s;
    a.key = heads_of(*key);
  }
  if (gw_status s = check_rotary(rotary, head_dim, what, &a.rotary); s != GW_OK) return s;
  if (a.rotary.kind != kNone && !positions) return fail(GW_INVALID_ARGUMENT, what + " requires positions");
  if (!(epsilon >= 0.F)) return fail(GW_INVALID_ARGUMENT, what + " requires an epsilon of 0 or more");
  a.rows = rows;
  a.width = head_dim;
  a.positions = positions;
  a.epsilon = epsilon;
  GW_CUDA_CHECK(launch_norm_rotary(a, as_stream(stream)), what);
  return GW_OK;
}

gw_status gw_kv_cache_append(const gw_kv_cache* cache, const gw_sequences* batch, const gw_head_rows* key,
                             const gw_head_rows* value, const gw_head_rows* query, const int32_t* positions,
                             const gw_rotary* rotary, float epsilon, void* stream) {
  clear_error();
  const std::string what = "cache append";
  if (gw_status s = check_cache(cache, "cache append"); s != GW_OK) return s;
  if (gw_status s = check_batch(batch, "cache append"); s != GW_OK) return s;
  if (batch->rows == 0 || batch->sequences == 0) return GW_OK;
  const uint32_t width = cache->head_dim;
  if (gw_status s = check_heads(key, false, width, what); s != GW_OK) return s;
  if (gw_status s = check_heads(value, false, width, what); s != GW_OK) return s;
  if (key->heads != cache->kv_heads || value->heads != cache->kv_heads)
    return fail(GW_INVALID_ARGUMENT, what + " requires keys and values of the cache's heads");
  Append a{};
  if (gw_status s = check_rotary(rotary, width, what, &a.rotary); s != GW_OK) return s;
  if (!(epsilon >= 0.F)) return fail(GW_INVALID_ARGUMENT, what + " requires an epsilon of 0 or more");
  NormRotary q{};
  if (query) {
    if (gw_status s = check_heads(query, true, width, what); s != GW_OK) return s;
    q.query = heads_of(*query);
    q.rows = batch->rows;
    q.width = width;
    q.positions = positions;
    q.batch = *batch;
    q.rotary = a.rotary;
    q.epsilon = epsilon;
  }
  a.cache = *cache;
  a.batch = *batch;
  a.batch.page_table_entries = page_entries(*batch);
  a.key = heads_of(*key);
  a.value = heads_of(*value);
  a.positions = positions;
  a.epsilon = epsilon;
  const cudaStream_t s = as_stream(stream);
  g_append_ran[current_device_slot()] = true;
  if (query) GW_CUDA_CHECK(launch_norm_rotary(q, s), "cache append (queries)");
  const bool whole = a.rotary.kind == kWhole;
  const auto launch = width == 128   ? (whole ? &launch_append<16, 1, true> : &launch_append<16, 1, false>)
                      : width == 256 ? (whole ? &launch_append<32, 1, true> : &launch_append<32, 1, false>)
                                     : (whole ? &launch_append<32, 2, true> : &launch_append<32, 2, false>);
  GW_CUDA_CHECK(launch(a, s), what);
  return GW_OK;
}

}  // extern "C"
