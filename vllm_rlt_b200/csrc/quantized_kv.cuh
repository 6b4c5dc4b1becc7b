// A paged key/value cache in 8 bits: codes in e4m3, a scale for each page and head, value = code * scale.  What the kernels that fill it
// and read it share: its argument block, its conversions and the rows of a packed step.
//
// Scales that the store kernel writes are powers of two, so that x / scale and a change of scale are exact in fp32 and every code is
// rounded once.  Readers take a key's scale as it is, and a value's inside the range of those (value_scale_of).
#pragma once

#include <cuda_fp8.h>
#include <math.h>

#include "common.cuh"

namespace rlt {

constexpr int kMinScaleExponent = -100, kMaxScaleExponent = 100;
constexpr float kLargestCode = 448.0f;
// A context is split at fixed positions, whatever the batch: a row's bits are its own.  1024 tokens at first, so that a few ordinary contexts make
// enough parts for all SMs; 2048 from 4096 on, where a part's costs (references found anew, its sums written and joined) weigh more.
constexpr int kShortPart = 1024, kShortParts = 4, kLongPart = 2048;
// A window of up to kWholeWindow keys is one part wherever it lies: its rows need no joining, and an item's ends are paid once for it.  Split / whole,
// us: 96 requests of three rows, 1000 keys, 64-wide heads 75.6 / 61.7; 16 of one row, 1000 keys, 8 heads of 128 21 / 15; one request, 1800 keys 16.5 / 16.7.
constexpr int kWholeWindow = 1900;
__host__ __device__ __forceinline__ bool whole_window(int window) { return window > 0 && window <= kWholeWindow; }
__host__ __device__ __forceinline__ int part_of(int token, int window) {
  if (whole_window(window)) return 0;
  return token < kShortParts * kShortPart ? token / kShortPart : kShortParts + (token - kShortParts * kShortPart) / kLongPart;
}
__host__ __device__ __forceinline__ int part_begin(int part, int window) {
  if (whole_window(window)) return part > 0 ? 0x7fffffff : 0;
  return part <= kShortParts ? part * kShortPart : kShortParts * kShortPart + (part - kShortParts) * kLongPart;
}

struct QuantizedCache {
  uint8_t* key;
  uint8_t* value;
  float* key_scale;             // [pages][kv_heads], row stride scale_stride
  float* value_scale;
  int64_t block_stride;         // bytes between pages of this layer's view
  int64_t token_stride;
  int64_t scale_stride;
  int64_t num_pages;
  int block;
  int kv_heads;
  int dim;
};

// A step's rows: rows cu[s] .. cu[s + 1] - 1 belong to sequence s and stand at its last positions, row i of n_s at lengths[s] - n_s + i.
struct PackedRows {
  const int32_t* tables;        // [sequences, width]
  const int32_t* lengths;       // [sequences], tokens with the step's
  const int32_t* cu;            // [sequences + 1]
  int sequences;
  int width;
  int total;                    // rows of the step
  int row0, rows;               // of which a launch does rows row0 .. rows - 1
  const int32_t* only = nullptr;        // [sequences + 1]: where 0 the sequence has no rows, the last one 0: none has; nullptr: all have theirs
  const uint32_t* gave_up = nullptr;    // of the kernel that scored the others: where not 0 a wait of it ran out, and all sequences have their rows again
};

struct QuantizedAttentionArgs {
  QuantizedCache cache;
  PackedRows step;
  const void* q;
  void* out;
  int64_t q_stride;             // elements between rows
  int64_t out_stride;
  int q_heads;
  int dtype;
  float scale;                  // multiplies q . k
  int window;                   // 0: all keys before a row
  float* partials;              // [row][query head][parts][partial_stride]: O, then its reference exponent M and sum l
  int parts;                    // parts that a row's keys can span
};

// Floats of one partial: O (dim, rounded up to whole float4), M, l, two unused.
__host__ __device__ inline int partial_stride(int dim) { return (dim + 3) / 4 * 4 + 4; }

// Parts that a row's keys can span in a table of so many tokens, behind a window: w keys lie in at most ceil((w - 1) / part) + 1 parts of one size.
inline int parts_of(int64_t capacity, int window) {
  const int all = part_of(static_cast<int>(capacity) - 1, window) + 1;
  const int64_t seen = window > 0 ? (static_cast<int64_t>(window) + 2 * kShortPart - 2) / kShortPart : all;
  return static_cast<int>(seen < all ? seen : all);
}

__device__ __forceinline__ bool has_rows(const PackedRows& p, int s) { return p.only == nullptr || (static_cast<uint32_t>(p.only[s]) | *p.gave_up) != 0; }

// The rows of sequence s that a launch does, kept inside the step's, and the sequence's length with the last of them.
__device__ __forceinline__ void rows_of(const PackedRows& p, int s, int* first, int* count, int* length) {
  const int begin = min(max(p.cu[s], 0), p.total), end = min(max(p.cu[s + 1], begin), p.total), last = min(end, p.rows);
  *first = max(begin, p.row0);
  *count = has_rows(p, s) ? max(last - *first, 0) : 0;
  const int64_t tokens = static_cast<int64_t>(p.lengths[s]) - (end - last);
  *length = static_cast<int>(tokens < -0x7fffffff ? -0x7fffffff : tokens);
}

// The sequence of a row: the last one that starts at or before it (a row behind the last sequence is in none of them).
__device__ __forceinline__ int sequence_at(const int32_t* cu, int sequences, int row) {
  int lo = 0, hi = sequences;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= row) lo = mid; else hi = mid;
  }
  return lo;
}

// Tokens that a row of the tables can address; the host keeps the product within 32 bits.
__device__ __forceinline__ int table_tokens(const PackedRows& p, int block) { return p.width * block; }

// Keys that a row sees: positions low .. keys - 1.  A length that its table cannot address is cut to what it can.
__device__ __forceinline__ void keys_of(const PackedRows& p, int block, int window, int length, int first, int count, int row, int* low, int* keys) {
  const int64_t seen = static_cast<int64_t>(length) - count + (row - first) + 1;
  *keys = static_cast<int>(seen < 0 ? 0 : (seen < table_tokens(p, block) ? seen : table_tokens(p, block)));
  *low = window > 0 ? max(*keys - window, 0) : 0;
}

__device__ __forceinline__ float2 decode_pair(uint16_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(codes, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ float decode_one(uint8_t code) {
  const __half_raw h = __nv_cvt_fp8_to_halfraw(code, __NV_E4M3);
  return __half2float(*reinterpret_cast<const __half*>(&h));
}
// Nearest even, beyond the largest code the largest code; NaN stays NaN.
__device__ __forceinline__ uint16_t encode_pair(float2 x) { return __nv_cvt_float2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ uint8_t encode_one(float x) { return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3); }

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

// The smallest e with largest <= 448 * 2^e, inside the exponents that a scale may have: 448 = 1.75 * 2^8, so the exponent of `largest` less
// eight, and one more when its significand is above 1.75.
__device__ __forceinline__ int scale_exponent(float largest) {
  if (!(largest > 0.0f)) return kMinScaleExponent;
  const int bits = __float_as_int(largest), e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return min(max(e, kMinScaleExponent), kMaxScaleExponent);
}

// The smallest power of two that is not below a scale, as its exponent.
__device__ __forceinline__ int exponent_above(float scale) {
  if (!(scale > 0.0f)) return kMinScaleExponent;
  const int bits = __float_as_int(scale), e = (bits >> 23) - 127 + ((bits & 0x7fffff) != 0 ? 1 : 0);
  return min(max(e, kMinScaleExponent), kMaxScaleExponent);
}

// The scale of values that every reader goes by: zero, or 2^-100 .. 2^100 (one beyond an end counts as that end, which keeps weight / scale and its
// sums over a context within fp32); what is negative or NaN is no size, and NaN.
__device__ __forceinline__ float value_scale_of(float scale) {
  if (scale == 0.0f) return 0.0f;
  return scale > 0.0f ? fminf(fmaxf(scale, power_of_two(kMinScaleExponent)), power_of_two(kMaxScaleExponent)) : NAN;
}

inline bool quantized_cache_valid(const QuantizedCache& c) {
  return c.num_pages >= 0 && c.block > 0 && c.kv_heads > 0 && c.dim > 0 && c.dim <= 256 &&
         c.token_stride >= static_cast<int64_t>(c.kv_heads) * c.dim && c.block_stride >= c.token_stride * c.block && c.scale_stride >= c.kv_heads;
}

// quantized_attention_sm100.cu: 64- and 128-wide heads, fp16 / bf16 queries, pages of whole 16-token tiles.
bool quantized_tiles_supported(const QuantizedAttentionArgs& a);
int launch_quantized_tiles(const QuantizedAttentionArgs& a, int max_new, cudaStream_t stream);

}  // namespace rlt
