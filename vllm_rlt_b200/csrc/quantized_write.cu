// New keys and values into an 8-bit paged cache.
//
// For a page that gets rows, per head, K and V apart:
//   a = max |x| over the new rows' finite elements,   e = the smallest exponent with a <= 448 * 2^e
//   scale = 2^e for a page that starts with these rows (one stands at offset 0), else max(2^e, the old scale rounded up to a power of two)
//   code = e4m3(x / scale) to nearest even; what is not finite becomes NaN
// When the scale grows, the tokens in front of the new rows are rounded again at the new one: with powers of two that moves their exponents,
// and only codes below 2^-14 of the largest are rounded a second time.
//
// A run is what one sequence writes to one page in a call; a warp takes a run of one head, so the maximum is one warp's reduction and
// nothing is shared between warps.  Runs are found by their first rows: a CTA looks at kWindow rows, and does the keys or the values.
//
// Bound by its traffic for prompts: 16 of 128 to 1024 rows, 16 heads of 128 in bf16, 105 MB, take 27.8 us (3.8 TB/s; 34.5 with keys and values in
// one CTA, 60 when every run was read twice with one load in flight).  What is left is the start (the rows' sequences, their tables: four dependent
// reads) and the tail of two waves of CTAs (1070 of them, four an SM).  One row of each of 128 requests, 8 heads: 4.6 us, a launch and those reads.
#include <type_traits>

#include "quantized_kv.cuh"

namespace rlt {
namespace {

constexpr int kThreads = 256;
constexpr int kHeld = 8;                // pieces of a run that a lane keeps in registers
constexpr int kStaged = 2048;           // sequence bounds kept in shared memory

struct Run {
  int row;          // its first row
  int count;
  int offset;       // of the first row in the page
  int64_t page;
};

// kVec elements as they are stored.
template <typename T, int kVec>
struct Piece {
  static constexpr int kWords = kVec == 1 ? 1 : kVec * static_cast<int>(sizeof(T)) / 4;
  static constexpr bool kPairs = sizeof(T) == 2;
  // |x| as an unsigned number grows with |x|; from here on it is infinite or NaN
  static constexpr uint32_t kNotFinite = sizeof(T) == 4 ? 0x7f800000u : (std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u);
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kVec == 1) {
      if constexpr (kPairs) w[0] = *reinterpret_cast<const uint16_t*>(p);
      else w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) {
        const uint4 a = reinterpret_cast<const uint4*>(p)[i];
        w[4 * i] = a.x; w[4 * i + 1] = a.y; w[4 * i + 2] = a.z; w[4 * i + 3] = a.w;
      }
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  // the largest of `top` and the |x|, for 16-bit types in two halves
  __device__ __forceinline__ uint32_t fold(uint32_t top) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) top = kPairs ? __vmaxu2(top, w[i] & 0x7fff7fffu) : max(top, w[i] & 0x7fffffffu);
    return top;
  }
  __device__ __forceinline__ float at(int i) const {
    T x;
    if constexpr (kPairs) {
      const uint16_t half = static_cast<uint16_t>(w[i >> 1] >> (16 * (i & 1)));
      x = *reinterpret_cast<const T*>(&half);
    } else {
      x = *reinterpret_cast<const T*>(&w[i]);
    }
    return Elem<T>::to_float(x);
  }
};

template <typename T>
__device__ __forceinline__ float of_bits(uint32_t bits) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(bits);
  const uint16_t half = static_cast<uint16_t>(bits);
  return Elem<T>::to_float(*reinterpret_cast<const T*>(&half));
}

template <int kVec>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&x)[kVec]) {
  if constexpr (kVec == 1) {
    *p = encode_one(x[0]);
  } else {
    uint2 w;
    w.x = encode_pair(make_float2(x[0], x[1])) | static_cast<uint32_t>(encode_pair(make_float2(x[2], x[3]))) << 16;
    w.y = encode_pair(make_float2(x[4], x[5])) | static_cast<uint32_t>(encode_pair(make_float2(x[6], x[7]))) << 16;
    *reinterpret_cast<uint2*>(p) = w;
  }
}

template <int kVec>
__device__ __forceinline__ void rescale_codes(uint8_t* p, float ratio) {
  float x[kVec];
  if constexpr (kVec == 1) {
    x[0] = decode_one(*p) * ratio;
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    const uint32_t words[2] = {w.x, w.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 pair = decode_pair(static_cast<uint16_t>(words[i >> 1] >> (16 * (i & 1))));
      x[2 * i] = pair.x * ratio;
      x[2 * i + 1] = pair.y * ratio;
    }
  }
  store_codes<kVec>(p, x);
}

template <typename T, int kVec, int kWindow>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 4 : 2)
quantized_write_kernel(QuantizedCache c, PackedRows step, const T* __restrict__ k, int64_t k_stride, const T* __restrict__ v, int64_t v_stride) {
  __shared__ int32_t s_cu[kStaged + 1];
  __shared__ Run s_runs[kWindow];
  __shared__ int s_count;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool staged = step.sequences <= kStaged;
  if (threadIdx.x == 0) s_count = 0;
  for (int i = threadIdx.x; staged && i <= step.sequences; i += kThreads) s_cu[i] = step.cu[i];
  __syncthreads();
  const int row = blockIdx.x * kWindow + threadIdx.x;
  if (threadIdx.x < kWindow && row < step.rows) {
    const int s = sequence_at(staged ? s_cu : step.cu, step.sequences, row);
    int first, count, length;
    rows_of(step, s, &first, &count, &length);
    const int64_t position = static_cast<int64_t>(length) - count + (row - first);
    if (row >= first && row < first + count && position >= 0 && position < table_tokens(step, c.block)) {
      const int entry = static_cast<int>(position) / c.block, offset = static_cast<int>(position) - entry * c.block;
      if (row == first || offset == 0) {
        const int64_t page = step.tables[static_cast<int64_t>(s) * step.width + entry];
        if (page >= 0 && page < c.num_pages) {
          Run run;
          run.row = row; run.count = min(first + count - row, c.block - offset); run.offset = offset; run.page = page;
          s_runs[atomicAdd(&s_count, 1)] = run;          // in any order: runs share nothing
        }
      }
    }
  }
  __syncthreads();
  const int per_row = c.dim / kVec, tasks = s_count * c.kv_heads;
  for (int task = warp; task < tasks; task += kThreads / 32) {
    const Run run = s_runs[task / c.kv_heads];
    const int head = task % c.kv_heads;
    const bool value = blockIdx.y;
    const T* src = (value ? v : k) + run.row * (value ? v_stride : k_stride) + static_cast<int64_t>(head) * c.dim;
    const int64_t src_stride = value ? v_stride : k_stride;
    uint8_t* page = (value ? c.value : c.key) + run.page * c.block_stride + static_cast<int64_t>(head) * c.dim;
    float* scale_at = (value ? c.value_scale : c.key_scale) + run.page * c.scale_stride + head;
    const float old = run.offset == 0 ? 0.0f : *scale_at;
    // The run in chunks of kHeld pieces a lane, all of a chunk's loads in flight together; the last chunk (of sixteen tokens with 128
    // elements there is one) stays in registers for the second pass.
    using P = Piece<T, kVec>;
    const int items = run.count * per_row, chunks = (items + 32 * kHeld - 1) / (32 * kHeld), step_rows = 32 / per_row, step_at = 32 % per_row;
    P x[kHeld];
    auto each = [&](int chunk, auto&& what) {              // what(j, token of the run, piece of the row) for the lane's pieces of a chunk
      int i = chunk * 32 * kHeld + lane, t = i / per_row, at = i - t * per_row;
#pragma unroll
      for (int j = 0; j < kHeld; ++j) {
        if (i < items) what(j, t, at);
        i += 32; t += step_rows; at += step_at;
        if (at >= per_row) { at -= per_row; ++t; }
      }
    };
    auto load = [&](int chunk) {
#pragma unroll
      for (int j = 0; j < kHeld; ++j) x[j].clear();
      each(chunk, [&](int j, int t, int at) { x[j].load(src + t * src_stride + at * kVec); });
    };
    uint32_t top = 0;
    for (int chunk = 0; chunk < chunks; ++chunk) {
      load(chunk);
#pragma unroll
      for (int j = 0; j < kHeld; ++j) top = x[j].fold(top);
    }
    if (P::kPairs) top = max(top & 0xffffu, top >> 16);
    top = __reduce_max_sync(0xffffffffu, top);
    const bool finite = top < P::kNotFinite;
    float largest = of_bits<T>(top);
    if (!finite) {                                         // rare: once more, for the finite ones
      largest = 0.0f;
      for (int chunk = 0; chunk < chunks; ++chunk) {
        load(chunk);
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
#pragma unroll
          for (int k = 0; k < kVec; ++k) {
            const float m = fabsf(x[j].at(k));
            if (m < INFINITY) largest = fmaxf(largest, m);
          }
        }
      }
      largest = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(largest)));
    }
    int e = scale_exponent(largest);
    if (run.offset != 0) e = max(e, exponent_above(old));
    const float scale = power_of_two(e), inverse = power_of_two(-e);
    if (run.offset != 0 && scale != old) {
      const float ratio = old * inverse;
      for (int i = lane; i < run.offset * per_row; i += 32) rescale_codes<kVec>(page + (i / per_row) * c.token_stride + (i % per_row) * kVec, ratio);
    }
    if (lane == 0 && (run.offset == 0 || scale != old)) *scale_at = scale;
    uint8_t* to = page + run.offset * c.token_stride;
    for (int chunk = chunks - 1; chunk >= 0; --chunk) {
      if (chunk < chunks - 1) load(chunk);
      each(chunk, [&](int j, int t, int at) {
        float y[kVec];
#pragma unroll
        for (int k = 0; k < kVec; ++k) y[k] = x[j].at(k) * inverse;
        if (!finite) {
#pragma unroll
          for (int k = 0; k < kVec; ++k) y[k] = fabsf(x[j].at(k)) < INFINITY ? y[k] : NAN;
        }
        store_codes<kVec>(to + t * c.token_stride + at * kVec, y);
      });
    }
  }
}

template <typename T>
int launch(const QuantizedCache& c, const PackedRows& step, const void* k, int64_t k_stride, const void* v, int64_t v_stride, cudaStream_t stream) {
  const size_t es = sizeof(T);
  const bool wide = c.dim % 8 == 0 && c.block_stride % 8 == 0 && c.token_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(c.key) & 7u) == 0 &&
                    (reinterpret_cast<uintptr_t>(c.value) & 7u) == 0 && aligned16(k) && aligned16(v) && k_stride * es % 16 == 0 && v_stride * es % 16 == 0;
  // Long portions have a run every `block` rows; short ones one for nearly every row.
  const bool many = step.rows >= 8 * static_cast<int64_t>(step.sequences);
  const T *kp = static_cast<const T*>(k), *vp = static_cast<const T*>(v);
  const unsigned grid = static_cast<unsigned>(many ? (step.rows + 15) / 16 : step.rows);
  if (wide && many) quantized_write_kernel<T, 8, 16><<<dim3(grid, 2), kThreads, 0, stream>>>(c, step, kp, k_stride, vp, v_stride);
  else if (wide) quantized_write_kernel<T, 8, 1><<<dim3(grid, 2), kThreads, 0, stream>>>(c, step, kp, k_stride, vp, v_stride);
  else if (many) quantized_write_kernel<T, 1, 16><<<dim3(grid, 2), kThreads, 0, stream>>>(c, step, kp, k_stride, vp, v_stride);
  else quantized_write_kernel<T, 1, 1><<<dim3(grid, 2), kThreads, 0, stream>>>(c, step, kp, k_stride, vp, v_stride);
  return launch_status("quantized_write_kernel");
}

}  // namespace
}  // namespace rlt

extern "C" RLT_API int rlt_quantized_kv_write(void* key_cache, void* value_cache, float* key_scale, float* value_scale, int64_t block_stride,
                                              int64_t token_stride, int64_t scale_stride, int64_t num_blocks, int block_size, int kv_heads,
                                              int head_dim, const void* k, int64_t k_stride, const void* v, int64_t v_stride, int dtype,
                                              const int32_t* block_tables, const int32_t* lengths, const int32_t* cu_rows, int sequences,
                                              int table_width, int rows, rlt_stream_t stream) {
  using namespace rlt;
  RLT_REQUIRE(dtype_valid(dtype), "quantized_kv_write: rows must be float32, float16 or bfloat16");
  QuantizedCache c;
  c.key = static_cast<uint8_t*>(key_cache); c.value = static_cast<uint8_t*>(value_cache); c.key_scale = key_scale; c.value_scale = value_scale;
  c.block_stride = block_stride; c.token_stride = token_stride; c.scale_stride = scale_stride; c.num_pages = num_blocks; c.block = block_size;
  c.kv_heads = kv_heads; c.dim = head_dim;
  RLT_REQUIRE(quantized_cache_valid(c), "quantized_kv_write: cache must be [pages, block, kv_heads, dim <= 256] with a contiguous [kv_heads, dim] tail");
  RLT_REQUIRE(sequences >= 0 && rows >= 0 && table_width >= 0, "quantized_kv_write: invalid shape");
  if (rows == 0 || sequences == 0 || table_width == 0 || num_blocks == 0) return RLT_OK;
  RLT_REQUIRE(key_cache && value_cache && key_scale && value_scale && k && v && block_tables && lengths && cu_rows, "quantized_kv_write: null pointer");
  RLT_REQUIRE(static_cast<int64_t>(table_width) * block_size <= 0x7fffffff, "quantized_kv_write: positions beyond 32 bits");
  const int64_t row = static_cast<int64_t>(kv_heads) * head_dim;
  RLT_REQUIRE(k_stride >= row && v_stride >= row, "quantized_kv_write: rows must be [rows, kv_heads, head_dim] with a contiguous tail");
  PackedRows step;
  step.tables = block_tables; step.lengths = lengths; step.cu = cu_rows; step.sequences = sequences; step.width = table_width;
  step.total = step.rows = rows; step.row0 = 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  RLT_DISPATCH_DTYPE(dtype, T, return launch<T>(c, step, k, k_stride, v, v_stride, s));
}
