// Attention over an 8-bit paged cache: the kernel for every shape, the joining of parts, and the expansion of pages that long portions
// attend over with the 16-bit prompt kernels.
//
//   s_t = scale * q . (key_scale[page] * key_code[t]),   p = softmax over the keys a row sees,   out = sum_t p_t * value_scale[page] * value_code[t]
//
// Contexts are split at fixed positions.  A part leaves O = sum 2^(s_t - M) v_t, M and l = sum 2^(s_t - M) in fp32 (s in log2
// units); rows whose keys lie in one part are finished by the kernel that scored them, the others by the merge.
#include "attention.cuh"
#include "quantized_kv.cuh"

namespace rlt {
namespace {

constexpr int kWarps = 4;
constexpr float kToLog2 = 1.4426950408889634f;

// ---- any shape: one CTA per (row, query head, part) ---------------------------------------------------
// A lane scores a key of its own (32 at a time: five shuffles per 32 keys instead of per key), then the warp adds up the 32 values with its
// lanes across the head.  kDims: elements of a head per lane.  In fp32 throughout: this is the kernel of 32-bit queries, and of head sizes,
// page sizes and layouts that the tiles do not take.
template <typename T, int kDims>
__global__ void __launch_bounds__(kWarps * 32)
quantized_rows_kernel(QuantizedAttentionArgs a) {
  __shared__ float s_q[kDims * 32];
  __shared__ float s_o[kWarps][kDims * 32];
  __shared__ float s_m[kWarps], s_l[kWarps];
  const QuantizedCache& c = a.cache;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = static_cast<int>(blockIdx.x % a.parts);
  const int64_t pair = blockIdx.x / a.parts;
  const int row = static_cast<int>(pair / a.q_heads), head = static_cast<int>(pair % a.q_heads), kv_head = head / (a.q_heads / c.kv_heads);
  const int s = sequence_at(a.step.cu, a.step.sequences, row);
  int first, count, low, keys;
  rows_of(a.step, s, &first, &count);
  if (row < first || row >= first + count) return;                    // in no sequence: left as it was
  keys_of(a.step, c.block, a.window, s, first, count, row, &low, &keys);
  const int first_part = part_of(low), last_part = keys > 0 ? part_of(keys - 1) : first_part;
  if (first_part + part > last_part) return;
  const int begin = max(low, part_begin(first_part + part)), end = min(keys, part_begin(first_part + part + 1));

  const T* q = static_cast<const T*>(a.q) + row * a.q_stride + static_cast<int64_t>(head) * c.dim;
  for (int d = threadIdx.x; d < kDims * 32; d += kWarps * 32) s_q[d] = d < c.dim ? Elem<T>::to_float(q[d]) * (a.scale * kToLog2) : 0.0f;
  __syncthreads();
  const int32_t* table = a.step.tables + static_cast<int64_t>(s) * a.step.width;
  float m = -INFINITY, l = 0.0f, o[kDims];
#pragma unroll
  for (int j = 0; j < kDims; ++j) o[j] = 0.0f;
  for (int base = begin + warp * 32; base < end; base += kWarps * 32) {
    const int token = base + lane;
    float score = -INFINITY, value_scale = 0.0f;
    const uint8_t* value = nullptr;
    if (token < end) {
      const int entry = token / c.block;
      const int64_t page = table[entry];
      score = 0.0f;                                                   // a page that does not exist holds zeros
      if (page >= 0 && page < c.num_pages) {
        const int64_t at = page * c.block_stride + (token - entry * c.block) * c.token_stride + static_cast<int64_t>(kv_head) * c.dim;
        const uint8_t* key = c.key + at;
        value = c.value + at;
        value_scale = c.value_scale[page * c.scale_stride + kv_head];
        for (int d = 0; d < c.dim; ++d) score = fmaf(decode_one(key[d]), s_q[d], score);
        score *= c.key_scale[page * c.scale_stride + kv_head];
      }
    }
    float top = score;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float next = fmaxf(m, top), zero = next == -INFINITY ? 0.0f : next, keep = exp2f(m - zero);
    const float p = exp2f(score - zero);
    m = next;
    l = fmaf(l, keep, p);                                             // a lane's own share of the sum
#pragma unroll
    for (int j = 0; j < kDims; ++j) o[j] *= keep;
    const float weight = p * value_scale;
    for (int i = 0; i < 32 && base + i < end; ++i) {
      const float w = __shfl_sync(0xffffffffu, weight, i);
      const uint8_t* v = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(value), i));
      if (v == nullptr) continue;
#pragma unroll
      for (int j = 0; j < kDims; ++j)
        if (lane + 32 * j < c.dim) o[j] = fmaf(w, decode_one(v[lane + 32 * j]), o[j]);
    }
  }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
#pragma unroll
  for (int j = 0; j < kDims; ++j) s_o[warp][lane + 32 * j] = o[j];
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
  __syncthreads();
  float big = -INFINITY;
  for (int w = 0; w < kWarps; ++w) big = fmaxf(big, s_m[w]);
  const float zero = big == -INFINITY ? 0.0f : big;
  float total = 0.0f;
  for (int w = 0; w < kWarps; ++w) total = fmaf(s_l[w], exp2f(s_m[w] - zero), total);
  const bool whole = first_part == last_part;
  float* partial = whole ? nullptr : a.partials + (pair * a.parts + part) * partial_stride(c.dim);
  T* out = static_cast<T*>(a.out) + row * a.out_stride + static_cast<int64_t>(head) * c.dim;
  for (int d = threadIdx.x; d < c.dim; d += kWarps * 32) {
    float x = 0.0f;
    for (int w = 0; w < kWarps; ++w) x = fmaf(s_o[w][d], exp2f(s_m[w] - zero), x);
    if (whole) out[d] = Elem<T>::from_float(keys > low ? x / total : 0.0f);
    else partial[d] = x;
  }
  if (!whole && threadIdx.x == 0) {
    float* end_of = partial + partial_stride(c.dim) - 4;
    end_of[0] = big;
    end_of[1] = total;
  }
}

// ---- joining parts -----------------------------------------------------------------------------------
// out = sum_c O_c 2^(M_c - M) / sum_c l_c 2^(M_c - M), M the largest M_c.  One warp per (row, query head), parts in order; eight parts'
// loads are in flight together.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
quantized_merge_kernel(QuantizedAttentionArgs a) {
  grid_dependency_wait();
  const QuantizedCache& c = a.cache;
  const int lane = threadIdx.x & 31;
  const int64_t pair = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (pair >= static_cast<int64_t>(a.step.rows) * a.q_heads) return;
  const int row = static_cast<int>(pair / a.q_heads);
  const int s = sequence_at(a.step.cu, a.step.sequences, row);
  int first, count, low, keys;
  rows_of(a.step, s, &first, &count);
  if (row < first || row >= first + count) return;
  keys_of(a.step, c.block, a.window, s, first, count, row, &low, &keys);
  const int parts = keys > 0 ? part_of(keys - 1) - part_of(low) + 1 : 1;
  if (parts < 2) return;
  const int stride = partial_stride(c.dim), quads = (stride - 4) / 4;
  const float* part = a.partials + pair * a.parts * stride;
  float big = -INFINITY, total = 0.0f;
  float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
  for (int c0 = 0; c0 < parts; c0 += 8) {
    float2 ml[8];
    float4 o[8][2];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float* p = part + static_cast<int64_t>(min(c0 + i, parts - 1)) * stride;
      ml[i] = *reinterpret_cast<const float2*>(p + stride - 4);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (lane + 32 * j < quads) o[i][j] = reinterpret_cast<const float4*>(p)[lane + 32 * j];
    }
    float next = big;
#pragma unroll
    for (int i = 0; i < 8; ++i) next = fmaxf(next, ml[i].x);          // the last part's again behind the end
    // l goes by 2^x in two steps: between parts whose values differ by far in size the factor may be 0 in fp32 where l times it is not
    const float zero = next == -INFINITY ? 0.0f : next, root = exp2f(0.5f * (big - zero)), keep = root * root;
    big = next;
    total = total * root * root;
#pragma unroll
    for (int j = 0; j < 2; ++j) { acc[j].x *= keep; acc[j].y *= keep; acc[j].z *= keep; acc[j].w *= keep; }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (c0 + i >= parts) break;
      const float half = exp2f(0.5f * (ml[i].x - zero)), f = half * half;
      total += ml[i].y * half * half;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (lane + 32 * j < quads) {
          acc[j].x = fmaf(o[i][j].x, f, acc[j].x); acc[j].y = fmaf(o[i][j].y, f, acc[j].y);
          acc[j].z = fmaf(o[i][j].z, f, acc[j].z); acc[j].w = fmaf(o[i][j].w, f, acc[j].w);
        }
      }
    }
  }
  T* out = static_cast<T*>(a.out) + row * a.out_stride + (pair - static_cast<int64_t>(row) * a.q_heads) * c.dim;
  const float inverse = 1.0f / total;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int d = 4 * (lane + 32 * j);
    if (d < c.dim) out[d] = Elem<T>::from_float(acc[j].x * inverse);
    if (d + 1 < c.dim) out[d + 1] = Elem<T>::from_float(acc[j].y * inverse);
    if (d + 2 < c.dim) out[d + 2] = Elem<T>::from_float(acc[j].z * inverse);
    if (d + 3 < c.dim) out[d + 3] = Elem<T>::from_float(acc[j].w * inverse);
  }
}

template <typename T>
int launch_rows(const QuantizedAttentionArgs& a, cudaStream_t stream) {
  const int64_t pairs = static_cast<int64_t>(a.step.rows) * a.q_heads;
  if (pairs * a.parts > 0x7fffffffll) {
    set_last_error_text("quantized_attention: too many rows, heads and parts of a context for one launch");
    return RLT_ERR_UNSUPPORTED;
  }
  const unsigned grid = static_cast<unsigned>(pairs * a.parts);
  if (a.cache.dim <= 64) quantized_rows_kernel<T, 2><<<grid, kWarps * 32, 0, stream>>>(a);
  else if (a.cache.dim <= 128) quantized_rows_kernel<T, 4><<<grid, kWarps * 32, 0, stream>>>(a);
  else quantized_rows_kernel<T, 8><<<grid, kWarps * 32, 0, stream>>>(a);
  return launch_status("quantized_rows_kernel");
}

template <typename T>
int launch_merge(const QuantizedAttentionArgs& a, cudaStream_t stream) {
  const int64_t pairs = static_cast<int64_t>(a.step.rows) * a.q_heads;
  return launch_dependent("quantized_merge_kernel", quantized_merge_kernel<T>, dim3(static_cast<unsigned>((pairs + kWarps - 1) / kWarps)), dim3(kWarps * 32), 0,
                          stream, a);
}

// ---- expansion ---------------------------------------------------------------------------------------
// The tokens of every sequence as 16-token pages of T, sequence s in pages s * width16 .., and the tables that say so.  Bound by its
// traffic: a byte read, two (four) written.
template <typename T, bool kWide>
__global__ void __launch_bounds__(256)
quantized_expand_kernel(QuantizedCache c, PackedRows step, T* key, T* value, int32_t* tables, int width16) {
  const int s = blockIdx.y;
  const int64_t length = step.lengths[s];
  const int tokens = static_cast<int>(length < 0 ? 0 : (length < table_tokens(step, c.block) ? length : table_tokens(step, c.block)));
  const int32_t* table = step.tables + static_cast<int64_t>(s) * step.width;
  constexpr int kVec = kWide ? 8 : 1;
  const int row = c.kv_heads * c.dim, per_row = row / kVec;
  for (int p = blockIdx.x; p * 16 < tokens; p += gridDim.x) {
    const int64_t to = static_cast<int64_t>(s) * width16 + p;
    if (threadIdx.x == 0) tables[to] = static_cast<int32_t>(to);
    const int here = min(tokens - p * 16, 16);
    for (int i = threadIdx.x; i < here * per_row; i += 256) {
      const int t = i / per_row, at = (i - t * per_row) * kVec, token = p * 16 + t, entry = token / c.block;
      const int64_t page = table[entry];
      const bool there = page >= 0 && page < c.num_pages;
      const int64_t from = there ? page * c.block_stride + (token - entry * c.block) * c.token_stride + at : 0;
      const int64_t scale_at = there ? page * c.scale_stride + at / c.dim : 0;
      const float ks = there ? c.key_scale[scale_at] : 0.0f, vs = there ? c.value_scale[scale_at] : 0.0f;
      const int64_t dst = (to * 16 + t) * row + at;
      if constexpr (kWide) {
        const uint2 kw = there ? *reinterpret_cast<const uint2*>(c.key + from) : make_uint2(0u, 0u);
        const uint2 vw = there ? *reinterpret_cast<const uint2*>(c.value + from) : make_uint2(0u, 0u);
        const uint32_t words[4] = {kw.x, kw.y, vw.x, vw.y};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          T x[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 pair = decode_pair(static_cast<uint16_t>(words[2 * h + (j >> 1)] >> (16 * (j & 1))));
            x[2 * j] = Elem<T>::from_float(pair.x * (h ? vs : ks));
            x[2 * j + 1] = Elem<T>::from_float(pair.y * (h ? vs : ks));
          }
          T* out = (h ? value : key) + dst;
#pragma unroll
          for (int j = 0; j < static_cast<int>(8 * sizeof(T) / 16); ++j) reinterpret_cast<uint4*>(out)[j] = reinterpret_cast<const uint4*>(x)[j];
        }
      } else {
        key[dst] = Elem<T>::from_float(there ? decode_one(c.key[from]) * ks : 0.0f);
        value[dst] = Elem<T>::from_float(there ? decode_one(c.value[from]) * vs : 0.0f);
      }
    }
  }
}

template <typename T>
int launch_expand(const QuantizedCache& c, const PackedRows& step, void* key, void* value, int32_t* tables, int width16, int sm_count, cudaStream_t stream) {
  const bool wide = c.dim % 8 == 0 && c.block_stride % 8 == 0 && c.token_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(c.key) & 7u) == 0 &&
                    (reinterpret_cast<uintptr_t>(c.value) & 7u) == 0 && aligned16(key) && aligned16(value);
  const int across = 8 * sm_count / step.sequences + 1;
  const dim3 grid(static_cast<unsigned>(width16 < across ? width16 : across), static_cast<unsigned>(step.sequences));
  if (wide) quantized_expand_kernel<T, true><<<grid, 256, 0, stream>>>(c, step, static_cast<T*>(key), static_cast<T*>(value), tables, width16);
  else quantized_expand_kernel<T, false><<<grid, 256, 0, stream>>>(c, step, static_cast<T*>(key), static_cast<T*>(value), tables, width16);
  return launch_status("quantized_expand_kernel");
}

int read_args(QuantizedAttentionArgs& a, const void* key_cache, const void* value_cache, const float* key_scale, const float* value_scale,
              int64_t block_stride, int64_t token_stride, int64_t scale_stride, int64_t num_blocks, int block_size, int kv_heads, int head_dim, int dtype,
              const int32_t* block_tables, const int32_t* lengths, const int32_t* cu_rows, int sequences, int table_width, int rows) {
  QuantizedCache& c = a.cache;
  c.key = static_cast<uint8_t*>(const_cast<void*>(key_cache)); c.value = static_cast<uint8_t*>(const_cast<void*>(value_cache));
  c.key_scale = const_cast<float*>(key_scale); c.value_scale = const_cast<float*>(value_scale);
  c.block_stride = block_stride; c.token_stride = token_stride; c.scale_stride = scale_stride; c.num_pages = num_blocks; c.block = block_size;
  c.kv_heads = kv_heads; c.dim = head_dim;
  a.dtype = dtype;
  a.step.tables = block_tables; a.step.lengths = lengths; a.step.cu = cu_rows; a.step.sequences = sequences; a.step.width = table_width; a.step.rows = rows;
  RLT_REQUIRE(dtype_valid(dtype), "quantized_attention: dtype must be float32, float16 or bfloat16");
  RLT_REQUIRE(quantized_cache_valid(c), "quantized_attention: cache must be [pages, block, kv_heads, dim <= 256] with a contiguous [kv_heads, dim] tail");
  RLT_REQUIRE(sequences >= 0 && rows >= 0 && table_width >= 0, "quantized_attention: invalid shape");
  RLT_REQUIRE(static_cast<int64_t>(table_width) * block_size <= (1 << 26), "quantized_attention: tables of more than 2^26 tokens");
  RLT_REQUIRE(rows == 0 || sequences == 0 || (block_tables && lengths && cu_rows), "quantized_attention: null pointer");
  return RLT_OK;
}

}  // namespace
}  // namespace rlt

extern "C" RLT_API size_t rlt_quantized_attention_workspace_bytes(int rows, int q_heads, int head_dim, int block_size, int table_width, int window) {
  using namespace rlt;
  if (rows <= 0 || q_heads <= 0 || head_dim <= 0 || block_size <= 0 || table_width <= 0) return 0;
  const int parts = parts_of(static_cast<int64_t>(table_width) * block_size, window);
  return parts < 2 ? 0 : sizeof(float) * static_cast<size_t>(rows) * q_heads * parts * partial_stride(head_dim);
}

extern "C" RLT_API int rlt_quantized_attention(const void* q, int64_t q_stride, void* out, int64_t out_stride, const void* key_cache,
                                               const void* value_cache, const float* key_scale, const float* value_scale, int64_t block_stride,
                                               int64_t token_stride, int64_t scale_stride, int64_t num_blocks, int block_size, int q_heads,
                                               int kv_heads, int head_dim, int dtype, const int32_t* block_tables, const int32_t* lengths,
                                               const int32_t* cu_rows, int sequences, int table_width, int rows, int max_new, float scale, int window,
                                               void* workspace, size_t workspace_bytes, rlt_stream_t stream) {
  using namespace rlt;
  QuantizedAttentionArgs a = {};
  int status = read_args(a, key_cache, value_cache, key_scale, value_scale, block_stride, token_stride, scale_stride, num_blocks, block_size, kv_heads,
                         head_dim, dtype, block_tables, lengths, cu_rows, sequences, table_width, rows);
  if (status != RLT_OK) return status;
  RLT_REQUIRE(q_heads > 0 && q_heads % kv_heads == 0, "quantized_attention: query heads must be a positive multiple of KV heads");
  RLT_REQUIRE(window >= 0 && max_new >= 0, "quantized_attention: window and max_new must not be negative");
  if (rows == 0 || sequences == 0) return RLT_OK;
  const int64_t width = static_cast<int64_t>(q_heads) * head_dim;
  RLT_REQUIRE(q && out && key_cache && value_cache && key_scale && value_scale && table_width > 0, "quantized_attention: null pointer or empty tables");
  RLT_REQUIRE(q_stride >= width && out_stride >= width, "quantized_attention: row strides smaller than a row");
  a.q = q; a.q_stride = q_stride; a.out = out; a.out_stride = out_stride; a.q_heads = q_heads; a.scale = scale; a.window = window;
  a.parts = parts_of(static_cast<int64_t>(table_width) * block_size, window);
  a.partials = static_cast<float*>(workspace);
  if (workspace_bytes < rlt_quantized_attention_workspace_bytes(rows, q_heads, head_dim, block_size, table_width, window) ||
      (a.parts > 1 && (workspace == nullptr || !aligned16(workspace)))) {
    set_last_error_text("quantized_attention: workspace missing, misaligned or too small");
    return RLT_ERR_WORKSPACE;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  status = quantized_tiles_supported(a) ? launch_quantized_tiles(a, max_new, s) : RLT_ERR_UNSUPPORTED;
  if (status == RLT_ERR_UNSUPPORTED) RLT_DISPATCH_DTYPE(dtype, T, status = launch_rows<T>(a, s));
  if (status != RLT_OK || a.parts < 2) return status;
  RLT_DISPATCH_DTYPE(dtype, T, return launch_merge<T>(a, s));
}

extern "C" RLT_API int rlt_quantized_kv_expand(const void* key_cache, const void* value_cache, const float* key_scale, const float* value_scale,
                                               int64_t block_stride, int64_t token_stride, int64_t scale_stride, int64_t num_blocks, int block_size,
                                               int kv_heads, int head_dim, const int32_t* block_tables, const int32_t* lengths, int sequences,
                                               int table_width, void* key_pages, void* value_pages, int32_t* page_tables, int pages_width, int dtype,
                                               rlt_stream_t stream) {
  using namespace rlt;
  QuantizedAttentionArgs a = {};
  int status = read_args(a, key_cache, value_cache, key_scale, value_scale, block_stride, token_stride, scale_stride, num_blocks, block_size, kv_heads,
                         head_dim, dtype, block_tables, lengths, lengths, sequences, table_width, 1);
  if (status != RLT_OK || sequences == 0 || table_width == 0) return status;
  RLT_REQUIRE(key_cache && value_cache && key_scale && value_scale && key_pages && value_pages && page_tables, "quantized_kv_expand: null pointer");
  RLT_REQUIRE(static_cast<int64_t>(pages_width) * 16 >= static_cast<int64_t>(table_width) * block_size &&
                  static_cast<int64_t>(pages_width) * sequences <= 0x7fffffff, "quantized_kv_expand: page tables too narrow, or too many pages");
  RLT_REQUIRE(sequences <= 65535, "quantized_kv_expand: at most 65535 sequences");
  DeviceInfo info;
  status = current_device_info(&info);
  if (status != RLT_OK) return status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  RLT_DISPATCH_DTYPE(dtype, T, return launch_expand<T>(a.cache, a.step, key_pages, value_pages, page_tables, pages_width, info.sm_count, s));
}
