// Attention over an 8-bit paged cache: the kernel for every shape, the joining of parts, and the expansion of pages for long portions.
//
//   s_t = scale * q . (key_scale[page] * key_code[t]),   p = softmax over the keys a row sees,   out = sum_t p_t * value_scale[page] * value_code[t]
//
// Contexts are split at fixed positions.  A part leaves O = sum 2^(s_t - M) v_t, M and l = sum 2^(s_t - M) in fp32 (s in log2
// units); rows whose keys lie in one part are finished by the kernel that scored them, the others by the merge.
#include <algorithm>

#include "attention.cuh"
#include "quantized_kv.cuh"

namespace rlt {
namespace {

constexpr int kWarps = 4;
constexpr float kToLog2 = 1.4426950408889634f;

// ---- any shape: one CTA per (row, query head, part) ---------------------------------------------------
// A lane scores a key of its own (32 at a time: five shuffles per 32 keys instead of per key), then the warp adds up the 32 values with its
// lanes across the head.  kDims: elements of a head per lane.  In fp32 throughout: this is the kernel of 32-bit queries, and of head sizes,
// page sizes and layouts that the tiles do not take.  Bound by its loads of single codes: 64 contexts of 512 to 4096 tokens, 16 rows of 16 heads
// each, take 10 ms here and 0.15 ms in the tiles.
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
  const int row = a.step.row0 + static_cast<int>(pair / a.q_heads), head = static_cast<int>(pair % a.q_heads), kv_head = head / (a.q_heads / c.kv_heads);
  const int s = sequence_at(a.step.cu, a.step.sequences, row);
  int first, count, length, low, keys;
  rows_of(a.step, s, &first, &count, &length);
  if (row < first || row >= first + count) return;                    // in no sequence: left as it was
  keys_of(a.step, c.block, a.window, length, first, count, row, &low, &keys);
  const int first_part = part_of(low, a.window), last_part = keys > 0 ? part_of(keys - 1, a.window) : first_part;
  if (first_part + part > last_part) return;
  const int begin = max(low, part_begin(first_part + part, a.window)), end = min(keys, part_begin(first_part + part + 1, a.window));

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
        value_scale = value_scale_of(c.value_scale[page * c.scale_stride + kv_head]);
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
// loads are in flight together.  Bound by latency: a search, the bounds and length it gives, the parts.  With a binary search instead of 32
// candidates at a time it took 6 us more behind 1024 rows of 64 sequences.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
quantized_merge_kernel(QuantizedAttentionArgs a) {
  grid_dependency_wait();
  if (!has_rows(a.step, a.step.sequences)) return;
  const QuantizedCache& c = a.cache;
  const int lane = threadIdx.x & 31;
  const int64_t pair = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  if (pair >= static_cast<int64_t>(a.step.rows - a.step.row0) * a.q_heads) return;
  const int at = static_cast<int>(pair / a.q_heads), row = a.step.row0 + at;
  // the row's sequence, 32 candidates at a time: what a warp waits for is dependent reads
  int s = 0, past = a.step.sequences;
  while (past - s > 1) {
    const int step = (past - s + 31) / 32, at = s + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, lane == 0 || (at < past && a.step.cu[at] <= row));
    s += (31 - __clz(below)) * step;
    past = min(s + step, past);
  }
  int first, count, length, low, keys;
  rows_of(a.step, s, &first, &count, &length);
  if (row < first || row >= first + count) return;
  keys_of(a.step, c.block, a.window, length, first, count, row, &low, &keys);
  const int parts = keys > 0 ? part_of(keys - 1, a.window) - part_of(low, a.window) + 1 : 1;
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
  T* out = static_cast<T*>(a.out) + row * a.out_stride + (pair - static_cast<int64_t>(at) * a.q_heads) * c.dim;
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
  const int64_t pairs = static_cast<int64_t>(a.step.rows - a.step.row0) * a.q_heads;
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
  const int64_t pairs = static_cast<int64_t>(a.step.rows - a.step.row0) * a.q_heads;
  return launch_dependent("quantized_merge_kernel", quantized_merge_kernel<T>, dim3(static_cast<unsigned>((pairs + kWarps - 1) / kWarps)), dim3(kWarps * 32), 0,
                          stream, a);
}

// ---- long portions -----------------------------------------------------------------------------------
// Tiles of at most sixteen rows read and convert a context once for each of them; a portion of hundreds of rows is bound by that, not by its
// products.  So its pages are expanded into bf16 once, which has room for every code times 2^-100 .. 2^100 without a rounding, and the
// prompt kernel of 16-bit caches scores them in tiles of 256 rows.  What that kernel would get wrong is left to the tiles of this one: a
// sequence with a value that is NaN (its weight of 0 in rows that do not see it would make them NaN), with a page scale that is no power of
// two (its values would be rounded), or with a length beyond its table (rows are cut one by one here) is marked, and scored behind it.  So is a
// sequence with a short portion beside long ones, and its pages stay as they are: a single token's context would be expanded for one row, and walked by
// one CTA a head.  With all of them expanded / with the long ones, us, 32 heads over 8 of 128: 1000 rows beside ten single tokens on 50000 keys each
// 2855 / 248, on 2000 keys 158 / 90; 4000 rows beside forty on 4000 962 / 407; 2000 rows beside ten on 16 keys 115 / 131.
//
// A CTA takes pages of 16 tokens of one sequence: sequence s in pages s * width16 .. of `key` and `value`, and the tables, lengths and row
// bounds that say so.  Bound by its traffic, a byte read and two written: 4 contexts of 5117 tokens, 8 heads of 128, 126 MB in 19.2 us (6.5 TB/s),
// before 78 us of the prompt kernel for 1021 rows of 16 heads each; the tiles took 431 us for all of it.
struct Expanded {
  __nv_bfloat16* key;
  __nv_bfloat16* value;
  int32_t* tables;              // [sequences, width16]
  int32_t* lengths;             // [sequences]
  int32_t* cu;                  // [sequences + 1]
  int32_t* marked;              // [sequences + 1], zero before; the last: some sequence is
  int width16;
  int least;                    // rows of a portion that is long
};

// Of four codes in a word: the top bit of each that is NaN (all seven bits under its sign are set).
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
__device__ __forceinline__ bool plain_scale(float scale) {
  const uint32_t bits = __float_as_uint(scale);
  return (bits & 0x807fffffu) == 0 && bits >= static_cast<uint32_t>(kMinScaleExponent + 127) << 23 && bits <= static_cast<uint32_t>(kMaxScaleExponent + 127) << 23;
}

__global__ void __launch_bounds__(256)
quantized_expand_kernel(QuantizedCache c, PackedRows step, Expanded x) {
  const int s = blockIdx.y, capacity = table_tokens(step, c.block);
  int first, count, length;
  rows_of(step, s, &first, &count, &length);
  const bool expands = count >= x.least;
  const int tokens = expands ? min(max(length, 0), capacity) : 0;       // (the prompt kernel gives a short portion's rows zeros, which do not stay)
  const int32_t* table = step.tables + static_cast<int64_t>(s) * step.width;
  bool marks = expands ? length > capacity : count > 0;
  if (blockIdx.x == 0) {
    // bounds inside the rows that never fall, whatever stands in cu: the prompt kernel's list of tiles has room for those
    __shared__ int s_most[8];
    int most = 0;
    for (int i = threadIdx.x; i <= s; i += 256) most = max(most, min(step.cu[i], step.total));
    most = static_cast<int>(__reduce_max_sync(0xffffffffu, static_cast<unsigned>(max(most, 0))));
    if ((threadIdx.x & 31) == 0) s_most[threadIdx.x >> 5] = most;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < 8; ++i) most = max(most, s_most[i]);
      x.cu[s] = most;
      x.lengths[s] = tokens;
      if (s == step.sequences - 1) x.cu[s + 1] = max(most, min(step.cu[s + 1], step.total));
    }
  }
  const int row = c.kv_heads * c.dim, per_row = row / 16;
  for (int p = blockIdx.x; p * 16 < tokens; p += gridDim.x) {
    const int64_t to = static_cast<int64_t>(s) * x.width16 + p;
    const int entry = p * 16 / c.block, place = p * 16 - entry * c.block, here = min(tokens - p * 16, 16);      // (pages are whole sixteens)
    const int64_t page = table[entry];
    const bool there = page >= 0 && page < c.num_pages;
    if (threadIdx.x == 0) x.tables[to] = static_cast<int32_t>(to);
    for (int i = threadIdx.x; i < here * per_row; i += 256) {
      const int t = i / per_row, at = (i - t * per_row) * 16;
      const int64_t from = there ? page * c.block_stride + (place + t) * c.token_stride + at : 0, dst = (to * 16 + t) * row + at;
      const int64_t scale_at = there ? page * c.scale_stride + at / c.dim : 0;
      const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
      const uint4 kw = there ? *reinterpret_cast<const uint4*>(c.key + from) : zero, vw = there ? *reinterpret_cast<const uint4*>(c.value + from) : zero;
      const float ks = there ? c.key_scale[scale_at] : 1.0f, vs = there ? c.value_scale[scale_at] : 1.0f;
      marks |= (nan_codes(vw.x) | nan_codes(vw.y) | nan_codes(vw.z) | nan_codes(vw.w)) != 0 || !plain_scale(ks) || !plain_scale(vs);
      const uint32_t words[8] = {kw.x, kw.y, kw.z, kw.w, vw.x, vw.y, vw.z, vw.w};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float scale = h ? vs : ks;
        uint32_t out[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 pair = decode_pair(static_cast<uint16_t>(words[4 * h + (j >> 1)] >> (16 * (j & 1))));
          const __nv_bfloat162 two = __floats2bfloat162_rn(pair.x * scale, pair.y * scale);
          out[j] = *reinterpret_cast<const uint32_t*>(&two);
        }
        uint4* to16 = reinterpret_cast<uint4*>((h ? x.value : x.key) + dst);
        to16[0] = make_uint4(out[0], out[1], out[2], out[3]);
        to16[1] = make_uint4(out[4], out[5], out[6], out[7]);
      }
    }
  }
  if (__syncthreads_or(marks) && threadIdx.x == 0) x.marked[s] = x.marked[step.sequences] = 1;
}

// Rows whose partials are written and joined at a time: tables are as wide as the longest context may become, so their room goes by that.
constexpr size_t kMostPartials = size_t{2} << 30;
size_t partial_bytes(int q_heads, int parts, int dim) { return parts < 2 ? 0 : sizeof(float) * static_cast<size_t>(q_heads) * parts * partial_stride(dim); }
int rows_at_a_time(int rows, int q_heads, int parts, int dim) {
  const size_t each = partial_bytes(q_heads, parts, dim), fit = each == 0 ? static_cast<size_t>(rows) : (kMostPartials > each ? kMostPartials / each : 1);
  return static_cast<size_t>(rows) < fit ? rows : static_cast<int>(fit);
}

constexpr size_t kMostExpanded = size_t{4} << 30;      // bytes of expanded pages: tables are as wide as the longest context may become
constexpr int kLongRows = 64, kLongPasses = 8;         // of a portion that is expanded: its rows, and passes of the tiles over its context

// Whether a step's portions are long enough, and what the expansion takes of the workspace.
struct Expansion {
  bool used;
  int width16;
  size_t key, value, tables, lengths, cu, marked, prompt, partials;      // offsets
};
size_t aligned_up(size_t n) { return (n + 255) / 256 * 256; }
Expansion expansion_of(int rows, int sequences, int max_new, int q_heads, int kv_heads, int dim, int block, int width, int window, int dtype) {
  Expansion e = {};
  if (max_new <= 16 || window != 0 || dtype != RLT_BF16 || (dim != 64 && dim != 128) || block % 16 != 0 || kv_heads <= 0 || sequences <= 0 || sequences > 65535) return e;
  // The tiles pass over a context once for sixteen pairs of a row and a head; the prompt kernel has a CTA for 256 rows of a head, however many
  // of them there are, and walks the context alone.  us, tiles / expanded, heads of 128: 16 portions of 128 rows on 4096 tokens, 16 of 16
  // heads 570 / 338, 4 such portions 153 / 128, 4 of 1021 rows on 5120 tokens 431 / 119; with fewer rows 16 of 64, 292 / 331, 16 of 32 in
  // groups of four heads 291 / 359; with few CTAs 1 of 256 on 512 tokens 25 / 31, 1 of 64 in groups of four on 131072 tokens 911 / 1990.
  const int64_t passes = static_cast<int64_t>(rows) * (q_heads / kv_heads) / 16;
  const bool pays = passes >= static_cast<int64_t>(kLongPasses) * sequences && rows >= static_cast<int64_t>(kLongRows) * sequences && (static_cast<int64_t>(rows) / 256 + sequences) * q_heads >= 64;
  e.width16 = static_cast<int>(static_cast<int64_t>(width) * block / 16);
  const size_t pages = static_cast<size_t>(sequences) * e.width16, bytes = pages * 16 * kv_heads * dim * 2;
  if (!pays || 2 * bytes > kMostExpanded || pages > 0x7fffffff) return e;
  e.used = true;
  e.value = e.key + aligned_up(bytes);
  e.tables = e.value + aligned_up(bytes);
  e.lengths = e.tables + aligned_up(pages * 4);
  e.cu = e.lengths + aligned_up(static_cast<size_t>(sequences) * 4);
  e.marked = e.cu + aligned_up(static_cast<size_t>(sequences + 1) * 4);
  e.prompt = e.marked + aligned_up(static_cast<size_t>(sequences + 1) * 4);
  e.partials = e.prompt + aligned_up(prefill_sm100_workspace_bytes(rows, sequences));
  return e;
}

// Scores a step over expanded pages; *scored: false where the prompt kernel does not take its tensors, and nothing was launched that counts.
int launch_expanded(const QuantizedAttentionArgs& a, const Expansion& e, unsigned char* workspace, int sm_count, bool* scored, cudaStream_t stream) {
  const QuantizedCache& c = a.cache;
  *scored = false;
  if (c.block_stride % 16 != 0 || c.token_stride % 16 != 0 || !aligned16(c.key) || !aligned16(c.value)) return RLT_OK;
  Expanded x;
  x.key = reinterpret_cast<__nv_bfloat16*>(workspace + e.key); x.value = reinterpret_cast<__nv_bfloat16*>(workspace + e.value);
  x.tables = reinterpret_cast<int32_t*>(workspace + e.tables); x.lengths = reinterpret_cast<int32_t*>(workspace + e.lengths);
  x.cu = reinterpret_cast<int32_t*>(workspace + e.cu); x.marked = reinterpret_cast<int32_t*>(workspace + e.marked); x.width16 = e.width16;
  const int group = a.q_heads / c.kv_heads;
  x.least = std::max(kLongRows, (16 * kLongPasses + group - 1) / group);
  AttentionArgs p;
  p.q = a.q; p.out = a.out; p.key_cache = x.key; p.value_cache = x.value;
  p.token_stride = static_cast<int64_t>(c.kv_heads) * c.dim; p.block_stride = 16 * p.token_stride; p.num_blocks = static_cast<int64_t>(a.step.sequences) * e.width16;
  p.block_size = 16; p.q_heads = a.q_heads; p.kv_heads = c.kv_heads; p.head_dim = c.dim; p.dtype = a.dtype; p.block_tables = x.tables;
  p.table_rows = a.step.sequences; p.table_width = e.width16; p.context_lengths = x.lengths; p.cu_seqlens_q = x.cu; p.rows = a.step.total;
  p.value_dim = c.dim; p.v_block_stride = p.block_stride; p.v_token_stride = p.token_stride; p.q_stride = a.q_stride; p.out_stride = a.out_stride;
  p.terms.scale = a.scale;
  if (!(a.scale > 0.0f) || !prefill_sm100_supported(p)) return RLT_OK;      // (there a scale of 0 means the usual one, and the largest score is taken before it)
  RLT_CUDA_TRY(cudaMemsetAsync(x.marked, 0, static_cast<size_t>(a.step.sequences + 1) * 4, stream));
  const int across = 8 * sm_count / a.step.sequences + 1;
  quantized_expand_kernel<<<dim3(static_cast<unsigned>(e.width16 < across ? e.width16 : across), static_cast<unsigned>(a.step.sequences)), 256, 0, stream>>>(
      c, a.step, x);
  int status = launch_status("quantized_expand_kernel");
  if (status != RLT_OK) return status;
  status = launch_prefill_sm100(p, workspace + e.prompt, e.partials - e.prompt, stream);
  *scored = status == RLT_OK;
  return status == RLT_ERR_UNSUPPORTED ? RLT_OK : status;
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
  a.step.tables = block_tables; a.step.lengths = lengths; a.step.cu = cu_rows; a.step.sequences = sequences; a.step.width = table_width; a.step.total = a.step.rows = rows; a.step.row0 = 0;
  RLT_REQUIRE(dtype_valid(dtype), "quantized_attention: dtype must be float32, float16 or bfloat16");
  RLT_REQUIRE(quantized_cache_valid(c), "quantized_attention: cache must be [pages, block, kv_heads, dim <= 256] with a contiguous [kv_heads, dim] tail");
  RLT_REQUIRE(sequences >= 0 && rows >= 0 && table_width >= 0, "quantized_attention: invalid shape");
  RLT_REQUIRE(static_cast<int64_t>(table_width) * block_size <= (1 << 26), "quantized_attention: tables of more than 2^26 tokens");
  RLT_REQUIRE(rows == 0 || sequences == 0 || (block_tables && lengths && cu_rows), "quantized_attention: null pointer");
  return RLT_OK;
}

}  // namespace
}  // namespace rlt

extern "C" RLT_API size_t rlt_quantized_attention_workspace_bytes(int rows, int sequences, int max_new, int q_heads, int kv_heads, int head_dim,
                                                                  int block_size, int table_width, int window, int dtype) {
  using namespace rlt;
  if (rows <= 0 || sequences <= 0 || q_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || table_width <= 0) return 0;
  const int parts = parts_of(static_cast<int64_t>(table_width) * block_size, window);
  const Expansion e = expansion_of(rows, sequences, max_new, q_heads, kv_heads, head_dim, block_size, table_width, window, dtype);
  return e.partials + static_cast<size_t>(rows_at_a_time(rows, q_heads, parts, head_dim)) * partial_bytes(q_heads, parts, head_dim);
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
  const Expansion e = expansion_of(rows, sequences, max_new, q_heads, kv_heads, head_dim, block_size, table_width, window, dtype);
  a.partials = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + e.partials);
  const size_t needed = rlt_quantized_attention_workspace_bytes(rows, sequences, max_new, q_heads, kv_heads, head_dim, block_size, table_width, window, dtype);
  if (workspace_bytes < needed || (needed > 0 && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0))) {
    set_last_error_text("quantized_attention: workspace missing, misaligned or too small");
    return RLT_ERR_WORKSPACE;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (e.used) {
    DeviceInfo info;
    status = current_device_info(&info);
    if (status != RLT_OK) return status;
    bool scored = false;
    status = launch_expanded(a, e, static_cast<unsigned char*>(workspace), info.sm_count, &scored, s);
    if (status != RLT_OK) return status;
    if (scored) {
      a.step.only = reinterpret_cast<const int32_t*>(static_cast<unsigned char*>(workspace) + e.marked);
      a.step.gave_up = reinterpret_cast<const uint32_t*>(static_cast<unsigned char*>(workspace) + e.prompt) + 1;      // the prompt kernels' error word
    }
  }
  const bool tiles = quantized_tiles_supported(a);
  const int each = rows_at_a_time(rows, q_heads, a.parts, head_dim);
  for (int64_t row = 0; row < rows; row += each) {
    a.step.row0 = static_cast<int>(row);
    a.step.rows = static_cast<int>(rows - row < each ? rows : row + each);
    status = tiles ? launch_quantized_tiles(a, max_new, s) : RLT_ERR_UNSUPPORTED;
    if (status == RLT_ERR_UNSUPPORTED) RLT_DISPATCH_DTYPE(dtype, T, status = launch_rows<T>(a, s));
    if (status == RLT_OK && a.parts > 1) RLT_DISPATCH_DTYPE(dtype, T, status = launch_merge<T>(a, s));
    if (status != RLT_OK) return status;
  }
  return RLT_OK;
}
