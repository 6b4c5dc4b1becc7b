// Attention over an 8-bit paged cache for short portions (decoding, verification): 64- and 128-wide heads, fp16 / bf16 queries, pages of whole
// 16-token tiles.
//
// Work.  An item is up to 16 query rows of one key/value head — (row, query head of the group) pairs of one sequence — over one part of its
// context (kPartTokens at fixed positions).  Items are dealt to one CTA per SM in a fixed order that every CTA derives from the lengths: no work
// list, no atomics, no second launch before the first byte is read.
//
// Data flow.  A producer warp copies 32 tokens at a time (keys and values of two 16-token tiles, one TMA box each) into a ring of stages that runs
// on across items, so the loads never stop; eight consumer warps take the stages in turn, by position.  Codes go from shared memory to the
// tensor cores through one conversion: e4m3 is exact in half precision.
//   S = Q K^T     m16n8k16, rows x tokens.  The head's elements are dealt to the products' k so that a lane's sixteen are one 16-byte load.
//   O^T += V^T P^T   m16n8k16, elements x rows: S's accumulators are P^T's operand as they are, and V, which lies token by token, needs only a
//                    byte permutation of two rows: the elements are dealt to the products' m like the head's elements above.
// Queries are brought to half precision at their own row's power of two (bf16 and fp16 rows lose nothing but what is 2^-24 of the row's largest).
// A key's scale multiplies its score; a value's scale goes into its weight's exponent, so a weight is 2^(s + log2 scale_v - R) and the sum l of the
// weights divides it out again.  R is a row's reference: it moves only when a weight would pass 2^15, and then so that the largest is 2^8.
// Weights are rounded to half precision (2^-11) for the second product; at 2^8 .. 2^15 for the largest, what is lost below half precision's
// smallest numbers is 2^-33 of it.  Scores, R, l and O are fp32.
//
// The eight warps' results of an item are added in shared memory in the order of the warps, so a row's bits depend on positions only, not on
// the batch, the other rows of its item or the part's length.
//
// Bound by the bytes of keys and values.
#include <cuda.h>

#include "quantized_kv.cuh"
#include "sm100_primitives.cuh"

namespace rlt {
namespace {

constexpr int kConsumers = 8;
constexpr int kThreads = (kConsumers + 4) * 32;  // whole warpgroups, so that registers can move from the producer's to the consumers'
constexpr int kConsumerRegisters = 208, kProducerRegisters = 80;
static_assert(kConsumers * 32 * kConsumerRegisters + 4 * 32 * kProducerRegisters <= kThreads * 168, "what a block of this size is launched with");
constexpr int kSlots = 16;              // stages in the ring
constexpr int kStageTokens = 32;
constexpr int kBatch = 1024;            // sequences whose items are laid out at a time
constexpr float kHighest = 15.0f;       // log2 of the largest weight that is kept
constexpr float kFresh = 8.0f;          // log2 of the largest weight when a row's reference moves

template <int kD, int kRowTiles>
struct __align__(1024) Shared {
  static constexpr int kRows = 8 * kRowTiles, kStride = kD + 4;
  unsigned char stages[kSlots][2][2][16 * kD];      // [tile of the stage][lower / upper cache][token][element], swizzled by the copy
  float sums[kConsumers][kRows][kStride];           // O, R, l of each warp
  float4 scales[kSlots][2];                         // per tile: key scale, log2 of the value scale, its inverse
  unsigned long long full[kSlots], empty[kSlots];
  int items[kBatch + 1];                            // items in front of a sequence of the batch
  int first[kBatch], count[kBatch], base[kBatch];   // its rows, and the keys its first row sees (below 1: none)
};

struct Item {
  int s, first, count, base, kv_head, pair0, pairs, part;
  int begin;        // first token of the first stage
  int end;          // behind the last visible token of the part
  int stages;
};

__device__ __forceinline__ int clamp_keys(int keys, int capacity) { return max(min(keys, capacity), 0); }

// A sequence's parts and row tiles.
struct Spread {
  int first_part, parts, tiles;
};
template <int kRows>
__device__ __forceinline__ Spread spread_of(int count, int base, int group, int window, int capacity) {
  Spread x;
  const int top = clamp_keys(base + count - 1, capacity), low = window > 0 ? max(clamp_keys(base, capacity) - window, 0) : 0;
  x.first_part = low / kPartTokens;
  x.parts = top > 0 ? (top - 1) / kPartTokens - x.first_part + 1 : 1;
  x.tiles = (count * group + kRows - 1) / kRows;
  return x;
}

__device__ __forceinline__ void tma_tile_pair(uint32_t dst, const CUtensorMap* map, int token, int head, int page, uint32_t bar, uint64_t policy) {
  asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, %4, %5, %6}], [%7], %8;"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(token), "r"(head), "r"(0), "r"(page), "r"(bar), "l"(policy) : "memory");
}
__device__ __forceinline__ void tma_tile(uint32_t dst, const CUtensorMap* map, int token, int head, int page, uint32_t bar, uint64_t policy) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, %4, %5}], [%6], %7;"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(token), "r"(head), "r"(page), "r"(bar), "l"(policy) : "memory");
}

// Two codes (the low or the high half of a word) as packed half precision.
__device__ __forceinline__ uint32_t halves_low(uint32_t w) {
  uint32_t h;
  asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %1;\ncvt.rn.f16x2.e4m3x2 %0, lo;\n}\n" : "=r"(h) : "r"(w));
  return h;
}
__device__ __forceinline__ uint32_t halves_high(uint32_t w) {
  uint32_t h;
  asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %1;\ncvt.rn.f16x2.e4m3x2 %0, hi;\n}\n" : "=r"(h) : "r"(w));
  return h;
}
__device__ __forceinline__ uint4 load_shared16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ uint2 load_shared8(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}
// 0x80 in every byte that is a NaN code.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory"); }

__device__ __forceinline__ void block_sync() { asm volatile("bar.sync 2, %0;" ::"n"(kThreads) : "memory"); }

// The token of a 16-token tile that column or row i < 8 of a product stands for (and 8 more for the next eight).  For 64-wide heads two tokens
// share a 128-byte line, and this order keeps the lanes of a load in different banks.
template <int kD>
__device__ __forceinline__ int token_of(int i) {
  return kD == 64 ? static_cast<int>((0x65742130u >> (4 * i)) & 7u) : i;
}

template <typename T, int kD, int kRowTiles, bool kJoint>
__global__ void __launch_bounds__(kThreads, 1)
quantized_tiles_kernel(const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map, QuantizedAttentionArgs a, float scale_log2,
                       int key_first) {
  using Sm = Shared<kD, kRowTiles>;
  constexpr int kRows = Sm::kRows, kTileBytes = 16 * kD, kSteps = kD / 16;      // k steps of S, m tiles of O^T
  extern __shared__ unsigned char smem_raw[];
  Sm& sm = *reinterpret_cast<Sm*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const QuantizedCache& c = a.cache;
  const int group = a.q_heads / c.kv_heads, capacity = a.step.width * c.block;
  const uint32_t full = smem_u32(sm.full), empty = smem_u32(sm.empty);

  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) { mbar_init(full + 8 * i, 1); mbar_init(empty + 8 * i, 1); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  grid_dependency_wait();
  grid_dependency_release();

  unsigned stage = 0;          // stages of all items before the current one
  bool failed = false;
  int batch = 0, sequences = 0;

  // The items of the next sequences, by all threads; their number.
  auto lay_out = [&]() {
    sequences = min(a.step.sequences - batch, kBatch);
    block_sync();              // the batch before is done with
    for (int i = threadIdx.x; i < sequences; i += kThreads) {
      int first, count;
      rows_of(a.step, batch + i, &first, &count);
      const int64_t base = static_cast<int64_t>(a.step.lengths[batch + i]) - count + 1;
      sm.first[i] = first;
      sm.count[i] = count;
      sm.base[i] = static_cast<int>(base < -0x20000000 ? -0x20000000 : (base > 0x20000000 ? 0x20000000 : base));
      const Spread x = spread_of<kRows>(count, sm.base[i], group, a.window, capacity);
      sm.items[i] = count > 0 ? x.parts * x.tiles * c.kv_heads : 0;
    }
    block_sync();
    if (warp == 0) {
      int before = 0;
      for (int i0 = 0; i0 < sequences; i0 += 32) {
        const int mine = i0 + lane < sequences ? sm.items[i0 + lane] : 0;
        int sum = mine;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
          const int o = __shfl_up_sync(0xffffffffu, sum, x);
          if (lane >= x) sum += o;
        }
        if (i0 + lane < sequences) sm.items[i0 + lane] = before + sum - mine;
        before += __shfl_sync(0xffffffffu, sum, 31);
      }
      if (lane == 0) sm.items[sequences] = before;
    }
    block_sync();
    return sm.items[sequences];
  };

  // The last sequence whose items start at or before i, 32 candidates at a time; then the item's place among its own.
  auto item_at = [&](int i) {
    int lo = 0, hi = sequences;
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32, at = lo + lane * step;
      const unsigned below = __ballot_sync(0xffffffffu, at < hi && sm.items[at] <= i);
      lo += (31 - __clz(below)) * step;
      hi = min(lo + step, hi);
    }
    Item x;
    x.s = batch + lo; x.first = sm.first[lo]; x.count = sm.count[lo]; x.base = sm.base[lo];
    const Spread spread = spread_of<kRows>(x.count, x.base, group, a.window, capacity);
    const int local = i - sm.items[lo], rest = local / c.kv_heads, chunk = rest / spread.tiles;
    x.kv_head = local - rest * c.kv_heads;
    x.part = spread.first_part + chunk;
    x.pair0 = (rest - chunk * spread.tiles) * kRows;
    x.pairs = min(x.count * group - x.pair0, kRows);
    const int top = clamp_keys(x.base + (x.pair0 + x.pairs - 1) / group, capacity);
    const int low = a.window > 0 ? max(clamp_keys(x.base + x.pair0 / group, capacity) - a.window, 0) : 0;
    const int from = max(low, x.part * kPartTokens);
    x.end = min(top, (x.part + 1) * kPartTokens);
    x.begin = from / kStageTokens * kStageTokens;
    x.stages = x.end > from ? (x.end - x.begin + kStageTokens - 1) / kStageTokens : 0;
    return x;
  };

  if (warp >= kConsumers) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProducerRegisters));
    for (; batch < a.step.sequences; batch += kBatch) {
      const int total = lay_out();
      if (warp > kConsumers) continue;
      // ---- producer: lane l holds pages and scales of the item's tiles l and l + 32 ----
      const uint64_t policy = policy_evict_first();
      auto load_pages = [&](const Item& x, int (&page)[2]) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int token = x.begin + 16 * (lane + 32 * k);
          page[k] = x.stages > 0 && token < x.end ? a.step.tables[static_cast<int64_t>(x.s) * a.step.width + token / c.block] : -1;
        }
      };
      // a page outside the cache reads as zeros, which is what the copies of it bring too
      auto load_scales = [&](const Item& x, const int (&page)[2], float (&ks)[2], float (&vs)[2]) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const bool there = page[k] >= 0 && page[k] < c.num_pages;
          ks[k] = there ? c.key_scale[page[k] * c.scale_stride + x.kv_head] : 0.0f;
          vs[k] = there ? c.value_scale[page[k] * c.scale_stride + x.kv_head] : 0.0f;
        }
      };
      int page[2], next_page[2];
      float ks[2], vs[2], next_ks[2], next_vs[2];
      Item x, next;
      int i = blockIdx.x;
      if (i < total) {
        x = item_at(i);
        load_pages(x, page);
        load_scales(x, page, ks, vs);
      }
      while (i < total && !failed) {
        const int i_next = i + gridDim.x;
        const bool more = i_next < total;
        if (more) {
          next = item_at(i_next);
          load_pages(next, next_page);
        }
        bool scales_asked = false;
        for (int j = 0; j < x.stages; ++j) {
          const unsigned n = stage + j, slot = n % kSlots;
          if (n >= kSlots && !mbar_wait(empty + 8 * slot, (n / kSlots - 1) & 1)) { failed = true; break; }
          const int tile = 2 * j + (lane & 1), set = tile >> 5;
          const bool mine = lane >> 1 == (j & 15) && x.begin + 16 * tile < x.end;
          if (mine) {
            // a scale that is no positive number within 2^-100 .. 2^100 is brought there: codes of a page of scale 0 then add nothing
            const float v = fminf(fmaxf(set ? vs[1] : vs[0], 7.8886090522101181e-31f), 1.2676506002282294e30f);
            sm.scales[slot][lane & 1] = make_float4(set ? ks[1] : ks[0], log2f(v), 1.0f / v, 0.0f);
          }
          __syncwarp();
          if (mine) {
            const int token = x.begin + 16 * tile, at = token % c.block, id = set ? page[1] : page[0];
            const uint32_t bar = full + 8 * slot, dst = smem_u32(&sm.stages[slot][lane & 1][0][0]);
            if ((lane & 1) == 0) mbar_expect_tx(bar, (token + 16 < x.end ? 4 : 2) * kTileBytes);
            if constexpr (kJoint) {
              tma_tile_pair(dst, &key_map, at, x.kv_head, id, bar, policy);
            } else {
              tma_tile(dst, &key_map, at, x.kv_head, id, bar, policy);
              tma_tile(dst + kTileBytes, &value_map, at, x.kv_head, id, bar, policy);
            }
          }
          if (more && j == 2) { load_scales(next, next_page, next_ks, next_vs); scales_asked = true; }
        }
        stage += x.stages;
        if (more) {
          if (!scales_asked) load_scales(next, next_page, next_ks, next_vs);
          x = next;
#pragma unroll
          for (int k = 0; k < 2; ++k) { page[k] = next_page[k]; ks[k] = next_ks[k]; vs[k] = next_vs[k]; }
        }
        i = i_next;
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kConsumerRegisters));
    for (; batch < a.step.sequences; batch += kBatch) {
      const int total = lay_out();
      // ---- consumers ----
      for (int i = blockIdx.x; i < total; i += gridDim.x) {
        const Item x = item_at(i);
        // rows g and g + 8 of the item, as products of rows x tokens have them
        int keys[2], low[2];
        float row_scale[2];
        uint32_t q[kSteps][kRowTiles * 2];
#pragma unroll
        for (int r = 0; r < kRowTiles; ++r) {
          const int pair = x.pair0 + g + 8 * r;
          const bool live = g + 8 * r < x.pairs;
          const int row = (live ? pair : x.pair0) / group, head = x.kv_head * group + (live ? pair : x.pair0) - row * group;
          keys[r] = live ? clamp_keys(x.base + row, capacity) : capacity;       // rows that are none see everything, and nothing is masked for them
          low[r] = live && a.window > 0 ? max(keys[r] - a.window, 0) : 0;
          const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (x.first + row) * a.q_stride + static_cast<int64_t>(head) * kD + kD / 4 * t);
          uint4 raw[kD / 32];
#pragma unroll
          for (int k = 0; k < kD / 32; ++k) raw[k] = live ? src[k] : make_uint4(0u, 0u, 0u, 0u);
          float largest = 0.0f;
#pragma unroll
          for (int k = 0; k < kD / 32; ++k) {
            const T* e = reinterpret_cast<const T*>(&raw[k]);
#pragma unroll
            for (int j = 0; j < 8; ++j) largest = fmaxf(largest, fabsf(Elem<T>::to_float(e[j])));
          }
          largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
          largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
          const int e = largest < INFINITY && largest > 0.0f ? min(max((__float_as_int(largest) >> 23) - 127, -126), 126) : 0;
          const float down = power_of_two(-e);
          row_scale[r] = scale_log2 * power_of_two(e);
#pragma unroll
          for (int k = 0; k < kD / 32; ++k) {
            const T* el = reinterpret_cast<const T*>(&raw[k]);
#pragma unroll
            for (int j = 0; j < 4; ++j)            // element pairs 2j, 2j + 1: k step 2k + j / 2, first or second k half
              q[2 * k + (j >> 1)][(j & 1) * kRowTiles + r] = pack2<false>(Elem<T>::to_float(el[2 * j]) * down, Elem<T>::to_float(el[2 * j + 1]) * down);
          }
        }
        const int top_keys = clamp_keys(x.base + (x.pair0 + x.pairs - 1) / group, capacity), least_keys = clamp_keys(x.base + x.pair0 / group, capacity);
        const int least_low = a.window > 0 ? max(least_keys - a.window, 0) : 0, top_low = a.window > 0 ? max(top_keys - a.window, 0) : 0;

        float o[kSteps][kRowTiles][4];
#pragma unroll
        for (int m = 0; m < kSteps; ++m)
#pragma unroll
          for (int r = 0; r < kRowTiles; ++r) { o[m][r][0] = 0.f; o[m][r][1] = 0.f; o[m][r][2] = 0.f; o[m][r][3] = 0.f; }
        float ref[kRowTiles], l[kRowTiles];
#pragma unroll
        for (int r = 0; r < kRowTiles; ++r) { ref[r] = -INFINITY; l[r] = 0.f; }
        float largest_scale = -INFINITY;

        const int first_stage = x.begin / kStageTokens;                  // of all the context's: the warp of a stage goes by its position
        for (int j = (warp - first_stage) & (kConsumers - 1); j < x.stages; j += kConsumers) {
          const unsigned n = stage + j, slot = n % kSlots;
          if (failed ? !mbar_try_wait(full + 8 * slot, (n / kSlots) & 1) : !mbar_wait(full + 8 * slot, (n / kSlots) & 1)) failed = true;
          if (!failed) {
            const int token0 = x.begin + j * kStageTokens;
            const bool two = token0 + 16 < x.end;
            const uint32_t tile_at[2] = {smem_u32(&sm.stages[slot][0][0][0]), smem_u32(&sm.stages[slot][1][0][0])};
            // scores, in log2 units and relative to the row's reference
            float s[2][2][4];
            float inverse[2], log2_scale[2];
            bool far[2] = {false, false};        // values so much smaller than others' that their weights pass below fp32, but not their keys' share of l
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              if (u == 1 && !two) {
#pragma unroll
                for (int k = 0; k < 4; ++k) { s[1][0][k] = -INFINITY; s[1][1][k] = -INFINITY; }
                inverse[1] = 0.0f;
                break;
              }
              const uint32_t keys_at = tile_at[u] + (key_first ? 0 : kTileBytes);
#pragma unroll
              for (int k = 0; k < 4; ++k) { s[u][0][k] = 0.f; s[u][1][k] = 0.f; }
#pragma unroll
              for (int h = 0; h < kD / 64; ++h) {
                uint32_t w[2][4];
#pragma unroll
                for (int n8 = 0; n8 < 2; ++n8) {
                  const int token = token_of<kD>(g) + 8 * n8;
                  const uint32_t chunk = kD == 128 ? static_cast<uint32_t>((2 * t + h) ^ (token & 7)) : static_cast<uint32_t>(t ^ ((token >> 1) & 3));
                  const uint4 v = load_shared16(keys_at + token * kD + chunk * 16);
                  w[n8][0] = v.x; w[n8][1] = v.y; w[n8][2] = v.z; w[n8][3] = v.w;
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  uint32_t qa[4];
                  qa[0] = q[4 * h + k][0];
                  qa[1] = kRowTiles == 2 ? q[4 * h + k][1] : 0u;
                  qa[2] = q[4 * h + k][kRowTiles];
                  qa[3] = kRowTiles == 2 ? q[4 * h + k][kRowTiles + 1] : 0u;
#pragma unroll
                  for (int n8 = 0; n8 < 2; ++n8) mma_16816<false>(s[u][n8], qa, halves_low(w[n8][k]), halves_high(w[n8][k]));
                }
              }
              const float4 scales = sm.scales[slot][u];
              inverse[u] = scales.z;
              log2_scale[u] = scales.y;
              largest_scale = fmaxf(largest_scale, scales.y);
              far[u] = scales.y < largest_scale - 60.0f;
#pragma unroll
              for (int r = 0; r < kRowTiles; ++r) {
                const float factor = row_scale[r] * scales.x, shift = scales.y - (ref[r] == -INFINITY ? 0.0f : ref[r]);
#pragma unroll
                for (int n8 = 0; n8 < 2; ++n8) {
                  s[u][n8][2 * r] = fmaf(s[u][n8][2 * r], factor, shift);
                  s[u][n8][2 * r + 1] = fmaf(s[u][n8][2 * r + 1], factor, shift);
                }
              }
              const int tile0 = token0 + 16 * u;
              if (tile0 + 16 > least_keys || tile0 < top_low) {
#pragma unroll
                for (int n8 = 0; n8 < 2; ++n8) {
#pragma unroll
                  for (int k = 0; k < 2; ++k) {
                    const int token = tile0 + token_of<kD>(2 * t + k) + 8 * n8;
#pragma unroll
                    for (int r = 0; r < kRowTiles; ++r)
                      if (token >= keys[r] || token < low[r]) s[u][n8][2 * r + k] = -INFINITY;
                  }
                }
              }
            }
            // a row's reference moves when a weight would pass 2^kHighest
            float top[kRowTiles];
            bool moves = false;
#pragma unroll
            for (int r = 0; r < kRowTiles; ++r) {
              top[r] = fmaxf(fmaxf(fmaxf(s[0][0][2 * r], s[0][0][2 * r + 1]), fmaxf(s[0][1][2 * r], s[0][1][2 * r + 1])),
                             fmaxf(fmaxf(s[1][0][2 * r], s[1][0][2 * r + 1]), fmaxf(s[1][1][2 * r], s[1][1][2 * r + 1])));
              moves |= top[r] > (ref[r] == -INFINITY ? -INFINITY : kHighest);
            }
            if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
              for (int r = 0; r < kRowTiles; ++r) {
                float most = top[r];
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                const bool fresh = ref[r] == -INFINITY, move = most > (fresh ? -INFINITY : kHighest);
                const float by = move ? most - kFresh : 0.0f, root = move && !fresh ? exp2f(-0.5f * by) : 1.0f, keep = root * root;
                if (move) ref[r] = (fresh ? 0.0f : ref[r]) + by;
                l[r] = l[r] * root * root;            // in two steps: where a page of far larger values moved the reference, keep may be 0 in fp32 and l not
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                  for (int n8 = 0; n8 < 2; ++n8) { s[u][n8][2 * r] -= by; s[u][n8][2 * r + 1] -= by; }
                const float keep0 = __shfl_sync(0xffffffffu, keep, 8 * t), keep1 = __shfl_sync(0xffffffffu, keep, 8 * t + 4);
#pragma unroll
                for (int m = 0; m < kSteps; ++m) { o[m][r][0] *= keep0; o[m][r][1] *= keep1; o[m][r][2] *= keep0; o[m][r][3] *= keep1; }
              }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              if (u == 1 && !two) break;
              uint32_t p[kRowTiles][2];
#pragma unroll
              for (int r = 0; r < kRowTiles; ++r) {
                const float p0 = fast_exp2(s[u][0][2 * r]), p1 = fast_exp2(s[u][0][2 * r + 1]), p2 = fast_exp2(s[u][1][2 * r]), p3 = fast_exp2(s[u][1][2 * r + 1]);
                if (!far[u]) {
                  l[r] = fmaf((p0 + p1) + (p2 + p3), inverse[u], l[r]);
                } else {
                  const float back = log2_scale[u];
                  l[r] += (fast_exp2(s[u][0][2 * r] - back) + fast_exp2(s[u][0][2 * r + 1] - back)) +
                          (fast_exp2(s[u][1][2 * r] - back) + fast_exp2(s[u][1][2 * r + 1] - back));
                }
                p[r][0] = pack2<false>(p0, p1);
                p[r][1] = pack2<false>(p2, p3);
              }
              // values of tokens 2t, 2t + 1 and the same of the upper eight, elements g * kD / 8 ..
              const uint32_t values_at = tile_at[u] + (key_first ? kTileBytes : 0);
              uint32_t w[4][kD / 32];
              int tokens[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int token = tokens[k] = token_of<kD>(2 * t + (k & 1)) + 8 * (k >> 1);
                if constexpr (kD == 128) {
                  const uint4 v = load_shared16(values_at + token * kD + ((g ^ (token & 7)) << 4));
                  w[k][0] = v.x; w[k][1] = v.y; w[k][2] = v.z; w[k][3] = v.w;
                } else {
                  const uint2 v = load_shared8(values_at + token * kD + (((g >> 1) ^ ((token >> 1) & 3)) << 4) + (g & 1) * 8);
                  w[k][0] = v.x; w[k][1] = v.y;
                }
              }
              const int tile0 = token0 + 16 * u;
              if (tile0 + 16 > least_keys || tile0 < top_low) {
                // Slots that no row of the item sees may hold anything, and a weight of zero times NaN is NaN: they are cleared.  NaN that some
                // rows see and others do not goes to those that do, by a product of its own over ones.
                uint32_t nans = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const bool seen = tile0 + tokens[k] < top_keys && tile0 + tokens[k] >= least_low;
#pragma unroll
                  for (int j = 0; j < kD / 32; ++j) {
                    if (!seen) w[k][j] = 0u;
                    nans |= nan_codes(w[k][j]);
                  }
                }
                if (__any_sync(0xffffffffu, nans != 0u)) {
                  uint32_t sees[kRowTiles][2];
#pragma unroll
                  for (int r = 0; r < kRowTiles; ++r) {
#pragma unroll
                    for (int n8 = 0; n8 < 2; ++n8) {
                      const int at0 = tile0 + token_of<kD>(2 * t) + 8 * n8, at1 = tile0 + token_of<kD>(2 * t + 1) + 8 * n8;
                      sees[r][n8] = (at0 < keys[r] && at0 >= low[r] ? 0x3c00u : 0u) | (at1 < keys[r] && at1 >= low[r] ? 0x3c000000u : 0u);
                    }
                  }
#pragma unroll
                  for (int j = 0; j < kD / 32; ++j) {
                    uint32_t ones[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                      const uint32_t marks = nan_codes(w[k][j]) >> 7;
                      ones[k] = marks * 0x38u;
                      w[k][j] &= ~(marks * 0xffu);
                    }
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                      const uint32_t x0 = __byte_perm(ones[0], ones[1], half ? 0x7362 : 0x5140), x1 = __byte_perm(ones[2], ones[3], half ? 0x7362 : 0x5140);
                      const uint32_t va[4] = {halves_low(x0), halves_high(x0), halves_low(x1), halves_high(x1)};
#pragma unroll
                      for (int r = 0; r < kRowTiles; ++r) {
                        float hits[4] = {0.f, 0.f, 0.f, 0.f};
                        mma_16816<false>(hits, va, sees[r][0], sees[r][1]);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                          if (hits[k] > 0.0f) o[2 * j + half][r][k] = NAN;
                      }
                    }
                  }
                }
              }
#pragma unroll
              for (int j = 0; j < kD / 32; ++j) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                  const uint32_t x0 = __byte_perm(w[0][j], w[1][j], half ? 0x7362 : 0x5140), x1 = __byte_perm(w[2][j], w[3][j], half ? 0x7362 : 0x5140);
                  const uint32_t va[4] = {halves_low(x0), halves_high(x0), halves_low(x1), halves_high(x1)};
#pragma unroll
                  for (int r = 0; r < kRowTiles; ++r) mma_16816<false>(o[2 * j + half][r], va, p[r][0], p[r][1]);
                }
              }
            }
          }
          __syncwarp();          // every lane's reads are done
          if (lane == 0) mbar_arrive(empty + 8 * slot);
        }

        // the warps' sums, in the order of the warps
        if (((warp - first_stage) & (kConsumers - 1)) < x.stages) {
          constexpr int kMine = kD / 8;                                  // elements g * kMine .. of rows 2t, 2t + 1 of each tile
#pragma unroll
          for (int r = 0; r < kRowTiles; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (t == 0) {
              sm.sums[warp][8 * r + g][kD] = failed ? 0.0f : ref[r];
              sm.sums[warp][8 * r + g][kD + 1] = failed ? NAN : l[r];
            }
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
              for (int m = 0; m < kSteps; m += 2)
                *reinterpret_cast<float4*>(&sm.sums[warp][8 * r + 2 * t + k][g * kMine + 2 * m]) =
                    make_float4(o[m][r][k], o[m][r][k + 2], o[m + 1][r][k], o[m + 1][r][k + 2]);
          }
        }
        consumers_sync();
        {
          constexpr int kPerRow = kConsumers * 32 / kRows, kEach = kD / kPerRow;
          static_assert(kEach % 2 == 0, "whole pairs of elements per thread");
          const int r = threadIdx.x / kPerRow, d0 = (threadIdx.x % kPerRow) * kEach;
          if (r < x.pairs) {
            const int pair = x.pair0 + r, row = pair / group, head = x.kv_head * group + pair - row * group;
            const int row_keys = clamp_keys(x.base + row, capacity), row_low = a.window > 0 ? max(row_keys - a.window, 0) : 0;
            const int first_part = row_low / kPartTokens, last_part = row_keys > 0 ? (row_keys - 1) / kPartTokens : first_part;
            if (x.part >= first_part && x.part <= last_part) {
              float big = -INFINITY;
#pragma unroll
              for (int w = 0; w < kConsumers; ++w)
                if (((w - first_stage) & (kConsumers - 1)) < x.stages) big = fmaxf(big, sm.sums[w][r][kD]);
              const float zero = big == -INFINITY ? 0.0f : big;
              float sum = 0.0f, acc[kEach];
#pragma unroll
              for (int k = 0; k < kEach; ++k) acc[k] = 0.0f;
#pragma unroll
              for (int w = 0; w < kConsumers; ++w) {
                if (((w - first_stage) & (kConsumers - 1)) >= x.stages) continue;
                const float* from = sm.sums[w][r];
                const float root = exp2f(0.5f * (from[kD] - zero)), f = root * root;
                sum += from[kD + 1] * root * root;
#pragma unroll
                for (int k = 0; k < kEach; k += 2) {
                  const float2 v = *reinterpret_cast<const float2*>(from + d0 + k);
                  acc[k] = fmaf(v.x, f, acc[k]);
                  acc[k + 1] = fmaf(v.y, f, acc[k + 1]);
                }
              }
              const int64_t at = static_cast<int64_t>(x.first + row) * a.q_heads + head;
              if (first_part == last_part) {
                const float scale = row_keys > row_low ? 1.0f / sum : 0.0f;
                uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + (x.first + row) * a.out_stride + static_cast<int64_t>(head) * kD + d0);
#pragma unroll
                for (int k = 0; k < kEach; k += 2) out[k / 2] = pack2<std::is_same<T, __nv_bfloat16>::value>(acc[k] * scale, acc[k + 1] * scale);
              } else {
                float* partial = a.partials + (at * a.parts + x.part - first_part) * partial_stride(kD);
#pragma unroll
                for (int k = 0; k < kEach; k += 2) *reinterpret_cast<float2*>(partial + d0 + k) = make_float2(acc[k], acc[k + 1]);
                if (d0 == 0) *reinterpret_cast<float2*>(partial + kD) = make_float2(big, sum);
              }
            }
          }
        }
        consumers_sync();        // the sums are read before the next item's are written
        stage += x.stages;
      }
    }
  }
  // a wait that gave up left NaN; copies still in flight land before the shared memory is given back
  if (failed && warp < kConsumers)
    for (int i = 0; i < kSlots; ++i)
      if (!mbar_wait(full + 8 * i, 0) && !mbar_wait(full + 8 * i, 1)) break;
}

// ---- host ---------------------------------------------------------------------------------------
// One cache as [pages][kv_heads][block][dim] bytes in boxes of 16 tokens of one head; with `distance` both caches, that far apart, as one tensor
// whose boxes hold a tile of each.
int make_tile_map(CUtensorMap* map, const void* base, const QuantizedCache& c, uint64_t distance) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (fn == nullptr) return RLT_ERR_UNSUPPORTED;
  cuuint64_t dims[5], strides[4];
  cuuint32_t box[5], element[5] = {1, 1, 1, 1, 1};
  int rank = 0;
  auto add = [&](uint64_t size, uint64_t stride, uint32_t in_box) {
    dims[rank] = size;
    box[rank] = in_box;
    if (rank > 0) strides[rank - 1] = stride;
    ++rank;
  };
  add(c.dim, 1, c.dim);
  add(c.block, c.token_stride, 16);
  add(c.kv_heads, c.dim, 1);
  if (distance != 0) add(2, distance, 2);
  add(c.num_pages, c.block_stride, 1);
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(base), dims, strides, box, element, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        c.dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? RLT_OK : RLT_ERR_UNSUPPORTED;
}

template <typename T, int kD, int kRowTiles>
int launch(const QuantizedAttentionArgs& a, cudaStream_t stream) {
  const QuantizedCache& c = a.cache;
  DeviceInfo info;
  int status = current_device_info(&info);
  if (status != RLT_OK) return status;
  const uintptr_t k = reinterpret_cast<uintptr_t>(c.key), v = reinterpret_cast<uintptr_t>(c.value);
  const bool key_first = k < v;
  const uint64_t distance = key_first ? v - k : k - v;
  CUtensorMap key_map, value_map;
  const bool joint = distance != 0 && distance % 16 == 0 && distance < (1ull << 40) &&
                     make_tile_map(&key_map, key_first ? c.key : c.value, c, distance) == RLT_OK;
  if (joint) {
    value_map = key_map;
  } else if (make_tile_map(&key_map, c.key, c, 0) != RLT_OK || make_tile_map(&value_map, c.value, c, 0) != RLT_OK) {
    return RLT_ERR_UNSUPPORTED;
  }
  const size_t smem = sizeof(Shared<kD, kRowTiles>) + 1024;
  auto kernel = joint ? quantized_tiles_kernel<T, kD, kRowTiles, true> : quantized_tiles_kernel<T, kD, kRowTiles, false>;
  RLT_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  return launch_dependent("quantized_tiles_kernel", kernel, dim3(static_cast<unsigned>(info.sm_count)), dim3(kThreads), smem, stream, key_map, value_map, a,
                          static_cast<float>(1.4426950408889634 * a.scale), joint && !key_first ? 0 : 1);
}

template <typename T>
int launch_for(const QuantizedAttentionArgs& a, int max_new, cudaStream_t stream) {
  // up to eight rows an item: half the registers and products
  const bool few = static_cast<int64_t>(max_new) * (a.q_heads / a.cache.kv_heads) <= 8;
  if (a.cache.dim == 128) return few ? launch<T, 128, 1>(a, stream) : launch<T, 128, 2>(a, stream);
  return few ? launch<T, 64, 1>(a, stream) : launch<T, 64, 2>(a, stream);
}

}  // namespace

bool quantized_tiles_supported(const QuantizedAttentionArgs& a) {
  const QuantizedCache& c = a.cache;
  if (a.dtype == RLT_F32 || (c.dim != 64 && c.dim != 128) || c.block % 16 != 0 || c.num_pages < 1 || c.num_pages > 0x7fffffff) return false;
  if (c.token_stride % 16 != 0 || c.block_stride % 16 != 0 || !aligned16(c.key) || !aligned16(c.value)) return false;
  if (a.q_stride % 8 != 0 || !aligned16(a.q) || a.out_stride % 2 != 0 || (reinterpret_cast<uintptr_t>(a.out) & 3u) != 0) return false;
  const int64_t group = a.q_heads / c.kv_heads, tiles = (static_cast<int64_t>(a.step.rows) * group + 7) / 8 + a.step.sequences;
  return tiles * c.kv_heads * a.parts <= 0x7fffffff && static_cast<int64_t>(a.step.rows) * group <= 0x7fffffff;     // items are counted in 32 bits
}

int launch_quantized_tiles(const QuantizedAttentionArgs& a, int max_new, cudaStream_t stream) {
  if (a.dtype == RLT_BF16) return launch_for<__nv_bfloat16>(a, max_new, stream);
  return launch_for<__half>(a, max_new, stream);
}

}  // namespace rlt
