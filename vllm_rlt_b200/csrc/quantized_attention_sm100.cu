// Attention over an 8-bit paged cache for short portions (decoding, verification): 64- and 128-wide heads, fp16 / bf16 queries, pages of whole
// 16-token tiles.  The codes are operands of the 5th-generation tensor cores as they lie in their pages: no conversion anywhere (converting
// them to half precision took 77 % of the conversion pipe's time at 28 % of the memory's rate).
//
// Work.  An item is up to kRows query rows — (row, query head of the group) pairs of one sequence — of 128 bytes of heads (one 128-wide key/value
// head or two 64-wide ones) over one part of the context (at fixed positions).  Items are dealt to one CTA per SM in an order that every
// CTA derives from the lengths: no work list, no atomics, no launch before the first byte is read.
//
// Products.  Keys and values are the M operands, so a handful of rows is the N and nothing is padded to a tensor tile:
//   S^T = K Q^T        lanes = 128 tokens, columns = rows;       O^T += V^T P^T     lanes = 128 value elements, V^T read MN-major
// Two 64-wide heads share the 128 bytes of a token.  Each has a product of its own over its half of K and of the queries' lines, into columns of its
// own: over the whole line, zeros in a query's other half would meet what the other head holds there, and 0 * NaN is NaN.  (O^T needs no such split:
// an output element comes from its own value element, and the others are not stored.)
// Q and P have more bits than a code, so both are sums of three: x = h + m / 32 + l / 1024, each rounded to four significant bits, what is
// left going to the next: the columns of an operand are the three parts of its rows, and the parts of a result are added in fp32.  A query row
// is brought to its own power of two first (the largest element in 2^7 .. 2^8); bf16 and fp16 rows lose what is 2^-27 of that.
//
// Softmax.  A key's scale multiplies its score; a value's goes into its weight's exponent, so a weight is
// p = 2^(s + log2 scale_v - R) and l = sum p / scale_v.  R is a row's reference: it moves when a weight would pass 2^kHighest, and then so
// that the largest is 2^kFresh.  Rounding p to three parts leaves 2^-12 of it, and below 2^-20 nothing: 2^-26 of a row's largest weight.
// Scores, R, l and O are fp32.
//
// Roles.  Two groups of four or eight warps take tiles of 128 tokens in turn, each with scores, weights, references and sums of its own; one warp
// issues S^T products, one O^T products, four or eight the copies (a ring of tiles that runs on across items; keys give their place back before
// their values), two prepare the queries of the next items, four write the results; three items are under way.  Which group a tile belongs to
// goes by its position, so a row's bits do not depend on the batch or on the other rows of its item.
//
// What bounds it.  The bytes of keys and values would take 1440 cycles a tile (32 KB) of an SM; with sixteen rows an item the warps issue about 4800
// instructions for one (half of them the softmax's, a quarter what an item costs at its ends), at 2.4 a cycle.  Measured, heads of 128, bf16:
//   64 requests, 16 rows of 16 heads each, contexts of 512 to 4096        157 us, 4.0 TB/s of keys and values
//   128 requests, a row of 32 heads over 8, contexts of 100 to 2048        66 us, 4.5 TB/s (items of four rows: the chain of a tile's waits)
//   4 requests, 5 rows of 32 heads over 8, contexts of 65000 to 131072    265 us, 3.1 TB/s (20 rows are two items: every tile is scored twice)
// (a call's time with the joining of its parts, 5 to 10 us of it).  With items found by every warp for itself, four copy warps at all sizes and
// weights stored byte by byte: 189, 78 and 315 us.  With the codes converted to half precision and multiplied by the warps (mma.sync): 342,
// 176 and 642 us.
#include <cuda.h>

#include "quantized_kv.cuh"
#include "sm100_primitives.cuh"

namespace rlt {
namespace {

constexpr int kGroups = 2;
constexpr int kPieces = 8;              // of 16 tokens, in a tile
constexpr int kQueryWarps = 2;          // half of the rows each
// The warps of a block for items of so many rows: a softmax thread has a token and up to eight rows.  Behind the groups come the warps that copy, issue
// S^T, issue O^T, prepare queries, and join and write results (four, from a multiple of four on).
template <int kRows>
struct Roles {
  static constexpr int kMine = kRows < 8 ? kRows : 8, kHalves = kRows / kMine;
  static constexpr int kGroupWarps = 4 * kHalves, kGroupThreads = 32 * kGroupWarps;
  static constexpr bool kSplit = kHalves == 1;                                               // half of eight warps copy keys, half values; else four copy both
  static constexpr int kCopyWarps = kSplit ? 8 : 4;
  static constexpr int kCopy = kGroups * kGroupWarps, kScore = kCopy + kCopyWarps, kValue = kScore + 1, kQuery = kScore + 2, kResult = kScore + 4;
  static constexpr int kControl = kCopyWarps + 8;
  static constexpr int kThreads = 32 * (kResult + 4);
  static constexpr int kLaunched = 65536 / kThreads / 8 * 8;                               // registers of a thread
  // The softmax gets what the others leave of the launch's.  With 48 for them the copies and the results spilled: 1 to 2 % slower; with 40, 9 %.
  static constexpr int kControlRegisters = kHalves == 2 ? 56 : 72;
  static constexpr int kSoftmaxRegisters = (kThreads * kLaunched - 32 * kControl * kControlRegisters) / (kGroups * kGroupThreads) / 8 * 8;
};
constexpr int kDeep = 3;                // items between their queries and their results
constexpr int kTile = 128;              // tokens
constexpr int kTileBytes = kTile * 128; // of keys, or of values
static_assert(kPieces * 16 == kTile);
constexpr int kSlots = 10;              // tiles of keys or of values in the ring, in turn
constexpr int kScaleSlots = 8;          // tiles' scales; see the copies
constexpr int kBatch = 256;             // sequences whose items are laid out at a time
static_assert(kWholeWindow + 16 - 1 + kTile - 1 <= kLongPart, "the window of an item's rows, from the start of a tile, is a part at most");
constexpr int kList = 48;               // items of this CTA that are looked up at a time
constexpr float kHighest = 8.0f, kFresh = 6.0f;
constexpr float kFaint = -100.0f;       // log2 of a weight whose product with 1 / scale_v may leave fp32
constexpr float kWide = 30.0f;          // log2 of a value scale that makes that possible

struct alignas(16) Item {
  int s, first, count, base;
  int unit;         // 128 bytes of heads
  int pair0;        // the first pair of the item; pairs of every head of the unit
  int pairs;
  int part;
  int from, end;    // tokens of the part that some row sees
  int all_from, all_end;      // and those that every row sees
  int begin;        // the first tile's first token
  int tiles;
};

enum { kNowhere, kOutput, kZero, kPartial };

// The work of a batch of sequences: cells (part, row tile) of whole parts in front of a sequence; then the last parts, largest first.
struct Work {
  int whole_before[kBatch + 1], last_before[kBatch + 1], order[kBatch];
  alignas(8) int2 size[kBatch];                       // a sequence's cells of whole parts; the tiles of its last part and, in the low 24 bits, its row tiles
  int first[kBatch], count[kBatch], base[kBatch];     // a sequence's rows, and the keys its first row sees (below 1: none)
};

template <int kRows>
struct __align__(1024) Shared {
  static constexpr int kN = (3 * kRows + 15) / 16 * 16;         // three parts of every row, in whole sixteens
  unsigned char ring[kSlots][kTileBytes];             // [token][128 bytes], swizzled by the copy: keys of a tile, its values, the next tile's keys ..
  unsigned char q[kDeep][kN * 128];                   // [item][part of a row][128 elements], of two heads [item][part of a head's row][64 elements of each]
  unsigned char p[kGroups][2][kN * 128];              // of a group's tiles in turn: [16 parts of rows][128 tokens][16 bytes]
  uint32_t raw_q[kRows][64];                          // the next item's queries as they are
  float4 scales[kScaleSlots][2][kPieces];             // by head and 16 tokens: key scale, log2 of the value scale, its inverse, 0 where it is 0 (and 1)
  alignas(8) unsigned char wide[kScaleSlots][kPieces];      // a value scale of the piece is beyond 2^+-kWide
  Item list[kList];
  // of an item
  alignas(16) float row_scale[kDeep][kRows];          // of the scores
  int keys[kDeep][kRows], low[kDeep][kRows];          // what a row sees of the part
  int64_t to[kDeep][kRows];                           // where its result goes: elements into the output, or floats into the partials
  int kind[kDeep][kRows];                             // kNowhere, kOutput, kZero, kPartial
  alignas(16) float ref[kDeep][kGroups][kRows];
  float l[kDeep][kGroups][4][kRows];        // of each group; l of each quarter of its tokens
  alignas(16) uint32_t nan_value[kDeep][kGroups][kRows][4];      // elements that a row gets NaN in
  int marked[kDeep][kGroups];                         // there are some
  // of a group's tile
  alignas(16) float folded[kGroups][4][kRows];
  alignas(16) float by[kGroups][kRows];
  alignas(16) float root[kGroups][kRows];       // of a move of references: added to them (by); the root of what O and l are multiplied by
  uint32_t fresh[kGroups][2];                         // rows of a half without a reference yet
  unsigned moved[kGroups][2];                         // the turn of a half's last move of a reference that had been there
  float4 result[4][kRows];                            // of each result warp: the groups' factors and the address that a row goes to
  // A waiter may be a phase of a barrier behind, never two (a phase and the one after the next look alike): what has two buffers has two barriers.
  unsigned long long full[kSlots], empty[kSlots], q_full[kDeep], q_empty[kDeep], done[kDeep], s_ready[kGroups], s_free[kGroups], p_ready[kGroups][2], o_done[kGroups][2];
  uint32_t tmem_base;
  Work work;
};

// Bounded wait for a phase of a barrier: false after two million polls (a poll is suspended for up to a microsecond, which leaves the issue slots to
// other warps).  Few instructions: the roles' loops together have to stay within the instruction caches.  With unrolled polls at every wait they did
// not, and every phase took three to ten times as long.
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity) {
#pragma unroll 1
  for (int polls = 0; polls < 2000000; ++polls) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok) : "r"(bar), "r"(parity), "r"(1000u) : "memory");
    if (ok != 0) return true;
  }
  return false;
}

__device__ __forceinline__ int clamp_keys(int keys, int capacity) { return max(min(keys, capacity), 0); }

struct Spread {
  int first_part, parts, tiles;
};
// A sequence's parts, and the row tiles of `each` pairs.
__device__ __forceinline__ Spread spread_of(int each, int count, int base, int group, int window, int capacity) {
  Spread x;
  const int top = clamp_keys(base + count - 1, capacity), low = window > 0 ? max(clamp_keys(base, capacity) - window, 0) : 0;
  x.first_part = part_of(low, window);
  x.parts = top > 0 ? part_of(top - 1, window) - x.first_part + 1 : 1;
  x.tiles = (count * group + each - 1) / each;
  return x;
}

// The last i < n with before[i] <= x, 32 candidates at a time.
__device__ __forceinline__ int find(const int* before, int n, int x) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = n;
#pragma unroll 1
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, at = lo + lane * step;
    const unsigned below = __ballot_sync(0xffffffffu, at < hi && before[at] <= x);
    lo += (31 - __clz(below)) * step;
    hi = min(lo + step, hi);
  }
  return lo;
}

// Item i of a batch, by a whole warp.
__device__ __noinline__ Item find_item(const Work* work, int batch, int sequences, int whole, int i, int units, int each, int group, int window, int capacity) {
  const int cell = i / units;
  int lo, local;
  if (cell < whole) {
    lo = find(work->whole_before, sequences, cell);
    local = cell - work->whole_before[lo];
  } else {
    const int k = find(work->last_before, sequences, cell - whole);
    lo = work->order[k];
    local = cell - whole - work->last_before[k];
  }
  Item x;
  x.s = batch + lo; x.first = work->first[lo]; x.count = work->count[lo]; x.base = work->base[lo];
  const Spread spread = spread_of(each, x.count, x.base, group, window, capacity);
  const int chunk = cell < whole ? local / spread.tiles : spread.parts - 1;
  x.unit = i - cell * units;
  x.part = spread.first_part + chunk;
  x.pair0 = (cell < whole ? local - chunk * spread.tiles : local) * each;
  x.pairs = min(x.count * group - x.pair0, each);
  const int least = clamp_keys(x.base + x.pair0 / group, capacity), top = clamp_keys(x.base + (x.pair0 + x.pairs - 1) / group, capacity);
  x.from = max(window > 0 ? max(least - window, 0) : 0, part_begin(x.part, window));
  x.end = min(top, part_begin(x.part + 1, window));
  x.all_from = max(window > 0 ? max(top - window, 0) : 0, x.from);
  x.all_end = min(least, x.end);
  x.begin = x.from / kTile * kTile;
  x.tiles = x.end > x.from ? (x.end - x.begin + kTile - 1) / kTile : 0;
  return x;
}

__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int token, int page, uint32_t bar, uint64_t policy) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%2, %3, %4}], [%5], %6;"
               ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(token), "r"(page), "r"(bar), "l"(policy) : "memory");
}
// An operand of 16-byte pieces of its rows with the columns 16 bytes apart: `rows` bytes between pieces of 16 rows, `columns` between groups of eight
// columns; no swizzle.
__device__ __forceinline__ uint64_t piece_desc(uint32_t addr, uint32_t columns, uint32_t rows) {
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | static_cast<uint64_t>(columns >> 4) << 16 | static_cast<uint64_t>(rows >> 4) << 32 | 1ull << 46;
}
// D[tmem] (+)= A[smem] * B[smem] of e4m3 codes, one elected thread; 32 codes of K.
__device__ __forceinline__ void code_product(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n"
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// kCount columns into x[kFirst] ..
template <int kCount, int kFirst = 0, int kSize>
__device__ __forceinline__ void load_columns(uint32_t at, float (&x)[kSize]) {
  uint32_t r[kCount];
  if constexpr (kCount == 8) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(at));
  } else {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
  }
#pragma unroll
  for (int i = 0; i < kCount; ++i) x[kFirst + i] = __uint_as_float(r[i]);
}
template <int kCount>
__device__ __forceinline__ void store_columns(uint32_t at, const float (&x)[kCount]) {
  uint32_t r[kCount];
#pragma unroll
  for (int i = 0; i < kCount; ++i) r[i] = __float_as_uint(x[i]);
  if constexpr (kCount == 8) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
  } else {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
  }
}
// A group's barrier, with the OR of a predicate.
template <int kGroupThreads>
__device__ __forceinline__ bool any_of_group(int group, bool mine) {
  uint32_t any;
  asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbarrier.cta.red.or.pred q, %2, %3, p;\nselp.u32 %0, 1, 0, q;\n}\n"
               : "=r"(any) : "r"(mine ? 1u : 0u), "r"(1 + group), "n"(kGroupThreads) : "memory");
  return any != 0;
}

// Two numbers as packed codes of their three parts, x = h + m / 32 + l / 1024 for |x| <= 256: x in half precision (2^-11 of it, or 2^-25), then
// h and m rounded by the conversion to a code; what each leaves, times 32, is exact in half precision.
__device__ __forceinline__ void three_parts(float x0, float x1, uint32_t (&codes)[3]) {
  const __half2 whole = __floats2half2_rn(x0, x1), minus = __float2half2_rn(-32.0f), times = __float2half2_rn(32.0f);
  __half2 left = whole;
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    const __half2_raw raw = *reinterpret_cast<const __half2_raw*>(&left);
    const __nv_fp8x2_storage_t code = __nv_cvt_halfraw2_to_fp8x2(raw, __NV_SATFINITE, __NV_E4M3);
    codes[k] = code;
    if (k < 2) {
      const __half2_raw back = __nv_cvt_fp8x2_to_halfraw2(code, __NV_E4M3);
      left = __hfma2(*reinterpret_cast<const __half2*>(&back), minus, __hmul2(left, times));
    }
  }
}
__device__ __forceinline__ void store_shared8(uint32_t at, uint2 x) { asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(at), "r"(x.x), "r"(x.y) : "memory"); }
__device__ __forceinline__ void store_shared16(uint32_t at, uint4 x) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x.x), "r"(x.y), "r"(x.z), "r"(x.w) : "memory");
}
__device__ __forceinline__ float4 load_shared16f(uint32_t at) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
  return v;
}

// Adds kCount values up over the lanes of a warp, all of them at once: at every step a lane gives half of its values away and takes the other half's
// partners.  Returns value row_after_fold(lane) of them, complete, in every lane.
template <int kCount>
__device__ __forceinline__ float fold_rows(float (&v)[kCount], int lane) {
  int bit = 16;
#pragma unroll
  for (int half = kCount / 2; half > 0; half /= 2, bit /= 2) {
    const bool upper = lane & bit;
#pragma unroll
    for (int i = 0; i < half; ++i) {
      const float give = upper ? v[i] : v[i + half], stay = upper ? v[i + half] : v[i];
      v[i] = stay + __shfl_xor_sync(0xffffffffu, give, bit);
    }
  }
  float x = v[0];
  for (; bit > 0; bit /= 2) x += __shfl_xor_sync(0xffffffffu, x, bit);
  return x;
}
__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
template <int kCount>
__device__ __forceinline__ int row_after_fold(int lane) { return lane / (32 / kCount); }
// 0x80 in every byte that is a NaN code.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// kDim: 128, or 64 with two heads side by side, whose pairs are rows 0 .. kRows / 2 - 1 and kRows / 2 .. of an item.
template <typename T, int kDim, int kRows>
__global__ void __launch_bounds__(Roles<kRows>::kThreads, 1)
quantized_tiles_kernel(const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map, QuantizedAttentionArgs a, float scale_log2,
                       int box) {
  using Sm = Shared<kRows>;
  using Role = Roles<kRows>;
  constexpr int kThreads = Role::kThreads, kGroupWarps = Role::kGroupWarps, kHalves = Role::kHalves;
  constexpr int kCopyWarp = Role::kCopy, kScoreWarp = Role::kScore, kValueWarp = Role::kValue, kQueryWarp = Role::kQuery, kResultWarp = Role::kResult;
  const auto block_sync = [] { asm volatile("bar.sync 4, %0;" ::"n"(kThreads) : "memory"); };
  const auto group_any = [](int group, bool mine) { return any_of_group<Role::kGroupThreads>(group, mine); };
  constexpr int kHeads = 128 / kDim, kEach = kRows / kHeads, kN = Sm::kN;
  constexpr int kHeadN = (3 * kEach + 15) / 16 * 16;         // columns of a head's scores: three parts of its rows, in whole sixteens
  static_assert(kHeadN * kHeads <= 64 && kHeadN <= kN, "columns of a group's scores (a head's share of them is 64 / kHeads), lines of an item's queries");
  // tensor memory: 64 columns for the scores of each group, then for its outputs of the items under way
  constexpr uint32_t kScores = 0, kOutputs = kGroups * 64, kColumns = 512;
  static_assert(kOutputs + kGroups * kDeep * 64 <= kColumns, "tensor memory");
  extern __shared__ unsigned char smem_raw[];
  Sm& sm = *reinterpret_cast<Sm*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const QuantizedCache& c = a.cache;
  const int group_heads = a.q_heads / c.kv_heads, capacity = a.step.width * c.block, units = (c.kv_heads + kHeads - 1) / kHeads;

  if (warp == kScoreWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem_base)), "r"(kColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == kCopyWarp && lane < 2)
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(lane ? &value_map : &key_map)) : "memory");
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSlots; ++i) { mbar_init(smem_u32(&sm.full[i]), 4); mbar_init(smem_u32(&sm.empty[i]), 1); }
    for (int i = 0; i < kDeep; ++i) {
      mbar_init(smem_u32(&sm.q_full[i]), kQueryWarps);
      mbar_init(smem_u32(&sm.q_empty[i]), 4);                              // the result warps
      mbar_init(smem_u32(&sm.done[i]), 2 + kGroups * kGroupWarps);        // the last product's completion, the warp of S^T and each softmax warp
    }
    for (int i = 0; i < kGroups; ++i) {
      mbar_init(smem_u32(&sm.s_ready[i]), 1);
      mbar_init(smem_u32(&sm.s_free[i]), kGroupWarps);
      for (int k = 0; k < 2; ++k) {
        mbar_init(smem_u32(&sm.p_ready[i][k]), kGroupWarps);
        mbar_init(smem_u32(&sm.o_done[i][k]), 1);
      }
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
#pragma unroll 1
  for (int i = threadIdx.x; i < kDeep * kGroups * kRows * 4; i += kThreads) (&sm.nan_value[0][0][0][0])[i] = 0u;
  if (threadIdx.x < kDeep * kGroups) (&sm.marked[0][0])[threadIdx.x] = 0;
  grid_dependency_wait();
  grid_dependency_release();
  tcgen05_before_sync();
  __syncthreads();
  tcgen05_after_sync();
  const uint32_t tmem = sm.tmem_base;

  unsigned done_items = 0, done_tiles = 0, done_of[kGroups] = {0u, 0u};   // items, tiles, and tiles of each group before the current item
  bool failed = false;
  int sequences = 0, whole = 0;      // of the batch: sequences, cells of whole parts

  // The items of sequences batch .., by all threads; their number.  Cells of whole parts come first, then every sequence's last part, those with the
  // most tiles first: dealt in this order, one CTA has about as many tiles as another.  The heads of a cell go to neighbouring CTAs at a time.
  auto lay_out = [&](int batch) {
    static_assert(2 * (kBatch + 1) * sizeof(int) <= sizeof(sm.list), "the list is not in use meanwhile");
    int *const places = reinterpret_cast<int*>(sm.list), *const last_sums = places + kBatch + 1;      // among the last parts, and the cells in front there
    sequences = min(a.step.sequences - batch, kBatch);
    block_sync();              // the batch before is done with
#pragma unroll 1
    for (int i = threadIdx.x; i < sequences; i += kThreads) {
      int first, count, length;
      rows_of(a.step, batch + i, &first, &count, &length);
      const int64_t base = static_cast<int64_t>(length) - count + 1;
      sm.work.first[i] = first;
      sm.work.count[i] = count;
      sm.work.base[i] = static_cast<int>(base < -0x20000000 ? -0x20000000 : (base > 0x20000000 ? 0x20000000 : base));
      const Spread x = spread_of(kEach, count, sm.work.base[i], group_heads, a.window, capacity);
      const int top = clamp_keys(sm.work.base[i] + count - 1, capacity), low = a.window > 0 ? max(clamp_keys(sm.work.base[i], capacity) - a.window, 0) : 0;
      const int last_tiles = top > 0 ? (top - 1 - max(part_begin(part_of(top - 1, a.window), a.window), low / kTile * kTile)) / kTile + 1 : 0;
      sm.work.size[i] = make_int2(count > 0 ? (x.parts - 1) * x.tiles : 0, min(last_tiles, 127) << 24 | x.tiles);
    }
#pragma unroll 1
    for (int i = threadIdx.x; i <= sequences; i += kThreads) sm.work.whole_before[i] = places[i] = last_sums[i] = 0;
    block_sync();
    // A sequence's place, and what lies in front of it, by comparing it with all the others: a lane has a sequence, and the warps a share of the others
    // each.  The sum of all stands behind the last.
    const int blocks = sequences / 32 + 1, shares = kThreads / 32 / blocks, share = warp / blocks, i = warp % blocks * 32 + lane;
    if (share < shares && i <= sequences) {
      const int each = (sequences + shares - 1) / shares, mine = i < sequences ? sm.work.size[i].y >> 24 : -1;
      int place = 0, whole_before = 0, last_sum = 0;
#pragma unroll 4
      for (int k = share * each; k < min((share + 1) * each, sequences); ++k) {
        const int2 other = sm.work.size[k];
        if (k < i) whole_before += other.x;
        if (other.y >> 24 > mine || (other.y >> 24 == mine && k < i)) { ++place; last_sum += other.y & 0xffffff; }
      }
      atomicAdd(&sm.work.whole_before[i], whole_before);
      atomicAdd(&places[i], place);
      atomicAdd(&last_sums[i], last_sum);
    }
    block_sync();
#pragma unroll 1
    for (int k = threadIdx.x; k <= sequences; k += kThreads) {
      const int place = places[k];
      sm.work.last_before[place] = last_sums[k];
      if (k < sequences) sm.work.order[place] = k;
    }
    block_sync();
    whole = sm.work.whole_before[sequences];
    return (whole + sm.work.last_before[sequences]) * units;
  };

  // Items of this CTA that are looked up together, from its item `base` of the batch on.  The control warps do it, an item each in turn, between two
  // barriers of the block.
  auto items_of = [&](int base, int total) {
    return min((total - static_cast<int>(blockIdx.x) + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x) - base, kList);
  };
  auto look_up = [&](int batch, int base, int items) {
#pragma unroll 1
    for (int k = warp - kCopyWarp; k < items; k += Role::kControl) {
      const Item x = find_item(&sm.work, batch, sequences, whole, blockIdx.x + (base + k) * gridDim.x, units, kEach, group_heads, a.window, capacity);
      if (lane == 0) sm.list[k] = x;
    }
  };
  auto group_of = [&](const Item& x, int j) { return (x.begin / kTile + j) & 1; };
  auto tiles_of = [&](const Item& x, int group) { return (x.tiles + (group_of(x, 0) == group ? 1 : 0)) / 2; };
  auto buffer = [&]() { return done_items % kDeep; };
  auto phase = [&]() { return (done_items / kDeep) & 1; };
  auto pass = [&](const Item& x) {
    ++done_items;
    done_tiles += x.tiles;
    done_of[0] += tiles_of(x, 0);
    done_of[1] += tiles_of(x, 1);
  };

  // (a loop for each: what runs with a kind's registers stays apart from the other's)
  if (warp >= kCopyWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Role::kControlRegisters));
#pragma unroll 1
    for (int batch = 0, base = 0, total = 0; batch < a.step.sequences; base += kList) {
    if (base == 0) total = lay_out(batch);
    else block_sync();          // the items before are done with
    const int items = items_of(base, total);
    look_up(batch, base, items);
    block_sync();
    if (items < kList) { batch += kBatch; base = -kList; }
    if (warp >= kCopyWarp && warp < kScoreWarp) {
      static_assert(2 * kScaleSlots >= kSlots + 2, "tile n + kScaleSlots is copied after the values of tile n are done with");
      // ---- copies: a warp has two pieces of every tile, its lane 2j + i pages and scales of piece i of tile j of an item (a part has up to sixteen) ----
      // What a copy costs is its issue: a warp alone has an instruction in four or five cycles, a box takes about 200 and the wait in front 270, of 1440
      // that the memory gives a tile.  So nothing that waits for the memory stands between the copies of two items (a next item's pages are read when
      // an item's copies begin, and its scales when its first keys have gone out), and pieces that no row sees are copied too, as zeros from a page that
      // does not exist.
      constexpr bool kSplit = Role::kSplit;
      const uint64_t policy = policy_evict_first();
      const int which = kSplit ? (warp - kCopyWarp) / 4 : 0, piece0 = (warp - kCopyWarp) % 4 * 2, piece = piece0 + (lane & 1);
      const int boxes = box == 16 ? 2 : ((16 * piece0) % box == 0 ? 1 : 0);      // that start with this warp's pieces
      int next_page = -1, next_place = 0;
      float next_key[kHeads], next_value[kHeads];
      auto look = [&](const Item& next) {
        const int token = next.begin + (lane >> 1) * kTile + 16 * piece, entry = token / c.block;
        const bool seen = lane < 2 * next.tiles && (token & -box) < next.end && (token | (box - 1)) >= next.from;      // (a box lies in one page)
        next_place = token - entry * c.block;
        next_page = seen ? a.step.tables[static_cast<int64_t>(next.s) * a.step.width + entry] : -1;
      };
      auto load_scales = [&](const Item& next) {
#pragma unroll
        for (int h = 0; h < kHeads; ++h) {
          const int64_t at = next_page * c.scale_stride + min(next.unit * kHeads + h, c.kv_heads - 1);
          // a page outside the cache reads as zeros, which is what the copies of it bring too
          const bool there = next_page >= 0 && next_page < c.num_pages;
          next_key[h] = there ? c.key_scale[at] : 0.0f;
          next_value[h] = there ? c.value_scale[at] : 1.0f;
        }
      };
      unsigned slot = (2 * done_tiles + which) % kSlots, turn = (2 * done_tiles + which) / kSlots & 1, scale_slot = done_tiles % kScaleSlots;
      if (items > 0) {
        look(sm.list[0]);
        if (!kSplit || which == 1) load_scales(sm.list[0]);
      }
#pragma unroll 1
      for (int it = 0; it < items && !failed; ++it) {
        const int page = next_page, place = next_place, tiles = sm.list[it].tiles, heads_at = sm.list[it].unit * 128;
        float4 scales[kHeads];                                            // as the softmax takes them
        bool wide = false;
        auto convert = [&] {
#pragma unroll
          for (int h = 0; h < kHeads; ++h) {
            // a scale of 0 goes as the smallest one, its weights as nothing; one that is NaN makes the scores NaN for the rows that see its tokens
            const float given = value_scale_of(next_value[h]), v = fmaxf(given, power_of_two(kMinScaleExponent));
            const int e = (__float_as_int(v) >> 23) - 127;
            const float significand = __int_as_float((__float_as_int(v) & 0x007fffff) | 0x3f800000);      // 1 for powers of two: exact then
            const float exponent = given >= 0.0f ? static_cast<float>(e) + __log2f(significand) : NAN;
            scales[h] = make_float4(next_key[h], exponent, power_of_two(-e) * __frcp_rn(significand), given == 0.0f ? 0.0f : 1.0f);
            wide |= fabsf(exponent) > kWide;
          }
        };
        const bool more = it + 1 < items;
        const Item& next = sm.list[more ? it + 1 : it];
        if (more) look(next);
#pragma unroll 1
        for (int j = 0; j < tiles && !failed; ++j) {
          const int page0 = __shfl_sync(0xffffffffu, page, 2 * j), place0 = __shfl_sync(0xffffffffu, place, 2 * j);
          const int page1 = __shfl_sync(0xffffffffu, page, 2 * j + 1), place1 = place0 + 16 == c.block ? 0 : place0 + 16;      // (of a box of its own: in this page or the next)
#pragma unroll
          for (int values = which; values <= (kSplit ? which : 1); ++values) {
            if (!wait_for(smem_u32(&sm.empty[slot]), turn ^ 1)) { failed = true; break; }                 // (at first the phase before a barrier's first: over)
            if (values) {
              if (j == 0) {                                                // (the first item's are still on their way when its keys are copied)
                convert();
                if (more) load_scales(next);
              }
              // The slots of the tile kScaleSlots before are free: its values gave theirs back before this tile's could be copied.
              if ((lane >> 1) == j) {
#pragma unroll
                for (int h = 0; h < kHeads; ++h) sm.scales[scale_slot][h][piece] = scales[h];
                sm.wide[scale_slot][piece] = wide;
              }
              scale_slot = (scale_slot + 1) % kScaleSlots;
              __syncwarp();                                                // the scales are written
            }
            if (lane == 0) {
              const uint32_t bar = smem_u32(&sm.full[slot]), dst = smem_u32(sm.ring[slot]) + piece0 * 2048;
              const CUtensorMap* map = values ? &value_map : &key_map;
              mbar_expect_tx(bar, static_cast<uint32_t>(boxes * box) * 128);
              if (boxes > 0) {
                tma_box(dst, map, heads_at, place0, page0, bar, policy);
                if (boxes > 1) tma_box(dst + 2048, map, heads_at, place1, page1, bar, policy);
              }
            }
            slot += kSplit ? 2 : 1;
            if (slot >= kSlots) { slot -= kSlots; turn ^= 1; }
          }
        }
        if (tiles == 0 && more && (!kSplit || which == 1)) load_scales(next);
        done_tiles += tiles;
      }
    } else if (warp == kScoreWarp) {
      // ---- S^T of a tile, once its keys and the item's queries are there and its group has read the scores of the tile before ----
      constexpr uint32_t kIdesc = (1u << 4) | (static_cast<uint32_t>(kHeadN >> 3) << 17) | (static_cast<uint32_t>(kTile >> 4) << 24);
      constexpr int kSteps = 4 / kHeads;      // of 32 codes, in a head
#pragma unroll 1
      for (int it = 0; it < items && !failed; ++it) {
        const unsigned at = buffer();
        bool ok = wait_for(smem_u32(&sm.q_full[at]), phase());
        const Item x = sm.list[it];
        {
          const uint64_t q_desc = umma_desc(smem_u32(sm.q[at]), 16, 1024);
          unsigned of[kGroups] = {done_of[0], done_of[1]};
#pragma unroll 1
          for (int j = 0; j < x.tiles; ++j) {
            const int group = group_of(x, j);
            const unsigned h = 2 * (done_tiles + j), slot = h % kSlots, mine = group ? of[1] : of[0];
            ok = ok && (mine == 0 || wait_for(smem_u32(&sm.s_free[group]), (mine - 1) & 1));
            ok = ok && wait_for(smem_u32(&sm.full[slot]), (h / kSlots) & 1);
            if (!__all_sync(0xffffffffu, ok)) { failed = true; break; }
            tcgen05_after_sync();
            const uint64_t k_desc = umma_desc(smem_u32(sm.ring[slot]), 16, 1024);
            if (elect_one()) {
#pragma unroll
              for (int ks = 0; ks < 4; ++ks)
                code_product(tmem + kScores + group * 64 + ks / kSteps * 32, k_desc + static_cast<uint64_t>(ks * 2), q_desc + static_cast<uint64_t>(ks * 2), kIdesc,
                             ks % kSteps > 0);
              umma_commit(smem_u32(&sm.s_ready[group]));
              umma_commit(smem_u32(&sm.empty[slot]));
            }
            __syncwarp();
            if (group) ++of[1]; else ++of[0];
          }
        }
        if (!__all_sync(0xffffffffu, ok)) failed = true;
        // (nothing else holds an item without tiles back until this warp has seen its queries' phase)
        if (!failed && lane == 0) mbar_arrive(smem_u32(&sm.done[at]));
        pass(x);
      }
    } else if (warp == kValueWarp) {
      // ---- O^T of a tile, once its group's weights are there; its completion gives the stage back ----
      constexpr uint32_t kIdesc = (1u << 4) | (1u << 15) | (1u << 16) | (static_cast<uint32_t>(kN >> 3) << 17) | (static_cast<uint32_t>(128 >> 4) << 24);
#pragma unroll 1
      for (int it = 0; it < items && !failed; ++it) {
        const unsigned at = buffer();
        if (!__all_sync(0xffffffffu, wait_for(smem_u32(&sm.q_full[at]), phase()))) { failed = true; break; }
        const Item x = sm.list[it];
#pragma unroll 1
        for (int j = 0; j < x.tiles; ++j) {
          const int group = group_of(x, j);
          const unsigned h = 2 * (done_tiles + j) + 1, slot = h % kSlots, mine = (group ? done_of[1] : done_of[0]) + j / 2;
          if (!__all_sync(0xffffffffu, wait_for(smem_u32(&sm.full[slot]), (h / kSlots) & 1) && wait_for(smem_u32(&sm.p_ready[group][mine & 1]), (mine >> 1) & 1))) { failed = true; break; }
          tcgen05_after_sync();
          const uint64_t v_desc = umma_desc(smem_u32(sm.ring[slot]), kTileBytes, 1024), p_desc = piece_desc(smem_u32(sm.p[group][mine & 1]), 128, kTile * 16);
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              code_product(tmem + kOutputs + (at * kGroups + group) * 64, v_desc + static_cast<uint64_t>(ks * 4096 >> 4), p_desc + static_cast<uint64_t>(ks * 32 * 16 >> 4), kIdesc,
                           (j >= 2 || ks > 0) ? 1u : 0u);
            umma_commit(smem_u32(&sm.o_done[group][mine & 1]));
            umma_commit(smem_u32(&sm.empty[slot]));
          }
          __syncwarp();
        }
        // (an item without all of its products is never done: the result warps give up on it and leave NaN)
        if (!failed && elect_one()) umma_commit(smem_u32(&sm.done[at]));
        __syncwarp();
        pass(x);
      }
    } else if (warp >= kQueryWarp && warp < kQueryWarp + kQueryWarps) {
      // ---- the queries of an item in three parts, half of the rows each; what its rows see ----
      const int first_row = (warp - kQueryWarp) * (kRows / kQueryWarps);
#pragma unroll 1
      for (int it = 0; it < items && !failed; ++it) {
        const Item x = sm.list[it];
        const unsigned buf = buffer();
        // Twice: result warps that are waiting give up themselves meanwhile and go on, so every item gets the places where their NaN goes.
        const uint32_t empty = smem_u32(&sm.q_empty[buf]), before = phase() ^ 1;
        if (done_items >= kDeep && !__all_sync(0xffffffffu, wait_for(empty, before) || wait_for(empty, before))) { failed = true; break; }
        constexpr int kMine = kDim / 32;            // elements of a lane
        // lane r has row r's place in the item
        const int my_head = x.unit * kHeads + lane % kRows / kEach, my_pair = x.pair0 + lane % kEach, my_row = my_pair / group_heads;
        const bool my_live = lane % kEach < x.pairs && my_head < c.kv_heads;
        const int64_t head = static_cast<int64_t>(my_head) * group_heads + my_pair - my_row * group_heads, at_row = x.first + my_row;
        const int64_t my_source = my_live ? at_row * a.q_stride + head * kDim : -1;
        // all rows on their way at once, a lane's kMine elements of each
#pragma unroll 1
        for (int r = first_row; r < first_row + kRows / kQueryWarps; ++r) {
          const int64_t source = __shfl_sync(0xffffffffu, my_source, r);
          const T* src = static_cast<const T*>(a.q) + (source < 0 ? 0 : source) + lane * kMine;
          asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(smem_u32(&sm.raw_q[r][lane * (kMine / 2)])), "l"(src), "n"(kMine * 2), "r"(source < 0 ? 0 : kMine * 2) : "memory");
        }
        asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
        __syncwarp();
#pragma unroll 1
        for (int r = first_row; r < first_row + kRows / kQueryWarps; ++r) {
          {
            uint32_t raw[kMine / 2];
#pragma unroll
            for (int w = 0; w < kMine / 2; ++w) raw[w] = sm.raw_q[r][lane * (kMine / 2) + w];
            float v[kMine];
            uint32_t top = 0;
#pragma unroll
            for (int w = 0; w < kMine; ++w) {
              v[w] = Elem<T>::to_float(reinterpret_cast<const T*>(raw)[w]);
              top = max(top, static_cast<uint32_t>(__float_as_int(v[w])) & 0x7fffffffu);
            }
            top = __reduce_max_sync(0xffffffffu, top);
            const bool odd = top >= 0x7f800000u;    // a row with an element that is not finite has no scores that are: its references, and so its output, become NaN
            const int e = top > 0 && !odd ? max(static_cast<int>(top >> 23) - 127 - 7, -126) : 0;
            const float up = odd ? 0.0f : power_of_two(-e);
            if (lane == 0) sm.row_scale[buf][r] = odd ? NAN : scale_log2 * power_of_two(e);
            uint32_t codes[kMine / 2][3];
#pragma unroll
            for (int w = 0; w < kMine / 2; ++w) three_parts(odd ? 0.0f : v[2 * w] * up, odd ? 0.0f : v[2 * w + 1] * up, codes[w]);
            // element lane * kMine of a 128-byte line whose 16-byte pieces are swizzled by the line; of two heads, each has a half of a line
            const int byte = r / kEach * kDim + lane * kMine;
#pragma unroll
            for (int part = 0; part < 3; ++part) {
              const int line = part * kEach + r % kEach;
              const uint32_t at = smem_u32(sm.q[buf]) + line * 128 + (byte ^ ((line & 7) << 4));
              if constexpr (kDim == 128) {
                asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(codes[0][part] | codes[kMine / 2 - 1][part] << 16) : "memory");
              } else {
                asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(static_cast<uint16_t>(codes[0][part])) : "memory");
              }
            }
          }
        }
        if (first_row == 0 && lane < kRows) {
          const int sees = clamp_keys(x.base + my_row, capacity), low = a.window > 0 ? max(sees - a.window, 0) : 0;
          const int first_part = part_of(low, a.window), last_part = sees > 0 ? part_of(sees - 1, a.window) : first_part;
          sm.keys[buf][lane] = my_live ? min(sees, x.end) : x.end;          // of the part; rows that are none see all of it, and nothing is masked for them
          sm.low[buf][lane] = my_live ? max(low, x.from) : x.from;
          int kind = kNowhere;
          if (my_live && x.part >= first_part && x.part <= last_part) kind = first_part < last_part ? kPartial : (sees > low ? kOutput : kZero);
          sm.kind[buf][lane] = kind;
          sm.to[buf][lane] = kind == kPartial ? (((at_row - a.step.row0) * a.q_heads + head) * a.parts + x.part - first_part) * partial_stride(kDim) : at_row * a.out_stride + head * kDim;
        }
        fence_async_proxy();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.q_full[buf]));
        pass(x);
      }
    } else if (warp >= kResultWarp) {
      // ---- results: an element of the values per thread; both groups' parts added up ----
      const int own = threadIdx.x & (kTile - 1), row = lane % kRows;
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
#pragma unroll 1
      for (int it = 0; it < items; ++it) {
        const unsigned buf = buffer();
        if (!failed && !wait_for(smem_u32(&sm.done[buf]), phase())) failed = true;
        failed = __any_sync(0xffffffffu, failed);
        tcgen05_after_sync();
        const Item x = sm.list[it];
        const bool has0 = tiles_of(x, 0) > 0, has1 = tiles_of(x, 1) > 0;
        // a lane has a row's factors: 2^(R - max R) of each group, over the joined sum where this is the row's only part
        const int kind = sm.kind[buf][row];
        const int64_t to = sm.to[buf][row];
        {
          const float ref0 = has0 ? sm.ref[buf][0][row] : -INFINITY, ref1 = has1 ? sm.ref[buf][1][row] : -INFINITY;
          const float big = fmaxf(ref0, ref1), zero = big == -INFINITY ? 0.0f : big;
          const float root0 = fast_exp2(0.5f * (ref0 - zero)), root1 = fast_exp2(0.5f * (ref1 - zero));
          float sum = 0.0f;
          if (has0) sum = ((sm.l[buf][0][0][row] + sm.l[buf][0][1][row]) + (sm.l[buf][0][2][row] + sm.l[buf][0][3][row])) * root0 * root0;
          if (has1) sum += ((sm.l[buf][1][0][row] + sm.l[buf][1][1][row]) + (sm.l[buf][1][2][row] + sm.l[buf][1][3][row])) * root1 * root1;
          const float scale = failed ? NAN : (kind == kPartial ? 1.0f : (kind == kOutput ? __frcp_rn(sum) : 0.0f));
          const uint64_t at = kind == kPartial ? reinterpret_cast<uint64_t>(a.partials + to) : reinterpret_cast<uint64_t>(static_cast<T*>(a.out) + to);
          if (lane < kRows)
            sm.result[warp & 3][row] = make_float4(root0 * root0 * scale, root1 * root1 * scale, __uint_as_float(static_cast<uint32_t>(at)), __uint_as_float(static_cast<uint32_t>(at >> 32)));
          if (kind == kPartial && lane < kRows && (warp & 3) == 0) *reinterpret_cast<float2*>(a.partials + to + kDim) = make_float2(big, sum);
        }
        const uint32_t partial = __ballot_sync(0xffffffffu, kind == kPartial), nowhere = __ballot_sync(0xffffffffu, kind == kNowhere);
        const bool marked = (sm.marked[buf][0] | sm.marked[buf][1]) != 0;
        __syncwarp();
        const uint32_t outputs0 = tmem + lanes + kOutputs + (buf * kGroups) * 64, outputs1 = outputs0 + 64;
#pragma unroll 1
        for (int r0 = 0; r0 < kRows; r0 += 4) {
          if (((nowhere >> r0) & 15) == 15) continue;
          const int d = kHeads == 2 ? own - 64 * (r0 / kEach) : own;      // of two heads, a thread's element may be the other one's
          float acc0[4], m0[4], rest0[4], acc1[4], m1[4], rest1[4];
          load_columns<4>(outputs0 + r0, acc0);
          load_columns<4>(outputs0 + kRows + r0, m0);
          load_columns<4>(outputs0 + 2 * kRows + r0, rest0);
          load_columns<4>(outputs1 + r0, acc1);
          load_columns<4>(outputs1 + kRows + r0, m1);
          load_columns<4>(outputs1 + 2 * kRows + r0, rest1);
          tmem_load_wait();
          if (kHeads == 2 && (d < 0 || d >= kDim)) continue;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int r = r0 + k;
            const float4 of = load_shared16f(smem_u32(&sm.result[warp & 3][r]));
            const float o0 = fmaf(fmaf(rest0[k], 0.03125f, m0[k]), 0.03125f, acc0[k]), o1 = fmaf(fmaf(rest1[k], 0.03125f, m1[k]), 0.03125f, acc1[k]);
            float value = has0 ? o0 * of.x : 0.0f;                         // (a group without tiles has left nothing there)
            if (has1) value = fmaf(o1, of.y, value);
            if (marked && ((sm.nan_value[buf][0][r][own >> 5] | sm.nan_value[buf][1][r][own >> 5]) >> (own & 31)) & 1) value = NAN;
            const uint64_t at = static_cast<uint64_t>(__float_as_uint(of.z)) | static_cast<uint64_t>(__float_as_uint(of.w)) << 32;
            if ((partial >> r) & 1) reinterpret_cast<float*>(at)[d] = value;
            else if (!((nowhere >> r) & 1)) reinterpret_cast<T*>(at)[d] = Elem<T>::from_float(value);
          }
        }
        tcgen05_before_sync();
        if (marked) {
          asm volatile("bar.sync 3, 128;" ::: "memory");                   // the four warps have read them
          if (own < kGroups * kRows)
            *reinterpret_cast<uint4*>(&sm.nan_value[buf][own / kRows][own % kRows][0]) = make_uint4(0u, 0u, 0u, 0u);
          if (own < kGroups) sm.marked[buf][own] = 0;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.q_empty[buf]));
        pass(x);
      }
    }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Role::kSoftmaxRegisters));
#pragma unroll 1
    for (int batch = 0, base = 0, total = 0; batch < a.step.sequences; base += kList) {
      if (base == 0) total = lay_out(batch);
      else block_sync();
      const int items = items_of(base, total);
      block_sync();
      if (items < kList) { batch += kBatch; base = -kList; }
      // ---- softmax: a thread has a token and all or half of the rows (of two heads then: one head's) ----
      constexpr int kMine = Role::kMine, kOfHead = kHeads == 2 && kHalves == 1 ? kEach : kMine;       // rows of a thread that share a head's scales
      const int group = warp / kGroupWarps, half = kHalves == 2 ? (warp >> 2) & 1 : 0, own = threadIdx.x & (kTile - 1), row0 = half * kMine;
      const int waits = warp % kGroupWarps;        // what this warp waits for in its group
      const uint32_t lanes = (static_cast<uint32_t>((warp & 3) * 32) << 16) + group * 64;      // and columns
      const uint32_t scores_at = tmem + lanes + kScores + (kHeads == 2 ? half * 32 : row0);
      // a part of this thread's scores (of two heads' rows, half are the other head's)
      auto load_scores = [&](int part, float (&x)[kMine]) {
        load_columns<kOfHead>(scores_at + part * kEach, x);
        if constexpr (kOfHead < kMine) load_columns<kOfHead, kOfHead>(scores_at + 32 + part * kEach, x);
      };
      // where this thread's weights go: its token's line of 16 bytes, a half's eight of them
      const uint32_t first_weights = smem_u32(sm.p[group][0]) + own * 16 + half * 8;
      const int folded_row = row0 + row_after_fold<kMine>(lane);
      const bool folds = lane % (32 / kMine) == 0;
#pragma unroll 1
      for (int it = 0; it < items; ++it) {
        const unsigned buf = buffer();
        failed = group_any(group, failed || (waits == 0 && !wait_for(smem_u32(&sm.q_full[buf]), phase())));
        const Item x = sm.list[it];
        const uint32_t outputs_at = tmem + lanes + kOutputs + buf * kGroups * 64 + row0;
        const int mine = tiles_of(x, group);
        const unsigned before = group ? done_of[1] : done_of[0];
        float ref[kMine], l[kMine];
#pragma unroll
        for (int r = 0; r < kMine; ++r) { ref[r] = 0.0f; l[r] = 0.0f; }
        uint32_t fresh = (1u << kMine) - 1;          // rows without a reference yet
        if (own == 0) { sm.fresh[group][half] = fresh; sm.moved[group][half] = 0xffffffffu; }      // (read behind barriers)
        bool wide = false;                           // so has a tile had a scale beyond 2^+-kWide
#pragma unroll 1
        for (int k = 0; k < mine; ++k) {
          const int j = 2 * k + (group_of(x, 0) == group ? 0 : 1);
          const unsigned h = 2 * (done_tiles + j) + 1, turn = before + k, scale_slot = (done_tiles + j) % kScaleSlots;
          const int token0 = x.begin + j * kTile, token = token0 + own;
          // The tile's scales are there with its keys and its values.  Only the values can be waited for: they keep their place until this group's
          // weights have met them, while that of the keys may have been filled again (and its barrier be a whole turn on).
          // The product of the tile before the last is waited for as well (it has read the weights that this tile's replace).  A warp each waits for the
          // three, and all at the group's barrier, which costs no issue slots.
          bool ok = true;
          if (waits < 3 && !failed) {
            const uint32_t bar = waits == 0 ? smem_u32(&sm.s_ready[group]) : (waits == 1 ? smem_u32(&sm.full[h % kSlots]) : smem_u32(&sm.o_done[group][turn & 1]));
            ok = wait_for(bar, waits == 0 ? turn & 1 : (waits == 1 ? (h / kSlots) & 1 : ((turn >> 1) & 1) ^ 1));      // (before the first product: over)
          }
          if (group_any(group, !ok)) failed = true;
          tcgen05_after_sync();
          float s[kMine], m[kMine], rest[kMine];
          load_scores(0, s);
          load_scores(1, m);
          load_scores(2, rest);
          float4 scale_of[kMine / kOfHead];
#pragma unroll
          for (int h = 0; h < kMine / kOfHead; ++h) scale_of[h] = load_shared16f(smem_u32(&sm.scales[scale_slot][kHeads == 2 && kHalves == 2 ? half : h][own >> 4]));
          const uint2 any_wide = *reinterpret_cast<const uint2*>(sm.wide[scale_slot]);
          wide |= (any_wide.x | any_wide.y) != 0;
          tmem_load_wait();
          tcgen05_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sm.s_free[group]));
#pragma unroll
          for (int r = 0; r < kMine; r += 4) {
            const float4 row_scale = load_shared16f(smem_u32(&sm.row_scale[buf][row0 + r]));
            const float2 part = make_float2(0.03125f, 0.03125f);
#pragma unroll
            for (int i2 = 0; i2 < 4; i2 += 2) {
              const float4& scale = scale_of[(r + i2) / kOfHead];
              const float2 keys_scale = make_float2(scale.x, scale.x), exponent = make_float2(scale.y, scale.y);
              float2 raw = fma_pair(make_float2(rest[r + i2], rest[r + i2 + 1]), part, make_float2(m[r + i2], m[r + i2 + 1]));
              raw = fma_pair(raw, part, make_float2(s[r + i2], s[r + i2 + 1]));
              const float2 factor = mul_pair(i2 ? make_float2(row_scale.z, row_scale.w) : make_float2(row_scale.x, row_scale.y), keys_scale);
              raw = fma_pair(raw, factor, sub_pair(exponent, make_float2(ref[r + i2], ref[r + i2 + 1])));
              s[r + i2] = raw.x;
              s[r + i2 + 1] = raw.y;
            }
          }
          const bool ragged = token0 + kTile > x.all_end || token0 < x.all_from;
          if (ragged) {
#pragma unroll
            for (int r = 0; r < kMine; ++r)
              if (token >= sm.keys[buf][row0 + r] || token < sm.low[buf][row0 + r]) s[r] = -INFINITY;
          }
          float top = fmaxf(s[0], s[1]);
#pragma unroll
          for (int r = 2; r < kMine; r += 2) top = max3(top, s[r], s[r + 1]);
          // (the first tile, and rows that have not seen a key: always; the other half's rows need it as well)
          if (group_any(group, top > kHighest || fresh != 0)) {
#pragma unroll
            for (int r = 0; r < kMine; r += 4) {
              const float4 most = make_float4(warp_max(s[r]), warp_max(s[r + 1]), warp_max(s[r + 2]), warp_max(s[r + 3]));
              if (lane == 0) *reinterpret_cast<float4*>(&sm.folded[group][warp & 3][row0 + r]) = most;
            }
            group_any(group, false);
            if (own < kMine) {                     // a row each
              const int r = row0 + own;
              const float most = fmaxf(fmaxf(sm.folded[group][0][r], sm.folded[group][1][r]), fmaxf(sm.folded[group][2][r], sm.folded[group][3][r]));
              const bool first = (fresh >> own) & 1, move = most > (first ? -INFINITY : kHighest);
              const float by = move ? most - kFresh : 0.0f;
              sm.by[group][r] = by;
              sm.root[group][r] = move ? (first ? 0.0f : fast_exp2(-0.5f * by)) : 1.0f;     // 0: there is nothing yet
              if (move && first) atomicAnd(&sm.fresh[group][half], ~(1u << own));
              if (move && !first) sm.moved[group][half] = turn;
            }
            group_any(group, false);
            fresh = sm.fresh[group][half];
#pragma unroll
            for (int r = 0; r < kMine; r += 4) {
              const float4 by = load_shared16f(smem_u32(&sm.by[group][row0 + r])), root = load_shared16f(smem_u32(&sm.root[group][row0 + r]));
              ref[r] += by.x; ref[r + 1] += by.y; ref[r + 2] += by.z; ref[r + 3] += by.w;
              s[r] -= by.x; s[r + 1] -= by.y; s[r + 2] -= by.z; s[r + 3] -= by.w;
              // in two steps: where a page of far larger values moved the reference, the whole factor may be 0 in fp32 and l not
              l[r] = l[r] * root.x * root.x; l[r + 1] = l[r + 1] * root.y * root.y; l[r + 2] = l[r + 2] * root.z * root.z; l[r + 3] = l[r + 3] * root.w * root.w;
            }
            const bool moves = sm.moved[group][half] == turn;
            if (moves && k > 0) {                  // the same for the warps of a half; the output is at rest once the product before is complete
              if (!failed && !wait_for(smem_u32(&sm.o_done[group][(turn - 1) & 1]), ((turn - 1) >> 1) & 1)) failed = true;
              __syncwarp();
              tcgen05_after_sync();
#pragma unroll 1
              for (int part = 0; part < 3; ++part) {
                float o[kMine];
                load_columns<kMine>(outputs_at + part * kRows, o);
                tmem_load_wait();
#pragma unroll
                for (int r = 0; r < kMine; ++r) o[r] *= sm.root[group][row0 + r] * sm.root[group][row0 + r];
                store_columns<kMine>(outputs_at + part * kRows, o);
              }
              tmem_store_wait();
              tcgen05_before_sync();
            }
          }
          const uint32_t weights = first_weights + (turn & 1) * (kN * 128);
          uint32_t codes[kMine / 2][3];
#pragma unroll
          for (int r = 0; r < kMine; r += 2) {
            const float4& scale = scale_of[r / kOfHead];
            float2 p;
            if (!wide) {
              p = make_float2(fast_exp2(s[r]), fast_exp2(s[r + 1]));
              const float2 sum = fma_pair(p, make_float2(scale.z, scale.z), make_float2(l[r], l[r + 1]));
              l[r] = sum.x;
              l[r + 1] = sum.y;
            } else {
              // a weight that is nothing beside the largest may still be a share of l, where its page's values are that much smaller
              const bool faint0 = s[r] < kFaint, faint1 = s[r + 1] < kFaint;
              p = make_float2(fast_exp2(faint0 ? s[r] - scale.y : s[r]), fast_exp2(faint1 ? s[r + 1] - scale.y : s[r + 1]));
              l[r] = fmaf(p.x, faint0 ? 1.0f : scale.z, l[r]);
              l[r + 1] = fmaf(p.y, faint1 ? 1.0f : scale.z, l[r + 1]);
              p = make_float2(faint0 ? 0.0f : p.x * scale.w, faint1 ? 0.0f : p.y * scale.w);
            }
            three_parts(p.x, p.y, codes[r / 2]);
          }
          // a part of this thread's rows: 4 or 8 bytes; of four rows all parts share a line, of eight rows two do
          uint32_t words[3][kMine / 4];
#pragma unroll
          for (int k3 = 0; k3 < 3; ++k3)
#pragma unroll
            for (int w = 0; w < kMine / 4; ++w) words[k3][w] = __byte_perm(codes[2 * w][k3], codes[2 * w + 1][k3], 0x5410);
          if constexpr (kRows == 4) {
            store_shared16(weights, make_uint4(words[0][0], words[1][0], words[2][0], 0u));
          } else if constexpr (kRows == 8) {
            store_shared16(weights, make_uint4(words[0][0], words[0][1], words[1][0], words[1][1]));
            store_shared8(weights + kTile * 16, make_uint2(words[2][0], words[2][1]));
          } else {
#pragma unroll
            for (int k3 = 0; k3 < 3; ++k3) store_shared8(weights + k3 * (kTile * 16), make_uint2(words[k3][0], words[k3][1]));
          }
          if (ragged) {
            // Slots that no row of the item sees may hold anything, and a weight of zero times NaN is NaN: they are cleared.  NaN in a token that some
            // rows see and others do not is cleared too, and kept for those that do.  (Of two threads of a token, each takes 64 bytes.)
            unsigned char* value = sm.ring[h % kSlots] + own * 128;
            const bool seen = token >= x.from && token < x.end;
#pragma unroll 1
            for (int b = 8 / kHalves * half; b < 8 / kHalves * (half + 1); ++b) {
              uint4* at = reinterpret_cast<uint4*>(value + ((b ^ (own & 7)) << 4));
              const uint4 w = *at;
              if (!seen) {
                *at = make_uint4(0u, 0u, 0u, 0u);
              } else if (nan_codes(w.x) | nan_codes(w.y) | nan_codes(w.z) | nan_codes(w.w)) {
                sm.marked[buf][group] = 1;
                uint32_t* words = reinterpret_cast<uint32_t*>(at);
#pragma unroll 1
                for (int k4 = 0; k4 < 4; ++k4) {
                  const uint32_t marks = nan_codes(words[k4]) >> 7;
                  const uint32_t bits = (marks & 1) | ((marks >> 7) & 2) | ((marks >> 14) & 4) | ((marks >> 21) & 8);
#pragma unroll 1
                  for (int r = 0; r < kRows; ++r)
                    if ((kHeads == 1 || r / kEach == b / 4) && token < sm.keys[buf][r] && token >= sm.low[buf][r])
                      atomicOr(&sm.nan_value[buf][group][r][b >> 1], bits << (16 * (b & 1) + 4 * k4));
                  words[k4] &= ~(marks * 0xffu);
                }
              }
            }
          }
          fence_async_proxy();
          tcgen05_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&sm.p_ready[group][turn & 1]));
        }

        // what the result warps need
        if (mine > 0) {
          const float total = fold_rows<kMine>(l, lane);
          if (folds) sm.l[buf][group][warp & 3][folded_row] = failed ? NAN : total;
          if (own == 0) {
#pragma unroll
            for (int r = 0; r < kMine; ++r)
              if ((fresh >> r) & 1) ref[r] = -INFINITY;
#pragma unroll
            for (int r = 0; r < kMine; r += 4) *reinterpret_cast<float4*>(&sm.ref[buf][group][row0 + r]) = make_float4(ref[r], ref[r + 1], ref[r + 2], ref[r + 3]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.done[buf]));
        pass(x);
      }
    }
  }
  // a wait that gave up left NaN in the rows of its item and of those behind it (a result warp's own, at the latest); copies still in flight land before the shared memory is given back
  if (failed && warp >= kCopyWarp && warp < kScoreWarp)
    for (int i = 0; i < kSlots; ++i)
      if (!wait_for(smem_u32(&sm.full[i]), 0) && !wait_for(smem_u32(&sm.full[i]), 1)) break;
  tcgen05_before_sync();
  __syncthreads();
  if (warp == kScoreWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kColumns) : "memory");
}

// ---- host ---------------------------------------------------------------------------------------
// A cache as [pages][tokens][bytes of all heads], in boxes of 128 bytes and `box` tokens, swizzled; heads behind the last read as zeros.
int make_code_map(CUtensorMap* map, const void* base, const QuantizedCache& c, int box) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (fn == nullptr) return RLT_ERR_UNSUPPORTED;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(c.kv_heads) * c.dim, static_cast<cuuint64_t>(c.block), static_cast<cuuint64_t>(c.num_pages)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(c.token_stride), static_cast<cuuint64_t>(c.block_stride)};
  const cuuint32_t in_box[3] = {128, static_cast<cuuint32_t>(box), 1}, element[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, in_box, element, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? RLT_OK : RLT_ERR_UNSUPPORTED;
}

template <typename T, int kDim, int kRows>
int launch(const QuantizedAttentionArgs& a, cudaStream_t stream) {
  const QuantizedCache& c = a.cache;
  DeviceInfo info;
  int status = current_device_info(&info);
  if (status != RLT_OK) return status;
  int box = 16;                                     // tokens of a copy: as many as a page and a tile share
  while (box < kTile && c.block % (2 * box) == 0) box *= 2;
  CUtensorMap key_map, value_map;
  if (make_code_map(&key_map, c.key, c, box) != RLT_OK || make_code_map(&value_map, c.value, c, box) != RLT_OK) return RLT_ERR_UNSUPPORTED;
  constexpr size_t smem = sizeof(Shared<kRows>) + 1024;
  static_assert(smem <= 227 * 1024, "shared memory of a block");
  auto kernel = quantized_tiles_kernel<T, kDim, kRows>;
  RLT_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  return launch_dependent("quantized_tiles_kernel", kernel, dim3(static_cast<unsigned>(info.sm_count)), dim3(Roles<kRows>::kThreads), smem, stream, key_map, value_map, a,
                          static_cast<float>(1.4426950408889634 * a.scale), box);
}

template <typename T>
int launch_for(const QuantizedAttentionArgs& a, int max_new, cudaStream_t stream) {
  // Rows of an item: the fewest that a portion's fit in (two heads of 64 share an item's rows).
  const int64_t pairs = static_cast<int64_t>(max_new) * (a.q_heads / a.cache.kv_heads) * (128 / a.cache.dim);
  if (a.cache.dim == 128) return pairs <= 4 ? launch<T, 128, 4>(a, stream) : (pairs <= 8 ? launch<T, 128, 8>(a, stream) : launch<T, 128, 16>(a, stream));
  return pairs <= 8 ? launch<T, 64, 8>(a, stream) : launch<T, 64, 16>(a, stream);
}

}  // namespace

bool quantized_tiles_supported(const QuantizedAttentionArgs& a) {
  const QuantizedCache& c = a.cache;
  if (a.dtype == RLT_F32 || (c.dim != 64 && c.dim != 128) || c.block % 16 != 0 || c.num_pages < 1 || c.num_pages > 0x7fffffff) return false;
  if (c.token_stride % 16 != 0 || c.block_stride % 16 != 0 || !aligned16(c.key) || !aligned16(c.value)) return false;
  if (a.q_stride % 4 != 0 || (reinterpret_cast<uintptr_t>(a.q) & 7u) != 0) return false;
  const int64_t group = a.q_heads / c.kv_heads, tiles = (static_cast<int64_t>(a.step.total) * group + 3) / 4 + a.step.sequences;
  return tiles * c.kv_heads * a.parts <= 0x7fffffff && static_cast<int64_t>(a.step.total) * group <= (1 << 25);     // items are counted in 32 bits, a sequence's row tiles in 24
}

int launch_quantized_tiles(const QuantizedAttentionArgs& a, int max_new, cudaStream_t stream) {
  if (a.dtype == RLT_BF16) return launch_for<__nv_bfloat16>(a, max_new, stream);
  return launch_for<__half>(a, max_new, stream);
}

}  // namespace rlt
