// Where a step's rows go, on the GPU: pages claimed from a stack of free ones, the block tables that grow by them, and the position and
// slot of every row; and the way back, pages that requests no longer need pushed onto the stack again.
//
//   before_s = sum of the counts in front of s            (rows of request s: before_s .. before_s + count_s - 1)
//   need_s   = max(ceil((length_s + count_s) / block) - held_s, 0), off_s its sum in front of s
//   page k of the step (k = off_s + j) = free_pages[free_count - 1 - k], entry held_s + j of request s
//
// One launch of one cluster.  Every CTA forms both sums over all requests for itself, in shared memory (n words each: cheaper than a
// second launch or a pass through global memory); the cluster's barrier then stands between the last read of the state and its first
// write, so the state is updated in place without a copy.  Entries and rows are dealt to all threads of the cluster, which find their
// request by a search in shared memory.  What bounds it is latency: two dependent reads, two block-wide barriers and one search.  The launch
// for a full house (1024 requests, 1 to 37 rows each, about 19500 rows) takes 9.3 us, giving the pages back 4.6; a step of 64 single rows 4.7 and
// 3.3.  A Python call of either is 19 us.
#include <cooperative_groups.h>

#include "common.cuh"

namespace rlt {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 1024;
constexpr int kMaxRequests = 8192;      // sums in shared memory: 96 KB

struct SlotArgs {
  const int32_t* lengths;
  const int32_t* counts;        // nullptr: pages are given back
  int requests;
  int32_t* tables;
  int width;
  int block;
  int32_t* held;                // nullptr: the tables are complete, nothing is claimed
  int32_t* free_pages;
  int free_capacity;
  int32_t* free_count;
  int rows;
  int32_t* cu;
  int32_t* new_lengths;
  int32_t* positions;
  int32_t* row_seq;
  int64_t* write_blocks;
  int64_t* write_offsets;
  int32_t* active_rows;
  int32_t* status;
};

// Exclusive sums over the block's threads of two numbers each, and their totals.
__device__ __forceinline__ void block_sums(long long& a, long long& b, long long& total_a, long long& total_b) {
  __shared__ long long s_a[kThreads / 32], s_b[kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long mine_a = a, mine_b = b;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const long long oa = __shfl_up_sync(0xffffffffu, a, x), ob = __shfl_up_sync(0xffffffffu, b, x);
    if (lane >= x) { a += oa; b += ob; }
  }
  if (lane == 31) { s_a[warp] = a; s_b[warp] = b; }
  __syncthreads();
  long long wa = s_a[lane], wb = s_b[lane];
  total_a = wa; total_b = wb;
  if (lane >= warp) { wa = 0; wb = 0; }
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) {
    total_a += __shfl_xor_sync(0xffffffffu, total_a, x);
    total_b += __shfl_xor_sync(0xffffffffu, total_b, x);
    wa += __shfl_xor_sync(0xffffffffu, wa, x);
    wb += __shfl_xor_sync(0xffffffffu, wb, x);
  }
  a += wa - mine_a;
  b += wb - mine_b;
}

// The last i < n with sums[i] <= x; sums[0] = 0 <= x.
__device__ __forceinline__ int last_at_or_below(const int* sums, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// Pages that hold the first `tokens` tokens; a length below zero holds none.
__device__ __forceinline__ int pages_of(int tokens, int block) { return tokens <= 0 ? 0 : (tokens - 1) / block + 1; }

__global__ void __launch_bounds__(kThreads, 1)
step_slots_kernel(SlotArgs a) {
  extern __shared__ int s_words[];
  int *before = s_words, *off = before + a.requests, *held = off + a.requests;
  const cg::cluster_group cluster = cg::this_cluster();
  const int n = a.requests, per = (n + kThreads - 1) / kThreads, begin = threadIdx.x * per, end = min(begin + per, n);
  const long long capacity = static_cast<long long>(a.width) * a.block;
  const int available = a.held == nullptr ? 0 : *a.free_count;

  long long rows = 0, need = 0;
  int bad = available < 0 || available > a.free_capacity;
  for (int s = begin; s < end; ++s) {
    const int length = a.lengths[s], count = max(a.counts[s], 0);
    const long long after = static_cast<long long>(length) + count;
    bad |= length < 0 || after > capacity;
    rows += count;
    if (a.held != nullptr) {
      const int h = a.held[s];
      bad |= h < 0 || h > a.width;
      held[s] = h;
      need += max(pages_of(static_cast<int>(min(after, 0x7fffffffll)), a.block) - h, 0);
    }
  }
  long long total_rows, total_need;
  block_sums(rows, need, total_rows, total_need);
  const bool refused = __syncthreads_or(bad) != 0 || total_rows > a.rows || total_need > available;
  if (!refused) {
    for (int s = begin; s < end; ++s) {
      const int length = a.lengths[s], count = max(a.counts[s], 0);
      before[s] = static_cast<int>(rows);
      rows += count;
      if (a.held != nullptr) {
        off[s] = static_cast<int>(need);
        need += max(pages_of(length + count, a.block) - held[s], 0);
      }
    }
  }
  cluster.sync();                                       // all of the cluster have read the state (and see their own sums)

  const int at = cluster.block_rank() * kThreads + threadIdx.x, step = cluster.num_blocks() * kThreads;
  const int active = refused ? 0 : static_cast<int>(total_rows), claimed = refused ? 0 : static_cast<int>(total_need);
  for (int s = at; s < n; s += step) {
    const int length = a.lengths[s], count = refused ? 0 : max(a.counts[s], 0);
    a.cu[s] = refused ? 0 : before[s];
    a.new_lengths[s] = length + count;
    if (a.held != nullptr && !refused) a.held[s] = max(held[s], pages_of(length + count, a.block));
  }
  if (at == 0) {
    a.cu[n] = active;
    *a.active_rows = active;
    *a.status = refused ? 1 : 0;
    if (claimed > 0) *a.free_count = available - claimed;
  }
  for (int k = at; k < claimed; k += step) {
    const int s = last_at_or_below(off, n, k);
    a.tables[static_cast<int64_t>(s) * a.width + held[s] + k - off[s]] = a.free_pages[available - 1 - k];
  }
  for (int r = at; r < a.rows; r += step) {
    int position = 0, owner = -1, offset = 0;
    int64_t page = -1;
    if (r < active) {
      owner = last_at_or_below(before, n, r);
      position = a.lengths[owner] + r - before[owner];
      const int entry = position / a.block;
      offset = position - entry * a.block;
      // an entry of this step is taken from the stack, not from the table that other threads are filling
      page = a.held != nullptr && entry >= held[owner] ? a.free_pages[available - 1 - (off[owner] + entry - held[owner])]
                                                       : a.tables[static_cast<int64_t>(owner) * a.width + entry];
    }
    a.positions[r] = position;
    a.row_seq[r] = owner;
    a.write_blocks[r] = page;
    a.write_offsets[r] = offset;
  }
}

// Request s keeps the pages of its first lengths[s] tokens; page k of those given back (in the order of the requests and their tables)
// goes to place free_count + total - 1 - k, so that what was claimed last is claimed next, and claiming then giving back restores the stack.
__global__ void __launch_bounds__(kThreads, 1)
return_pages_kernel(SlotArgs a) {
  extern __shared__ int s_words[];
  int *off = s_words, *keep = off + a.requests;
  const cg::cluster_group cluster = cg::this_cluster();
  const int n = a.requests, per = (n + kThreads - 1) / kThreads, begin = threadIdx.x * per, end = min(begin + per, n);
  const int count = *a.free_count;
  long long given = 0, unused = 0;
  int bad = 0;
  for (int s = begin; s < end; ++s) {
    const int h = a.held[s];
    bad |= h < 0 || h > a.width;
    keep[s] = min(pages_of(a.lengths[s], a.block), h);
    given += h - keep[s];
  }
  long long total, unused_total;
  block_sums(given, unused, total, unused_total);
  const bool refused = __syncthreads_or(bad) != 0 || count < 0 || count + total > a.free_capacity;
  if (!refused) {
    for (int s = begin; s < end; ++s) {
      off[s] = static_cast<int>(given);
      given += a.held[s] - keep[s];
    }
  }
  cluster.sync();
  const int at = cluster.block_rank() * kThreads + threadIdx.x, step = cluster.num_blocks() * kThreads;
  if (at == 0) {
    *a.status = refused ? 1 : 0;
    if (!refused && total > 0) *a.free_count = count + static_cast<int>(total);
  }
  if (refused) return;
  for (int s = at; s < n; s += step) a.held[s] = keep[s];
  for (int k = at; k < static_cast<int>(total); k += step) {
    const int s = last_at_or_below(off, n, k);
    a.free_pages[count + static_cast<int>(total) - 1 - k] = a.tables[static_cast<int64_t>(s) * a.width + keep[s] + k - off[s]];
  }
}

// words: of shared memory for each request.
int launch(const char* what, void (*kernel)(SlotArgs), const SlotArgs& a, int words, int64_t work, cudaStream_t stream) {
  // The limit is the process's: always that of the most requests, so that no thread's call lowers what another is about to launch with (and whatever the
  // size, since without it the kernel's static memory counts against the usual 48 KB too).
  RLT_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, words * static_cast<int>(sizeof(int)) * kMaxRequests));
  const size_t smem = static_cast<size_t>(words) * sizeof(int) * a.requests;
  // Few rows are one CTA's work; a cluster's barrier costs more than a second pass over them.
  const unsigned ctas = work <= 2 * kThreads ? 1 : 8;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(ctas); config.blockDim = dim3(kThreads); config.dynamicSmemBytes = smem; config.stream = stream;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = ctas; attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute; config.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&config, kernel, a);
  if (err != cudaSuccess) {
    cudaGetLastError();
    set_last_error(what, err);
    return RLT_ERR_CUDA;
  }
  return RLT_OK;
}

}  // namespace
}  // namespace rlt

extern "C" RLT_API int rlt_step_slots(const int32_t* lengths, const int32_t* counts, int requests, int32_t* tables, int table_width, int block_size,
                                      int32_t* held, const int32_t* free_pages, int free_capacity, int32_t* free_count, int rows, int32_t* cu,
                                      int32_t* new_lengths, int32_t* positions, int32_t* row_seq, int64_t* write_blocks, int64_t* write_offsets,
                                      int32_t* active_rows, int32_t* status, rlt_stream_t stream) {
  using namespace rlt;
  RLT_REQUIRE(requests >= 0 && table_width >= 0 && block_size > 0 && rows >= 0 && free_capacity >= 0, "step_slots: invalid shape");
  RLT_REQUIRE(requests <= kMaxRequests, "step_slots: at most 8192 requests");
  RLT_REQUIRE(cu && active_rows && status && (requests == 0 || (lengths && counts && new_lengths)), "step_slots: null pointer");
  RLT_REQUIRE(requests == 0 || table_width == 0 || tables != nullptr, "step_slots: null pointer");
  RLT_REQUIRE(rows == 0 || (positions && row_seq && write_blocks && write_offsets), "step_slots: null pointer");
  RLT_REQUIRE(held == nullptr || (free_count && (free_capacity == 0 || free_pages)), "step_slots: held pages need the stack of free ones");
  RLT_REQUIRE(static_cast<int64_t>(table_width) * block_size <= 0x7fffffff, "step_slots: positions beyond 32 bits");
  SlotArgs a = {};
  a.lengths = lengths; a.counts = counts; a.requests = requests; a.tables = tables; a.width = table_width; a.block = block_size; a.held = held;
  a.free_pages = const_cast<int32_t*>(free_pages); a.free_capacity = free_capacity; a.free_count = free_count; a.rows = rows; a.cu = cu;
  a.new_lengths = new_lengths; a.positions = positions; a.row_seq = row_seq; a.write_blocks = write_blocks; a.write_offsets = write_offsets;
  a.active_rows = active_rows; a.status = status;
  return launch("step_slots_kernel", step_slots_kernel, a, 3, rows, static_cast<cudaStream_t>(stream));
}

extern "C" RLT_API int rlt_return_pages(const int32_t* lengths, int requests, const int32_t* tables, int table_width, int block_size, int32_t* held,
                                        int32_t* free_pages, int free_capacity, int32_t* free_count, int32_t* status, rlt_stream_t stream) {
  using namespace rlt;
  RLT_REQUIRE(requests >= 0 && table_width >= 0 && block_size > 0 && free_capacity >= 0, "return_pages: invalid shape");
  RLT_REQUIRE(requests <= kMaxRequests, "return_pages: at most 8192 requests");
  RLT_REQUIRE(free_count && status && (requests == 0 || (lengths && held)) && (requests == 0 || table_width == 0 || tables) &&
                  (free_capacity == 0 || free_pages), "return_pages: null pointer");
  SlotArgs a = {};
  a.lengths = lengths; a.requests = requests; a.tables = const_cast<int32_t*>(tables); a.width = table_width; a.block = block_size; a.held = held;
  a.free_pages = free_pages; a.free_capacity = free_capacity; a.free_count = free_count; a.status = status;
  return launch("return_pages_kernel", return_pages_kernel, a, 2, static_cast<int64_t>(requests) * 8, static_cast<cudaStream_t>(stream));
}
