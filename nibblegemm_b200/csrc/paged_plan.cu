// Plan of one step over a paged KV cache, built on the GPU from the requests'
// lengths, so that a serving loop (or a CUDA graph of it) never reads them back:
//   blocks[b] = ceil((cached[b] + new[b]) / page)
//   need[b]   = max(0, blocks[b] - held[b]) pages to take; 0 if the blocks do not fit the
//               table's row: such a request gets nothing, and its pages are left to the others
//   off       = exclusive prefix sum of need over the requests, in order
//   granted b : the blocks fit, and need[b] == 0 or off[b] + need[b] <= free pages left
//   table[b, held[b] + i] = free[cursor + off[b] + i]
//   slot(b, i) = table[b, (cached + i) / page] * page + (cached + i) % page
//   position(b, i) = cached[b] + depth of node i (no tree: + i)
//   mask(b, i) : bit j set iff node j is an ancestor of node i, or i itself
//
// Every CTA scans the lengths itself (a few loads per thread; the alternative,
// a scan kernel and a second launch, costs more than re-reading 12 B per
// request from L2) and keeps both prefix sums in shared memory; a token or a
// fresh page then finds its request by binary search there.
//
// Bound: without trees, the launch and three dependent rounds of loads (lengths, table, free
// pages): 1000 requests with 32,000 new tokens 5.0 us on a B200; the bytes alone would take 0.05 us.
// With trees, the walk to the root: one dependent load for every level above a node.  16 trees of
// 32 nodes take 4.1 us (random ones) or 6.1 (chains, 31 levels), 16 chains of 64 nodes 8.6, 4
// of 512 59 and one of 4096 506 us; one node with 4095 children 11.7.
#include <algorithm>
#include <mutex>

#include "paged_common.cuh"

namespace ngb {
namespace {

constexpr int kPlanThreads = 256;
constexpr int kPlanMostTokens = (1 << 30) - 1;  // cached or new, of a request: their sum is an int
constexpr int kPlanMaxBatch = 16384;  // two int prefix sums per request: 128 KB of shared memory

struct PlanArgs {
  const int* cached;
  const int* new_lens;
  const int* held;
  int* table;
  long long table_stride;
  int table_width;
  const int* free_pages;
  int num_free;
  const int* cursor;
  const int* parents;
  int B, tokens, page_shift, mask_words;
  int* cu_new;
  int* slots;
  int* positions;
  int* kv_lens;
  int* held_out;
  int* taken;
  unsigned long long* mask;
  unsigned int* err;
};

// Last index b in [0, B) with prefix[b] <= x (prefix is non-decreasing, prefix[0] = 0 <= x).
__device__ __forceinline__ int find_request(const int* prefix, int B, int x) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

struct Pair {
  long long a, b;
};

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PlanArgs p) {
  extern __shared__ int plan_smem[];
  int* cu = plan_smem;             // [B + 1] tokens before request b
  int* ends = plan_smem + p.B + 1; // [B + 1] pages needed before request b
  __shared__ Pair warp_sum[kPlanThreads / 32];
  __shared__ int taken_s;
  pdl_launch_next();
  pdl_wait_previous();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int B = p.B, ps = 1 << p.page_shift;
  const int used = p.cursor ? min(max(*p.cursor, 0), p.num_free) : 0;
  const int available = p.num_free - used;

  auto lengths = [&](int b, int& cached, int& fresh, int& held, int& blocks, int& need) {
    cached = p.cached[b];
    fresh = p.new_lens[b];
    held = p.held[b];
    if (cached < 0 || fresh < 0 || held < 0 || cached > kPlanMostTokens || fresh > kPlanMostTokens) {
      atomicOr(p.err, kErrBadIndex);
      cached = min(max(cached, 0), kPlanMostTokens);
      fresh = min(max(fresh, 0), kPlanMostTokens);
      held = max(held, 0);
    }
    // (rounded up without a sign: the sum may lie less than a page below 2^31)
    blocks = static_cast<int>((static_cast<unsigned>(cached + fresh) + ps - 1) >> p.page_shift);
    need = blocks <= p.table_width ? max(0, blocks - held) : 0;
  };

  // ---- both prefix sums: a contiguous run of requests per thread
  const int per = (B + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(B, tid * per), b1 = min(B, b0 + per);
  Pair mine = {0, 0};
  for (int b = b0; b < b1; ++b) {
    int cached, fresh, held, blocks, need;
    lengths(b, cached, fresh, held, blocks, need);
    mine.a += fresh;
    mine.b += need;
  }
  Pair inc = mine;
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, inc.a, o), b = __shfl_up_sync(0xffffffffu, inc.b, o);
    if (lane >= o) {
      inc.a += a;
      inc.b += b;
    }
  }
  if (lane == 31) warp_sum[warp] = inc;
  if (tid == 0) taken_s = 0;
  __syncthreads();
  Pair run = {inc.a - mine.a, inc.b - mine.b};
  for (int w = 0; w < warp; ++w) {
    run.a += warp_sum[w].a;
    run.b += warp_sum[w].b;
  }
  const bool first = blockIdx.x == 0;
  int taken = 0;
  // Sums past the capacity (an error, flagged) or past 2^31 are held at a bound
  // that still reads as "beyond the end".
  auto clip = [](long long v, long long top) { return static_cast<int>(v < top ? v : top); };
  for (int b = b0; b < b1; ++b) {
    int cached, fresh, held, blocks, need;
    lengths(b, cached, fresh, held, blocks, need);
    cu[b] = clip(run.a, p.tokens);
    ends[b] = clip(run.b, 0x7fffffff);
    const bool granted = (need == 0 || run.b + need <= available) && blocks <= p.table_width;
    run.a += fresh;
    run.b += need;
    if (granted && need) taken = max(taken, clip(run.b, available));
    if (first) {
      p.cu_new[b] = cu[b];
      p.kv_lens[b] = granted ? cached + fresh : 0;
      p.held_out[b] = granted ? max(held, blocks) : held;
    }
    if (b == B - 1) {
      cu[B] = clip(run.a, p.tokens);
      ends[B] = clip(run.b, 0x7fffffff);
      if (first) {
        p.cu_new[B] = cu[B];
        if (run.a > p.tokens) atomicOr(p.err, kErrBadIndex);
      }
    }
  }
  if (taken) atomicMax(&taken_s, taken);
  __syncthreads();
  if (first && tid == 0) *p.taken = taken_s;

  const int stride = gridDim.x * kPlanThreads, start = blockIdx.x * kPlanThreads + tid;
  // ---- fresh pages into the table
  const int fresh_pages = min(ends[B], available);
  for (int j = start; j < fresh_pages; j += stride) {
    const int b = find_request(ends, B, j);
    int cached, fresh, held, blocks, need;
    lengths(b, cached, fresh, held, blocks, need);
    if (ends[b] + need > available) continue;  // not granted
    const int col = held + j - ends[b];
    p.table[static_cast<size_t>(b) * p.table_stride + col] = p.free_pages[used + j];
  }
  // ---- tokens
  const int total = cu[B];
  for (int t = start; t < p.tokens; t += stride) {
    if (t >= total) {  // rows beyond the last request's tokens
      p.slots[t] = -1;
      p.positions[t] = 0;
      for (int w = 0; w < p.mask_words; ++w) p.mask[static_cast<size_t>(t) * p.mask_words + w] = 0;
      continue;
    }
    const int b = find_request(cu, B, t);
    const int i = t - cu[b];
    int cached, fresh, held, blocks, need;
    lengths(b, cached, fresh, held, blocks, need);
    const bool granted =
        (need == 0 || static_cast<long long>(ends[b]) + need <= available) && blocks <= p.table_width;
    int slot = -1;
    if (granted) {
      const int at = cached + i, blk = at >> p.page_shift;
      const int page = blk < held ? p.table[static_cast<size_t>(b) * p.table_stride + blk]
                                  : p.free_pages[used + ends[b] + blk - held];
      if (page < 0 || page > (0x7fffffff >> p.page_shift))
        atomicOr(p.err, kErrBadIndex);
      else
        slot = (page << p.page_shift) + (at & (ps - 1));
    }
    p.slots[t] = slot;
    if (!p.parents) {
      p.positions[t] = cached + i;
      continue;
    }
    // Walk to the root: a parent's index is below its child's, so the walk ends.
    int depth = 0;
    unsigned long long bits = 0;
    int word = i >> 6;
    if (p.mask_words) {
      if (word >= p.mask_words) atomicOr(p.err, kErrBadIndex);
      for (int w = word + 1; w < p.mask_words; ++w) p.mask[static_cast<size_t>(t) * p.mask_words + w] = 0;
    }
    for (int node = i;;) {
      if ((node >> 6) != word) {  // bits of a lower word: this one is complete
        if (word < p.mask_words) p.mask[static_cast<size_t>(t) * p.mask_words + word] = bits;
        for (int w = word - 1; w > (node >> 6); --w)
          if (w < p.mask_words) p.mask[static_cast<size_t>(t) * p.mask_words + w] = 0;
        word = node >> 6;
        bits = 0;
      }
      bits |= 1ull << (node & 63);
      int up = p.parents[cu[b] + node];
      if (up >= node || up < -1) {  // not a tree in topological order
        atomicOr(p.err, kErrBadIndex);
        up = -1;
      }
      if (up < 0) break;
      node = up;
      ++depth;
    }
    if (word < p.mask_words) p.mask[static_cast<size_t>(t) * p.mask_words + word] = bits;
    for (int w = word - 1; w >= 0; --w)
      if (w < p.mask_words) p.mask[static_cast<size_t>(t) * p.mask_words + w] = 0;
    p.positions[t] = cached + depth;
  }
}

}  // namespace
}  // namespace ngb

extern "C" int ng_paged_plan(const int* cached, const int* new_lens, const int* held, int* block_table,
                             long long table_stride, int table_width, const int* free_pages, int num_free,
                             const int* cursor, const int* parents, int B, int num_tokens, int page_size,
                             int mask_words, int* cu_new, int* slots, int* positions, int* kv_lens,
                             int* held_out, int* taken, long long* mask, void* stream) {
  using namespace ngb;
  if (!cached || !new_lens || !held || !block_table || !cu_new || !kv_lens || !held_out || !taken)
    return NG_ERR_NULL_POINTER;
  if (num_tokens > 0 && (!slots || !positions)) return NG_ERR_NULL_POINTER;
  if (num_free > 0 && !free_pages) return NG_ERR_NULL_POINTER;
  if (mask_words > 0 && num_tokens > 0 && (!parents || !mask)) return NG_ERR_NULL_POINTER;
  if (B < 1 || B > kPlanMaxBatch || num_tokens < 0 || num_tokens > (1 << 30) || num_free < 0 ||
      table_width < 1 || table_stride < table_width || !page_size_ok(page_size))
    return NG_ERR_BAD_SHAPE;
  if (mask_words < 0 || mask_words > 64) return NG_ERR_BAD_ARGUMENT;
  DeviceInfo dev;
  if (int st = current_device_info(&dev)) return st;
  const size_t smem = 2 * (static_cast<size_t>(B) + 1) * sizeof(int);
  static std::once_flag once[kMaxDevices];
  std::call_once(once[dev.device], [] {
    cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         2 * (kPlanMaxBatch + 1) * static_cast<int>(sizeof(int)));
  });
  const PlanArgs a{cached, new_lens, held, block_table, table_stride, table_width, free_pages, num_free, cursor,
                   parents, B, num_tokens, log2_of(page_size), mask_words, cu_new, slots, positions, kv_lens,
                   held_out, taken, reinterpret_cast<unsigned long long*>(mask), dev.err};
  const int grid = std::max(1, std::min(dev.sm_count, (num_tokens + kPlanThreads - 1) / kPlanThreads));
  return launch_chained(paged_plan_kernel, dim3(grid), dim3(kPlanThreads), smem,
                        static_cast<cudaStream_t>(stream), a);
}
