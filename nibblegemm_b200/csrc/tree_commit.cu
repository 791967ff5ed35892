// Greedy acceptance of a drafted tree and the move of its cache rows.
//   path_0 = 0 (the request's last known token, the root);
//   path_{i+1} = the first child c of path_i with draft[c] == next[path_i];
//   the walk ends at a node without such a child, or at max_path nodes.
// Then, for every layer, cache row (before + i) <- row (before + path_i), with
// before = kv - n the rows in front of the tree: the kept nodes become the
// context's last rows and the rest is free to be written over.  path is
// increasing and path_i >= i, so a row that a move has written is never the source of a later
// move (path_j >= j > i): the rows of a few moves can be read together, and
// no buffer is needed.
//
// One CTA per (request, layer, share of the heads); every CTA repeats the walk
// rather than wait for another kernel (several layers a CTA, to walk less often,
// measured no faster).  The walk is bound by latency, so all nodes
// look up at once whether they follow their parent, each parent keeps its first such child
// (an atomic minimum, whose order does not matter), and the path is a chase through shared
// memory: two rounds of global loads instead of two for every node of the path.
// Trees of more nodes than fit there are walked with a ballot over the children.
//
// Bound: latency for few trees (4 of 32 nodes, 32 layers: 3.6 us on a B200), then HBM (64
// of 64 nodes: 7.1 us; 31 MB move, 1.84 rows a tree, which alone would take 4.7 us).
#include <algorithm>

#include "paged_common.cuh"

namespace ngb {
namespace {

constexpr int kCommitThreads = 128;
constexpr int kCommitMaxPath = 512;
constexpr int kCommitNodes = 2048;  // nodes of a tree whose children are found in shared memory

struct CommitArgs {
  const long long* draft;
  const int* parents;
  const long long* next;
  const int* cu;
  const int* kv;
  const int* table;
  long long table_stride;
  int table_width;
  uint4* k_cache;
  uint4* v_cache;
  long long s_layer, s_page, s_row, s_head;  // in 16-byte units
  int B, T, Hkv, vecs, num_pages, page_shift, max_path;
  int* accepted;
  int* path;
  long long* bonus;
  int* kv_out;
  unsigned int* err;
};

__global__ void __launch_bounds__(kCommitThreads) tree_commit_kernel(const CommitArgs p) {
  __shared__ int path[kCommitMaxPath];
  __shared__ int child[kCommitNodes];
  __shared__ long long from[kCommitMaxPath], to[kCommitMaxPath];  // 16-byte units in a layer, -1: not mapped
  __shared__ int count_s;
  pdl_launch_next();
  pdl_wait_previous();
  const int b = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31;
  const int first = min(max(p.cu[b], 0), p.T), end = min(max(p.cu[b + 1], first), p.T);
  const int n = end - first;
  const int kv = p.kv[b];
  const bool any = n > 0 && kv >= n;
  if (any && n <= kCommitNodes) {
    for (int c = tid; c < n; c += kCommitThreads) child[c] = n;
    __syncthreads();
    for (int c = tid; c < n; c += kCommitThreads) {
      const int up = p.parents[first + c];
      if (up >= 0 && up < c && p.draft[first + c] == p.next[first + up]) atomicMin(&child[up], c);
    }
    __syncthreads();
  }
  if (tid < 32) {
    int count = 0;
    if (any) {
      int cur = 0;
      for (;;) {
        if (lane == 0) path[count] = cur;
        ++count;
        if (count >= p.max_path) break;
        int found = n;
        if (n <= kCommitNodes) {
          found = child[cur];
        } else {
          const long long want = p.next[first + cur];
          for (int c0 = cur + 1; c0 < n && found == n; c0 += 32) {  // children come after their parent
            const int c = c0 + lane;
            const bool hit = c < n && p.parents[first + c] == cur && p.draft[first + c] == want;
            const unsigned vote = __ballot_sync(0xffffffffu, hit);
            if (vote) found = c0 + __ffs(vote) - 1;
          }
        }
        if (found == n) break;
        cur = found;
      }
    }
    __syncwarp();
    if (lane == 0) count_s = count;
    if (blockIdx.y == 0 && blockIdx.z == 0) {
      if (lane == 0) {
        p.accepted[b] = count;
        p.bonus[b] = count ? p.next[first + path[count - 1]] : -1;
        p.kv_out[b] = count ? kv - n + count : kv;
        if (n > 0 && kv < n && kv != 0) atomicOr(p.err, kErrBadIndex);
      }
      for (int i = lane; i < p.max_path; i += 32)
        p.path[static_cast<size_t>(b) * p.max_path + i] = i < count ? path[i] : -1;
    }
  }
  __syncthreads();
  const int count = count_s, before = kv - n;
  const int* row = p.table + static_cast<size_t>(b) * p.table_stride;
  auto offset = [&](int at) -> long long {  // of cache row `at`
    const int blk = at >> p.page_shift;
    const int page = blk < p.table_width ? row[blk] : -1;
    if (page < 0 || page >= p.num_pages) return -1;
    return page * p.s_page + (at & ((1 << p.page_shift) - 1)) * p.s_row;
  };
  for (int i = tid; i < count; i += kCommitThreads) {
    from[i] = to[i] = -1;
    if (path[i] != i) {
      from[i] = offset(before + path[i]);
      to[i] = offset(before + i);
      if (from[i] < 0 || to[i] < 0) {
        atomicOr(p.err, kErrBadIndex);
        from[i] = -1;
      }
    }
  }
  __syncthreads();
  constexpr int kBatch = 4;  // moves whose rows are read together
  const int columns = p.Hkv * p.vecs;
  for (int col = blockIdx.z * kCommitThreads + tid; col < columns; col += gridDim.z * kCommitThreads) {
    const size_t at = static_cast<size_t>(blockIdx.y) * p.s_layer + static_cast<size_t>(col / p.vecs) * p.s_head +
                      col % p.vecs;
    for (int i0 = 0; i0 < count; i0 += kBatch) {
      uint4 k[kBatch], v[kBatch];
#pragma unroll
      for (int q = 0; q < kBatch; ++q)
        if (i0 + q < count && from[i0 + q] >= 0) {
          k[q] = p.k_cache[at + from[i0 + q]];
          v[q] = p.v_cache[at + from[i0 + q]];
        }
#pragma unroll
      for (int q = 0; q < kBatch; ++q)
        if (i0 + q < count && from[i0 + q] >= 0) {
          p.k_cache[at + to[i0 + q]] = k[q];
          p.v_cache[at + to[i0 + q]] = v[q];
        }
    }
  }
}

}  // namespace
}  // namespace ngb

extern "C" int ng_tree_commit(const long long* draft, const int* parents, const long long* next,
                              const int* cu_new, const int* kv_lens, const int* block_table,
                              long long table_stride, int table_width, void* k_cache, void* v_cache,
                              long long stride_layer, long long stride_page, long long stride_row,
                              long long stride_head, int dtype, int B, int T, int layers, int Hkv, int D,
                              int num_pages, int page_size, int max_path, int* accepted, int* path,
                              long long* bonus, int* kv_out, void* stream) {
  using namespace ngb;
  if (!draft || !parents || !next || !cu_new || !kv_lens || !block_table || !k_cache || !v_cache || !accepted ||
      !path || !bonus || !kv_out)
    return NG_ERR_NULL_POINTER;
  if (!act_dtype_ok(dtype)) return NG_ERR_BAD_DTYPE;
  if (B < 1 || T < 1 || layers < 1 || layers > 65535 || Hkv < 1 || D < 8 || D % 8 || num_pages < 1 ||
      table_width < 1 || table_stride < table_width || !page_size_ok(page_size))
    return NG_ERR_BAD_SHAPE;
  const CacheStrides cs{stride_page, stride_row, stride_head};
  if (!cache_strides_ok(cs) || stride_layer % 8 || stride_layer < 0) return NG_ERR_BAD_SHAPE;
  if (max_path < 1 || max_path > kCommitMaxPath) return NG_ERR_BAD_ARGUMENT;
  if (!aligned(k_cache, 16) || !aligned(v_cache, 16)) return NG_ERR_MISALIGNED;
  DeviceInfo dev;
  if (int st = current_device_info(&dev)) return st;
  const CommitArgs a{draft, parents, next, cu_new, kv_lens, block_table, table_stride, table_width,
                     static_cast<uint4*>(k_cache), static_cast<uint4*>(v_cache), stride_layer / 8,
                     stride_page / 8, stride_row / 8, stride_head / 8, B, T, Hkv, D / 8, num_pages,
                     log2_of(page_size), max_path, accepted, path, bonus, kv_out, dev.err};
  const int shares = std::min(64, std::max(1, (Hkv * (D / 8) + kCommitThreads - 1) / kCommitThreads));
  return launch_chained(tree_commit_kernel, dim3(B, layers, shares), dim3(kCommitThreads), 0,
                        static_cast<cudaStream_t>(stream), a);
}
