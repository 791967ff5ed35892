// Attention of drafted trees, chains or single tokens over a paged KV cache.
#include <algorithm>

#include "paged_common.cuh"

namespace ngb {
namespace {

struct TreeAttnArgs {
  const uint16_t* q;
  long long q_token, q_head;
  const uint16_t* k;
  const uint16_t* v;
  CacheStrides cs;
  const int* table;
  long long table_stride;
  int table_width;
  const int* kv_lens;
  const int* cu;
  const unsigned long long* mask;
  int mask_words;
  uint16_t* out;
  float* lse;
  int B, T, Hq, Hkv, num_pages, page_shift;
  float scale;
  unsigned int* err;
};

// One warp per (token, query head): keys one at a time, online softmax.
template <bool BF16, int D>
__global__ void __launch_bounds__(128) tree_attn_simple(const TreeAttnArgs p) {
  constexpr int kPer = D / 32;
  pdl_launch_next();
  pdl_wait_previous();
  const int lane = threadIdx.x & 31;
  const long long gw = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int t = static_cast<int>(gw / p.Hq), h = static_cast<int>(gw % p.Hq);
  if (t >= p.T) return;
  int b = 0;
  for (int i = 0; i < p.B; ++i)
    if (p.cu[i] <= t) b = i;
  const int first = p.cu[b], n = min(p.cu[b + 1], p.T) - first, i = t - first;
  const bool live = i < n;
  const int kv = live ? p.kv_lens[b] : 0, ctx = max(0, kv - n);
  const int kh = h / (p.Hq / p.Hkv);
  auto ld = [](const uint16_t* x) {
    return BF16 ? __uint_as_float(static_cast<uint32_t>(*x) << 16) : __half2float(__ushort_as_half(*x));
  };
  float q[kPer], acc[kPer], mx = -INFINITY, sum = 0.f;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    q[j] = ld(p.q + t * p.q_token + h * p.q_head + lane + 32 * j) * p.scale;
    acc[j] = 0.f;
  }
  for (int key = 0; key < kv; ++key) {
    const int node = key - ctx;
    if (node >= 0) {
      if (!p.mask ? node > i
                  : node >= p.mask_words * 64 ||
                        !((p.mask[static_cast<size_t>(t) * p.mask_words + (node >> 6)] >> (node & 63)) & 1))
        continue;
    }
    const int blk = key >> p.page_shift;
    const int page = blk < p.table_width ? p.table[b * p.table_stride + blk] : -1;
    if (page < 0 || page >= p.num_pages) {
      if (lane == 0) atomicOr(p.err, kErrBadIndex);
      continue;
    }
    const size_t at = page * p.cs.page + (key & ((1 << p.page_shift) - 1)) * p.cs.row + kh * p.cs.head;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) s += q[j] * ld(p.k + at + lane + 32 * j);
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float nm = fmaxf(mx, s), base = nm == -INFINITY ? 0.f : nm;
    const float corr = expf(mx - base), pw = expf(s - base);
    sum = sum * corr + pw;
#pragma unroll
    for (int j = 0; j < kPer; ++j) acc[j] = acc[j] * corr + pw * ld(p.v + at + lane + 32 * j);
    mx = nm;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint16_t* o = p.out + (static_cast<size_t>(t) * p.Hq + h) * D;
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    o[lane + 32 * j] = static_cast<uint16_t>(pack_pair<BF16>(sum == 0.f ? 0.f : acc[j] * inv, 0.f) & 0xFFFFu);
  if (p.lse && lane == 0) p.lse[static_cast<size_t>(t) * p.Hq + h] = sum == 0.f ? -INFINITY : mx + logf(sum);
}

template <bool BF16, int D>
int launch_tree_attn(const TreeAttnArgs& a, cudaStream_t st) {
  const long long warps = static_cast<long long>(a.T) * a.Hq;
  return launch_chained(tree_attn_simple<BF16, D>, dim3(static_cast<unsigned>((warps + 3) / 4)), dim3(128), 0, st, a);
}

}  // namespace
}  // namespace ngb

extern "C" size_t ng_tree_attn_workspace_bytes(int D) {
  if (D != 64 && D != 128) return 0;
  return 256;
}

extern "C" int ng_tree_attn(const void* q, long long q_stride_token, long long q_stride_head,
                            const void* k_cache, const void* v_cache, long long stride_page,
                            long long stride_row, long long stride_head, const int* block_table,
                            long long table_stride, int table_width, const int* kv_lens, const int* cu_new,
                            const long long* mask, int mask_words, void* out, float* lse, int dtype, int B,
                            int T, int Hq, int Hkv, int D, int num_pages, int page_size, float scale,
                            void* workspace, size_t workspace_bytes, void* stream) {
  using namespace ngb;
  if (!q || !k_cache || !v_cache || !block_table || !kv_lens || !cu_new || !out || !workspace)
    return NG_ERR_NULL_POINTER;
  if (!act_dtype_ok(dtype)) return NG_ERR_BAD_DTYPE;
  if (B < 1 || T < 1 || Hq < 1 || Hkv < 1 || Hq % Hkv || Hq / Hkv > 128 || (D != 64 && D != 128) ||
      num_pages < 1 || table_width < 1 || table_stride < table_width || !page_size_ok(page_size) ||
      static_cast<long long>(T) * Hq > (1LL << 30))
    return NG_ERR_BAD_SHAPE;
  const CacheStrides cs{stride_page, stride_row, stride_head};
  if (!cache_strides_ok(cs) || q_stride_token % 8 || q_stride_head % 8 || q_stride_token < 0 || q_stride_head < 0)
    return NG_ERR_BAD_SHAPE;
  if (!(scale > 0.f) || !(scale < INFINITY) || mask_words < 0 || (mask && mask_words < 1))
    return NG_ERR_BAD_ARGUMENT;
  if (workspace_bytes < ng_tree_attn_workspace_bytes(D)) return NG_ERR_BAD_ARGUMENT;
  if (!aligned(q, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(out, 16) ||
      !aligned(mask, 8) || !aligned(workspace, 256))
    return NG_ERR_MISALIGNED;
  DeviceInfo dev;
  if (int st = current_device_info(&dev)) return st;
  const TreeAttnArgs a{static_cast<const uint16_t*>(q), q_stride_token, q_stride_head,
                       static_cast<const uint16_t*>(k_cache), static_cast<const uint16_t*>(v_cache), cs,
                       block_table, table_stride, table_width, kv_lens, cu_new,
                       reinterpret_cast<const unsigned long long*>(mask), mask_words,
                       static_cast<uint16_t*>(out), lse, B, T, Hq, Hkv, num_pages, log2_of(page_size), scale,
                       dev.err};
  auto st = static_cast<cudaStream_t>(stream);
  if (D == 128)
    return dtype == NG_DTYPE_BF16 ? launch_tree_attn<true, 128>(a, st) : launch_tree_attn<false, 128>(a, st);
  return dtype == NG_DTYPE_BF16 ? launch_tree_attn<true, 64>(a, st) : launch_tree_attn<false, 64>(a, st);
}
