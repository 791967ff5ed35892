// Per-head RMSNorm of the queries and keys, rotation by position, and append of
// K and V to a paged cache, in one pass over the fused projection's output:
//   x = qkv[m] = q heads | k heads | v heads, D values each
//   y = x * rsqrt(mean(x^2) + eps) * w            (q and k heads; no weight: y = x)
//   (y_i, y_{i+r/2}) -> (y_i c - y_{i+r/2} s, y_{i+r/2} c + y_i s),  i < r/2
//   q -> q_out[m], k and v -> cache rows slots[m] (a negative slot: not stored)
// with (c, s) the cosine and sine of 2 pi * frac(pos * turn_i).  turn_i comes as
// a whole number of 2^-64 turns, so pos * turn_i modulo one turn is one wrapping
// 64-bit multiply, exact at every position; an fp32 product pos * theta^(-2i/r)
// is off by 6e-3 rad at position 100,000.
//
// A row of D values is held by D / 8 lanes, 16 bytes each, so a warp works on
// 256 / D rows at a time; the sum of squares is a shuffle reduction within the
// row and the rotation partner is a shuffle across half of the rotated lanes.  A
// warp keeps one token, so its cosines and sines are computed once for its rows.
#include <algorithm>

#include "paged_common.cuh"

namespace ngb {
namespace {

constexpr int kNrThreads = 128;

struct NormRopeArgs {
  const uint16_t* qkv;
  long long qkv_stride;
  const uint16_t* q_weight;
  const uint16_t* k_weight;
  const long long* turns;
  const int* positions;
  const int* slots;
  uint16_t* q_out;
  uint16_t* k_cache;
  uint16_t* v_cache;
  CacheStrides cs;
  int M, Hq, Hkv, rot, page_shift, chunks;
  long long num_rows;  // pages * page size
  float eps;
  unsigned int* err;
};

template <bool BF16, int D>
__global__ void __launch_bounds__(kNrThreads) qk_norm_rope_kernel(const NormRopeArgs p) {
  constexpr int kLanes = D / 8;        // lanes per row
  constexpr int kRows = 32 / kLanes;   // rows per warp and iteration
  pdl_launch_next();
  pdl_wait_previous();
  const int lane = threadIdx.x & 31, l = lane % kLanes, sub = lane / kLanes;
  const int gw = blockIdx.x * (kNrThreads / 32) + (threadIdx.x >> 5);
  const int m = gw / p.chunks, chunk = gw % p.chunks;
  if (m >= p.M) return;
  const int rows = p.Hq + 2 * p.Hkv;
  const int steps = (rows + kRows - 1) / kRows;
  const int s0 = steps * chunk / p.chunks, s1 = steps * (chunk + 1) / p.chunks;

  const int half8 = p.rot / 16;  // lanes of the rotated first half
  const bool rotated = l < 2 * half8, low = l < half8;
  const int partner = rotated ? (low ? lane + half8 : lane - half8) : lane;
  float cs[8], sn[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) cs[j] = 1.f, sn[j] = 0.f;
  if (rotated) {
    const unsigned long long pos = static_cast<unsigned long long>(static_cast<long long>(p.positions[m]));
    const long long* t = p.turns + (low ? l : l - half8) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int phase = static_cast<int>(static_cast<unsigned long long>(t[j]) * pos >> 32);
      sincospif(static_cast<float>(phase) * 4.656612873077393e-10f, &sn[j], &cs[j]);  // 2^-31 half turns
      if (low) sn[j] = -sn[j];
    }
  }
  uint4 wq = make_uint4(0, 0, 0, 0), wk = wq;
  const bool normed = p.q_weight != nullptr;
  if (normed) {
    wq = ld_ro_v4(p.q_weight + l * 8);
    wk = ld_ro_v4(p.k_weight + l * 8);
  }
  const int slot = p.slots[m];
  const bool stored = slot >= 0 && slot < p.num_rows;
  if (slot >= p.num_rows && l == 0) atomicOr(p.err, kErrBadIndex);
  const size_t cache_row = stored ? static_cast<size_t>(slot >> p.page_shift) * p.cs.page +
                                        static_cast<size_t>(slot & ((1 << p.page_shift) - 1)) * p.cs.row
                                  : 0;
  const uint16_t* src = p.qkv + static_cast<size_t>(m) * p.qkv_stride;
  for (int s = s0; s < s1; ++s) {
    const int r = s * kRows + sub;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (r < rows) x = ld_ro_v4(src + static_cast<size_t>(r) * D + l * 8);
    float f[8];
    unpack8<BF16>(x, f);
    if (normed) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += f[j] * f[j];
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float inv = rsqrtf(ss * (1.f / D) + p.eps);
      float w[8];
      unpack8<BF16>(r < p.Hq ? wq : wk, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = f[j] * inv * w[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float other = __shfl_sync(0xffffffffu, f[j], partner);
      f[j] = f[j] * cs[j] + (rotated ? other * sn[j] : 0.f);
    }
    if (r < p.Hq) {
      *reinterpret_cast<uint4*>(p.q_out + (static_cast<size_t>(m) * p.Hq + r) * D + l * 8) = pack8<BF16>(f);
    } else if (r < rows && stored) {
      if (r < p.Hq + p.Hkv)
        *reinterpret_cast<uint4*>(p.k_cache + cache_row + (r - p.Hq) * p.cs.head + l * 8) = pack8<BF16>(f);
      else
        *reinterpret_cast<uint4*>(p.v_cache + cache_row + (r - p.Hq - p.Hkv) * p.cs.head + l * 8) = x;
    }
  }
}

template <bool BF16, int D>
int launch_norm_rope(NormRopeArgs a, const DeviceInfo& dev, cudaStream_t st) {
  constexpr int kRows = 256 / D;
  const int steps = (a.Hq + 2 * a.Hkv + kRows - 1) / kRows;
  // Few tokens: one step a warp, to spread the rows over the SMs.  Many: one
  // warp a token, so the sines are computed once.
  const long long want = static_cast<long long>(dev.sm_count) * 32;
  a.chunks = static_cast<int>(std::max<long long>(1, std::min<long long>(steps, want / a.M)));
  const long long warps = static_cast<long long>(a.M) * a.chunks;
  const long long blocks = (warps + kNrThreads / 32 - 1) / (kNrThreads / 32);
  return launch_chained(qk_norm_rope_kernel<BF16, D>, dim3(static_cast<unsigned>(blocks)), dim3(kNrThreads), 0,
                        st, a);
}

}  // namespace
}  // namespace ngb

extern "C" int ng_qk_norm_rope_append(const void* qkv, long long qkv_stride, const void* q_weight,
                                      const void* k_weight, const long long* turns, int rotary_dim,
                                      const int* positions, const int* slots, void* q_out, void* k_cache,
                                      void* v_cache, long long stride_page, long long stride_row,
                                      long long stride_head, int dtype, int M, int Hq, int Hkv, int D,
                                      int num_pages, int page_size, float eps, void* stream) {
  using namespace ngb;
  if (!qkv || !positions || !slots || !q_out || !k_cache || !v_cache) return NG_ERR_NULL_POINTER;
  if ((q_weight == nullptr) != (k_weight == nullptr) || (rotary_dim > 0 && !turns)) return NG_ERR_NULL_POINTER;
  if (!act_dtype_ok(dtype)) return NG_ERR_BAD_DTYPE;
  if (M < 1 || Hq < 1 || Hkv < 1 || (D != 64 && D != 128 && D != 256) || num_pages < 1 ||
      !page_size_ok(page_size) || M > (1 << 24) || Hq + 2 * Hkv > (1 << 16))
    return NG_ERR_BAD_SHAPE;
  if (rotary_dim < 0 || rotary_dim > D || rotary_dim % 16) return NG_ERR_BAD_ARGUMENT;
  const CacheStrides cs{stride_page, stride_row, stride_head};
  if (!cache_strides_ok(cs) || qkv_stride % 8 || qkv_stride < static_cast<long long>(Hq + 2 * Hkv) * D)
    return NG_ERR_BAD_SHAPE;
  if (!aligned(qkv, 16) || !aligned(q_out, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16) ||
      !aligned(q_weight, 16) || !aligned(k_weight, 16) || !aligned(turns, 8))
    return NG_ERR_MISALIGNED;
  DeviceInfo dev;
  if (int st = current_device_info(&dev)) return st;
  const NormRopeArgs a{static_cast<const uint16_t*>(qkv), qkv_stride, static_cast<const uint16_t*>(q_weight),
                       static_cast<const uint16_t*>(k_weight), turns, positions, slots,
                       static_cast<uint16_t*>(q_out), static_cast<uint16_t*>(k_cache),
                       static_cast<uint16_t*>(v_cache), cs, M, Hq, Hkv, rotary_dim, log2_of(page_size), 1,
                       static_cast<long long>(num_pages) * page_size, eps, dev.err};
  auto st = static_cast<cudaStream_t>(stream);
  const bool bf = dtype == NG_DTYPE_BF16;
  switch (D) {
    case 64: return bf ? launch_norm_rope<true, 64>(a, dev, st) : launch_norm_rope<false, 64>(a, dev, st);
    case 128: return bf ? launch_norm_rope<true, 128>(a, dev, st) : launch_norm_rope<false, 128>(a, dev, st);
    default: return bf ? launch_norm_rope<true, 256>(a, dev, st) : launch_norm_rope<false, 256>(a, dev, st);
  }
}
