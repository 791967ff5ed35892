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
// 256 / D rows at a time.  Weight and rotation are folded into two factors per value,
//   out_i = inv (x_i (w_i c_i) + x_p (w_p s_i)),  p the partner of i, s_i signed,
// which a warp works out once for its token and section (q or k); the partner comes
// by a shuffle of the raw 16-bit values (four words for eight of them).  The sum of squares is a
// shuffle reduction within the row.  Each half of a rotated pair of lanes evaluates
// half of their common sines.  v rows are copied without being looked at.
//
// Bound: HBM for many tokens.  Four rows are loaded ahead (with one, the loads
// of a warp were exposed one after another: 56 us where four take 40; two, three and six
// are slower).  128 registers a thread, 16 warps an SM (20 of 96: 2000 tokens of 48 rows
// 14.0 us, not 11.7).  8192 tokens of 48 rows of 128, bf16, on a B200: 38.4 us, 5.2 TB/s;
// 976 tokens of 80 rows 9.5 us, one round of loads after another; 4 tokens 2.3 us, the
// launch.
#include <algorithm>

#include "paged_common.cuh"

namespace ngb {
namespace {

constexpr int kNrThreads = 128;
constexpr int kNrBlocks = 4;  // blocks an SM: 128 registers a thread

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
  int M, Hq, Hkv, rot, page_shift;
  int whole, chunks;  // tokens that one warp takes each; warps for each of the others
  long long num_rows;  // pages * page size
  float eps;
  unsigned int* err;
};

template <bool BF16, int D>
__global__ void __launch_bounds__(kNrThreads, kNrBlocks) qk_norm_rope_kernel(const NormRopeArgs p) {
  constexpr int kLanes = D / 8;        // lanes per row
  constexpr int kRows = 32 / kLanes;   // rows per warp and step
  constexpr int kAhead = 4;            // steps whose rows are loaded together
  pdl_launch_next();
  pdl_wait_previous();
  const int lane = threadIdx.x & 31, l = lane % kLanes, sub = lane / kLanes;
  const int gw = blockIdx.x * (kNrThreads / 32) + (threadIdx.x >> 5);
  const int chunks = gw < p.whole ? 1 : p.chunks, rest = gw - p.whole;
  const int m = gw < p.whole ? gw : p.whole + rest / chunks, chunk = gw < p.whole ? 0 : rest % chunks;
  if (m >= p.M) return;
  // Steps of the three sections, and this warp's run of them.
  const int q_steps = (p.Hq + kRows - 1) / kRows, k_steps = (p.Hkv + kRows - 1) / kRows;
  const int steps = q_steps + 2 * k_steps;
  const int s0 = steps * chunk / chunks, s1 = steps * (chunk + 1) / chunks;

  const uint16_t* src = p.qkv + static_cast<size_t>(m) * p.qkv_stride + l * 8;
  const int slot = p.slots[m];
  const bool stored = slot >= 0 && slot < p.num_rows;
  if (slot >= p.num_rows && lane == 0) atomicOr(p.err, kErrBadIndex);
  const size_t cache_row = stored ? static_cast<size_t>(slot >> p.page_shift) * p.cs.page +
                                        static_cast<size_t>(slot & ((1 << p.page_shift) - 1)) * p.cs.row + l * 8
                                  : 0;

  // The rows of up to kAhead steps from step s on, all of one section.
  auto end_of = [&](int section) { return section == 0 ? min(s1, q_steps) : section == 1 ? min(s1, q_steps + k_steps) : s1; };
  auto section_of = [&](int s) { return s < q_steps ? 0 : s < q_steps + k_steps ? 1 : 2; };
  auto row_of = [&](int section, int s) { return (s - (section ? q_steps + (section - 1) * k_steps : 0)) * kRows + sub; };
  auto load = [&](int s, uint4 (&x)[kAhead]) {
    const int section = section_of(s), heads = section ? p.Hkv : p.Hq, end = end_of(section);
    const uint16_t* rows = src + static_cast<size_t>(section ? p.Hq + (section - 1) * p.Hkv : 0) * D;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int r = row_of(section, s + i);
      x[i] = make_uint4(0, 0, 0, 0);
      if (s + i < end && r < heads) x[i] = ld_ro_v4(rows + static_cast<size_t>(r) * D);
    }
  };
  uint4 x[kAhead];
  load(s0, x);  // before the sines: they wait for the position, and these need not

  const int half8 = p.rot / 16;  // lanes of the rotated first half
  const bool rotated = l < 2 * half8, low = l < half8;
  const int other = low ? l + half8 : l - half8;  // the partner's place in the row
  const int partner = rotated ? lane - l + other : lane;
  const unsigned pairs = __ballot_sync(0xffffffffu, rotated);  // whole pairs of lanes
  const bool normed = p.q_weight != nullptr;
  float cs[8], sn[8];
  if (s0 < q_steps + k_steps) {
#pragma unroll
    for (int j = 0; j < 8; ++j) cs[j] = 1.f, sn[j] = 0.f;
    if (rotated) {
      // A pair of lanes has the same eight frequencies: the low lane evaluates the
      // first four, the high one the others.
      const unsigned long long pos = static_cast<unsigned long long>(static_cast<long long>(p.positions[m]));
      const long long* t = p.turns + (low ? l * 8 : other * 8 + 4);
      float c4[4], n4[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int phase = static_cast<int>(static_cast<unsigned long long>(t[j]) * pos >> 32);
        sincospif(static_cast<float>(phase) * 4.656612873077393e-10f, &n4[j], &c4[j]);  // 2^-31 half turns
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float co = __shfl_sync(pairs, c4[j], partner), no = __shfl_sync(pairs, n4[j], partner);
        cs[j] = low ? c4[j] : co;
        cs[4 + j] = low ? co : c4[j];
        sn[j] = low ? -n4[j] : no;
        sn[4 + j] = low ? -no : n4[j];
      }
    }
  }

  f2 fc[4], fs[4];
  int have = -1;  // section whose factors fc and fs are
  for (int s = s0; s < s1;) {
    const int section = section_of(s);
    const int next = min(s + kAhead, end_of(section));
    uint4 ahead[kAhead];
    if (next < s1) load(next, ahead);
    if (section == 2) {  // v rows, as they are
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int r = row_of(2, s + i);
        if (s + i < next && r < p.Hkv && stored)
          *reinterpret_cast<uint4*>(p.v_cache + cache_row + r * p.cs.head) = x[i];
      }
    } else if (section == 0 || stored) {
      if (section != have) {
        have = section;
        float wo[8], wp[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) wo[j] = wp[j] = 1.f;
        if (normed) {
          const uint16_t* w = section ? p.k_weight : p.q_weight;
          unpack8<BF16>(ld_ro_v4(w + l * 8), wo);
          unpack8<BF16>(ld_ro_v4(w + (rotated ? other : l) * 8), wp);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          fc[j] = f2_make(wo[2 * j] * cs[2 * j], wo[2 * j + 1] * cs[2 * j + 1]);
          fs[j] = f2_make(wp[2 * j] * sn[2 * j], wp[2 * j + 1] * sn[2 * j + 1]);
        }
      }
      const int heads = section ? p.Hkv : p.Hq;
      uint16_t* dst = section ? p.k_cache + cache_row : p.q_out + static_cast<size_t>(m) * p.Hq * D + l * 8;
      const long long dst_head = section ? p.cs.head : D;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (s + i >= next) break;
        const int r = row_of(section, s + i);
        uint4 y;
        y.x = __shfl_sync(0xffffffffu, x[i].x, partner);
        y.y = __shfl_sync(0xffffffffu, x[i].y, partner);
        y.z = __shfl_sync(0xffffffffu, x[i].z, partner);
        y.w = __shfl_sync(0xffffffffu, x[i].w, partner);
        if (!rotated) y = make_uint4(0, 0, 0, 0);  // (0 * inf would not be 0)
        float f[8], g[8];
        unpack8<BF16>(x[i], f);
        unpack8<BF16>(y, g);
        float inv = 1.f;
        if (normed) {
          f2 sq = f2_make(0.f, 0.f);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const f2 v = f2_make(f[2 * j], f[2 * j + 1]);
            sq = f2_fma(v, v, sq);
          }
          float lo, hi;
          f2_split(sq, lo, hi);
          float ss = lo + hi;
#pragma unroll
          for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          inv = rsqrtf(ss * (1.f / D) + p.eps);
        }
        const f2 inv2 = f2_make(inv, inv);
        float o[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f2 t = f2_fma(f2_make(f[2 * j], f[2 * j + 1]), fc[j],
                              f2_mul(f2_make(g[2 * j], g[2 * j + 1]), fs[j]));
          f2_split(f2_mul(t, inv2), o[2 * j], o[2 * j + 1]);
        }
        if (r < heads) *reinterpret_cast<uint4*>(dst + r * dst_head) = pack8<BF16>(o);
      }
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i) x[i] = ahead[i];
    s = next;
  }
}

template <bool BF16, int D>
int launch_norm_rope(NormRopeArgs a, const DeviceInfo& dev, cudaStream_t st) {
  constexpr int kRows = 256 / D;
  const int steps = (a.Hq + kRows - 1) / kRows + 2 * ((a.Hkv + kRows - 1) / kRows);
  // A warp that has a whole token works out its sines once, so as many tokens as fill the SMs
  // a whole number of times go to a warp each.  Those that are left over are shared by as
  // many warps as the SMs hold at once, but no more: 976 tokens of 80 rows take 10.7 us with
  // two warps a token, 13.2 with four, of which some wait for the others; 2500 of 48 rows
  // 19.1 us with a warp for every token, and 14.7 so.
  const int wave = dev.sm_count * kNrBlocks * (kNrThreads / 32);
  a.whole = a.M / wave * wave;
  const int rest = a.M - a.whole;
  a.chunks = rest ? std::min(steps, wave / rest) : 1;
  const long long warps = a.whole + static_cast<long long>(rest) * a.chunks;
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
                       static_cast<uint16_t*>(v_cache), cs, M, Hq, Hkv, rotary_dim, log2_of(page_size), 0, 1,
                       static_cast<long long>(num_pages) * page_size, eps, dev.err};
  auto st = static_cast<cudaStream_t>(stream);
  const bool bf = dtype == NG_DTYPE_BF16;
  switch (D) {
    case 64: return bf ? launch_norm_rope<true, 64>(a, dev, st) : launch_norm_rope<false, 64>(a, dev, st);
    case 128: return bf ? launch_norm_rope<true, 128>(a, dev, st) : launch_norm_rope<false, 128>(a, dev, st);
    default: return bf ? launch_norm_rope<true, 256>(a, dev, st) : launch_norm_rope<false, 256>(a, dev, st);
  }
}
