// Shared pieces of the paged-cache kernels (paged_plan.cu, qk_norm_rope.cu,
// tree_attn.cu, tree_commit.cu): 16-byte vectors of eight fp16 / bf16 values,
// the launch helper, and the argument checks the entry points share.
#pragma once

#include "ng_common.cuh"

namespace ngb {

// Eight consecutive 16-bit activations <-> fp32.
template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (BF16) {
      f[2 * j] = __uint_as_float(w[j] << 16);
      f[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    } else {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
      f[2 * j] = t.x;
      f[2 * j + 1] = t.y;
    }
  }
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

template <bool BF16>
__device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
  return make_uint4(pack_pair<BF16>(f[0], f[1]), pack_pair<BF16>(f[2], f[3]), pack_pair<BF16>(f[4], f[5]),
                    pack_pair<BF16>(f[6], f[7]));
}

// Programmatic dependent launch: the next kernel on the stream may launch; wait
// for the kernels before this one.
__device__ __forceinline__ void pdl_launch_next() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void pdl_wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename... KArgs, typename... Args>
inline int launch_chained(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                          Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return launch_status(cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...));
}

// Rows of a page: a power of two in [8, 1024].  8 rows of 128 bytes are one
// swizzle atom of the attention kernel's tiles, so a page never splits an atom.
inline bool page_size_ok(int p) { return p >= 8 && p <= 1024 && (p & (p - 1)) == 0; }
inline int log2_of(int p) { return 31 - __builtin_clz(static_cast<unsigned>(p)); }
inline bool act_dtype_ok(int d) { return d == NG_DTYPE_F16 || d == NG_DTYPE_BF16; }

// Element strides of one layer's cache, [pages, page_size, kv heads, D] with
// the last dimension contiguous.
struct CacheStrides {
  long long page, row, head;
};
inline bool cache_strides_ok(const CacheStrides& s) {
  return s.page > 0 && s.row > 0 && s.head > 0 && s.page % 8 == 0 && s.row % 8 == 0 && s.head % 8 == 0;
}

}  // namespace ngb
