// Compiled torch binding over the C ABI: the reference extension's three ops
// (gemv_w4a16, gemm_w4a16, dequant_w4; arvindcr4/nibblegemm csrc/bindings.cpp)
// taking tensors, with the argument checks, the output allocation, the device
// guard, the current-stream lookup and the per-stream workspace cache done in
// C++ (and the paged-cache ops of paged.py the same way) -- a few microseconds per call instead of the tens a Python + ctypes path
// costs.  The kernels are the ones of libnibblegemm_b200.so; this file only
// marshals.  Argument-check failures raise RuntimeError (TORCH_CHECK), as the
// reference's do; the library's own status is returned beside the output and
// the Python wrapper raises on a non-zero one.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <limits>
#include <mutex>
#include <optional>
#include <tuple>
#include <unordered_map>
#include <vector>

#include "nibblegemm_b200.h"

namespace {

int dtype_code(const torch::Tensor& t) {
  if (t.scalar_type() == torch::kHalf) return NG_DTYPE_F16;
  if (t.scalar_type() == torch::kBFloat16) return NG_DTYPE_BF16;
  TORCH_CHECK(false, "activations must be fp16 or bf16");
}

void check_weight(const torch::Tensor& Wq, const torch::Tensor& S, const torch::Device& dev) {
  TORCH_CHECK(Wq.is_cuda() && S.is_cuda(), "all tensors must live on CUDA");
  TORCH_CHECK(Wq.device() == dev && S.device() == dev, "all tensors must be on the same device");
  TORCH_CHECK(Wq.scalar_type() == torch::kInt, "packed weights must be int32");
  TORCH_CHECK(S.scalar_type() == torch::kHalf, "scales must be fp16");
  TORCH_CHECK(Wq.is_contiguous() && S.is_contiguous(), "inputs must be contiguous");
  TORCH_CHECK(Wq.dim() == 2 && S.dim() == 2, "expected 2-D inputs");
}

std::tuple<int64_t, int64_t, int64_t> check_act(const torch::Tensor& X, const torch::Tensor& Wq,
                                                const torch::Tensor& S, int64_t group_size) {
  TORCH_CHECK(X.is_cuda(), "all tensors must live on CUDA");
  check_weight(Wq, S, X.device());
  dtype_code(X);
  TORCH_CHECK(X.is_contiguous(), "inputs must be contiguous");
  TORCH_CHECK(X.dim() == 2, "expected 2-D inputs");
  const int64_t M = X.size(0), K = X.size(1), N = Wq.size(1);
  TORCH_CHECK(Wq.size(0) * 8 == K, "packed weight rows disagree with K");
  TORCH_CHECK(group_size > 0 && S.size(0) * group_size == K, "scale rows disagree with K/group_size");
  TORCH_CHECK(S.size(1) == N, "scale columns disagree with N");
  return {M, K, N};
}

torch::Tensor output(const std::optional<torch::Tensor>& out, int64_t M, int64_t N,
                     const torch::Tensor& X) {
  if (!out.has_value()) return torch::empty({M, N}, X.options());
  const auto& o = *out;
  TORCH_CHECK(o.dim() == 2 && o.size(0) == M && o.size(1) == N && o.scalar_type() == X.scalar_type() &&
                  o.device() == X.device() && o.is_contiguous(),
              "out must be a contiguous [M, N] tensor like X");
  return o;
}

// Kinds of workspace.
constexpr int kGemvWorkspace = 0, kGemmWorkspace = 1, kAttentionWorkspace = 2;

// The cached workspace of (device, stream, kind), grown on demand; one per stream,
// because calls sharing a workspace must not overlap on the GPU.  Those of the GEMV and the
// GEMM are zero-filled, once: every call leaves their counters at zero.  The attention needs
// no zeros, and its buffer has the size of its largest form from the start, so it never grows.
//
// A captured CUDA graph keeps the address, so
// * a buffer that was outgrown is never freed (each is at least twice the one before, so all
//   of them are less than twice the last);
// * no buffer is made by a capture, whose graph would own it and fill it with zeros again at
//   every replay (and at the replay only): one that is first asked for during a capture is made
//   beside it, on a stream that is not captured.
torch::Tensor workspace(const torch::Device& dev, cudaStream_t stream, int kind, size_t need) {
  // Heap-held and never destroyed: a static map of tensors would be torn down at
  // process exit after torch's CUDA allocator, and crash there.
  static std::mutex mu;
  static auto* cache = new std::unordered_map<uint64_t, std::vector<torch::Tensor>>();  // the last one is in use
  const uint64_t key = (reinterpret_cast<uint64_t>(stream) << 8) ^ (static_cast<uint64_t>(dev.index()) << 2) ^
                       static_cast<uint64_t>(kind);
  std::lock_guard<std::mutex> lock(mu);
  auto& all = (*cache)[key];
  const size_t have = all.empty() ? 0 : static_cast<size_t>(all.back().numel());
  if (have >= std::max<size_t>(need, 1)) return all.back();
  const c10::cuda::CUDAGuard guard(dev);
  const size_t least = kind == kAttentionWorkspace ? ng_tree_attn_workspace_bytes(128)
                       : kind == kGemvWorkspace    ? 4u << 20
                                                   : 1u << 20;
  const auto bytes = static_cast<int64_t>(std::max({need, 2 * have, least}));
  const auto options = torch::TensorOptions().dtype(torch::kUInt8).device(dev);
  auto make = [&] { return kind == kAttentionWorkspace ? torch::empty({bytes}, options) : torch::zeros({bytes}, options); };
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) {
    all.push_back(make());
  } else {
    const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
    auto beside = c10::cuda::getStreamFromPool(false, dev.index());
    auto captured = [&] {
      const c10::cuda::CUDAStreamGuard on(beside);
      return c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None;
    };
    for (int i = 0; i < 32 && captured(); ++i) beside = c10::cuda::getStreamFromPool(false, dev.index());  // it has 32
    TORCH_CHECK(!captured(), "no stream is left to make a workspace on beside the capture");
    {
      const c10::cuda::CUDAStreamGuard on(beside);
      all.push_back(make());
    }
    beside.synchronize();
  }
  return all.back();
}

// The attention's workspace for one call.  In a capture it comes from the graph's own
// memory: graphs captured on one stream may be replayed at the same time.
torch::Tensor attention_workspace(const torch::Device& dev, cudaStream_t stream, size_t need) {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None)
    return workspace(dev, stream, kAttentionWorkspace, need);
  return torch::empty({static_cast<int64_t>(need)}, torch::TensorOptions().dtype(torch::kUInt8).device(dev));
}

std::tuple<torch::Tensor, int64_t> gemv_w4a16(torch::Tensor X, torch::Tensor Wq, torch::Tensor S, int64_t group_size,
                         int64_t version, int64_t splits_override, int64_t threads_override,
                         int64_t algo, std::optional<torch::Tensor> out) {
  auto [M, K, N] = check_act(X, Wq, S, group_size);
  TORCH_CHECK(N % 4 == 0, "N must be a multiple of 4 for 128-bit weight loads");
  TORCH_CHECK(group_size == 64 || group_size == 128 || group_size == 256,
              "group_size must be 64, 128 or 256");
  TORCH_CHECK(M >= 1 && M <= 16, "gemv path supports 1 <= M <= 16; use gemm_w4a16 for larger M");
  TORCH_CHECK(version >= 0 && version <= 4, "version must be one of 0..4");
  // Version 3 of the reference ladder is version 4 pinned to one K split.
  const int splits = version == 3 ? 1 : static_cast<int>(splits_override);
  const c10::cuda::CUDAGuard guard(X.device());
  auto Y = output(out, M, N, X);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(X.device().index()).stream();
  auto ws = workspace(X.device(), stream, kGemvWorkspace, ng_gemv_workspace_bytes(1, static_cast<int>(N)));
  const int st = ng_gemv_w4a16(X.data_ptr(), dtype_code(X), Wq.data_ptr<int32_t>(),
                             reinterpret_cast<const uint16_t*>(S.data_ptr()), Y.data_ptr(),
                             static_cast<int>(M), static_cast<int>(K), static_cast<int>(N),
                             static_cast<int>(group_size), splits, static_cast<int>(threads_override),
                             static_cast<int>(algo), ws.data_ptr(), static_cast<size_t>(ws.numel()), stream);
  return {Y, st};
}

std::tuple<torch::Tensor, int64_t> gemm_w4a16(torch::Tensor X, torch::Tensor Wq, torch::Tensor S, int64_t group_size,
                         int64_t version, int64_t tile_tokens, std::optional<torch::Tensor> out) {
  auto [M, K, N] = check_act(X, Wq, S, group_size);
  TORCH_CHECK(version == 6 || version == 7, "version must be 6 or 7");
  const c10::cuda::CUDAGuard guard(X.device());
  auto Y = output(out, M, N, X);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(X.device().index()).stream();
  auto ws = workspace(X.device(), stream, kGemmWorkspace, ng_gemm_workspace_bytes(static_cast<int>(M), static_cast<int>(N)));
  const int st = ng_gemm_w4a16(X.data_ptr(), dtype_code(X), Wq.data_ptr<int32_t>(),
                             reinterpret_cast<const uint16_t*>(S.data_ptr()), Y.data_ptr(),
                             static_cast<int>(M), static_cast<int>(K), static_cast<int>(N),
                             static_cast<int>(group_size), static_cast<int>(tile_tokens), ws.data_ptr(),
                             static_cast<size_t>(ws.numel()), stream);
  return {Y, st};
}

std::tuple<torch::Tensor, int64_t> dequant_w4(torch::Tensor Wq, torch::Tensor S, int64_t group_size, bool fast,
                         std::optional<torch::ScalarType> out_dtype) {
  check_weight(Wq, S, Wq.device());
  const int64_t K = Wq.size(0) * 8, N = Wq.size(1);
  TORCH_CHECK(S.size(1) == N, "scale columns disagree with N");
  TORCH_CHECK(group_size > 0 && S.size(0) * group_size == K, "scale rows disagree with K/group_size");
  const auto dt = out_dtype.value_or(torch::kHalf);
  TORCH_CHECK(dt == torch::kHalf || dt == torch::kBFloat16, "out_dtype must be fp16 or bf16");
  const c10::cuda::CUDAGuard guard(Wq.device());
  auto out = torch::empty({K, N}, Wq.options().dtype(dt));
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(Wq.device().index()).stream();
  const int st = ng_dequant_w4(Wq.data_ptr<int32_t>(), reinterpret_cast<const uint16_t*>(S.data_ptr()),
                             out.data_ptr(), dt == torch::kHalf ? NG_DTYPE_F16 : NG_DTYPE_BF16,
                             static_cast<int>(K), static_cast<int>(N), static_cast<int>(group_size),
                             fast ? 1 : 0, stream);
  return {out, st};
}

// ---------------------------------------------------------------------------
// Paged KV cache and drafted trees.
// ---------------------------------------------------------------------------
void check_ints(const torch::Tensor& t, const torch::Device& dev, torch::ScalarType type, int64_t dim,
                const char* name) {
  TORCH_CHECK(t.device() == dev, name, " must be on ", dev);
  TORCH_CHECK(t.scalar_type() == type, name, " must be ", type);
  TORCH_CHECK(t.dim() == dim && t.is_contiguous(), name, " must be a contiguous ", dim, "-D tensor");
}

// A [.., pages, page_size, heads, D] cache pair: same type, shape and strides, D contiguous.
void check_caches(const torch::Tensor& K, const torch::Tensor& V, int64_t dim, const torch::Device& dev) {
  TORCH_CHECK(K.is_cuda() && K.device() == dev && V.device() == dev, "the caches must be on the same CUDA device");
  dtype_code(K);
  TORCH_CHECK(K.dim() == dim && V.dim() == dim, "the caches must be ", dim, "-D");
  TORCH_CHECK(K.sizes() == V.sizes() && K.strides() == V.strides() && K.scalar_type() == V.scalar_type(),
              "the K and V caches must have the same type, shape and strides");
  TORCH_CHECK(K.stride(dim - 1) == 1, "the caches' last dimension must be contiguous");
}

// Row stride of a block table whose rows are contiguous.
int64_t check_table(const torch::Tensor& t, const torch::Device& dev, int64_t B) {
  TORCH_CHECK(t.device() == dev && t.scalar_type() == torch::kInt && t.dim() == 2 && t.size(0) == B &&
                  t.stride(1) == 1 && t.size(1) >= 1,
              "block_table must be an int32 [requests, blocks] tensor with contiguous rows");
  return B > 1 ? t.stride(0) : std::max(t.stride(0), t.size(1));
}

// Several small outputs out of one allocation: each begins on a 16-byte boundary of
// `buffer` (uint8).  Made without the dispatcher, which takes most of a microsecond
// for each empty() or view.
class Slices {
 public:
  Slices(int64_t bytes, const torch::Device& dev)
      : buffer_(torch::empty({bytes}, torch::TensorOptions().dtype(torch::kUInt8).device(dev))) {}
  static int64_t padded(int64_t bytes) { return (bytes + 15) / 16 * 16; }
  torch::Tensor take(torch::IntArrayRef sizes, torch::ScalarType type) {
    int64_t n = 1;
    for (const auto s : sizes) n *= s;
    const int64_t item = static_cast<int64_t>(c10::elementSize(type));
    auto t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buffer_.storage()), buffer_.key_set(),
                                                      c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_storage_offset(used_ / item);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    used_ += padded(n * item);
    TORCH_INTERNAL_ASSERT(used_ <= buffer_.numel());
    return t;
  }

 private:
  torch::Tensor buffer_;
  int64_t used_ = 0;
};

std::tuple<std::vector<std::optional<torch::Tensor>>, int64_t> paged_plan(
    torch::Tensor cached, torch::Tensor fresh, torch::Tensor held, torch::Tensor table, torch::Tensor free_pages,
    int64_t page_size, int64_t num_tokens, std::optional<torch::Tensor> parents, int64_t mask_words,
    std::optional<torch::Tensor> cursor) {
  TORCH_CHECK(cached.is_cuda(), "all tensors must live on CUDA");
  const auto dev = cached.device();
  const int64_t B = cached.size(0);
  check_ints(cached, dev, torch::kInt, 1, "cached");
  check_ints(fresh, dev, torch::kInt, 1, "new");
  check_ints(held, dev, torch::kInt, 1, "held");
  check_ints(free_pages, dev, torch::kInt, 1, "free_pages");
  TORCH_CHECK(fresh.size(0) == B && held.size(0) == B, "cached, new and held must have one entry per request");
  const int64_t stride = check_table(table, dev, B);
  TORCH_CHECK(num_tokens >= 0 && num_tokens <= (1 << 30), "num_tokens out of range");
  TORCH_CHECK(mask_words == 0 || parents.has_value(), "a mask needs parents");
  if (parents.has_value()) {
    check_ints(*parents, dev, torch::kInt, 1, "parents");
    TORCH_CHECK(parents->size(0) == num_tokens, "parents must have num_tokens entries");
  }
  if (cursor.has_value()) {
    check_ints(*cursor, dev, torch::kInt, 1, "cursor");
    TORCH_CHECK(cursor->size(0) == 1, "cursor must have one entry");
  }
  const c10::cuda::CUDAGuard guard(dev);
  TORCH_CHECK(mask_words >= 0 && mask_words <= 64, "mask_words must be 0..64");
  const int64_t token = Slices::padded(num_tokens * 4), request = Slices::padded(B * 4);
  Slices slices(Slices::padded((B + 1) * 4) + 2 * token + 2 * request + 16 + Slices::padded(num_tokens * mask_words * 8),
                dev);
  auto cu = slices.take({B + 1}, torch::kInt), slots = slices.take({num_tokens}, torch::kInt),
       positions = slices.take({num_tokens}, torch::kInt), kv = slices.take({B}, torch::kInt),
       held_out = slices.take({B}, torch::kInt), taken = slices.take({1}, torch::kInt);
  std::optional<torch::Tensor> mask;
  if (mask_words > 0) mask = slices.take({num_tokens, mask_words}, torch::kLong);
  if (B == 0) {  // all tokens are rows past the last request's
    for (auto* t : {&cu, &positions, &taken}) t->zero_();
    slots.fill_(-1);
    if (mask) mask->zero_();
    return {{cu, slots, positions, kv, held_out, taken, mask}, 0};
  }
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  const int st = ng_paged_plan(
      cached.data_ptr<int>(), fresh.data_ptr<int>(), held.data_ptr<int>(), table.data_ptr<int>(), stride,
      static_cast<int>(table.size(1)), free_pages.data_ptr<int>(), static_cast<int>(free_pages.size(0)),
      cursor ? cursor->data_ptr<int>() : nullptr, parents ? parents->data_ptr<int>() : nullptr,
      static_cast<int>(B), static_cast<int>(num_tokens), static_cast<int>(page_size),
      static_cast<int>(mask_words), cu.data_ptr<int>(), slots.data_ptr<int>(), positions.data_ptr<int>(),
      kv.data_ptr<int>(), held_out.data_ptr<int>(), taken.data_ptr<int>(),
      mask ? reinterpret_cast<long long*>(mask->data_ptr<int64_t>()) : nullptr, stream);
  return {{cu, slots, positions, kv, held_out, taken, mask}, st};
}

std::tuple<torch::Tensor, int64_t> qk_norm_rope_append(
    torch::Tensor qkv, std::optional<torch::Tensor> q_weight, std::optional<torch::Tensor> k_weight,
    torch::Tensor turns, torch::Tensor positions, torch::Tensor slots, torch::Tensor K, torch::Tensor V,
    int64_t q_heads, double eps, std::optional<torch::Tensor> out) {
  TORCH_CHECK(qkv.is_cuda(), "all tensors must live on CUDA");
  const auto dev = qkv.device();
  check_caches(K, V, 4, dev);
  const int64_t M = qkv.size(0), Hkv = K.size(2), D = K.size(3);
  TORCH_CHECK(qkv.scalar_type() == K.scalar_type(), "qkv and the caches must have the same type");
  TORCH_CHECK(qkv.dim() == 2 && qkv.size(1) == (q_heads + 2 * Hkv) * D && qkv.stride(1) == 1,
              "qkv must be [tokens, (q_heads + 2 kv_heads) * D] with contiguous rows");
  check_ints(turns, dev, torch::kLong, 1, "turns");
  check_ints(positions, dev, torch::kInt, 1, "positions");
  check_ints(slots, dev, torch::kInt, 1, "slots");
  TORCH_CHECK(positions.size(0) == M && slots.size(0) == M, "positions and slots must have one entry per token");
  TORCH_CHECK(q_weight.has_value() == k_weight.has_value(), "give both norm weights or neither");
  for (const auto* w : {&q_weight, &k_weight})
    if (w->has_value())
      TORCH_CHECK((*w)->device() == dev && (*w)->scalar_type() == qkv.scalar_type() && (*w)->dim() == 1 &&
                      (*w)->size(0) == D && (*w)->is_contiguous(),
                  "a norm weight must be a contiguous [D] tensor of the type of qkv");
  if (out.has_value())
    TORCH_CHECK(out->device() == dev && out->scalar_type() == qkv.scalar_type() && out->is_contiguous() &&
                    out->sizes() == torch::IntArrayRef({M, q_heads, D}),
                "out must be a contiguous [tokens, q_heads, D] tensor like qkv");
  const c10::cuda::CUDAGuard guard(dev);
  auto q = out.has_value() ? *out : torch::empty({M, q_heads, D}, qkv.options());
  if (M == 0) return {q, 0};
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  const int st = ng_qk_norm_rope_append(
      qkv.data_ptr(), M > 1 ? qkv.stride(0) : qkv.size(1), q_weight ? q_weight->data_ptr() : nullptr,
      k_weight ? k_weight->data_ptr() : nullptr, reinterpret_cast<const long long*>(turns.data_ptr<int64_t>()),
      static_cast<int>(2 * turns.size(0)), positions.data_ptr<int>(), slots.data_ptr<int>(), q.data_ptr(),
      K.data_ptr(), V.data_ptr(), K.stride(0), K.stride(1), K.stride(2), dtype_code(qkv), static_cast<int>(M),
      static_cast<int>(q_heads), static_cast<int>(Hkv), static_cast<int>(D), static_cast<int>(K.size(0)),
      static_cast<int>(K.size(1)), static_cast<float>(eps), stream);
  return {q, st};
}

std::tuple<torch::Tensor, std::optional<torch::Tensor>, int64_t> tree_attention(
    torch::Tensor q, torch::Tensor K, torch::Tensor V, torch::Tensor table, torch::Tensor kv_lens,
    torch::Tensor cu_new, std::optional<torch::Tensor> mask, double scale, bool return_lse,
    std::optional<torch::Tensor> out) {
  TORCH_CHECK(q.is_cuda(), "all tensors must live on CUDA");
  const auto dev = q.device();
  check_caches(K, V, 4, dev);
  TORCH_CHECK(q.dim() == 3 && q.scalar_type() == K.scalar_type() && q.size(2) == K.size(3) && q.stride(2) == 1,
              "q must be [tokens, q_heads, D] of the caches' type with D contiguous");
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2), B = kv_lens.size(0);
  check_ints(kv_lens, dev, torch::kInt, 1, "kv_lens");
  check_ints(cu_new, dev, torch::kInt, 1, "cu_new");
  TORCH_CHECK(cu_new.size(0) == B + 1, "cu_new must have one entry more than kv_lens");
  const int64_t stride = check_table(table, dev, B);
  if (mask.has_value()) {
    check_ints(*mask, dev, torch::kLong, 2, "mask");
    TORCH_CHECK(mask->size(0) == T && mask->size(1) >= 1, "mask must be [tokens, words]");
  }
  if (out.has_value())
    TORCH_CHECK(out->device() == dev && out->scalar_type() == q.scalar_type() && out->is_contiguous() &&
                    out->sizes() == q.sizes(),
                "out must be a contiguous tensor like q");
  const c10::cuda::CUDAGuard guard(dev);
  auto y = out.has_value() ? *out : torch::empty({T, Hq, D}, q.options());
  std::optional<torch::Tensor> lse;
  if (return_lse) lse = torch::empty({T, Hq}, q.options().dtype(torch::kFloat));
  if (T == 0) return {y, lse, 0};
  if (B == 0) {  // tokens of no request see nothing
    y.zero_();
    if (lse) lse->fill_(-std::numeric_limits<float>::infinity());
    return {y, lse, 0};
  }
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  auto ws = attention_workspace(dev, stream, ng_tree_attn_workspace_bytes(static_cast<int>(D)));
  const int st = ng_tree_attn(
      q.data_ptr(), q.stride(0), q.stride(1), K.data_ptr(), V.data_ptr(), K.stride(0), K.stride(1), K.stride(2),
      table.data_ptr<int>(), stride, static_cast<int>(table.size(1)), kv_lens.data_ptr<int>(),
      cu_new.data_ptr<int>(), mask ? reinterpret_cast<const long long*>(mask->data_ptr<int64_t>()) : nullptr,
      mask ? static_cast<int>(mask->size(1)) : 0, y.data_ptr(), lse ? lse->data_ptr<float>() : nullptr,
      dtype_code(q), static_cast<int>(B), static_cast<int>(T), static_cast<int>(Hq), static_cast<int>(K.size(2)),
      static_cast<int>(D), static_cast<int>(K.size(0)), static_cast<int>(K.size(1)), static_cast<float>(scale),
      ws.data_ptr(), static_cast<size_t>(ws.numel()), stream);
  return {y, lse, st};
}

std::tuple<torch::Tensor, torch::Tensor, torch::Tensor, torch::Tensor, int64_t> tree_commit(
    torch::Tensor draft, torch::Tensor parents, torch::Tensor next, torch::Tensor cu_new, torch::Tensor kv_lens,
    torch::Tensor table, torch::Tensor K, torch::Tensor V, int64_t max_path) {
  TORCH_CHECK(draft.is_cuda(), "all tensors must live on CUDA");
  const auto dev = draft.device();
  TORCH_CHECK(K.dim() == 4 || K.dim() == 5, "the caches must be [layers, pages, page_size, heads, D] or one layer of it");
  const int64_t o = K.dim() - 4;
  check_caches(K, V, 4 + o, dev);
  check_ints(draft, dev, torch::kLong, 1, "draft");
  check_ints(next, dev, torch::kLong, 1, "next");
  check_ints(parents, dev, torch::kInt, 1, "parents");
  check_ints(cu_new, dev, torch::kInt, 1, "cu_new");
  check_ints(kv_lens, dev, torch::kInt, 1, "kv_lens");
  const int64_t B = kv_lens.size(0), T = draft.size(0);
  TORCH_CHECK(next.size(0) == T && parents.size(0) == T, "draft, parents and next must have one entry per token");
  TORCH_CHECK(cu_new.size(0) == B + 1, "cu_new must have one entry more than kv_lens");
  TORCH_CHECK(max_path >= 1 && max_path <= 512, "max_path must be 1..512");
  const int64_t stride = check_table(table, dev, B);
  const c10::cuda::CUDAGuard guard(dev);
  Slices slices(2 * Slices::padded(B * 4) + Slices::padded(B * max_path * 4) + Slices::padded(B * 8), dev);
  auto accepted = slices.take({B}, torch::kInt), path = slices.take({B, max_path}, torch::kInt),
       bonus = slices.take({B}, torch::kLong), kv_out = slices.take({B}, torch::kInt);
  if (B == 0) return {accepted, path, bonus, kv_out, 0};
  if (T == 0) {
    accepted.zero_();
    path.fill_(-1);
    bonus.fill_(-1);
    kv_out.copy_(kv_lens);
    return {accepted, path, bonus, kv_out, 0};
  }
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(dev.index()).stream();
  auto* ll = +[](torch::Tensor& t) { return reinterpret_cast<long long*>(t.data_ptr<int64_t>()); };
  const int st = ng_tree_commit(
      ll(draft), parents.data_ptr<int>(), ll(next), cu_new.data_ptr<int>(), kv_lens.data_ptr<int>(),
      table.data_ptr<int>(), stride, static_cast<int>(table.size(1)), K.data_ptr(), V.data_ptr(),
      o ? K.stride(0) : 0, K.stride(o), K.stride(o + 1), K.stride(o + 2), dtype_code(K), static_cast<int>(B),
      static_cast<int>(T), o ? static_cast<int>(K.size(0)) : 1, static_cast<int>(K.size(o + 2)),
      static_cast<int>(K.size(o + 3)), static_cast<int>(K.size(o)), static_cast<int>(K.size(o + 1)),
      static_cast<int>(max_path), accepted.data_ptr<int>(), path.data_ptr<int>(), ll(bonus),
      kv_out.data_ptr<int>(), stream);
  return {accepted, path, bonus, kv_out, st};
}

// The cached workspace a call on (device, stream) uses (for inspection).
torch::Tensor workspace_for(int64_t device_index, int64_t stream, int64_t kind, int64_t need) {
  return workspace(torch::Device(torch::kCUDA, static_cast<c10::DeviceIndex>(device_index)),
                   reinterpret_cast<cudaStream_t>(stream), static_cast<int>(kind), static_cast<size_t>(need));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("gemv_w4a16", &gemv_w4a16, "Decode-regime W4A16 GEMV (M <= 16).", py::arg("X"), py::arg("Wq"),
        py::arg("S"), py::arg("group_size"), py::arg("version") = 4, py::arg("splits_override") = 0,
        py::arg("threads_override") = 0, py::arg("algo") = 0, py::arg("out") = py::none());
  m.def("gemm_w4a16", &gemm_w4a16, "Prefill-regime W4A16 GEMM (tcgen05).", py::arg("X"), py::arg("Wq"),
        py::arg("S"), py::arg("group_size"), py::arg("version") = 6, py::arg("tile_tokens") = 0,
        py::arg("out") = py::none());
  m.def("workspace", &workspace_for, "The cached workspace of (device, stream); kind 0 = GEMV, 1 = GEMM (both zero-initialised), 2 = tree attention.",
        py::arg("device_index"), py::arg("stream"), py::arg("kind"), py::arg("need"));
  m.def("paged_plan", &paged_plan);
  m.def("qk_norm_rope_append", &qk_norm_rope_append);
  m.def("tree_attention", &tree_attention);
  m.def("tree_commit", &tree_commit);
  m.def("dequant_w4", &dequant_w4, "Packed INT4 to dense fp16 / bf16.", py::arg("Wq"), py::arg("S"),
        py::arg("group_size"), py::arg("fast") = true, py::arg("out_dtype") = py::none());
}
