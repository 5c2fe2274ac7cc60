// The paged 8-bit KV cache (host side): e4m3 codes [pages, KV heads, page size, head dim]
// for K and for V, and one fp32 scale for each (page, KV head) of each.  `KvPool` checks
// the tensors once, keeps them alive, and launches the operators of kv_cache.cu and
// paged_attention.cu on the caller's current stream.
#pragma once

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda.h>
#include <torch/extension.h>

#include <stdexcept>
#include <string>
#include <tuple>

namespace sn {
namespace kv {

inline void need(bool ok, const char* what) {
  if (!ok) throw std::invalid_argument(what);
}

inline void need_ok(cudaError_t e, const char* what) {
  if (e != cudaSuccess) throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

inline bool is_16bit(const at::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf;
}

class KvPool {
 public:
  KvPool(at::Tensor k, at::Tensor v, at::Tensor k_scale, at::Tensor v_scale);

  void append(const at::Tensor& k, const at::Tensor& v, const at::Tensor& slots);
  at::Tensor rope_append(const at::Tensor& qkv, const at::Tensor& cos_t, const at::Tensor& sin_t,
                         const at::Tensor& positions, const at::Tensor& slots, const c10::optional<at::Tensor>& q_out);
  std::tuple<at::Tensor, at::Tensor> read(const at::Tensor& slots, at::ScalarType dtype,
                                          const c10::optional<at::Tensor>& k_out,
                                          const c10::optional<at::Tensor>& v_out);
  std::tuple<at::Tensor, c10::optional<at::Tensor>> attention(const at::Tensor& q, const at::Tensor& tables,
                                                              const at::Tensor& lengths, double scale, int64_t window,
                                                              const c10::optional<at::Tensor>& out, bool want_lse);

  int attention_launches(int64_t sequences, int64_t tokens, int64_t hq, int64_t width) const;

  at::Tensor k, v, k_scale, v_scale;
  at::Tensor err;  // one int32: nonzero after a wait of the attention kernel ran out
  int64_t pages;
  int heads, page_size, dim;

 private:
  CUtensorMap make_map(const at::Tensor& codes) const;
  CUtensorMap k_map_, v_map_;  // made by the first attention call
  bool mapped_ = false;

  void need_device(const at::Tensor& t, const char* what) const {
    if (t.device() != k.device()) throw std::invalid_argument(std::string(what) + " must be on the cache's device");
  }
  void need_cuda() const { need(k.is_cuda(), "the cache is not on a CUDA device"); }
  cudaStream_t stream() const { return at::cuda::getCurrentCUDAStream(k.device().index()).stream(); }
};

}  // namespace kv
}  // namespace sn
