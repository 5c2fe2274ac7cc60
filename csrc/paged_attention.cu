// Decode attention over the paged 8-bit KV cache (sm_100a).
//
//   out[b, t, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale * q . k_j - max)
//
// over the keys j < lengths[b] that token t of the sequence's last T tokens sees: j <=
// lengths[b] - T + t, and j > lengths[b] - T + t - window where there is a window.  k_j and
// v_j are code * scale of j's page and KV head.  Rows that see no key give 0, lse -inf.
//
// This form: one block per (sequence, token, query head); 4 warps take every 4th key, each
// lane a slice of the head; running maximum and sum per warp, joined at the end.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "sparknet/kv_pool.h"

namespace {

constexpr int kWarps = 4;

struct AttnArgs {
  const void* q;
  void* out;
  float* lse;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int *tables, *lengths;
  int64_t q_b, q_t, q_h, table_row, pages;
  int T, hq, hkv, page_size, width, window;
  float scale_log2;
};

__device__ __forceinline__ float value1(uint8_t c) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(c)));
  return __low2float(*reinterpret_cast<__half2*>(&h));
}

template <class T, int D>
__global__ void __launch_bounds__(kWarps * 32) k_attention(AttnArgs a) {
  constexpr int E = D / 32;
  __shared__ float sm[kWarps], sl[kWarps], so[kWarps][D];
  const int h = blockIdx.x, t = blockIdx.y, b = blockIdx.z;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, kvh = h / (a.hq / a.hkv);
  const T* q = static_cast<const T*>(a.q) + b * a.q_b + t * a.q_t + h * a.q_h;
  float qf[E], o[E] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) qf[e] = float(q[lane * E + e]);
  const int64_t len = min(int64_t(a.lengths[b]), int64_t(a.width) * a.page_size);
  const int64_t end = len - a.T + t + 1, begin = a.window ? max(int64_t(0), end - a.window) : 0;
  for (int64_t j = begin + warp; j < end; j += kWarps) {
    const int page = a.tables[b * a.table_row + j / a.page_size];
    if (page < 0 || page >= a.pages) continue;
    const int64_t block = int64_t(page) * a.hkv + kvh, at = (block * a.page_size + j % a.page_size) * D + lane * E;
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) s += qf[e] * value1(a.kc[at + e]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= a.ks[block] * a.scale_log2;
    const float m2 = fmaxf(m, s), old = m == m2 ? 1.0f : exp2f(m - m2), p = exp2f(s - m2), vs = a.vs[block];
    l = l * old + p;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * old + p * vs * value1(a.vc[at + e]);
    m = m2;
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[warp][lane * E + e] = o[e];
  __syncthreads();
  if (int(threadIdx.x) >= D) return;
  float mm = -INFINITY, ll = 0.0f, oo = 0.0f;
  for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sm[w]);
  for (int w = 0; w < kWarps; ++w) {
    const float c = sm[w] == mm ? 1.0f : exp2f(sm[w] - mm);  // equal infinities too: NaN sums stay NaN
    ll += c * sl[w];
    oo += c * so[w][threadIdx.x];
  }
  const int64_t row = (int64_t(b) * a.T + t) * a.hq + h;
  static_cast<T*>(a.out)[row * D + threadIdx.x] = T(ll != 0.0f ? oo / ll : 0.0f);
  if (a.lse && threadIdx.x == 0) a.lse[row] = ll != 0.0f ? (mm + log2f(ll)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace

namespace sn {
namespace kv {

std::tuple<at::Tensor, c10::optional<at::Tensor>> KvPool::attention(const at::Tensor& q, const at::Tensor& tables,
                                                                    const at::Tensor& lengths, double scale,
                                                                    int64_t window,
                                                                    const c10::optional<at::Tensor>& out,
                                                                    bool want_lse) {
  need(q.dim() == 3 || q.dim() == 4, "q must be [sequences, heads, head_dim] or [sequences, tokens, heads, head_dim]");
  const bool many = q.dim() == 4;
  const int64_t n = q.size(0), T = many ? q.size(1) : 1, hq = q.size(many ? 2 : 1);
  need(q.size(many ? 3 : 2) == dim, "q's head_dim differs from the cache's");
  need(hq >= 1 && hq % heads == 0, "query heads must be a multiple of the cache's KV heads");
  need(is_16bit(q), "q must be bfloat16 or float16");
  need(n <= 4096 && T >= 1 && T * (hq / heads) <= 4096, "paged_decode_attention takes up to 4096 sequences and up to 4096 query rows for a KV head");
  for (int i = 0; i + 1 < q.dim(); ++i)
    need(q.size(i) <= 1 || q.stride(i) % 8 == 0, "q must have strides that are multiples of 8 elements");
  need(q.stride(q.dim() - 1) == 1 && aligned16(q.data_ptr()), "q must be 16-byte aligned with contiguous rows");
  need(tables.dim() == 2 && tables.size(0) == n && tables.size(1) >= 1 && tables.scalar_type() == at::kInt &&
           (tables.stride(1) == 1 || tables.size(1) == 1),
       "block_tables must be int32 [sequences, pages] with contiguous rows");
  need(tables.size(1) * page_size < (int64_t(1) << 30), "block_tables are limited to 2^30 tokens a sequence");
  need(lengths.dim() == 1 && lengths.size(0) == n && lengths.scalar_type() == at::kInt && lengths.is_contiguous(),
       "lengths must be contiguous int32 [sequences]");
  need(window >= 0 && window < (int64_t(1) << 30), "window must be in 0..2^30 (0: none)");
  need(std::isfinite(scale), "scale must be finite");
  if (out)
    need(out->sizes() == q.sizes() && out->scalar_type() == q.scalar_type() && out->is_contiguous() &&
             aligned16(out->data_ptr()),
         "out must be contiguous, of q's shape and type");
  need_device(q, "q");
  need_device(tables, "block_tables");
  need_device(lengths, "lengths");
  if (out) need_device(*out, "out");
  need_cuda();
  c10::cuda::CUDAGuard guard(k.device());
  at::Tensor o = out ? *out : at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  c10::optional<at::Tensor> lse;
  if (want_lse) lse = at::empty(q.sizes().slice(0, q.dim() - 1), q.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous));
  if (n == 0) return {o, lse};
  AttnArgs a{};
  a.q = q.data_ptr();
  a.out = o.data_ptr();
  a.lse = lse ? lse->data_ptr<float>() : nullptr;
  a.kc = static_cast<const uint8_t*>(k.data_ptr());
  a.vc = static_cast<const uint8_t*>(v.data_ptr());
  a.ks = k_scale.data_ptr<float>();
  a.vs = v_scale.data_ptr<float>();
  a.tables = tables.data_ptr<int>();
  a.lengths = lengths.data_ptr<int>();
  a.q_b = q.stride(0);
  a.q_t = many ? q.stride(1) : 0;
  a.q_h = q.stride(many ? 2 : 1);
  a.table_row = tables.stride(0);
  a.pages = pages;
  a.T = int(T);
  a.hq = int(hq);
  a.hkv = heads;
  a.page_size = page_size;
  a.width = int(tables.size(1));
  a.window = int(window);
  a.scale_log2 = float(scale * 1.4426950408889634);
  const dim3 grid(hq, T, n);
  if (q.scalar_type() == at::kBFloat16) {
    if (dim == 128) k_attention<__nv_bfloat16, 128><<<grid, kWarps * 32, 0, stream()>>>(a);
    else k_attention<__nv_bfloat16, 64><<<grid, kWarps * 32, 0, stream()>>>(a);
  } else {
    if (dim == 128) k_attention<__half, 128><<<grid, kWarps * 32, 0, stream()>>>(a);
    else k_attention<__half, 64><<<grid, kWarps * 32, 0, stream()>>>(a);
  }
  need_ok(cudaGetLastError(), "paged_decode_attention launch");
  return {o, lse};
}

}  // namespace kv
}  // namespace sn
