// Writing and reading the paged 8-bit KV cache (sm_100a).
//
// The format.  K and V each are e4m3 codes [pages, Hkv, page size, D] with one scale for
// each (page, KV head): value = code * scale.  A scale is 2^e with the smallest e >= -100
// for which every finite |x| of its block is at most 448 * 2^e (448 is e4m3's largest
// value).  e4m3 is a floating type, so a scale that is a power of two costs no precision
// above its subnormals, and multiplying by it is exact.  A token's slot is
// page * page_size + place in the page.
//
// Appending to a page that holds tokens already may need a larger scale: the older
// codes c become RN(c * old / new), exact for powers of two but for values that fall
// into e4m3's subnormals (below 2^-6 of the new scale).  A scale never shrinks while a
// page fills; rows that begin at place 0 start the page, and its scale, afresh.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "sparknet/kv_pool.h"

namespace py = pybind11;

namespace {

constexpr int kThreads = 256;
constexpr int kMinExponent = -100;

// --- conversions ------------------------------------------------------------------------
__device__ __forceinline__ float2 to_float2(uint32_t w, __nv_bfloat16) {
  __nv_bfloat162 h = *reinterpret_cast<__nv_bfloat162*>(&w);
  return __bfloat1622float2(h);
}
__device__ __forceinline__ float2 to_float2(uint32_t w, __half) {
  __half2 h = *reinterpret_cast<__half2*>(&w);
  return __half22float2(h);
}
__device__ __forceinline__ uint32_t from_float2(float a, float b, __nv_bfloat16) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t from_float2(float a, float b, __half) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

template <class T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = to_float2(u[i], T());
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

// Two floats to two e4m3 codes (low byte first): nearest even, infinities saturate to
// +-448, NaN stays NaN.
__device__ __forceinline__ uint32_t codes2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}

// Two e4m3 codes to two floats, exactly (through fp16, which holds every e4m3 value).
__device__ __forceinline__ float2 values2(uint32_t codes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(uint16_t(codes)));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}

// 2^e, the smallest scale (e >= kMinExponent) with amax <= 448 * 2^e, from amax's bits:
// amax = m * 2^x with 1 <= m < 2, and 448 = 1.75 * 2^8.
__device__ __forceinline__ float scale_for(float amax) {
  const int bits = __float_as_int(amax);
  int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  e = max(e, kMinExponent);
  return __int_as_float((e + 127) << 23);
}

struct AppendArgs {
  const void *k, *v, *q;        // rows of one 16-bit type
  int64_t k_row, k_head, v_row, v_head, q_row, q_head;  // strides in elements
  void* q_out;                  // [n, Hq, D] contiguous (rope only)
  const int *slots, *positions;
  const float *cos_t, *sin_t;   // [table rows, D / 2] (rope only)
  uint8_t *kc, *vc;
  float *ks, *vs;
  int64_t slots_in_pool;
  int n, hq, hkv, page_size, rows_per_block, table_rows, q_blocks;
};

// Chunk `c` (8 elements) of a row of D, rotated (rotate-half form) if ROPE.  Products and
// sums round separately, as an unfused fp32 computation does.
template <class T, int D, bool ROPE>
__device__ __forceinline__ void load_chunk(const T* row, int c, const float* cos_row, const float* sin_row,
                                           float (&x)[8]) {
  load8(row + c * 8, x);
  if constexpr (ROPE) {
    constexpr int H = D / 16;  // chunks in half a row
    const bool low = c < H;
    const int pc = low ? c + H : c - H, tc = low ? c : c - H;
    float y[8];
    load8(row + pc * 8, y);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float cs = cos_row[tc * 8 + i], sn = sin_row[tc * 8 + i];
      const float own = __fmul_rn(x[i], cs), other = __fmul_rn(y[i], sn);
      x[i] = low ? __fsub_rn(own, other) : __fadd_rn(own, other);
    }
  }
}

// One block: the runs of rows that begin in its `rows_per_block` rows, one KV head; half
// the threads do K, half V.  A run is rows with consecutive slots in one page, so one block
// sees all that a call adds to a page and head.
template <class T, int D, bool ROPE>
__global__ void __launch_bounds__(kThreads) k_append(AppendArgs a) {
  constexpr int kChunks = D / 8, kSide = kThreads / 2, kRows = kSide / kChunks;
  constexpr int kHeld = 4;  // passes over a run that stay in registers
  __shared__ float warp_max[kThreads / 32];
  const int r0 = blockIdx.x * a.rows_per_block, r1 = min(a.n, r0 + a.rows_per_block);
  if constexpr (ROPE) {
    if (int(blockIdx.y) >= a.hkv) {  // rotate q
      const int part = blockIdx.y - a.hkv;
      const T* q = static_cast<const T*>(a.q);
      T* out = static_cast<T*>(a.q_out);
      const int total = (r1 - r0) * a.hq * kChunks;
      for (int i = part * kThreads + threadIdx.x; i < total; i += a.q_blocks * kThreads) {
        const int c = i % kChunks, h = i / kChunks % a.hq, r = r0 + i / kChunks / a.hq;
        const int pos = min(max(a.positions[r], 0), a.table_rows - 1);
        float x[8];
        load_chunk<T, D, true>(q + r * a.q_row + h * a.q_head, c, a.cos_t + int64_t(pos) * (D / 2),
                               a.sin_t + int64_t(pos) * (D / 2), x);
        uint4 w;
        w.x = from_float2(x[0], x[1], T());
        w.y = from_float2(x[2], x[3], T());
        w.z = from_float2(x[4], x[5], T());
        w.w = from_float2(x[6], x[7], T());
        *reinterpret_cast<uint4*>(out + (int64_t(r) * a.hq + h) * D + c * 8) = w;
      }
      return;
    }
  }
  const int h = blockIdx.y, lane = threadIdx.x & 31;
  const bool is_v = threadIdx.x >= kSide;
  const int tid = threadIdx.x % kSide, c = tid % kChunks, first = tid / kChunks;
  const T* src = static_cast<const T*>(is_v ? a.v : a.k) + h * (is_v ? a.v_head : a.k_head);
  const int64_t stride = is_v ? a.v_row : a.k_row;
  const int ps = a.page_size;

  auto values = [&](int r, float(&x)[8]) {
    if (ROPE && !is_v) {
      const int pos = min(max(a.positions[r], 0), a.table_rows - 1);
      load_chunk<T, D, ROPE>(src + r * stride, c, a.cos_t + int64_t(pos) * (D / 2), a.sin_t + int64_t(pos) * (D / 2),
                             x);
    } else {
      load8(src + r * stride + c * 8, x);
    }
  };

  // which of the block's rows begin a run: every warp asks for itself
  for (int r32 = r0; r32 < r1; r32 += 32) {
    const int own = r32 + lane < r1 ? a.slots[r32 + lane] : -1;
    const int prior = r32 + lane < r1 && r32 + lane > 0 ? a.slots[r32 + lane - 1] : -1;
    uint32_t begins = __ballot_sync(0xffffffffu, own >= 0 && own < a.slots_in_pool &&
                                                     (own % ps == 0 || r32 + lane == 0 || prior != own - 1));
    for (; begins; begins &= begins - 1) {
      const int r = r32 + __ffs(begins) - 1, slot = __shfl_sync(0xffffffffu, own, __ffs(begins) - 1);
      const int place = slot % ps;
      const int64_t block = int64_t(slot / ps) * a.hkv + h;
      float* scale_at = (is_v ? a.vs : a.ks) + block;
      uint8_t* codes = (is_v ? a.vc : a.kc) + block * ps * D;
      const float old = place ? *scale_at : 0.0f;
      int count = 1;  // rows of the run
      for (;;) {
        const int j = count + lane;
        const bool on = place + j < ps && r + j < a.n && a.slots[r + j] == slot + j;
        const uint32_t m = __ballot_sync(0xffffffffu, on);
        if (m == 0xffffffffu) {
          count += 32;
          continue;
        }
        count += __ffs(~m) - 1;
        break;
      }

      float x[kHeld][8], amax = 0.0f;
      auto load_group = [&](int j0) {
#pragma unroll
        for (int p = 0; p < kHeld; ++p) {
          const int j = j0 + p * kRows + first;
          if (j < count) values(r + j, x[p]);
        }
      };
      for (int j0 = 0; j0 < count; j0 += kHeld * kRows) {
        load_group(j0);
#pragma unroll
        for (int p = 0; p < kHeld; ++p)
          if (j0 + p * kRows + first < count)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float m = fabsf(x[p][i]);
              amax = fmaxf(amax, m <= 3.4028234e38f ? m : 0.0f);  // finite values only
            }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      if (lane == 0) warp_max[threadIdx.x / 32] = amax;
      __syncthreads();
      const float* wm = warp_max + (is_v ? kSide / 32 : 0);
#pragma unroll
      for (int i = 0; i < kSide / 32; ++i) amax = fmaxf(amax, wm[i]);
      __syncthreads();  // warp_max is free for the next run
      const float fresh = scale_for(amax), scale = place ? fmaxf(old, fresh) : fresh;
      if (tid == 0) *scale_at = scale;

      if (place && scale > old) {  // the older rows in the larger scale
        const float shrink = old / scale;
        for (int i = tid; i < place * D / 16; i += kSide) {
          uint4* at = reinterpret_cast<uint4*>(codes) + i;
          uint4 w = *at;
          uint32_t* u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 lo = values2(u[e] & 0xffffu), hi = values2(u[e] >> 16);
            u[e] = codes2(lo.x * shrink, lo.y * shrink) | codes2(hi.x * shrink, hi.y * shrink) << 16;
          }
          *at = w;
        }
      }
      const float inv = 1.0f / scale;
      for (int j0 = 0; j0 < count; j0 += kHeld * kRows) {
        if (count > kHeld * kRows) load_group(j0);  // a run of one group is still held
#pragma unroll
        for (int p = 0; p < kHeld; ++p) {
          const int j = j0 + p * kRows + first;
          if (j < count) {
            uint2 w;
            w.x = codes2(x[p][0] * inv, x[p][1] * inv) | codes2(x[p][2] * inv, x[p][3] * inv) << 16;
            w.y = codes2(x[p][4] * inv, x[p][5] * inv) | codes2(x[p][6] * inv, x[p][7] * inv) << 16;
            *reinterpret_cast<uint2*>(codes + (place + j) * D + c * 8) = w;
          }
        }
      }
    }
  }
}

// --- read: slots -> rows of K and V -------------------------------------------------------
// 8 words to a 32-byte aligned address, one sector at once.
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// 16 codes times `scale` to 16 values.
template <class O>
__device__ __forceinline__ void store16(O* p, uint4 codes, float scale) {
  const uint32_t u[4] = {codes.x, codes.y, codes.z, codes.w};
  uint32_t w[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 a = values2(u[e] & 0xffffu), b = values2(u[e] >> 16);
    w[2 * e] = from_float2(a.x * scale, a.y * scale, O());
    w[2 * e + 1] = from_float2(b.x * scale, b.y * scale, O());
  }
  store32(p, w);
}
template <>
__device__ __forceinline__ void store16<float>(float* p, uint4 codes, float scale) {
  const uint32_t u[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    uint32_t w[8];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float2 a = values2(u[2 * g + e] & 0xffffu), b = values2(u[2 * g + e] >> 16);
      w[4 * e] = __float_as_uint(a.x * scale);
      w[4 * e + 1] = __float_as_uint(a.y * scale);
      w[4 * e + 2] = __float_as_uint(b.x * scale);
      w[4 * e + 3] = __float_as_uint(b.y * scale);
    }
    store32(p + 8 * g, w);
  }
}

// Thread: 16 elements of K and of V of one (row, head).  Rows without a slot read as zeros.
template <class O, int D>
__global__ void __launch_bounds__(kThreads) k_read(const uint8_t* __restrict__ kc, const uint8_t* __restrict__ vc,
                                                   const float* __restrict__ ks, const float* __restrict__ vs,
                                                   const int* __restrict__ slots, O* __restrict__ k_out,
                                                   O* __restrict__ v_out, int64_t total, int hkv, int page_shift,
                                                   int64_t slots_in_pool) {
  constexpr int kChunks = D / 16;
  const int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  if (i >= total) return;
  const int c = int(i % kChunks);
  const int64_t rh = i / kChunks, row = total < (int64_t(1) << 31) ? int64_t(uint32_t(rh) / uint32_t(hkv)) : rh / hkv;
  const int h = int(rh - row * hkv), slot = slots[row];
  uint4 kw = make_uint4(0, 0, 0, 0), vw = kw;
  float a = 0.0f, b = 0.0f;
  if (slot >= 0 && slot < slots_in_pool) {
    const int64_t block = int64_t(slot >> page_shift) * hkv + h;
    const int64_t at = ((block << page_shift) + (slot & ((1 << page_shift) - 1))) * D + c * 16;
    kw = *reinterpret_cast<const uint4*>(kc + at);
    vw = *reinterpret_cast<const uint4*>(vc + at);
    a = ks[block];
    b = vs[block];
  }
  store16(k_out + i * 16, kw, a);
  store16(v_out + i * 16, vw, b);
}

template <class T, int D, bool ROPE>
void launch_append(AppendArgs a, cudaStream_t st) {
  // enough rows to a block that prompts do not launch mostly idle blocks, few enough that a
  // decode step's rows go to blocks of their own
  int rows = 1;
  while (rows < a.page_size && int64_t(a.n) * a.hkv / rows > 148 * 16) rows *= 2;
  a.rows_per_block = rows;
  a.q_blocks = ROPE ? int(std::min<int64_t>((int64_t(rows) * a.hq * (D / 8) + kThreads - 1) / kThreads, 64)) : 0;
  const dim3 grid((a.n + rows - 1) / rows, a.hkv + a.q_blocks);
  k_append<T, D, ROPE><<<grid, kThreads, 0, st>>>(a);
  sn::kv::need_ok(cudaGetLastError(), "kv_append launch");
}

template <bool ROPE>
void append_by_type(const AppendArgs& a, at::ScalarType t, int dim, cudaStream_t st) {
  if (t == at::kBFloat16) {
    if (dim == 128) launch_append<__nv_bfloat16, 128, ROPE>(a, st);
    else launch_append<__nv_bfloat16, 64, ROPE>(a, st);
  } else {
    if (dim == 128) launch_append<__half, 128, ROPE>(a, st);
    else launch_append<__half, 64, ROPE>(a, st);
  }
}

}  // namespace

namespace sn {
namespace kv {

KvPool::KvPool(at::Tensor k_, at::Tensor v_, at::Tensor ks_, at::Tensor vs_)
    : k(std::move(k_)), v(std::move(v_)), k_scale(std::move(ks_)), v_scale(std::move(vs_)) {
  need(k.dim() == 4 && k.sizes() == v.sizes(), "k and v must be [pages, kv_heads, page_size, head_dim], both alike");
  need(k.scalar_type() == at::kFloat8_e4m3fn && v.scalar_type() == at::kFloat8_e4m3fn,
       "k and v must be float8_e4m3fn");
  need(k.is_contiguous() && v.is_contiguous(), "k and v must be contiguous");
  pages = k.size(0);
  heads = int(k.size(1));
  page_size = int(k.size(2));
  dim = int(k.size(3));
  need(page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128,
       "page_size must be 16, 32, 64 or 128");
  need(dim == 64 || dim == 128, "head_dim must be 64 or 128");
  need(pages >= 1 && k.size(1) >= 1 && k.size(1) <= 4096, "the cache needs at least one page and 1..4096 KV heads");
  need(pages * page_size <= INT32_MAX && pages * heads <= INT32_MAX,
       "the cache's slots and (page, KV head) pairs must number below 2^31");
  for (const at::Tensor* s : {&k_scale, &v_scale})
    need(s->dim() == 2 && s->size(0) == pages && s->size(1) == heads && s->scalar_type() == at::kFloat &&
             s->is_contiguous(),
         "scales must be contiguous float32 [pages, kv_heads]");
  need_device(v, "v");
  need_device(k_scale, "k_scale");
  need_device(v_scale, "v_scale");
  need(aligned16(k.data_ptr()) && aligned16(v.data_ptr()), "k and v must be 16-byte aligned");
  err = at::zeros({1}, k_scale.options().dtype(at::kInt));
}

static void need_rows(const at::Tensor& t, const char* what) {
  for (int i = 0; i + 1 < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) % 8) throw std::invalid_argument(std::string(what) + " must have strides that are multiples of 8 elements");
  if ((t.size(t.dim() - 1) > 1 && t.stride(t.dim() - 1) != 1) || !aligned16(t.data_ptr()))
    throw std::invalid_argument(std::string(what) + " must be 16-byte aligned with contiguous rows");
}

static void need_int32(const at::Tensor& t, int64_t n, const char* what) {
  if (t.dim() != 1 || t.size(0) != n || t.scalar_type() != at::kInt || !t.is_contiguous())
    throw std::invalid_argument(std::string(what) + " must be contiguous int32, one for each row");
}

void KvPool::append(const at::Tensor& kx, const at::Tensor& vx, const at::Tensor& slots) {
  need(kx.dim() == 3 && kx.sizes() == vx.sizes() && kx.size(1) == heads && kx.size(2) == dim,
       "k and v rows must be [n, kv_heads, head_dim], both alike");
  need(is_16bit(kx) && kx.scalar_type() == vx.scalar_type(), "k and v rows must be both bfloat16 or both float16");
  need(kx.size(0) <= INT32_MAX, "too many rows");
  need_rows(kx, "k rows");
  need_rows(vx, "v rows");
  need_int32(slots, kx.size(0), "slots");
  need_device(kx, "k rows");
  need_device(vx, "v rows");
  need_device(slots, "slots");
  need_cuda();
  if (kx.size(0) == 0) return;
  c10::cuda::CUDAGuard guard(k.device());
  AppendArgs a{};
  a.k = kx.data_ptr();
  a.v = vx.data_ptr();
  a.k_row = kx.stride(0);
  a.k_head = kx.stride(1);
  a.v_row = vx.stride(0);
  a.v_head = vx.stride(1);
  a.slots = slots.data_ptr<int>();
  a.kc = static_cast<uint8_t*>(k.data_ptr());
  a.vc = static_cast<uint8_t*>(v.data_ptr());
  a.ks = k_scale.data_ptr<float>();
  a.vs = v_scale.data_ptr<float>();
  a.slots_in_pool = pages * page_size;
  a.n = int(kx.size(0));
  a.hkv = heads;
  a.page_size = page_size;
  append_by_type<false>(a, kx.scalar_type(), dim, stream());
}

at::Tensor KvPool::rope_append(const at::Tensor& qkv, const at::Tensor& cos_t, const at::Tensor& sin_t,
                               const at::Tensor& positions, const at::Tensor& slots,
                               const c10::optional<at::Tensor>& q_out) {
  need(qkv.dim() == 2 && qkv.size(1) % dim == 0 && qkv.size(1) / dim > 2 * heads,
       "qkv must be [n, (heads + 2 kv_heads) * head_dim]");
  need(is_16bit(qkv), "qkv must be bfloat16 or float16");
  const int64_t n = qkv.size(0), hq = qkv.size(1) / dim - 2 * heads;
  need(n <= INT32_MAX && hq <= 4096, "too many rows or heads");
  need_rows(qkv, "qkv");
  for (const at::Tensor* t : {&cos_t, &sin_t})
    need(t->dim() == 2 && t->size(1) == dim / 2 && t->size(0) >= 1 && t->scalar_type() == at::kFloat &&
             t->is_contiguous() && t->size(0) == cos_t.size(0) && t->size(0) <= INT32_MAX,
         "cos and sin must be contiguous float32 [positions, head_dim / 2], both alike");
  need_int32(positions, n, "positions");
  need_int32(slots, n, "slots");
  if (q_out)
    need(q_out->dim() == 3 && q_out->size(0) == n && q_out->size(1) == hq && q_out->size(2) == dim &&
             q_out->scalar_type() == qkv.scalar_type() && q_out->is_contiguous() && aligned16(q_out->data_ptr()),
         "q_out must be contiguous [n, heads, head_dim] of qkv's type");
  need_device(qkv, "qkv");
  need_device(cos_t, "cos");
  need_device(sin_t, "sin");
  need_device(positions, "positions");
  need_device(slots, "slots");
  if (q_out) need_device(*q_out, "q_out");
  need_cuda();
  c10::cuda::CUDAGuard guard(k.device());
  at::Tensor q = q_out ? *q_out : at::empty({n, hq, dim}, qkv.options());
  if (n == 0) return q;
  AppendArgs a{};
  const char* base = static_cast<const char*>(qkv.data_ptr());
  a.q = base;
  a.k = base + hq * dim * 2;
  a.v = base + (hq + heads) * dim * 2;
  a.q_row = a.k_row = a.v_row = qkv.stride(0);
  a.q_head = a.k_head = a.v_head = dim;
  a.q_out = q.data_ptr();
  a.slots = slots.data_ptr<int>();
  a.positions = positions.data_ptr<int>();
  a.cos_t = cos_t.data_ptr<float>();
  a.sin_t = sin_t.data_ptr<float>();
  a.table_rows = int(cos_t.size(0));
  a.kc = static_cast<uint8_t*>(k.data_ptr());
  a.vc = static_cast<uint8_t*>(v.data_ptr());
  a.ks = k_scale.data_ptr<float>();
  a.vs = v_scale.data_ptr<float>();
  a.slots_in_pool = pages * page_size;
  a.n = int(n);
  a.hq = int(hq);
  a.hkv = heads;
  a.page_size = page_size;
  append_by_type<true>(a, qkv.scalar_type(), dim, stream());
  return q;
}

std::tuple<at::Tensor, at::Tensor> KvPool::read(const at::Tensor& slots, at::ScalarType dtype,
                                                const c10::optional<at::Tensor>& k_out,
                                                const c10::optional<at::Tensor>& v_out) {
  need(slots.dim() == 1, "slots must be contiguous int32, one for each row");
  need_int32(slots, slots.size(0), "slots");
  need(dtype == at::kBFloat16 || dtype == at::kHalf || dtype == at::kFloat,
       "dtype must be bfloat16, float16 or float32");
  const int64_t n = slots.size(0);
  for (const auto* o : {&k_out, &v_out})
    if (*o)
      need((*o)->dim() == 3 && (*o)->size(0) == n && (*o)->size(1) == heads && (*o)->size(2) == dim &&
               (*o)->scalar_type() == dtype && (*o)->is_contiguous() &&
               (reinterpret_cast<uintptr_t>((*o)->data_ptr()) & 31) == 0,
           "k_out and v_out must be contiguous, 32-byte aligned [n, kv_heads, head_dim] of the given dtype");
  need_device(slots, "slots");
  if (k_out) need_device(*k_out, "k_out");
  if (v_out) need_device(*v_out, "v_out");
  need_cuda();
  c10::cuda::CUDAGuard guard(k.device());
  const auto options = k.options().dtype(dtype);
  at::Tensor ko = k_out ? *k_out : at::empty({n, heads, dim}, options);
  at::Tensor vo = v_out ? *v_out : at::empty({n, heads, dim}, options);
  const int64_t total = n * heads * (dim / 16);
  if (total == 0) return {ko, vo};
  need((total + kThreads - 1) / kThreads <= INT32_MAX, "too many rows");
  const int grid = int((total + kThreads - 1) / kThreads);
  auto go = [&](auto zero, auto d) {
    using O = decltype(zero);
    k_read<O, decltype(d)::value><<<grid, kThreads, 0, stream()>>>(
        static_cast<const uint8_t*>(k.data_ptr()), static_cast<const uint8_t*>(v.data_ptr()),
        k_scale.data_ptr<float>(), v_scale.data_ptr<float>(), slots.data_ptr<int>(), static_cast<O*>(ko.data_ptr()),
        static_cast<O*>(vo.data_ptr()), total, heads, __builtin_ctz(page_size), pages * page_size);
  };
  auto by_dim = [&](auto zero) {
    if (dim == 128) go(zero, std::integral_constant<int, 128>());
    else go(zero, std::integral_constant<int, 64>());
  };
  if (dtype == at::kBFloat16) by_dim(__nv_bfloat16());
  else if (dtype == at::kHalf) by_dim(__half());
  else by_dim(float());
  need_ok(cudaGetLastError(), "kv_read launch");
  return {ko, vo};
}

}  // namespace kv
}  // namespace sn

void register_kv_cache(py::module_& m) {
  using sn::kv::KvPool;
  py::class_<KvPool, std::shared_ptr<KvPool>>(m, "KvPool")
      .def(py::init<at::Tensor, at::Tensor, at::Tensor, at::Tensor>(), py::arg("k"), py::arg("v"), py::arg("k_scale"),
           py::arg("v_scale"))
      .def("append", &KvPool::append, py::arg("k"), py::arg("v"), py::arg("slots"))
      .def("rope_append", &KvPool::rope_append, py::arg("qkv"), py::arg("cos"), py::arg("sin"), py::arg("positions"),
           py::arg("slots"), py::arg("q_out") = py::none())
      .def("read", &KvPool::read, py::arg("slots"), py::arg("dtype"), py::arg("k_out") = py::none(),
           py::arg("v_out") = py::none())
      .def("attention", &KvPool::attention, py::arg("q"), py::arg("block_tables"), py::arg("lengths"),
           py::arg("scale"), py::arg("window"), py::arg("out") = py::none(), py::arg("want_lse") = false)
      .def("attention_launches", &KvPool::attention_launches, py::arg("sequences"), py::arg("tokens"),
           py::arg("heads"), py::arg("width"))
      .def_readonly("k", &KvPool::k)
      .def_readonly("v", &KvPool::v)
      .def_readonly("k_scale", &KvPool::k_scale)
      .def_readonly("v_scale", &KvPool::v_scale)
      .def_readonly("err", &KvPool::err)
      .def_readonly("num_pages", &KvPool::pages)
      .def_readonly("kv_heads", &KvPool::heads)
      .def_readonly("page_size", &KvPool::page_size)
      .def_readonly("head_dim", &KvPool::dim);
}
