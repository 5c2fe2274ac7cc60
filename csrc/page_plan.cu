// Page planning for a paged KV cache: one launch turns the requests' lengths into block
// tables, the slot and position of every new token, and the next lengths (sm_100a).
//
// Free pages are a stack: free_pages[0 .. count).  The pages of finished requests are pushed
// in request order, then each request's new pages are popped from the top, in request order:
//
//   held  = ceil(length / page),  need = ceil((length + new) / page) - held
//   granted where need == 0 or the inclusive sum of need reaches at most the pages that are
//   free; the j-th page taken over all requests is free_pages[count - 1 - j].
//
// A request that would pass its table's width or the token rows is refused and takes part
// in no sum of pages.
//
// The work is two or three prefix sums over the requests and a map over the token rows; what
// bounds it is latency: the launch, two rounds of loads, the scans.  Few rows take one block
// of as many threads as there are rows or requests.  More take a cluster of 8 blocks: each
// block does the scans for itself (no exchange), finished requests' pages and token rows are
// shared out, and one cluster barrier lies between all reads of what the caller may have
// updated in place and its writes (1024 requests, 40,000 rows: 57.4 us in one block, of which
// most was one thread copying a finished request's pages; see the launch for the border).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <stdexcept>
#include <string>

namespace py = pybind11;

namespace {

constexpr int kThreads = 1024;
constexpr int kMaxRequests = 4096;

struct PlanArgs {
  const int *lengths, *fresh;  // tokens held, tokens to add
  const uint8_t* finished;     // or null
  int *tables, *free_pages;
  const int* free_count;
  int *slots, *positions, *starts, *lengths_out, *granted, *count_out;
  int requests, width, capacity, max_tokens, page_size;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}

// Exclusive prefix sum of x over the block, `total` its sum.  `sums` holds one word a warp.
__device__ __forceinline__ int64_t scan(int64_t x, int64_t* sums, int64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int64_t s = x;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int64_t t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  if (lane == 31) sums[warp] = s;
  __syncthreads();
  // every warp scans the warps' sums for itself
  int64_t w = lane < warps ? sums[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int64_t t = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += t;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const int64_t before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
  __syncthreads();  // sums is free
  return (warp ? before : 0) + s - x;
}

__global__ void __launch_bounds__(kThreads) k_plan(PlanArgs a) {
  extern __shared__ int shared[];
  int* starts = shared;                    // first token row of each request, and the end
  int* base = starts + a.requests + 1;     // tokens held
  int* taken = base + a.requests;          // pages taken by the requests before it; -1: refused
  int* add_of = taken + a.requests;        // new tokens; before that, places of finished requests' pages
  __shared__ int64_t sums[kThreads / 32];
  __shared__ int top;
  const int ps = a.page_size, shift = __ffs(ps) - 1, threads = blockDim.x;
  const int rank = cluster_rank(), blocks = cluster_size();
  if (blockIdx.x != rank) return;  // launched without its cluster: the first block does it all
  int64_t count = min(max(*a.free_count, 0), a.capacity);
  if (threadIdx.x == 0) top = 0;

  int64_t len_of = 0, fresh_of = 0;  // of request threadIdx.x
  bool done_of = false;
  if (int(threadIdx.x) < a.requests) {
    len_of = max(a.lengths[threadIdx.x], 0);
    fresh_of = max(a.fresh[threadIdx.x], 0);
    done_of = a.finished && a.finished[threadIdx.x];
  }
  auto load = [&](int b, int64_t& len, int64_t& add, bool& done) {
    len = add = 0;
    done = false;
    if (b >= a.requests) return;
    if (b == int(threadIdx.x)) {
      len = len_of;
      add = fresh_of;
      done = done_of;
    } else {
      len = max(a.lengths[b], 0);
      add = max(a.fresh[b], 0);
      done = a.finished && a.finished[b];
    }
  };

  if (a.finished) {  // push the pages of finished requests
    for (int b0 = 0; b0 < a.requests; b0 += threads) {
      const int b = b0 + threadIdx.x;
      int64_t len, add, total;
      bool done;
      load(b, len, add, done);
      const int64_t gone = done ? min((len + ps - 1) >> shift, int64_t(a.width)) : 0;
      const int64_t at = count + scan(gone, sums, total);
      if (b < a.requests) {
        add_of[b] = int(min(at, int64_t(a.capacity)));
        taken[b] = int(gone);
      }
      count = min(count + total, int64_t(a.capacity));
    }
    __syncthreads();
    // a warp looks at 32 requests and copies the pages of those that have any
    const int lane = threadIdx.x & 31, warps = blocks * threads / 32;
    for (int b0 = (rank * threads + threadIdx.x) / 32 * 32; b0 < a.requests; b0 += warps * 32) {
      const int mine = b0 + lane < a.requests ? taken[b0 + lane] : 0;
      for (uint32_t rest = __ballot_sync(0xffffffffu, mine > 0); rest; rest &= rest - 1) {
        const int b = b0 + __ffs(rest) - 1, gone = taken[b], at = add_of[b];
        const int* row = a.tables + int64_t(b) * a.width;
#pragma unroll 4
        for (int i = lane; i < gone; i += 32)
          if (at + i < a.capacity) a.free_pages[at + i] = row[i];
      }
    }
    __syncthreads();
  }

  int64_t pages = 0, rows = 0;
  for (int b0 = 0; b0 < a.requests; b0 += threads) {
    const int b = b0 + threadIdx.x;
    int64_t len, add, total;
    bool done;
    load(b, len, add, done);
    if (done) len = 0;
    const int64_t start = rows + scan(add, sums, total);
    rows += total;
    const int64_t after = (len + add + ps - 1) >> shift, held = (len + ps - 1) >> shift;
    const bool fits = after <= a.width && start + add <= a.max_tokens;
    const int64_t need = fits ? after - held : 0;
    const int64_t before = pages + scan(need, sums, total);
    pages += total;
    if (b < a.requests) {
      const bool ok = fits && (need == 0 || before + need <= count);
      starts[b] = int(min(start, int64_t(INT32_MAX)));
      base[b] = int(len);
      taken[b] = ok ? int(before) : -1;
      add_of[b] = int(add);
      if (ok && need) atomicMax(&top, int(before + need));
    }
  }
  if (threadIdx.x == 0) starts[a.requests] = int(min(rows, int64_t(INT32_MAX)));
  __syncthreads();
  // every block has read the caller's state, and the pushed pages are there
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");

  const int thread = rank * threads + threadIdx.x;
  for (int b = thread; b <= a.requests; b += blocks * threads) {
    a.starts[b] = starts[b];
    if (b == a.requests) {
      *a.count_out = int(count) - top;
      break;
    }
    const bool ok = taken[b] >= 0;
    a.granted[b] = ok ? add_of[b] : 0;
    a.lengths_out[b] = base[b] + (ok ? add_of[b] : 0);
  }
#pragma unroll 2
  for (int row = thread; row < a.max_tokens; row += blocks * threads) {
    int slot = -1, position = 0;
    if (row < starts[a.requests]) {
      int lo = 0, hi = a.requests - 1;  // the last request that starts at or before the row
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (starts[mid] <= row) lo = mid;
        else hi = mid - 1;
      }
      position = base[lo] + row - starts[lo];
      if (taken[lo] >= 0) {
        const int held = (base[lo] + ps - 1) >> shift, at = position >> shift, place = position & (ps - 1);
        int* entry = a.tables + int64_t(lo) * a.width + at;
        int page;
        if (at < held) {
          page = *entry;
        } else {
          page = a.free_pages[count - 1 - (taken[lo] + at - held)];
          if (place == 0) *entry = page;
        }
        slot = page * ps + place;
      }
    }
    a.slots[row] = slot;
    a.positions[row] = position;
  }
}

void need(bool ok, const char* what) {
  if (!ok) throw std::invalid_argument(what);
}

bool int32_vector(const at::Tensor& t, int64_t n) {
  return t.dim() == 1 && t.size(0) == n && t.scalar_type() == at::kInt && t.is_contiguous();
}

// -> (slots, positions, starts, lengths, granted, free_count)
std::vector<at::Tensor> plan_pages(const at::Tensor& lengths, const at::Tensor& fresh, at::Tensor& tables,
                                   at::Tensor& free_pages, const at::Tensor& free_count, int64_t page_size,
                                   int64_t max_tokens, const c10::optional<at::Tensor>& finished,
                                   const c10::optional<at::Tensor>& lengths_out,
                                   const c10::optional<at::Tensor>& count_out) {
  need(lengths.dim() == 1, "lengths must be contiguous int32 [requests]");
  const int64_t n = lengths.size(0);
  need(int32_vector(lengths, n), "lengths must be contiguous int32 [requests]");
  need(n >= 1 && n <= kMaxRequests, "plan_pages takes 1..4096 requests");
  need(int32_vector(fresh, n), "new_tokens must be contiguous int32 [requests]");
  need(tables.dim() == 2 && tables.size(0) == n && tables.size(1) >= 1 && tables.scalar_type() == at::kInt &&
           tables.is_contiguous(),
       "block_tables must be contiguous int32 [requests, pages]");
  need(free_pages.dim() == 1 && int32_vector(free_pages, free_pages.size(0)), "free_pages must be contiguous int32");
  need(int32_vector(free_count, 1), "free_count must be one int32");
  need(page_size == 16 || page_size == 32 || page_size == 64 || page_size == 128,
       "page_size must be 16, 32, 64 or 128");
  need(max_tokens >= 0 && max_tokens < (int64_t(1) << 30), "max_tokens must be in 0..2^30");
  need(tables.size(1) * page_size < (int64_t(1) << 30) && free_pages.size(0) < (int64_t(1) << 30),
       "the tables' width and the free list are limited to 2^30 tokens and pages");
  if (finished)
    need(finished->dim() == 1 && finished->size(0) == n && finished->scalar_type() == at::kBool &&
             finished->is_contiguous(),
         "finished must be contiguous bool [requests]");
  if (lengths_out) need(int32_vector(*lengths_out, n), "lengths_out must be contiguous int32 [requests]");
  if (count_out) need(int32_vector(*count_out, 1), "free_count_out must be one int32");
  for (const at::Tensor* t : {&fresh, static_cast<const at::Tensor*>(&tables),
                              static_cast<const at::Tensor*>(&free_pages), &free_count})
    need(t->device() == lengths.device(), "every tensor of a plan must be on one device");
  for (const auto* t : {&finished, &lengths_out, &count_out})
    need(!*t || (*t)->device() == lengths.device(), "every tensor of a plan must be on one device");
  need(lengths.is_cuda(), "the plan's tensors are not on a CUDA device");
  c10::cuda::CUDAGuard guard(lengths.device());
  // one allocation for what comes back
  const int64_t rows = (max_tokens + 3) / 4 * 4, reqs = (n + 4) / 4 * 4;
  at::Tensor all = at::empty({2 * rows + 3 * reqs + 4}, lengths.options());
  auto part = [&](int64_t at, int64_t len) { return all.narrow(0, at, len); };
  std::vector<at::Tensor> out = {part(0, max_tokens),
                                 part(rows, max_tokens),
                                 part(2 * rows, n + 1),
                                 lengths_out ? *lengths_out : part(2 * rows + reqs, n),
                                 part(2 * rows + 2 * reqs, n),
                                 count_out ? *count_out : part(2 * rows + 3 * reqs, 1)};
  PlanArgs a{};
  a.lengths = lengths.data_ptr<int>();
  a.fresh = fresh.data_ptr<int>();
  a.finished = finished ? reinterpret_cast<const uint8_t*>(finished->data_ptr<bool>()) : nullptr;
  a.tables = tables.data_ptr<int>();
  a.free_pages = free_pages.data_ptr<int>();
  a.free_count = free_count.data_ptr<int>();
  a.slots = out[0].data_ptr<int>();
  a.positions = out[1].data_ptr<int>();
  a.starts = out[2].data_ptr<int>();
  a.lengths_out = out[3].data_ptr<int>();
  a.granted = out[4].data_ptr<int>();
  a.count_out = out[5].data_ptr<int>();
  a.requests = int(n);
  a.width = int(tables.size(1));
  a.capacity = int(free_pages.size(0));
  a.max_tokens = int(max_tokens);
  a.page_size = int(page_size);
  // one block for what 1024 threads do in a round or two, else a cluster of 8
  const int64_t most = std::max(n, max_tokens);
  const int blocks = most <= 2048 ? 1 : 8;
  const int threads = int(std::min<int64_t>(kThreads, std::max<int64_t>(64, (most + 31) / 32 * 32)));
  const size_t smem = (4 * n + 1) * sizeof(int);
  if (smem > 46 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(k_plan, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               int((4 * kMaxRequests + 1) * sizeof(int)));
    if (e != cudaSuccess) throw std::runtime_error(std::string("plan_pages: ") + cudaGetErrorString(e));
  }
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(blocks);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = at::cuda::getCurrentCUDAStream().stream();
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim = {unsigned(blocks), 1, 1};
  config.attrs = &attribute;
  config.numAttrs = blocks > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&config, k_plan, a);
  if (e != cudaSuccess) throw std::runtime_error(std::string("plan_pages launch: ") + cudaGetErrorString(e));
  return out;
}

}  // namespace

void register_page_plan(py::module_& m) {
  m.def("plan_pages", &plan_pages, py::arg("lengths"), py::arg("new_tokens"), py::arg("block_tables"),
        py::arg("free_pages"), py::arg("free_count"), py::arg("page_size"), py::arg("max_tokens"),
        py::arg("finished") = py::none(), py::arg("lengths_out") = py::none(), py::arg("free_count_out") = py::none());
}
