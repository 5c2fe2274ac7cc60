// Decode attention over the paged 8-bit KV cache (sm_100a).
//
//   out[b, t, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale * q . k_j - max)
//
// over the keys j < lengths[b] that token t of the sequence's last T tokens sees: j <=
// lengths[b] - T + t, and j > lengths[b] - T + t - window where there is a window.  k_j and
// v_j are code * scale of j's page and KV head.  Rows that see no key give 0, lse -inf.
//
// The work is bound by reading the codes once (2 * D bytes a key and KV head).  The query
// rows that share a KV head (its group of query heads, for each of the T tokens) are
// handled together, 8 * NT rows at a time, so that a code is read once for all of them.
//
// * Tiles of 32 keys.  Each warp owns a ring of STAGES tiles in shared memory, filled by TMA
//   (plain per-CTA loads, one box per page piece, swizzled) and walks its own tiles: no
//   barrier between warps while keys stream by.
// * The tiles of all (sequence, KV head, row group) are one line, cut into equal chunks, one
//   for each block, whatever the lengths: no launch parameter depends on a length, a ragged
//   batch is balanced, and one long sequence fills the GPU.  A block that holds all of a
//   segment writes its output; pieces go to a workspace and k_merge joins them in order of
//   the blocks, so results do not depend on timing.  No counter needs to be zero: the workspace is
//   plain memory of this call.
// * Scores S^T = K Q^T and outputs O^T = V^T P^T by mma.m16n8k16: the keys (the head's
//   elements) are the 16 rows, so 8 query rows fill a tile and the codes, converted exactly to
//   fp16 in registers, are never padded.  Scale of K: on the scores.  Scale of V: on P,
//   relative to the largest seen so far (vref), so P is at most 2^14 in fp16 and a weight
//   keeps fp16's 11 bits down to 2^-28 of the largest.
// * q is brought to fp16 by a power of two of its row (exact for bf16 and fp16 but for
//   values 2^-28 below the row's largest, which lose bits).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cmath>

#include "sparknet/kv_pool.h"
#include "sparknet/tc_gemm.cuh"

namespace {

using sn::tc::smem_u32;

constexpr int kTile = 32;  // keys
// What a segment's beginning and end cost, in rounds of a block's warps over tiles: with 0, 1, 2
// and 3 rounds 64 ragged sequences to 8192 took 114, 99, 93 and 91 us.
constexpr int kPadRounds = 3;

struct AttnArgs {
  const void* q;
  void* out;
  float* lse;
  const float *ks, *vs;
  const int *tables, *lengths;
  float* part;     // [2 * blocks][rows][D] sums of weighted values
  float2* part_ml; // [2 * blocks][rows] (max in log2, sum)
  int* plan;       // places in a chunk, then each sequence's first place (one KV head and row group), and the end
  uint32_t* err;
  int64_t q_b, q_t, q_h, table_row;
  int pages, n, T, hq, hkv, group, row_groups, page_size, page_shift, width, window, direct, pad, resident;
  float scale_log2;
};

struct Span {  // tiles of one sequence that some row sees
  int len, first, tiles;
};

__device__ __forceinline__ Span span_of(const AttnArgs& a, int b) {
  Span s;
  s.len = min(max(a.lengths[b], 0), a.width << a.page_shift);
  s.first = a.window ? max(s.len - a.T + 1 - a.window, 0) / kTile : 0;
  s.tiles = s.len ? (s.len + kTile - 1) / kTile - s.first : 0;
  return s;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Four codes to two pairs of fp16.
__device__ __forceinline__ void halves_of_codes(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\t"
      "mov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(codes));
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t h;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h) : "f"(hi), "f"(lo));
  return h;
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// TMA: `rows` keys of one page and head, 3-D map (D, page size, pages * heads).
__device__ __forceinline__ void load_keys(uint32_t dst, const CUtensorMap* map, int place, int block, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(place), "r"(block), "r"(smem_u32(bar))
      : "memory");
}

// 4 bytes to shared memory without waiting; zero where `on` is false.
__device__ __forceinline__ void copy4(void* dst, const float* src, bool on) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 4 : 0)
               : "memory");
}

template <int D, int NT>
struct Layout {
  // warps of a block (two blocks to an SM) and tiles in each warp's ring: as many as registers
  // and shared memory hold
  static constexpr int kWarps = D == 64 ? (NT == 1 ? 8 : NT == 2 ? 6 : 4) : NT == 1 ? 6 : 4;
  static constexpr int kStages = D == 64 ? (NT == 1 ? 3 : 4) : 2;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kTileBytes = kTile * D;          // K or V
  static constexpr int kRing = kWarps * kStages * 2 * kTileBytes;
  static constexpr int kRows = 8 * NT;
  static constexpr int kPitch = D + 4;                  // floats; spreads the four lanes of a row over the banks
  static constexpr int kSumBytes = 2 * kRows * kPitch * 4;
  static constexpr int kQBytes = kRows * D * 2;
  struct alignas(16) Stage {
    float k_scale[2], v_scale[2];  // of the tile's two halves of 16 keys
    int on[2], pad[2];             // whether the half's page exists
  };
  static constexpr int kStageBytes = kWarps * kStages * int(sizeof(Stage));
  static constexpr int kBarBytes = kWarps * kStages * 8;
  static constexpr int kBytes = 1024 + kRing + kSumBytes + kQBytes + kStageBytes + kBarBytes;
};

// A place in the line.  A segment takes as many places as it has tiles, and `pad` more that
// stand for the time of its beginning and end.
struct Cursor {
  int b, h, rg, i, g;  // sequence, KV head, row group; place in the segment; place in the line
  Span s;
  __device__ __forceinline__ void step(const AttnArgs& a, int by, int end) {
    g += by;
    i += by;
    if (g >= end) return;
    while (i >= s.tiles + a.pad) {
      i -= s.tiles + a.pad;
      if (++rg == a.row_groups) {
        rg = 0;
        if (++h == a.hkv) {
          h = 0;
          do s = span_of(a, ++b);
          while (s.tiles == 0);
        }
      }
    }
  }
  // the next place that is a tile
  __device__ __forceinline__ void settle(const AttnArgs& a, int by, int end) {
    while (g < end && i >= s.tiles) step(a, by, end);
  }
};

__device__ __forceinline__ int cluster_rank() {
  int r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ int cluster_size() {
  int r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();  // the aligned form wants whole warps
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of this block's `p` in the shared memory of block `rank` of the cluster.
__device__ __forceinline__ uint32_t in_block(const void* p, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr));
  return v;
}
__device__ __forceinline__ float2 ld_cluster2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr));
  return v;
}

template <class T>
__device__ __forceinline__ float2 floats_of(uint32_t w);
template <>
__device__ __forceinline__ float2 floats_of<__nv_bfloat16>(uint32_t w) {
  return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w));
}
template <>
__device__ __forceinline__ float2 floats_of<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}
__device__ __forceinline__ uint32_t pair_of(float a, float b, __nv_bfloat16) { return sn::tc::pack_bf16x2(a, b); }
__device__ __forceinline__ uint32_t pair_of(float a, float b, __half) { return pack_half2(a, b); }

template <class T, int D, int NT>
__global__ void __launch_bounds__(Layout<D, NT>::kThreads, 2) k_attention(const __grid_constant__ CUtensorMap k_map,
                                                           const __grid_constant__ CUtensorMap v_map,
                                                           const AttnArgs a) {
  using L = Layout<D, NT>;
  constexpr int S = L::kStages, C = D / 16, W = L::kWarps;
  extern __shared__ uint8_t raw[];
  uint8_t* ring = raw + (1024 - (smem_u32(raw) & 1023)) % 1024;
  float* sums = reinterpret_cast<float*>(ring + L::kRing);
  uint2* qs = reinterpret_cast<uint2*>(ring + L::kRing + L::kSumBytes);  // [NT][C][32 lanes]: MMA B fragments
  auto* info = reinterpret_cast<typename L::Stage*>(ring + L::kRing + L::kSumBytes + L::kQBytes);
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + L::kRing + L::kSumBytes + L::kQBytes + L::kStageBytes);
  __shared__ float q_scale[L::kRows];                 // score factor of each row
  __shared__ float sm[W][L::kRows], sl[W][L::kRows];
  __shared__ float2 block_ml[L::kRows];               // (max, sum) of the block, for its cluster
  __shared__ int found[3], warp_tiles[W];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g8 = lane >> 2, t4 = lane & 3;
  const int hr_count = a.hkv * a.row_groups;

  // --- where this block's chunk lies: prefix sums of the sequences' tiles -------------------
  bars += warp * S;
  info += warp * S;
  ring += warp * S * 2 * L::kTileBytes;
  if (lane == 0) {
    for (int s = 0; s < S; ++s) sn::tc::mbar_init(&bars[s], 2);  // the loads' bytes, the scales' copies
    sn::tc::fence_barrier_init();
    if (warp == 0) {
      sn::tc::prefetch_tmap(&k_map);
      sn::tc::prefetch_tmap(&v_map);
    }
  }
  Cursor seg;  // the segment that the block computes
  int g0 = 0, g1 = 0;
  int split = 1, part = 0;  // blocks of a cluster that share the segment, and this one's place among them
  if (a.direct) {
    if (a.direct > 1) {
      split = cluster_size();
      part = cluster_rank();
      // launched without its cluster: the first block of each does it all
      if (split != a.direct && blockIdx.x % a.direct) return;
    }
    const int segment = blockIdx.x / a.direct;
    seg.b = segment / hr_count;
    seg.h = segment % hr_count / a.row_groups;
    seg.rg = segment % a.row_groups;
    seg.s = span_of(a, seg.b);
    const int share = (seg.s.tiles + split - 1) / split;
    g0 = seg.i = seg.g = min(part * share, seg.s.tiles);
    g1 = min(g0 + share, seg.s.tiles);
    __syncthreads();
  } else {
    // the total, then the sequence that holds the chunk's first tile
    int total = 0, chunk = 0, here = 0, mine = 0;
    for (int pass = 0; pass < 2; ++pass) {
      int before = 0;
      if (pass) {
        total *= hr_count;
        chunk = max((total + int(gridDim.x) - 1) / int(gridDim.x), W);  // a tile for each warp at least
        g0 = min(int(blockIdx.x) * chunk, total);
        g1 = min(total, g0 + chunk);
      }
      for (int b0 = 0; b0 < a.n; b0 += L::kThreads) {
        const int b = b0 + threadIdx.x;
        if (!pass || a.n > L::kThreads) {
          mine = b < a.n ? span_of(a, b).tiles : 0;
          mine += mine ? a.pad : 0;
          int sum = mine;
#pragma unroll
          for (int o = 1; o < 32; o *= 2) {
            const int up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
          }
          if (lane == 31) warp_tiles[warp] = sum;
          __syncthreads();
          here = before + sum - mine;  // places of the sequences before b
          for (int w = 0; w < W; ++w) {
            if (w < warp) here += warp_tiles[w];
            before += warp_tiles[w];
          }
          if (a.n > L::kThreads) __syncthreads();
        }
        if (pass) {
          if (mine && g0 >= here * hr_count && g0 < (here + mine) * hr_count) {
            found[0] = b;
            found[1] = here;
            found[2] = mine;
          }
          if (blockIdx.x == 0 && b < a.n) a.plan[1 + b] = here;
        }
      }
      if (!pass) total = before;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      a.plan[0] = chunk;
      a.plan[1 + a.n] = total / hr_count;
    }
    __syncthreads();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (g0 >= g1) return;
    const int rest = g0 - found[1] * hr_count, hr = rest / found[2];
    seg.b = found[0];
    seg.h = hr / a.row_groups;
    seg.rg = hr % a.row_groups;
    seg.i = rest % found[2];
    seg.g = g0;
    seg.s = span_of(a, seg.b);
  }
  Cursor ahead = seg;  // the next tile that this warp requests
  ahead.step(a, warp, g1);
  ahead.settle(a, W, g1);

  // --- requests ---------------------------------------------------------------------------
  const bool halves = a.page_size == 16;  // a tile is two pages
  struct Pages {
    int p[2];
  };
  auto look_up = [&](const Cursor& c) {
    Pages p;
    if (c.g < g1) {
      const int key = (c.s.first + c.i) * kTile;
      const int* table = a.tables + c.b * a.table_row;
      p.p[0] = table[key >> a.page_shift];
      p.p[1] = halves && key + 16 < c.s.len ? table[(key >> 4) + 1] : -1;
    }
    return p;
  };
  auto request = [&](const Cursor& c, const Pages& p, int stage) {
    if (lane == 0 && c.g < g1) {
      typename L::Stage& st = info[stage];
      uint64_t* bar = &bars[stage];
      const uint32_t dst = smem_u32(ring + stage * 2 * L::kTileBytes);
      const bool on0 = uint32_t(p.p[0]) < uint32_t(a.pages);
      const int z0 = on0 ? p.p[0] * a.hkv + c.h : 0;
      st.on[0] = on0;
      copy4(&st.k_scale[0], a.ks + z0, on0);
      copy4(&st.v_scale[0], a.vs + z0, on0);
      if (!halves) {
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
        sn::tc::mbar_expect_tx(bar, on0 ? 2 * L::kTileBytes : 0);
        if (on0) {
          const int place = (c.s.first + c.i) * kTile & (a.page_size - 1);
          load_keys(dst, &k_map, place, z0, bar);
          load_keys(dst + L::kTileBytes, &v_map, place, z0, bar);
        }
      } else {
        const bool on1 = uint32_t(p.p[1]) < uint32_t(a.pages);
        const int z1 = on1 ? p.p[1] * a.hkv + c.h : 0;
        st.on[1] = on1;
        copy4(&st.k_scale[1], a.ks + z1, on1);
        copy4(&st.v_scale[1], a.vs + z1, on1);
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
        sn::tc::mbar_expect_tx(bar, (on0 ? L::kTileBytes : 0) + (on1 ? L::kTileBytes : 0));
        if (on0) {
          load_keys(dst, &k_map, 0, z0, bar);
          load_keys(dst + L::kTileBytes, &v_map, 0, z0, bar);
        }
        if (on1) {
          load_keys(dst + L::kTileBytes / 2, &k_map, 0, z1, bar);
          load_keys(dst + L::kTileBytes * 3 / 2, &v_map, 0, z1, bar);
        }
      }
    }
  };
  Pages next;
  int pending = 0;  // requested tiles that are not consumed yet
  {
    Cursor at[S];
    Pages p[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      at[s] = ahead;
      p[s] = look_up(ahead);
      pending += ahead.g < g1;
      ahead.step(a, W, g1);
      ahead.settle(a, W, g1);
    }
    next = look_up(ahead);
#pragma unroll
    for (int s = 0; s < S; ++s) request(at[s], p[s], s);
  }

  // --- segments ---------------------------------------------------------------------------
  int stage = 0;
  uint32_t phase = 0;
  bool dead = false;  // a load did not arrive: compute nothing more
  // chunk c of row r of a tile lies at (c ^ swizzle(r)) * 16; this lane reads rows and chunks of
  // its own in each 8 x 8 matrix, chunk 0's address being the base that the others differ from
  // by an exclusive or
  const uint32_t lane_at = ((lane & 7) + ((lane >> 3) & 1) * 8) * D +
                           (((lane >> 4) ^ (D == 128 ? lane & 7 : (lane >> 1) & 3)) << 4);
  // A segment's q rows, brought to fp16 fragments in shared memory by the first NT warps (W is
  // at least NT): loaded before the previous segment's warps are joined, stored after.
  const int rows = a.T * a.group;
  uint2 q_raw[C];
  auto load_q = [&](const Cursor& c) {
    const int r = c.rg * L::kRows + warp * 8 + g8;
#pragma unroll
    for (int i = 0; i < C; ++i) q_raw[i] = make_uint2(0, 0);
    if (warp < NT && r < rows) {
      const int t = r / a.group;
      const T* q = static_cast<const T*>(a.q) + c.b * a.q_b + t * a.q_t + (c.h * a.group + r - t * a.group) * a.q_h;
#pragma unroll
      for (int i = 0; i < C; ++i) q_raw[i] = *reinterpret_cast<const uint2*>(q + i * 16 + t4 * 4);
    }
  };
  auto store_q = [&]() {
    if (warp >= NT) return;
    float amax = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const float2 x = floats_of<T>(q_raw[c].x), y = floats_of<T>(q_raw[c].y);
      amax = fmaxf(fmaxf(amax, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(y.x), fabsf(y.y)));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    // the row's largest to [2^14, 2^15); an infinite row keeps its values
    const int e = amax <= 3.4028234e38f ? max((__float_as_int(amax) >> 23) - 127, -100) : 14;
    const float up = __int_as_float((14 - e + 127) << 23);
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const float2 x = floats_of<T>(q_raw[c].x), y = floats_of<T>(q_raw[c].y);
      qs[(warp * C + c) * 32 + lane] = make_uint2(pack_half2(x.x * up, x.y * up), pack_half2(y.x * up, y.y * up));
    }
    if (t4 == 0) q_scale[warp * 8 + g8] = a.scale_log2 * __int_as_float((e - 14 + 127) << 23);
  };
  auto skip_empty = [&](Cursor& c) {  // past a segment of whose places only the pad is here
    while (c.g < g1 && c.i >= c.s.tiles) c.step(a, min(c.s.tiles + a.pad - c.i, g1 - c.g), g1);
  };
  if (!a.direct) skip_empty(seg);
  if (!a.direct && seg.g >= g1) return;
  load_q(seg);
  store_q();
  __syncthreads();
  do {
    const int places = min(seg.s.tiles + a.pad - seg.i, g1 - seg.g);
    const Span span = seg.s;
    const int b = seg.b, h = seg.h, r0 = seg.rg * L::kRows;
    const int i0 = seg.i, i1 = min(span.tiles, i0 + places);
    uint2 qf[NT <= 2 ? NT : 1][C];
    if constexpr (NT <= 2) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < C; ++c) qf[nt][c] = qs[(nt * C + c) * 32 + lane];
    }
    float o[NT][C][4], m[NT][2], l[NT][2], f[NT][2], vref = 0.0f;
    int limit[NT][2];  // the last key of rows 2 t4 and 2 t4 + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = r0 + nt * 8 + t4 * 2 + e;
        m[nt][e] = -INFINITY;
        l[nt][e] = 0.0f;
        f[nt][e] = q_scale[nt * 8 + t4 * 2 + e];
        limit[nt][e] = r < rows ? span.len - a.T + r / a.group : -1;
      }
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][c][e] = 0.0f;
    }
    const int least = a.window ? max(span.len - a.T + 1 - a.window, 0) : 0;  // first key that any row sees

    for (int i = i0 + (warp + W - (seg.g - g0) % W) % W; i < i1; i += W) {
      if (!dead) dead = !sn::tc::mbar_wait(&bars[stage], phase, a.err);
      if (dead) continue;
      const int j0 = (span.first + i) * kTile;
      {
        typename L::Stage st = info[stage];
        if (!halves) {
          st.k_scale[1] = st.k_scale[0];
          st.v_scale[1] = st.v_scale[0];
          st.on[1] = st.on[0];
        }
        const uint32_t kt = smem_u32(ring + stage * 2 * L::kTileBytes) + lane_at;
        const bool edge = j0 + kTile - 1 > span.len - a.T || (a.window && j0 <= span.len - 1 - a.window) ||
                          !(st.on[0] && st.on[1]);
        // scores of two times 16 keys
        float s[2][NT][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[mt][nt][e] = 0.0f;
#pragma unroll
          for (int c = 0; c < C; c += 2) {
            uint32_t x[4];
            ldsm4((kt ^ (c << 4)) + mt * 16 * D, x);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              uint32_t a0, a1, a2, a3;
              halves_of_codes(x[2 * u], a0, a2);
              halves_of_codes(x[2 * u + 1], a1, a3);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const uint2 q = NT <= 2 ? qf[NT <= 2 ? nt : 0][c + u] : qs[(nt * C + c + u) * 32 + lane];
                mma(s[mt][nt], a0, a1, a2, a3, q.x, q.y);
              }
            }
          }
        }
        // key of element e: j0 + 16 mt + g8 + 8 (e / 2), row 2 t4 + e % 2
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[mt][nt][e] *= st.k_scale[mt] * f[nt][e & 1];
        if (edge) {
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int key = j0 + mt * 16 + g8 + (e >> 1) * 8, last = limit[nt][e & 1];
                if (!(key <= last && (!a.window || key > last - a.window) && st.on[mt])) s[mt][nt][e] = -INFINITY;
              }
        }
        float top[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            top[nt][e] = fmaxf(fmaxf(s[0][nt][e], s[0][nt][e + 2]), fmaxf(s[1][nt][e], s[1][nt][e + 2]));
#pragma unroll
        for (int x = 4; x < 32; x *= 2)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              top[nt][e] = fmaxf(top[nt][e], __shfl_xor_sync(0xffffffffu, top[nt][e], x));
        const float vnew = fmaxf(vref, fmaxf(st.v_scale[0], st.v_scale[1]));
        const float vold = vnew > vref ? vref / vnew : 1.0f;
        vref = vnew;
        bool same = vold == 1.0f;
        float back[NT][2], base[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float best = fmaxf(m[nt][e], top[nt][e]);
            base[nt][e] = best == -INFINITY ? 0.0f : best;
            const float shrink = best == m[nt][e] ? 1.0f : ex2(m[nt][e] - best);
            same = same && shrink == 1.0f;
            m[nt][e] = best;
            l[nt][e] *= shrink;
            back[nt][e] = shrink * vold;
          }
        if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nt][c][e] *= back[nt][e & 1];
        }
        // weights, and their 8 x 8 pieces turned to the second product's operand
        const float vinv = vref > 0.0f ? 16384.0f / vref : 0.0f;
        uint32_t p[2][NT][2];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const float vf = st.v_scale[mt] * vinv;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              w[e] = ex2(s[mt][nt][e] - base[nt][e & 1]);
              l[nt][e & 1] += w[e];
            }
            p[mt][nt][0] = transpose8x8(pack_half2(w[0] * vf, w[1] * vf));
            p[mt][nt][1] = transpose8x8(pack_half2(w[2] * vf, w[3] * vf));
          }
        }
        // O^T += V^T P^T; a transposed piece holds elements (2 g8, 2 g8 + 1) of keys 2 t4, 2 t4 + 1
        bool odd = false;  // a NaN code among an edge tile's keys
        auto second = [&](auto masked) {
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            uint32_t keep[2];
            if constexpr (masked) {  // codes of keys that no row sees may be anything: they count as zero
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                const int key = j0 + mt * 16 + u * 8 + t4 * 2;
                keep[u] = (key >= least && key < span.len && st.on[mt] ? 0xffffu : 0u) |
                          (key + 1 >= least && key + 1 < span.len && st.on[mt] ? 0xffff0000u : 0u);
              }
            }
#pragma unroll
            for (int c = 0; c < C; c += 2) {
              uint32_t x[4];
              ldsm4_trans((kt ^ (c << 4)) + L::kTileBytes + mt * 16 * D, x);
              if constexpr (masked) {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                  x[u] &= keep[u & 1];
                  const uint32_t nan = __vcmpeq4(x[u] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                  odd = odd || nan;
                  x[u] &= ~nan;  // counted below for the rows that see it
                }
              }
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                uint32_t a0, a1, a2, a3;
                halves_of_codes(__byte_perm(x[2 * u], 0, 0x3120), a0, a1);
                halves_of_codes(__byte_perm(x[2 * u + 1], 0, 0x3120), a2, a3);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma(o[nt][c + u], a0, a1, a2, a3, p[mt][nt][0], p[mt][nt][1]);
              }
            }
          }
        };
        if (edge) second(std::true_type());
        else second(std::false_type());
        if (edge && __any_sync(0xffffffffu, odd)) {
          // rare: how many NaN codes each (element, row) sees, as products of ones and zeros
          for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float one[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int key = j0 + mt * 16 + g8 + (e >> 1) * 8, last = limit[nt][e & 1];
                one[e] = key <= last && (!a.window || key > last - a.window) && st.on[mt] ? 1.0f : 0.0f;
              }
              const uint32_t b0 = transpose8x8(pack_half2(one[0], one[1]));
              const uint32_t b1 = transpose8x8(pack_half2(one[2], one[3]));
#pragma unroll
              for (int c = 0; c < C; c += 2) {
                uint32_t x[4];
                ldsm4_trans((kt ^ (c << 4)) + L::kTileBytes + mt * 16 * D, x);
#pragma unroll
                for (int u = 0; u < 4; ++u)  // 1.0 in e4m3 where NaN
                  x[u] = __vcmpeq4(x[u] & 0x7f7f7f7fu, 0x7f7f7f7fu) & 0x38383838u;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                  uint32_t a0, a1, a2, a3;
                  halves_of_codes(__byte_perm(x[2 * u], 0, 0x3120), a0, a1);
                  halves_of_codes(__byte_perm(x[2 * u + 1], 0, 0x3120), a2, a3);
                  float hits[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                  mma(hits, a0, a1, a2, a3, b0, b1);
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    if (hits[e] > 0.0f) o[nt][c + u][e] = NAN;
                }
              }
            }
          }
        }
      }
      __syncwarp();  // every lane has read the stage
      pending += (ahead.g < g1) - 1;
      request(ahead, next, stage);
      ahead.step(a, W, g1);
      ahead.settle(a, W, g1);
      next = look_up(ahead);
      if (++stage == S) {
        stage = 0;
        phase ^= 1;
      }
    }

    Cursor following = seg;
    following.step(a, places, g1);
    if (!a.direct) skip_empty(following);
    if (following.g < g1) load_q(following);

    // --- join the warps ---------------------------------------------------------------------
#pragma unroll
    for (int x = 4; x < 32; x *= 2)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) l[nt][e] += __shfl_xor_sync(0xffffffffu, l[nt][e], x);
    if (g8 == 0) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          sm[warp][nt * 8 + t4 * 2 + e] = m[nt][e];
          sl[warp][nt * 8 + t4 * 2 + e] = l[nt][e];
        }
    }
    __syncthreads();
    auto largest = [&](int r) {
      float x = sm[0][r];
#pragma unroll
      for (int w = 1; w < W; ++w) x = fmaxf(x, sm[w][r]);
      return x;
    };
    float* mine = sums + (warp & 1) * L::kRows * L::kPitch;
#pragma unroll
    for (int pair = 0; pair < W / 2; ++pair) {  // the first two warps store, the others add
      if (warp / 2 == pair) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = nt * 8 + t4 * 2 + e;
            const float best = largest(r);
            const float weight = (m[nt][e] == best ? 1.0f : ex2(m[nt][e] - best)) * vref * (1.0f / 16384.0f);
#pragma unroll
            for (int c = 0; c < C; ++c) {
              float2* at = reinterpret_cast<float2*>(mine + r * L::kPitch + c * 16 + g8 * 2);
              float2 x = make_float2(o[nt][c][e] * weight, o[nt][c][2 + e] * weight);
              if (pair) {
                const float2 y = *at;
                x.x += y.x;
                x.y += y.y;
              }
              *at = x;
            }
          }
      }
      __syncthreads();
    }
    const bool whole = (i0 == 0 && i1 == span.tiles) || split > 1;
    const int slot = 2 * blockIdx.x + (g0 >= seg.g - i0 ? 0 : 1);  // at most the first and the last are pieces
    auto write = [&](int r, int d, const float4& v, float best, float sum) {
      const int t = (r0 + r) / a.group;
      const int64_t row = (int64_t(b) * a.T + t) * a.hq + h * a.group + r0 + r - t * a.group;
      const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + row * D + d) =
          make_uint2(pair_of(v.x * inv, v.y * inv, T()), pair_of(v.z * inv, v.w * inv, T()));
      if (a.lse && d == 0) a.lse[row] = sum != 0.0f ? (best + log2f(sum)) * 0.6931471805599453f : -INFINITY;
    };
    for (int x = threadIdx.x; x < L::kRows * (D / 4); x += L::kThreads) {
      const int r = x / (D / 4), d = x % (D / 4) * 4;
      if (r0 + r >= rows) break;
      const float best = largest(r);
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) sum += sl[w][r] * (sm[w][r] == best ? 1.0f : ex2(sm[w][r] - best));
      const float4 p = *reinterpret_cast<const float4*>(sums + r * L::kPitch + d);
      const float4 q = *reinterpret_cast<const float4*>(sums + (L::kRows + r) * L::kPitch + d);
      const float4 v = make_float4(p.x + q.x, p.y + q.y, p.z + q.z, p.w + q.w);
      if (split > 1) {
        *reinterpret_cast<float4*>(sums + r * L::kPitch + d) = v;
        if (d == 0) block_ml[r] = make_float2(best, sum);
      } else if (whole) {
        write(r, d, v, best, sum);
      } else {
        *reinterpret_cast<float4*>(a.part + (int64_t(slot) * L::kRows + r) * D + d) = v;
        if (d == 0) a.part_ml[slot * L::kRows + r] = make_float2(best, sum);
      }
    }
    if (split > 1) {  // join the blocks: each writes every split-th piece of the rows
      cluster_sync();
      for (int x = part * L::kThreads + threadIdx.x; x < L::kRows * (D / 4); x += split * L::kThreads) {
        const int r = x / (D / 4), d = x % (D / 4) * 4;
        if (r0 + r >= rows) break;
        float best = -INFINITY, sum = 0.0f;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int c = 0; c < split; ++c) best = fmaxf(best, ld_cluster2(in_block(&block_ml[r], c)).x);
        for (int c = 0; c < split; ++c) {
          const float2 ml = ld_cluster2(in_block(&block_ml[r], c));
          const float4 y = ld_cluster4(in_block(sums + r * L::kPitch + d, c));
          const float w = ml.x == best ? 1.0f : ex2(ml.x - best);
          sum += ml.y * w;
          v.x += y.x * w;
          v.y += y.y * w;
          v.z += y.z * w;
          v.w += y.w * w;
        }
        write(r, d, v, best, sum);
      }
      cluster_sync();  // no block leaves while another reads its sums
    }
    if (following.g < g1) store_q();
    __syncthreads();  // the sums are free, and q is there for the next segment
    seg = following;
  } while (seg.g < g1);
  if (dead)  // let this warp's copies land before it exits
    for (; pending > 0; --pending) {
      sn::tc::mbar_drain(&bars[stage], phase);
      if (++stage == S) {
        stage = 0;
        phase ^= 1;
      }
    }
}

// Joins the pieces of segments that lie in several blocks, in order of the blocks, and writes
// the rows of segments without keys.  One block: `rows_here` rows of one segment, `groups`
// groups of D / 4 threads for each, a group taking every groups-th piece.
template <class T, int D>
__global__ void __launch_bounds__(1024) k_merge(const AttnArgs a, int rows_per_segment, int groups) {
  extern __shared__ float4 shared[];
  constexpr int kLanes = D / 4;
  const int d = threadIdx.x % kLanes, group = threadIdx.x / kLanes % groups, row_here = threadIdx.x / (kLanes * groups);
  const int rows_here = blockDim.x / (kLanes * groups);
  const int hr_count = a.hkv * a.row_groups, b = blockIdx.x / hr_count, hr = blockIdx.x % hr_count;
  const int r = blockIdx.y * rows_here + row_here, rr = hr % a.row_groups * rows_per_segment + r;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int chunk = a.plan[0], before = a.plan[1 + b], places = a.plan[2 + b] - before, tiles = places ? places - a.pad : 0;
  const int begin = before * hr_count + hr * places;
  const int c0 = tiles ? begin / chunk : 0, c1 = tiles ? (begin + tiles - 1) / chunk : -1;
  if (c0 == c1) return;  // one block held it all
  const bool real = r < rows_per_segment && rr < a.T * a.group;
  float best = -INFINITY, sum = 0.0f;
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto slot_of = [&](int c) { return int64_t(2 * c + (c * chunk >= begin ? 0 : 1)) * rows_per_segment + r; };
  if (real) {
#pragma unroll 4
    for (int c = c0 + group; c <= c1; c += groups) best = fmaxf(best, a.part_ml[slot_of(c)].x);
#pragma unroll 4
    for (int c = c0 + group; c <= c1; c += groups) {
      const float2 ml = a.part_ml[slot_of(c)];
      const float w = ml.x == best ? 1.0f : ex2(ml.x - best);
      const float4 x = *reinterpret_cast<const float4*>(a.part + slot_of(c) * D + d * 4);
      sum += ml.y * w;
      v.x += x.x * w;
      v.y += x.y * w;
      v.z += x.z * w;
      v.w += x.w * w;
    }
  }
  if (groups > 1) {
    float2* sums = reinterpret_cast<float2*>(shared + blockDim.x);
    const int at = threadIdx.x / kLanes;
    shared[threadIdx.x] = v;
    if (d == 0) sums[at] = make_float2(best, sum);
    __syncthreads();
    if (group == 0) {
      for (int x = 1; x < groups; ++x) best = fmaxf(best, sums[at + x].x);
      v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      sum = 0.0f;
      for (int x = 0; x < groups; ++x) {
        const float2 ml = sums[at + x];
        const float w = ml.x == best ? 1.0f : ex2(ml.x - best);
        const float4 y = shared[threadIdx.x + x * kLanes];
        sum += ml.y * w;
        v.x += y.x * w;
        v.y += y.y * w;
        v.z += y.z * w;
        v.w += y.w * w;
      }
    }
  }
  if (group != 0 || !real) return;
  const int h = hr / a.row_groups;
  const int64_t row = (int64_t(b) * a.T + rr / a.group) * a.hq + h * a.group + rr % a.group;
  const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
  *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + row * D + d * 4) =
      make_uint2(pair_of(v.x * inv, v.y * inv, T()), pair_of(v.z * inv, v.w * inv, T()));
  if (a.lse && d == 0) a.lse[row] = sum != 0.0f ? (best + log2f(sum)) * 0.6931471805599453f : -INFINITY;
}

using sn::kv::need_ok;

// How many blocks share a segment that is not cut from the line, 0 to cut the line.  Where the
// tables hold few tiles, the blocks of one cluster take a segment and join through distributed
// shared memory: one launch, no workspace.  A cluster grows while its blocks hold more than
// about a tile a warp and the grid stays in one wave (8 sequences x 1024 keys, one KV head:
// 12.3 us in one block each, 14.5 us from the line, 8.4 us in clusters of 8); more than four
// such rounds a block go to the line, which balances them.
int direct_blocks(int64_t segments, int64_t tiles, int resident) {
  int blocks = 1;
  while (blocks < 8 && tiles > blocks * 6 && segments * blocks * 2 <= resident) blocks *= 2;
  return tiles <= blocks * 24 ? blocks : 0;
}

template <class T, int D, int NT>
void launch(AttnArgs a, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
  using L = Layout<D, NT>;
  auto kernel = k_attention<T, D, NT>;
  static std::atomic<uint64_t> ready{0};  // devices that allow the kernel its shared memory
  int device = 0;
  need_ok(cudaGetDevice(&device), "paged_decode_attention");
  const uint64_t bit = 1ull << (device & 63);
  if (!(ready.load() & bit)) {
    need_ok(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes),
            "paged_decode_attention");
    ready.fetch_or(bit);
  }
  const int segments = a.n * a.hkv * a.row_groups;
  int blocks = segments * std::max(a.direct, 1);
  if (!a.direct) {
    a.pad = kPadRounds * L::kWarps;
    const int places = segments * ((a.width * a.page_size + kTile - 1) / kTile + a.pad);  // at most
    blocks = std::min(a.resident, (places + L::kWarps - 1) / L::kWarps);
  }
  if (a.direct > 1) {
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(blocks);
    config.blockDim = dim3(L::kThreads);
    config.dynamicSmemBytes = L::kBytes;
    config.stream = st;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim = {unsigned(a.direct), 1, 1};
    config.attrs = &attribute;
    config.numAttrs = 1;
    need_ok(cudaLaunchKernelEx(&config, kernel, mk, mv, a), "paged_decode_attention launch");
    return;
  }
  kernel<<<blocks, L::kThreads, L::kBytes, st>>>(mk, mv, a);
  need_ok(cudaGetLastError(), "paged_decode_attention launch");
  if (a.direct) return;

  // pieces a segment is likely cut into, four of them a group
  const int rows = std::min(L::kRows, a.T * a.group);
  const int pieces = std::min(a.resident / segments + 2, a.width * a.page_size / kTile / L::kWarps + 2);
  int groups = 1;
  while (groups < 32 && groups * 4 < pieces) groups *= 2;
  int rows_here = 1;
  while (rows_here * 2 * groups * (D / 4) <= 256 && rows_here < rows) rows_here *= 2;
  const int threads = rows_here * groups * (D / 4);
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(segments, (rows + rows_here - 1) / rows_here);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = groups > 1 ? threads * sizeof(float4) + threads / (D / 4) * sizeof(float2) : 0;
  config.stream = st;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  need_ok(cudaLaunchKernelEx(&config, k_merge<T, D>, a, int(L::kRows), groups), "paged_decode_attention merge");
}

template <class T, int D>
void launch_rows(const AttnArgs& a, const CUtensorMap& mk, const CUtensorMap& mv, int nt, cudaStream_t st) {
  if (nt == 1) launch<T, D, 1>(a, mk, mv, st);
  else if (nt == 2) launch<T, D, 2>(a, mk, mv, st);
  else launch<T, D, 4>(a, mk, mv, st);
}

}  // namespace

namespace sn {
namespace kv {

// The map of one pool of codes as (head dim, page size, pages * heads) bytes; the box is the
// keys of a tile that lie in one page.
CUtensorMap KvPool::make_map(const at::Tensor& codes) const {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                              const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      return Encode(nullptr);
    return reinterpret_cast<Encode>(p);
  }();
  if (!encode) throw std::runtime_error("the driver offers no cuTensorMapEncodeTiled");
  CUtensorMap map;
  cuuint64_t dims[3] = {cuuint64_t(dim), cuuint64_t(page_size), cuuint64_t(pages) * cuuint64_t(heads)};
  cuuint64_t strides[2] = {cuuint64_t(dim), cuuint64_t(dim) * cuuint64_t(page_size)};
  cuuint32_t box[3] = {cuuint32_t(dim), cuuint32_t(std::min(page_size, kTile)), 1};
  cuuint32_t step[3] = {1, 1, 1};
  const CUresult r =
      encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, codes.data_ptr(), dims, strides, box, step,
             CU_TENSOR_MAP_INTERLEAVE_NONE, dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw std::runtime_error("cuTensorMapEncodeTiled failed: " + std::to_string(int(r)));
  return map;
}

int KvPool::attention_launches(int64_t sequences, int64_t tokens, int64_t hq, int64_t width) const {
  need_cuda();
  const int64_t rows = tokens * (hq / heads);
  const int nt = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
  const int64_t segments = sequences * heads * ((rows + 8 * nt - 1) / (8 * nt));
  const int resident = 2 * at::cuda::getDeviceProperties(k.device().index())->multiProcessorCount;
  return direct_blocks(segments, (width * page_size + kTile - 1) / kTile, resident) ? 1 : 2;
}

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
  need(n <= 4096 && T >= 1 && T * (hq / heads) <= 4096,
       "paged_decode_attention takes up to 4096 sequences and up to 4096 query rows for a KV head");
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
  const int64_t rows = T * (hq / heads);
  const int nt = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
  const int64_t row_groups = (rows + 8 * nt - 1) / (8 * nt), segments = n * heads * row_groups;
  need(segments * ((tables.size(1) * page_size + kTile - 1) / kTile + 8) < (int64_t(1) << 30),
       "the sequences' tables, KV heads and query rows together are too large for one call");
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
  if (want_lse)
    lse = at::empty(q.sizes().slice(0, q.dim() - 1),
                    q.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous));
  if (n == 0) return {o, lse};
  if (!mapped_) {
    k_map_ = make_map(k);
    v_map_ = make_map(v);
    mapped_ = true;
  }
  // two blocks of four warps fill an SM's shared memory
  const int resident = 2 * at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const int64_t parts = 2 * int64_t(resident) * 8 * nt;  // two pieces a block
  at::Tensor work = at::empty({parts * dim + parts * 2 + n + 2}, k_scale.options());
  AttnArgs a{};
  a.part = work.data_ptr<float>();
  a.part_ml = reinterpret_cast<float2*>(a.part + parts * dim);
  a.plan = reinterpret_cast<int*>(a.part + parts * dim + parts * 2);
  a.err = reinterpret_cast<uint32_t*>(err.data_ptr<int>());
  a.q = q.data_ptr();
  a.out = o.data_ptr();
  a.lse = lse ? lse->data_ptr<float>() : nullptr;
  a.ks = k_scale.data_ptr<float>();
  a.vs = v_scale.data_ptr<float>();
  a.tables = tables.data_ptr<int>();
  a.lengths = lengths.data_ptr<int>();
  a.q_b = q.stride(0);
  a.q_t = many ? q.stride(1) : 0;
  a.q_h = q.stride(many ? 2 : 1);
  a.table_row = tables.stride(0);
  a.pages = int(pages);
  a.n = int(n);
  a.resident = resident;
  a.T = int(T);
  a.hq = int(hq);
  a.hkv = heads;
  a.group = int(hq / heads);
  a.row_groups = int(row_groups);
  a.page_size = page_size;
  a.page_shift = __builtin_ctz(page_size);
  a.width = int(tables.size(1));
  a.window = int(window);
  a.scale_log2 = float(scale * 1.4426950408889634);
  a.direct = direct_blocks(segments, (tables.size(1) * page_size + kTile - 1) / kTile, resident);
  if (q.scalar_type() == at::kBFloat16) {
    if (dim == 128) launch_rows<__nv_bfloat16, 128>(a, k_map_, v_map_, nt, stream());
    else launch_rows<__nv_bfloat16, 64>(a, k_map_, v_map_, nt, stream());
  } else {
    if (dim == 128) launch_rows<__half, 128>(a, k_map_, v_map_, nt, stream());
    else launch_rows<__half, 64>(a, k_map_, v_map_, nt, stream());
  }
  return {o, lse};
}

}  // namespace kv
}  // namespace sn
