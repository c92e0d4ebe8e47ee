// Low-rank adapters of many requests beside a shared B1_0 projection
// (bonsai_b1_gemm_lora), for sm_100a:
//
//   y[t] = epi( W x[t] + scale_a * B_a (A_a x[t]) ),  a = the adapter of t's request
//
// A 1-bit weight cannot take an adapter in (its entries are +-scale), so the
// low-rank product runs beside it.
//   lora_shrink_kernel   low[t][r] = scale_a * sum_k A_a[r][k] x[t][k]   (f32)
//   lora_expand_kernel   delta[t][n] = sum_r B_a[n][r] low[t][r]         (f32)
//   B1_0 GEMM            acc += delta in the epilogue, before its mode
// low and delta stay in f32: nothing between x and the epilogue's own
// rounding is rounded.
#include "internal.cuh"

#include <cooperative_groups.h>

#include <algorithm>
#include <mutex>

namespace cg = cooperative_groups;

namespace bonsai {
namespace lora {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kChunk = 32;  // inputs per step of a warp: 16 bytes per thread and row

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

struct ShrinkParams {
  const __half* x;
  long long ldx;
  int tokens, k_in;
  const __half* down;         // [slots][r_pad][k_in]
  const LoraSlot* slot_info;  // [slots]
  int n_slots, r_pad;
  const int* cu;              // [n_reqs + 1]
  const int* slots;           // [n_reqs]
  int n_reqs;
  float* low;                 // [tokens][r_pad]
};

// Tile u of the requests' token tiles (tiles of `size` tokens that do not
// cross requests).  One warp; false where there are at most u tiles.
__device__ bool find_request(const int* cu, int n, int tokens, int size, int u, int& req, int& tile) {
  const int lane = threadIdx.x & 31;
  int base = 0;
  for (int i0 = 0; i0 < n; i0 += 32) {
    int c = 0;
    if (i0 + lane < n) {
      const int a = max(0, min(cu[i0 + lane], tokens)), b = max(a, min(cu[i0 + lane + 1], tokens));
      c = (b - a + size - 1) / size;
    }
    int incl = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, base + incl > u);
    if (past) {
      const int l = __ffs(past) - 1;
      req = i0 + l;
      tile = u - base - (__shfl_sync(0xffffffffu, incl, l) - __shfl_sync(0xffffffffu, c, l));
      return true;
    }
    base += __shfl_sync(0xffffffffu, incl, 31);
  }
  return false;
}

// A cluster of CTAs takes one tile of 16 * MW tokens of one request; the
// CTAs split K between them, and the 8 / MW warps of each 16-token row of
// warps split the CTA's share.  x and A go from global memory straight into
// the fragments of mma.m16n8k16: the order of k within a step is free as long
// as both operands share it, so each thread takes 8 consecutive k of its row
// (one 16-byte load) for two steps.  Bound by reading A (few tokens) or x
// (many).  Partial sums meet in shared memory, then across the cluster, in a
// fixed order.
template <int NT, int MW>  // NT: 8-rank tiles held
__global__ void __launch_bounds__(kThreads) lora_shrink_kernel(const ShrinkParams p) {
  constexpr int KW = kWarps / MW;
  constexpr int TM = 16 * MW;
  constexpr int R = NT * 8;
  extern __shared__ float red[];  // [KW][TM][R]
  __shared__ int found[2];
  cg::cluster_group cluster = cg::this_cluster();
  const int csize = (int)cluster.num_blocks(), crank = (int)cluster.block_rank();
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  if (warp == 0) {
    int req = -1, tile = 0;
    if (!find_request(p.cu, p.n_reqs, p.tokens, TM, (int)blockIdx.x / csize, req, tile)) req = -1;
    if (lane == 0) {
      found[0] = req;
      found[1] = tile;
    }
  }
  __syncthreads();
  const int req = found[0];
  if (req < 0) return;  // the whole cluster
  const int slot = p.slots[req];
  if (slot < 0 || slot >= p.n_slots) return;
  const LoraSlot info = p.slot_info[slot];
  const int nt = (info.rank + 7) / 8;
  if (nt == 0) return;
  const int end = min(p.cu[req + 1], p.tokens);
  const int t0 = max(0, p.cu[req]) + found[1] * TM;

  const int mw = warp % MW, kw = warp / MW;
  const int g = lane >> 2, c = lane & 3;
  const int ta = t0 + mw * 16 + g, tb = ta + 8;
  const __half* xa = p.x + (size_t)ta * p.ldx + c * 8;
  const __half* xb = p.x + (size_t)tb * p.ldx + c * 8;
  const __half* aw = p.down + ((size_t)slot * p.r_pad + g) * p.k_in + c * 8;
  const int chunks = p.k_in / kChunk;
  const int per = (chunks + csize - 1) / csize;
  const int c0 = crank * per, c1 = min(chunks, c0 + per);

  float acc[NT][4] = {};
  const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll 2
  for (int ch = c0 + kw; ch < c1; ch += KW) {
    const uint4 va = ta < end ? *reinterpret_cast<const uint4*>(xa + ch * kChunk) : zero;
    const uint4 vb = tb < end ? *reinterpret_cast<const uint4*>(xb + ch * kChunk) : zero;
    uint4 w[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
      w[i] = i < nt ? __ldg(reinterpret_cast<const uint4*>(aw + (size_t)i * 8 * p.k_in + ch * kChunk)) : zero;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      mma_f16(acc[i], va.x, vb.x, va.y, vb.y, w[i].x, w[i].y);
      mma_f16(acc[i], va.z, vb.z, va.w, vb.w, w[i].z, w[i].w);
    }
  }
  // accumulator i: rows g, g + 8 of the warp's 16 tokens, ranks 8 i + 2 c, + 1
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    float* d = red + ((size_t)kw * TM + mw * 16 + g) * R + i * 8 + c * 2;
    d[0] = acc[i][0];
    d[1] = acc[i][1];
    d[8 * R] = acc[i][2];
    d[8 * R + 1] = acc[i][3];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < TM * R; e += kThreads) {
    float s = red[e];
#pragma unroll
    for (int k = 1; k < KW; ++k) s += red[k * TM * R + e];
    red[e] = s;
  }
  cluster.sync();
  for (int e = crank * kThreads + threadIdx.x; e < TM * R; e += csize * kThreads) {
    const int t = t0 + e / R, r = e % R;
    float s = 0.f;
    for (int q = 0; q < csize; ++q) s += cluster.map_shared_rank(red, q)[e];
    if (t < end && r < p.r_pad) p.low[(size_t)t * p.r_pad + r] = info.scale * s;
  }
  cluster.sync();  // no CTA ends while another reads its shared memory
}

struct ExpandParams {
  const __half* up;           // [slots][n_rows][r_pad]
  const LoraSlot* slot_info;
  int n_slots, r_pad, n_rows, tokens;
  const int* cu;
  const int* slots;
  int n_reqs;
  const float* low;           // [tokens][r_pad]
  float* delta;               // [tokens][n_rows]
};

constexpr int kExpandTokens = 4;

// One thread per output row of 4 tokens: B rows are read once per run of
// tokens with the same adapter, low from shared memory.  Bound by reading B.
__global__ void __launch_bounds__(kThreads) lora_expand_kernel(const ExpandParams p) {
  __shared__ float low[kExpandTokens][128];
  __shared__ int slot_of[kExpandTokens];
  const int t0 = (int)blockIdx.x * kExpandTokens;
  const int n = (int)blockIdx.y * kThreads + threadIdx.x;
  if (threadIdx.x < kExpandTokens) {
    const int t = t0 + threadIdx.x;
    int slot = -1;
    if (t < p.tokens) {
      int lo = 0, hi = p.n_reqs;  // the last request that begins at or before t
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (p.cu[mid] <= t) lo = mid; else hi = mid;
      }
      if (t >= p.cu[lo] && t < p.cu[lo + 1]) slot = p.slots[lo];
      if (slot >= p.n_slots || (slot >= 0 && p.slot_info[slot].rank == 0)) slot = -1;
    }
    slot_of[threadIdx.x] = slot;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kExpandTokens * p.r_pad; i += kThreads) {
    const int j = i / p.r_pad, r = i % p.r_pad;
    low[j][r] = slot_of[j] >= 0 ? p.low[(size_t)(t0 + j) * p.r_pad + r] : 0.f;
  }
  __syncthreads();
  if (n >= p.n_rows) return;
  float acc[kExpandTokens] = {};
  for (int j0 = 0; j0 < kExpandTokens;) {
    const int slot = slot_of[j0];
    int j1 = j0 + 1;
    while (j1 < kExpandTokens && slot_of[j1] == slot) ++j1;
    if (slot >= 0) {
      const int rank = p.slot_info[slot].rank;
      const uint4* row = reinterpret_cast<const uint4*>(p.up + ((size_t)slot * p.n_rows + n) * p.r_pad);
#pragma unroll 4
      for (int r8 = 0; r8 < (rank + 7) / 8; ++r8) {
        const uint4 v = __ldg(row + r8);
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
        float b[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
          b[2 * i] = f.x;
          b[2 * i + 1] = f.y;
        }
#pragma unroll
        for (int j = 0; j < kExpandTokens; ++j)
          if (j >= j0 && j < j1) {
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[j] = fmaf(b[i], low[j][r8 * 8 + i], acc[j]);
          }
      }
    }
    j0 = j1;
  }
#pragma unroll
  for (int j = 0; j < kExpandTokens; ++j)
    if (t0 + j < p.tokens) p.delta[(size_t)(t0 + j) * p.n_rows + n] = acc[j];
}

template <int NT, int MW>
int shrink(const ShrinkParams& p, cudaStream_t st) {
  auto kern = lora_shrink_kernel<NT, MW>;
  constexpr int TM = 16 * MW;
  constexpr int smem = (kWarps / MW) * TM * NT * 8 * (int)sizeof(float);
  static std::once_flag once[64];
  cudaError_t e = cudaSuccess;
  std::call_once(once[device_slot()],
                 [&] { e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
  if (e != cudaSuccess) return cuda_status(e, "lora shrink set smem attribute");
  const long long seqs = std::min(p.n_reqs, p.tokens);
  const long long units = (p.tokens + seqs * (TM - 1)) / TM;
  // CTAs of a cluster split K: about two CTAs per SM, each warp at least one chunk
  int c = 8;
  while (c > 1 && (units * c > 2ll * num_sms() || (p.k_in / kChunk) / c < kWarps / MW)) c /= 2;
  if (units * c > 0x7fffffffll) return fail(-2, "b1_gemm_lora: too many tokens in one call");
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)c;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(units * c));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) return cuda_status(e, "lora_shrink_kernel launch");
  return launch_status("lora_shrink_kernel launch");
}

template <int MW>
int shrink_by_rank(const ShrinkParams& p, int max_rank, cudaStream_t st) {
  if (max_rank <= 16) return shrink<2, MW>(p, st);
  if (max_rank <= 32) return shrink<4, MW>(p, st);
  if (max_rank <= 64) return shrink<8, MW>(p, st);
  return shrink<16, MW>(p, st);
}

}  // namespace lora

int launch_b1_gemm_lora(const __half* x, long long ldx, int tokens, const B1Weight& w, const EpiSeg& seg,
                        const LoraDevice& set, const int* cu, const int* slots, int n_reqs, cudaStream_t st) {
  if (tokens == 0) return 0;
  if (n_reqs == 0) return launch_b1_gemm(x, ldx, tokens, w, &seg, 1, false, st);
  const size_t low_n = ((size_t)tokens * set.r_pad + 3) / 4 * 4;
  void* mem = nullptr;
  int rc = scratch_alloc(&mem, (low_n + (size_t)tokens * w.n_rows) * sizeof(float), "b1_gemm_lora", st);
  if (rc) return rc;
  float* scratch = static_cast<float*>(mem);
  float* delta = scratch + low_n;
  lora::ShrinkParams s{};
  s.x = x;
  s.ldx = ldx;
  s.tokens = tokens;
  s.k_in = w.k_in;
  s.down = set.down;
  s.slot_info = set.info;
  s.n_slots = set.n_slots;
  s.r_pad = set.r_pad;
  s.cu = cu;
  s.slots = slots;
  s.n_reqs = n_reqs;
  s.low = scratch;
  // 64-token tiles where the requests are long enough to fill them
  rc = tokens >= 32ll * n_reqs ? lora::shrink_by_rank<4>(s, set.max_rank, st)
                                   : lora::shrink_by_rank<1>(s, set.max_rank, st);
  if (rc == 0) {
    lora::ExpandParams e{};
    e.up = set.up;
    e.slot_info = set.info;
    e.n_slots = set.n_slots;
    e.r_pad = set.r_pad;
    e.n_rows = w.n_rows;
    e.tokens = tokens;
    e.cu = cu;
    e.slots = slots;
    e.n_reqs = n_reqs;
    e.low = scratch;
    e.delta = delta;
    const dim3 grid((unsigned)((tokens + lora::kExpandTokens - 1) / lora::kExpandTokens),
                    (unsigned)((w.n_rows + lora::kThreads - 1) / lora::kThreads));
    lora::lora_expand_kernel<<<grid, lora::kThreads, 0, st>>>(e);
    rc = launch_status("lora_expand_kernel launch");
  }
  if (rc == 0) rc = launch_b1_gemm(x, ldx, tokens, w, &seg, 1, false, st, nullptr, delta);
  scratch_free(mem, st);
  return rc;
}

}  // namespace bonsai
