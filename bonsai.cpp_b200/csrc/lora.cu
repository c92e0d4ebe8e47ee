// Low-rank adapters of many requests beside a shared B1_0 projection
// (bonsai_b1_gemm_lora), for sm_100a:
//
//   y[t] = epi( W x[t] + scale_a * B_a (A_a x[t]) ),  a = the adapter of t's request
//
// A 1-bit weight cannot take an adapter in (its entries are +-scale), so the
// low-rank product runs beside it.
// Two forms, chosen by the tokens per request:
//   few (decoding): low[t][r] = scale_a * sum_k A_a[r][k] x[t][k] by
//     lora_shrink_kernel, and the B1_0 GEMM's epilogue warps compute
//     B_a low while its products run (LORA_DELTA).  Each reads the adapters
//     once, and both are bound by latency: for the 64 tokens below 15 and 22 % of
//     DRAM's rate.
//   many (prompts, images): low by lora_shrink_tile_kernel (tcgen05), and
//     the B1_0 GEMM takes scale_a B_a low as extra k-blocks of its own
//     products, listed by lora_plan_kernel: no second pass over y.
// Measured (B200, a call among others): 64 requests of one token, 3072 -> 9216,
// ranks 8 to 64: 35 us; 4 requests of about 1100 tokens, 3072 -> 12288: 322-328
// us, 1.06 PFLOP/s, 20 of them the shrink; 24 of 5 to 160 tokens, 9216 -> 3072,
// f32: 172 us.
// low stays in f32, and the tensor cores take it and B in pieces that keep all
// of it (kLowPieces), so nothing between x and the epilogue's own rounding is
// rounded further, whatever its magnitude.
#include "internal.cuh"

#include "ptx.cuh"

#include <cooperative_groups.h>
#include <cudaTypedefs.h>

#include <algorithm>

namespace cg = cooperative_groups;

namespace bonsai {
int encode_tmap_2d_16b(CUtensorMap* map, const void* base, long long rows, long long cols, long long ld,
                       int box_cols, int box_rows, bool bf16);
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
  float* low;                 // [tokens][r_pad] (few tokens per request)
  uint32_t* low_pieces;       // bf16 [r_pad / 16][kLowParts][tokens][16] (many)
};

// The upper 8 bits of an f32 value's 24, as an f32 value; what is left of it is
// exact, and after three times nothing (the parts l1, l2, l3).  All of a value
// that is not finite is in its first part.
__device__ __forceinline__ float cut_piece(float& rest) {
  const float piece = __uint_as_float(__float_as_uint(rest) & 0xffff0000u);
  rest = (__float_as_uint(piece) & 0x7f800000u) == 0x7f800000u ? 0.f : rest - piece;
  return piece;
}

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

// ---- the form for few tokens per request
// A cluster of CTAs takes one tile of 16 tokens of one request; the CTAs split
// K between them, and their warps split the CTA's share.  x and A go from global memory straight into
// the fragments of mma.m16n8k16: the order of k within a step is free as long
// as both operands share it, so each thread takes 8 consecutive k of its row
// (one 16-byte load) for two steps.  Bound by latency (12 us, 15 % of DRAM's rate for
// 64 requests): request, slot, A and x one behind the other, then two barriers of
// the cluster.  Partial sums meet in shared memory, then across the cluster, in a
// fixed order.
template <int NT>  // 8-rank tiles held
__global__ void __launch_bounds__(kThreads, 2) lora_shrink_kernel(const ShrinkParams p) {
  constexpr int TM = 16;
  constexpr int R = NT * 8;
  extern __shared__ float red[];  // [kWarps][TM][R]
  __shared__ int found[2];
  cg::cluster_group cluster = cg::this_cluster();
  const int csize = (int)cluster.num_blocks(), crank = (int)cluster.block_rank();
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  griddep_wait();
  griddep_launch();
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

  const int g = lane >> 2, c = lane & 3;
  const int ta = t0 + g, tb = ta + 8;
  const __half* xa = p.x + (size_t)ta * p.ldx + c * 8;
  const __half* xb = p.x + (size_t)tb * p.ldx + c * 8;
  const __half* aw = p.down + ((size_t)slot * p.r_pad + g) * p.k_in + c * 8;
  const int chunks = p.k_in / kChunk;
  const int per = (chunks + csize - 1) / csize;
  const int c0 = crank * per, c1 = min(chunks, c0 + per);

  float acc[NT][4] = {};
  const uint4 zero = make_uint4(0, 0, 0, 0);
#pragma unroll NT <= 4 ? 4 : NT <= 8 ? 2 : 1
  for (int ch = c0 + warp; ch < c1; ch += kWarps) {
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
  // accumulator i: tokens g, g + 8, ranks 8 i + 2 c, + 1
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    float* d = red + ((size_t)warp * TM + g) * R + i * 8 + c * 2;
    d[0] = acc[i][0];
    d[1] = acc[i][1];
    d[8 * R] = acc[i][2];
    d[8 * R + 1] = acc[i][3];
  }
  __syncthreads();
  const int used = min(TM, end - t0) * R;  // of the tile's tokens
  for (int e = threadIdx.x; e < used; e += kThreads) {
    float s = red[e];
#pragma unroll
    for (int k = 1; k < kWarps; ++k) s += red[k * TM * R + e];
    red[e] = s;
  }
  cluster.sync();
  for (int e = crank * kThreads + threadIdx.x; e < used; e += csize * kThreads) {
    const int t = t0 + e / R, r = e % R;
    float s = 0.f;
    for (int q = 0; q < csize; ++q) s += cluster.map_shared_rank(red, q)[e];
    if (r < p.r_pad)  // what x leaves of A's rows past the rank (0 * inf) is no value
      p.low[(size_t)t * p.r_pad + r] = r < info.rank ? info.scale * s : 0.f;
  }
  cluster.sync();  // no CTA ends while another reads its shared memory
}

// ---- the form for many tokens per request
namespace tile {
constexpr int BM = 128;     // tokens
constexpr int BK = 64;      // inputs per stage
constexpr int STAGES = 4;
constexpr int X_BYTES = BM * BK * 2;
constexpr int NUM_THREADS = 192;  // TMA, MMA, 4 epilogue warps
constexpr int ACCS = 4;     // accumulators, taken in turn: short chains of f32 additions (the tensor core's truncate)
constexpr int kMaxRank = 128;
inline __host__ __device__ int tmem_cols(int r_pad) { return r_pad <= 16 ? 64 : r_pad <= 32 ? 128 : r_pad <= 64 ? 256 : 512; }

// Shared memory of a launch: stages of x and A; the partial sums (f32
// [r_pad][128 tokens]) take the stages' place once the products are done.  A
// CTA that takes all of the tensor memory takes all of the shared memory too,
// so that none waits for its columns (see TmemShare).
inline int smem_bytes(int r_pad) {
  if (tmem_cols(r_pad) == kTmemColumns) return kSmemMax;
  return 1024 + std::max(STAGES * (X_BYTES + r_pad * BK * 2), r_pad * BM * 4) + 256;
}
static_assert(1024 + STAGES * (X_BYTES + kMaxRank * BK * 2) + 256 <= kSmemMax && kMaxRank * BM * 4 <= kSmemMax - 1280,
              "shared memory of one CTA");
}  // namespace tile

// low of one 128-token tile of one request: x (128 x K) times A^T (K x rank) on
// the tensor cores.  A cluster's CTAs split K (the tiles of a batch of prompts
// are too few to fill the GPU otherwise) and add their parts through
// distributed shared memory in a fixed order.  Bound by latency (20-23 us; 15-22 %
// of DRAM's rate, 6-12 % of the tensor pipe).
__global__ void __launch_bounds__(tile::NUM_THREADS)
    lora_shrink_tile_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap amap,
                            const ShrinkParams p, int* err) {
  using namespace tile;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int stage_bytes = X_BYTES + p.r_pad * BK * 2;
  const int ring = max(STAGES * stage_bytes, p.r_pad * BM * 4);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + ring);
  uint64_t* empty = full + STAGES;
  uint64_t* done = empty + STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* found = reinterpret_cast<int*>(tmem_slot + 2);
  float* sums = reinterpret_cast<float*>(smem);

  cg::cluster_group cluster = cg::this_cluster();
  const int csize = (int)cluster.num_blocks(), crank = (int)cluster.block_rank();
  const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
  griddep_wait();
  if (warp == 0) {
    int req = -1, tl = 0;
    if (!find_request(p.cu, p.n_reqs, p.tokens, BM, (int)blockIdx.x / csize, req, tl)) req = -1;
    if (lane == 0) {
      found[0] = req;
      found[1] = tl;
    }
  }
  __syncthreads();
  const int req = found[0];
  if (req < 0) return;  // the whole cluster
  const int slot = p.slots[req];
  if (slot < 0 || slot >= p.n_slots) return;
  const LoraSlot info = p.slot_info[slot];
  if (info.rank == 0) return;
  const int n16 = (info.rank + 15) / 16;
  const int end = min(p.cu[req + 1], p.tokens);
  const int t0 = max(0, p.cu[req]) + found[1] * BM;
  const int blocks = (p.k_in + BK - 1) / BK, per = (blocks + csize - 1) / csize;
  const int b0 = min(blocks, crank * per), b1 = min(blocks, b0 + per);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      bar_init(&full[s], 1);
      bar_init(&empty[s], 1);
    }
    bar_init(done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, tmem_cols(p.r_pad));
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_launch();  // after the TMEM allocation: a dependent's could block it, and waits for this grid
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (elect_one()) {
      bool ok = true;
      for (int b = b0; b < b1; ++b) {
        const int it = b - b0, s = it % STAGES;
        if (!wait_bar(&empty[s], ((it / STAGES) & 1) ^ 1, abort_flag, err, DEV_ERR_TIMEOUT_TMA)) {
          ok = false;
          break;
        }
        uint8_t* st = smem + s * stage_bytes;
        bar_arrive_expect_tx(&full[s], (uint32_t)(X_BYTES + n16 * 16 * BK * 2));
        tma_load_2d(st, &xmap, &full[s], b * BK, t0);
        for (int i = 0; i < n16; ++i)  // 16 ranks per box: only the slot's own
          tma_load_2d(st + X_BYTES + i * 16 * BK * 2, &amap, &full[s], b * BK, slot * p.r_pad + i * 16);
      }
      if (!ok) {
        const unsigned long long w0 = globaltimer_ns();
        while (globaltimer_ns() - w0 < 1000000ull) {
        }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint32_t idesc = make_idesc_f16(BM, n16 * 16, 0, 0, 0);
      for (int b = b0; b < b1; ++b) {
        const int it = b - b0, s = it % STAGES;
        if (!wait_bar(&full[s], (it / STAGES) & 1, abort_flag, err, DEV_ERR_TIMEOUT_MMA)) break;
        tc_fence_after();
        const uint32_t xa = smem_u32(smem + s * stage_bytes), aa = xa + X_BYTES;
#pragma unroll
        for (int k16 = 0; k16 < BK / 16; ++k16)
          mma_ss(tmem + (it % ACCS) * p.r_pad, make_smem_desc(xa + k16 * 32, 16, 1024),
                 make_smem_desc(aa + k16 * 32, 16, 1024), idesc, it >= ACCS || k16 != 0 ? 1u : 0u);
        tc_commit(&empty[s]);
      }
      tc_commit(done);
      const uint32_t da = smem_u32(done);
      const unsigned long long w0 = globaltimer_ns();
      while (!bar_try_wait(da, 0)) {
        if (globaltimer_ns() - w0 > kWaitLimitNs) {
          if (err) atomicCAS(err, 0, DEV_ERR_TIMEOUT_MMA);
          break;
        }
      }
    }
  } else {
    const int q = warp & 3;
    const bool good = wait_bar(done, 0, abort_flag, err, DEV_ERR_TIMEOUT_EPILOGUE);
    if (__all_sync(0xffffffffu, good)) {
      tc_fence_after();
      for (int c = 0; c < n16 * 16; c += 16) {
        float v[16] = {};
        for (int a = 0; a < min(ACCS, b1 - b0); ++a) {
          uint32_t r[16];
          tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + a * p.r_pad + c, r);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] += __uint_as_float(r[i]);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) sums[(c + i) * BM + q * 32 + lane] = v[i];
      }
    }
    tc_fence_before();
  }
  cluster.sync();
  const int n = n16 * 8;  // pairs of ranks
  for (int e = crank * NUM_THREADS + threadIdx.x; e < n * BM; e += csize * NUM_THREADS) {
    const int row = e % BM, t = t0 + row, r = e / BM * 2;
    float a = 0.f, b = 0.f;
    for (int c = 0; c < csize; ++c) {
      const float* part = cluster.map_shared_rank(sums, c) + r * BM + row;
      a += part[0];
      b += part[BM];
    }
    if (t >= end) continue;
    a = r < info.rank ? a * info.scale : 0.f;  // what x leaves of A's rows past the rank (0 * inf) is no value
    b = r + 1 < info.rank ? b * info.scale : 0.f;
    uint32_t* dst = p.low_pieces + ((size_t)(r / 16 * kLowParts) * p.tokens + t) * 8 + r % 16 / 2;
    const size_t part = (size_t)p.tokens * 8;
    const uint32_t l1 = __byte_perm(__float_as_uint(cut_piece(a)), __float_as_uint(cut_piece(b)), 0x7632);
    dst[0] = l1;
    dst[part] = __byte_perm(__float_as_uint(cut_piece(a)), __float_as_uint(cut_piece(b)), 0x7632);
    dst[2 * part] = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
    dst[3 * part] = l1 & (((l1 & 0x7f80u) != 0x7f80u ? 0x0000ffffu : 0u) |
                          ((l1 & 0x7f800000u) != 0x7f800000u ? 0xffff0000u : 0u));
  }
  cluster.sync();  // no CTA ends while another reads its shared memory
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols(p.r_pad));
  }
}

// B [out][rank] into the chunks of a slot (LoraDevice::up), and the slot's rank
// and scale.  Rows [swiglu_from, out) go to alternating device rows, gate then
// value, as those of the B1_0 weight.
__global__ void lora_retile_kernel(const __half* __restrict__ src, LoraSlot info, int n_rows, int n_ftiles, int r_pad,
                                   int swiglu_from, __half* __restrict__ dst, LoraSlot* slot) {
  const int rank = info.rank;
  if (blockIdx.x == 0 && threadIdx.x == 0) {  // nonfinite is zero before this kernel
    slot->rank = rank;
    slot->scale = info.scale;
  }
  if (rank == 0) return;
  bool bad = false;
  const long long total = (long long)n_ftiles * 128 * r_pad;
  for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < total;
       i += (long long)gridDim.x * blockDim.x) {
    const int r16 = (int)(i % 16), row = (int)(i / 16 % 128);
    const int g = (int)(i / 2048 % (r_pad / 16)), ft = (int)(i / 2048 / (r_pad / 16));
    const int n = ft * 128 + row, r = g * 16 + r16;
    __half v = __float2half_rn(0.f);
    if (n < n_rows && r < rank) {
      int s = n;
      if (swiglu_from >= 0 && n >= swiglu_from) {
        const int j = n - swiglu_from;
        s = swiglu_from + ((j & 1) ? (n_rows - swiglu_from) / 2 + (j >> 1) : (j >> 1));
      }
      v = src[(size_t)s * rank + r];
      bad |= (__half_as_ushort(v) & 0x7c00) == 0x7c00;
    }
    dst[i] = v;
  }
  if (bad) atomicOr(&slot->nonfinite, 1);
}

// Lists the extra k-blocks of each token tile of the GEMM (LoraGemm): for
// every request with an adapter that has tokens in the tile, its ranks in
// groups of 16.  One warp per tile.
__global__ void lora_plan_kernel(const int* __restrict__ cu, const int* __restrict__ slots, int n_reqs, int tokens,
                                 const LoraSlot* __restrict__ slot_info, int n_slots, int tile_tokens, int n_tiles,
                                 int max_groups, int* __restrict__ group_count, int4* __restrict__ groups) {
  const int tile = (int)(blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32), lane = threadIdx.x & 31;
  griddep_wait();
  griddep_launch();
  if (tile >= n_tiles) return;
  const int t0 = tile * tile_tokens, t1 = min(tokens, t0 + tile_tokens);
  int lo = 0, hi = n_reqs;  // the last request that begins at or before t0
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (cu[mid] <= t0) lo = mid; else hi = mid;
  }
  int base = 0, any_bad = 0;
  for (int i0 = lo; i0 < n_reqs; i0 += 32) {
    const int i = i0 + lane;
    int slot = -1, n16 = 0, a = t1, b = t1, bad = 0;
    if (i < n_reqs) {
      a = max(t0, cu[i]);
      b = min(t1, cu[i + 1]);
      slot = slots[i];
      if (a < b && slot >= 0 && slot < n_slots) {
        n16 = (slot_info[slot].rank + 15) / 16;
        if (n16 > 0 && slot_info[slot].nonfinite) bad = kNonfinite;
      }
    }
    int incl = n16;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const int at = base + incl - n16;
    for (int j = 0; j < n16; ++j)
      if (at + j < max_groups) groups[(size_t)tile * max_groups + at + j] = make_int4(slot | bad, j * 16, a, b);
    base += __shfl_sync(0xffffffffu, incl, 31);
    any_bad |= __reduce_or_sync(0xffffffffu, bad);
    // past the tile once one of these 32 requests begins at or after its end
    if (__any_sync(0xffffffffu, i < n_reqs && cu[i] >= t1)) break;
  }
  if (lane == 0) group_count[tile] = min(base, max_groups) | any_bad;
}

int shrink_tiles(const ShrinkParams& p, cudaStream_t st) {
  CUtensorMap xmap, amap;
  int rc = encode_tmap_2d_16b(&xmap, p.x, p.tokens, p.k_in, p.ldx, tile::BK, tile::BM, false);
  if (!rc)
    rc = encode_tmap_2d_16b(&amap, p.down, (long long)p.n_slots * p.r_pad, p.k_in, p.k_in, tile::BK, 16, false);
  if (rc) return rc;
  static DeviceMemo<1> memo;
  int set = 0;
  const cudaError_t e = memo.get(0, &set, [](int*) {
    return cudaFuncSetAttribute(lora_shrink_tile_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                tile::smem_bytes(tile::kMaxRank));
  });
  if (e != cudaSuccess) return cuda_status(e, "lora shrink set smem attribute");
  const long long seqs = std::min(p.n_reqs, p.tokens);
  const long long units = (p.tokens + seqs * (tile::BM - 1)) / tile::BM;
  int c = 8;  // CTAs that split K: about three per SM's worth of them, each at least two stages
  while (c > 1 && (units * c > 3ll * num_sms() || p.k_in / tile::BK < 2 * c)) c /= 2;
  if (units * c > 0x7fffffffll) return fail(-2, "b1_gemm_lora: too many tokens in one call");
  ProfScope prof("lora_shrink", 0.0, 2.0 * p.tokens * p.k_in, st);  // x; the ranks are on the device
  return launch_after("lora_shrink_tile_kernel launch", lora_shrink_tile_kernel, dim3((unsigned)(units * c)),
                      dim3(tile::NUM_THREADS), (size_t)tile::smem_bytes(p.r_pad), c, st, xmap, amap, p,
                      device_error_word());
}

template <int NT>
int shrink(const ShrinkParams& p, cudaStream_t st) {
  auto kern = lora_shrink_kernel<NT>;
  constexpr int TM = 16;
  constexpr int smem = kWarps * TM * NT * 8 * (int)sizeof(float);
  static DeviceMemo<1> memo;
  int set = 0;
  const cudaError_t e = memo.get(0, &set, [&](int*) {
    return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  });
  if (e != cudaSuccess) return cuda_status(e, "lora shrink set smem attribute");
  const long long seqs = std::min(p.n_reqs, p.tokens);
  const long long units = (p.tokens + seqs * (TM - 1)) / TM;
  // CTAs of a cluster split K: about two CTAs per SM, each warp at least one chunk
  int c = 8;
  while (c > 1 && (units * c > 2ll * num_sms() || (p.k_in / kChunk) / c < kWarps)) c /= 2;
  if (units * c > 0x7fffffffll) return fail(-2, "b1_gemm_lora: too many tokens in one call");
  ProfScope prof("lora_shrink", 0.0, 2.0 * p.tokens * p.k_in, st);
  return launch_after("lora_shrink_kernel launch", kern, dim3((unsigned)(units * c)), dim3(kThreads), smem, c, st, p);
}

int shrink_by_rank(const ShrinkParams& p, int max_rank, cudaStream_t st) {
  if (max_rank <= 16) return shrink<2>(p, st);
  if (max_rank <= 32) return shrink<4>(p, st);
  if (max_rank <= 64) return shrink<8>(p, st);
  return shrink<16>(p, st);
}

}  // namespace lora

int lora_tmem_shares(TmemShare* s) {
  int n = 0;
  for (int r = 16; r <= lora::tile::kMaxRank; r += 16)
    s[n++] = {lora::tile::smem_bytes(r), lora::tile::tmem_cols(r)};
  return n;
}

int launch_lora_retile(const __half* up, const LoraSlot& info, const LoraDevice& set, int slot, cudaStream_t st) {
  const size_t n = (size_t)set.n_ftiles * 128 * set.r_pad;
  const unsigned blocks = info.rank == 0 ? 1u : (unsigned)std::min<size_t>((n + 255) / 256, 148 * 16);
  LoraSlot* slot_info = set.info + slot;
  const cudaError_t e = cudaMemsetAsync(&slot_info->nonfinite, 0, sizeof(int), st);
  if (e != cudaSuccess) return cuda_status(e, "lora_retile_kernel clear");
  lora::lora_retile_kernel<<<blocks, 256, 0, st>>>(up, info, set.n_rows, set.n_ftiles, set.r_pad, set.swiglu_from,
                                                   set.up + (size_t)slot * n, slot_info);
  return launch_status("lora_retile_kernel launch");
}

int launch_b1_gemm_lora(const __half* x, long long ldx, int tokens, const B1Weight& w, const EpiSeg& seg,
                        const LoraDevice& set, const int* cu, const int* slots, int n_reqs, cudaStream_t st) {
  if (tokens == 0) return 0;
  if (n_reqs == 0) return launch_b1_gemm(x, ldx, tokens, w, &seg, 1, false, st);
  LoraGemm g;
  // The few-form reads B once per token, the other takes extra k-blocks per
  // request and rank.  Both, few / many in us (calls of a graph), adapters of
  // its own for each request:
  //                    3072 -> 9216, f16               3072 -> 3072  9216 -> 3072, f32
  //   rank             8         32         128        32            32
  //   64 x 1 token     23 / 89   27 / 149   60 / 616   21 / 147      27 / 182
  //   64 x 4           52 / 60   65 / 88    166 / 346  37 / 88       81 / 124
  //   16 x 8           30 / 41   36 / 56    83 / 158   25 / 51       42 / 81
  //   64 x 8           93 / 63   122 / 92   307 / 304  65 / 60       158 / 98
  //   16 x 16          51 / 37   64 / 44    153 / 98   36 / 42       76 / 75
  //   1 x 64           21 / 24   25 / 25    50 / 32    19 / 25       25 / 55
  //   64 x 32          345 / 116 463 / 152  1159 / 358 179 / 83      438 / 192
  //   1 x 300, 63 x 1  72 / 91   93 / 146   237 / 550  38 / 144      82 / 183
  //   1 x 900, 127 x 1 185 / 164 248 / 283  617 / 1060 95 / 254      236 / 370
  // The average decides, at 8.  Near it either may be the faster, for 64 x 8 by
  // 1.6 times and for the last row, whose average is 8.03, by 2.7 times the one
  // that is not taken: the rule does not look at ranks, shapes or the longest
  // request.
  g.mode = tokens > 8ll * n_reqs ? LORA_BLOCKS : LORA_DELTA;
  // scratch: low (or its pieces), then the lists of extra blocks
  const size_t low_bytes = (size_t)tokens * set.r_pad * (g.mode == LORA_BLOCKS ? 2 * kLowParts : sizeof(float));
  const size_t low_n = (low_bytes + 15) / 16 * 4;
  size_t more = 0;
  int n_tiles = 0;
  if (g.mode == LORA_BLOCKS) {
    g.tile_tokens = b1_gemm_tile_tokens(tokens, w, seg.mode);
    n_tiles = (tokens + g.tile_tokens - 1) / g.tile_tokens;
    g.max_groups = set.r_pad / 16 * std::min(n_reqs, g.tile_tokens);
    more = (size_t)n_tiles * (g.max_groups * sizeof(int4) + sizeof(int));
  }
  void* mem = nullptr;
  int rc = scratch_alloc(&mem, low_n * sizeof(float) + more, "b1_gemm_lora", st);
  if (rc) return rc;
  float* low = static_cast<float*>(mem);
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
  s.low = low;
  s.low_pieces = reinterpret_cast<uint32_t*>(low);
  g.cu = cu;
  g.slots = slots;
  g.info = set.info;
  g.n_reqs = n_reqs;
  g.n_slots = set.n_slots;
  g.r_pad = set.r_pad;
  g.n_ftiles = set.n_ftiles;
  g.up = set.up;
  g.low = low;
  g.tokens = tokens;
  g.low_pieces = reinterpret_cast<const uint4*>(low);
  if (g.mode == LORA_BLOCKS) {
    int4* groups = reinterpret_cast<int4*>(low + low_n);
    int* count = reinterpret_cast<int*>(groups + (size_t)n_tiles * g.max_groups);
    g.groups = groups;
    g.group_count = count;
    ProfScope prof("lora_plan", 0.0, 0.0, st);
    rc = launch_after("lora_plan_kernel launch", lora::lora_plan_kernel, dim3((unsigned)((n_tiles + 7) / 8)),
                      dim3(256), 0, 1, st, cu, slots, n_reqs, tokens, set.info, set.n_slots, g.tile_tokens, n_tiles,
                      g.max_groups, count, groups);
    if (rc == 0) rc = lora::shrink_tiles(s, st);
  } else {
    rc = lora::shrink_by_rank(s, set.max_rank, st);
  }
  if (rc == 0) rc = launch_b1_gemm(x, ldx, tokens, w, &seg, 1, false, st, nullptr, &g);
  scratch_free(mem, st);
  return rc;
}

}  // namespace bonsai
