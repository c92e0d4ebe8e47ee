// Causal grouped-head attention of the text stage for sm_100a: over whole
// packed prompts (bonsai_prompt_attention) and of new tokens over a paged
// key/value cache (bonsai_paged_attention), plus the cache's append.
//
//   O[t, h] = sum_j p_j V[j, h / G],  p = softmax_j(scale * Q[t, h] . K[j, h / G])
//
// over the keys j that token t sees: those of its own sequence up to its own
// place (causal), or all of them.  G = n_heads / n_kv_heads query heads share
// one key/value head.
//
// One CTA = one sequence x one key/value head x one tile of 128 query rows,
// where a row is a (token, head of the group) pair: row r is token r / G, head
// r % G.  Taking the group's heads into the rows reads every key once for G
// heads, makes the causal triangle's diagonal G times narrower, and lets a
// single token fill G rows.  Two such CTAs share an SM: one's softmax runs
// beside the other's products and loads.
//   warps 0-3   softmax: thread i owns row i (TMEM lane i).  Online softmax
//               in the log2 domain; the running max moves (and O in TMEM is
//               rescaled) only when a block's max exceeds it by more than 8.
//               Warps without a row (a single token has G rows) take no part.
//   warp 4      TMA: Q once, then K and V blocks of 64 keys (128-byte
//               swizzle, 64-dim halves); paged: one box per page and half,
//               issued by one lane each, page indices read 32 at a time.
//   warp 5      one thread issues tcgen05.mma: S(j) = Q K_j^T (SMEM, SMEM),
//               O += P(j) V_j (P from TMEM, V MN-major); S runs two blocks
//               ahead (double-buffered).
//   warps 6-7   blocks that not every row sees whole (a causal diagonal, the
//               end of a sequence inside a block or page): V rows past the
//               sequence's end are zeroed in shared memory before the
//               product, since 0 * NaN would reach every row; V values of
//               keys that only some rows see are zeroed where they are not
//               finite, and the rows that do see them add them at the end.
// TMEM (256 columns): S(even) [0, 64) S(odd) [64, 128) O [128, 128 + HD);
// P(j) (16-bit pairs) overwrites the first 32 columns of its S.
#include "internal.cuh"
#include "ptx.cuh"

#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>

namespace bonsai {
namespace gemm {
PFN_cuTensorMapEncodeTiled_v12000 get_encode_fn();
}
namespace text {

constexpr int BQ = 128;   // query rows per CTA
constexpr int BKV = 64;   // keys per block
constexpr int RING = 2;   // K and V slots
constexpr int NUM_THREADS = 256;
constexpr int WARP_TMA = 4, WARP_MMA = 5, WARP_FIX = 6;
constexpr int TMEM_COLS = 256;
constexpr int S_COL = 0, O_COL = 128;
constexpr float kRescaleThreshold = 8.0f;
constexpr int kMaxSeqs = 8192;  // tile counts of a launch fit the K/V ring

template <int HD>
struct Cfg {
  static constexpr int HALVES = HD / 64;
  static constexpr int Q_HALF = BQ * 128;         // 128 rows x 64 dims
  static constexpr int Q_BYTES = HALVES * Q_HALF;
  static constexpr int KV_HALF = BKV * 128;
  static constexpr int KV_BYTES = HALVES * KV_HALF;
  static constexpr int SMEM_BYTES = 1024 + Q_BYTES + 2 * RING * KV_BYTES + 256;
};
static_assert(2 * RING * Cfg<64>::KV_BYTES >= kMaxSeqs * 4, "tile counts do not fit the ring");

struct Params {
  const int* cu;        // [n_seqs + 1] first query row of each sequence
  const int* ctx;       // [n_seqs] keys of each sequence (null: its query rows)
  const int* table;     // [n_seqs][table_ld] page indices (paged)
  long long table_ld;
  int table_width, page_shift, n_pages;
  int n_seqs, total_q, n_heads, n_kv, group, tile_tokens;
  int causal, splits;
  float scale_log2;     // softmax scale * log2(e)
  void* out;
  long long out_token, out_head;
  const void* v;        // values as the kernel's repair reads them
  long long v_page, v_token, v_head;
  float* part_o;        // [splits][total_q][n_heads][HD] (splits > 1)
  float* part_lse;      // [splits][total_q][n_heads]
  int* err;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool kBF16>
__device__ __forceinline__ uint32_t cvt2(float lo, float hi) {
  uint32_t y;
  if constexpr (kBF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}
template <bool kBF16>
__device__ __forceinline__ bool finite16(uint32_t h) {  // low 16 bits
  constexpr uint32_t e = kBF16 ? 0x7f80u : 0x7c00u;
  return (h & e) != e;
}
template <bool kBF16>
__device__ __forceinline__ float to_f32(uint16_t h) {
  if constexpr (kBF16)
    return __uint_as_float((uint32_t)h << 16);
  else
    return __half2float(__ushort_as_half(h));
}

__device__ __forceinline__ void tma_load_4d(void* dst, const void* map, uint64_t* bar, int c0,
                                            int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// Query tile b of a launch: tiles go by level (their index within their
// sequence), the highest level of all sequences first, so that under a causal
// mask the tiles with the most keys start first.  count[i] = tiles of
// sequence i (shared memory).  One warp; false where there are at most b tiles.
__device__ bool find_tile(const int* count, int n, int b, int& seq, int& level) {
  const int lane = (int)lane_id();
  auto at_least = [&](int lv) {  // tiles of level >= lv
    int c = 0;
    for (int i = lane; i < n; i += 32) c += max(0, count[i] - lv);
    return __reduce_add_sync(0xffffffffu, c);
  };
  int hi = 0;
  for (int i = lane; i < n; i += 32) hi = max(hi, count[i]);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (at_least(0) <= b) return false;
  int lo = 0, above = 0;  // at_least(lo) > b, at_least(hi) = above <= b
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    const int c = at_least(mid);
    if (c > b) {
      lo = mid;
    } else {
      hi = mid;
      above = c;
    }
  }
  int rank = b - above;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const uint32_t has = __ballot_sync(0xffffffffu, i0 + lane < n && count[i0 + lane] > lo);
    const int c = __popc(has);
    if (rank < c) {
      const bool mine = ((has >> lane) & 1u) && __popc(has & ((1u << lane) - 1u)) == rank;
      seq = i0 + __ffs(__ballot_sync(0xffffffffu, mine)) - 1;
      level = lo;
      return true;
    }
    rank -= c;
  }
  return false;
}

template <int HD, bool kBF16, bool kPaged>
__global__ void __launch_bounds__(NUM_THREADS, 2)
    text_attention_kernel(const __grid_constant__ CUtensorMap qmap,
                          const __grid_constant__ CUtensorMap kmap,
                          const __grid_constant__ CUtensorMap vmap, const Params p) {
  using C = Cfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* qs = smem;
  uint8_t* ks = qs + C::Q_BYTES;
  uint8_t* vs = ks + RING * C::KV_BYTES;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(vs + RING * C::KV_BYTES);
  uint64_t* k_full = q_full + 1;
  uint64_t* k_empty = k_full + RING;
  uint64_t* v_full = k_empty + RING;
  uint64_t* v_empty = v_full + RING;
  uint64_t* v_fixed = v_empty + RING;
  uint64_t* s_full = v_fixed + RING;
  uint64_t* p_ready = s_full + 2;
  uint64_t* pv_done = p_ready + 2;
  uint64_t* drain = pv_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* nonfinite = abort_flag + 1;
  int* found = const_cast<int*>(nonfinite) + 1;  // sequence (-1: none), level

  const int warp = threadIdx.x / 32;
  const int lane = (int)lane_id();
  const int split = (int)(blockIdx.x % (unsigned)p.splits);
  const int unit = (int)(blockIdx.x / (unsigned)p.splits);
  const int kvh = unit % p.n_kv;

  // ---- which tile
  int* count = reinterpret_cast<int*>(ks);
  for (int i = threadIdx.x; i < p.n_seqs; i += NUM_THREADS) {
    const int a = max(0, min(p.cu[i], p.total_q)), b = max(a, min(p.cu[i + 1], p.total_q));
    count[i] = (b - a + p.tile_tokens - 1) / p.tile_tokens;
  }
  __syncthreads();
  if (warp == 0) {
    int seq = -1, level = 0;
    if (!find_tile(count, p.n_seqs, unit / p.n_kv, seq, level)) seq = -1;
    if (lane == 0) {
      found[0] = seq;
      found[1] = level;
    }
  }
  fence_proxy_async_smem();  // the ring's next writer is the TMA
  __syncthreads();
  const int seq = found[0];
  if (seq < 0) return;
  const int q_begin = max(0, min(p.cu[seq], p.total_q));
  const int q_len = max(q_begin, min(p.cu[seq + 1], p.total_q)) - q_begin;
  int kv_len = q_len;
  if (kPaged) {
    const long long room = (long long)p.table_width << p.page_shift;
    kv_len = (int)max(0ll, min((long long)p.ctx[seq], room));
  }
  const int t0 = found[1] * p.tile_tokens;          // first token of the tile
  const int n_tok = min(p.tile_tokens, q_len - t0);
  const int first = kPaged ? p.ctx[seq] - q_len + t0 : t0;  // its place in the sequence
  // Keys [0, lim) are seen by a row; lim grows by one with each token.
  auto keys_seen = [&](int tok) {
    return p.causal ? max(0, min(kv_len, first + tok + 1)) : kv_len;
  };
  const int lim_min = keys_seen(0), lim_max = keys_seen(n_tok - 1);
  const int blocks = (lim_max + BKV - 1) / BKV;
  const int chunk = (blocks + p.splits - 1) / p.splits;
  const int j0 = split * chunk;
  const int nkv = max(0, min(blocks - j0, chunk));
  // Blocks [jb, nkv) hold a key that some row of the tile does not see.
  const int jb = max(0, lim_min / BKV - j0);

  const int row = warp * 32 + lane;  // softmax warps
  const int tok = row / p.group;
  const bool valid = warp < 4 && tok < n_tok && row < p.tile_tokens * p.group;
  const int head = kvh * p.group + row - tok * p.group;
  const size_t q_row = (size_t)(q_begin + t0 + tok);
  uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + q_row * p.out_token + (size_t)head * p.out_head;
  const size_t part = ((size_t)split * p.total_q + q_row) * p.n_heads + head;

  if (nkv == 0) {  // no key: zeros (or a partial of weight zero)
    if (valid) {
      if (p.splits > 1) {
        p.part_lse[part] = -INFINITY;
      } else {
        for (int i = 0; i < HD / 8; ++i) reinterpret_cast<uint4*>(dst)[i] = make_uint4(0, 0, 0, 0);
      }
    }
    return;
  }
  const int active = (n_tok * p.group + 31) / 32;  // softmax warps with a row

  if (threadIdx.x == 0) {
    bar_init(q_full, 1);
    for (int s = 0; s < RING; ++s) {
      bar_init(&k_full[s], 1);
      bar_init(&k_empty[s], 1);
      bar_init(&v_full[s], 1);
      bar_init(&v_empty[s], 1);
      bar_init(&v_fixed[s], 2);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(&s_full[i], 1);
      bar_init(&p_ready[i], active);
      bar_init(&pv_done[i], 1);
    }
    bar_init(drain, 1);
    *abort_flag = 0;
    *nonfinite = 0;
    fence_barrier_init();
  }
  if (warp == WARP_MMA) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == WARP_TMA) {
    if (lane == 0) {
      tma_prefetch_desc(&kmap);
      tma_prefetch_desc(&vmap);
      bar_arrive_expect_tx(q_full, (uint32_t)(p.group * p.tile_tokens * HD * 2));
      for (int h = 0; h < C::HALVES; ++h)
        tma_load_3d(qs + h * C::Q_HALF, &qmap, q_full, h * 64, kvh * p.group, q_begin + t0);
    }
    // Paged: a block of 64 keys takes 64 / page boxes (one where a page holds
    // more), and each half of the head dims its own; lane l issues box
    // l / HALVES, half l % HALVES.  `ent` = 32 consecutive page indices.
    const int box_shift = min(p.page_shift, 6);
    const int boxes = BKV >> box_shift;
    const int box = lane / C::HALVES, half = lane % C::HALVES;
    const bool issues = kPaged ? box < boxes : lane < C::HALVES;
    int ent = -1, ent_base = -1;
    auto load = [&](const void* map, uint8_t* ring, uint64_t* full, uint64_t* empty, int j) -> bool {
      const int s = j % RING;
      const int key0 = (j0 + j) * BKV;
      int page = 0;
      if constexpr (kPaged) {
        const int want = (key0 >> p.page_shift) & ~31;
        if (want != ent_base) {  // 64 keys never reach past 32 pages (page >= 8)
          ent_base = want;
          ent = want + lane < p.table_width ? p.table[(size_t)seq * p.table_ld + want + lane] : -1;
        }
        page = __shfl_sync(0xffffffffu, ent, (((key0 + (box << box_shift)) >> p.page_shift) - ent_base) & 31);
      }
      const bool good = wait_bar(&empty[s], ((j / RING) & 1) ^ 1, abort_flag, p.err, DEV_ERR_TIMEOUT_TMA);
      if (!__all_sync(0xffffffffu, good)) return false;
      if (lane == 0) bar_arrive_expect_tx(&full[s], C::KV_BYTES);
      __syncwarp();
      if (issues) {
        uint8_t* d = ring + s * C::KV_BYTES + half * C::KV_HALF;
        if constexpr (kPaged)
          tma_load_4d(d + (box << box_shift) * 128, map, &full[s], half * 64, kvh,
                      (key0 + (box << box_shift)) & ((1 << p.page_shift) - 1), page);
        else
          tma_load_3d(d, map, &full[s], half * 64, kvh, q_begin + key0);
      }
      return true;
    };
    // K runs two blocks ahead of V, as S does of P V: each load is asked for as
    // soon as its slot is free, two blocks' time before it is needed.
    bool ok = load(&kmap, ks, k_full, k_empty, 0) && (nkv == 1 || load(&kmap, ks, k_full, k_empty, 1));
    for (int j = 0; j < nkv && ok; ++j) {
      ok = load(&vmap, vs, v_full, v_empty, j);
      if (ok && j + 2 < nkv) ok = load(&kmap, ks, k_full, k_empty, j + 2);
    }
    if (!ok) {  // let copies in flight land before the shared memory is released
      const unsigned long long w0 = globaltimer_ns();
      while (globaltimer_ns() - w0 < 1000000ull) {
      }
    }
  } else if (warp == WARP_MMA) {
    if (elect_one()) {
      constexpr uint32_t idesc_s = make_idesc_f16(BQ, BKV, kBF16 ? 1 : 0, 0, 0);
      constexpr uint32_t idesc_o = make_idesc_f16(BQ, HD, kBF16 ? 1 : 0, 0, 1);
      auto issue_s = [&](int j) -> bool {
        const int s = j % RING;
        if (!wait_bar(&k_full[s], (j / RING) & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_MMA)) return false;
        tc_fence_after();
        const uint32_t qa = smem_u32(qs), ka = smem_u32(ks + s * C::KV_BYTES);
#pragma unroll
        for (int k16 = 0; k16 < HD / 16; ++k16)
          mma_ss(tmem + S_COL + (j & 1) * BKV,
                 make_smem_desc(qa + (k16 >> 2) * C::Q_HALF + (k16 & 3) * 32, 16, 1024),
                 make_smem_desc(ka + (k16 >> 2) * C::KV_HALF + (k16 & 3) * 32, 16, 1024), idesc_s,
                 k16 > 0 ? 1u : 0u);
        tc_commit(&s_full[j & 1]);
        tc_commit(&k_empty[s]);
        return true;
      };
      auto issue_pv = [&](int j) -> bool {
        const int s = j % RING;
        if (!wait_bar(&v_full[s], (j / RING) & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_MMA)) return false;
        if (!wait_bar(&v_fixed[s], (j / RING) & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_MMA)) return false;
        if (!wait_bar(&p_ready[j & 1], (j >> 1) & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_MMA)) return false;
        tc_fence_after();
        const uint32_t va = smem_u32(vs + s * C::KV_BYTES);
#pragma unroll
        for (int k16 = 0; k16 < BKV / 16; ++k16)
          mma_ts(tmem + O_COL, tmem + S_COL + (j & 1) * BKV + k16 * 8,
                 make_smem_desc(va + k16 * 16 * 128, C::KV_HALF, 1024), idesc_o,
                 (j > 0 || k16 > 0) ? 1u : 0u);
        tc_commit(&pv_done[j & 1]);
        tc_commit(&v_empty[s]);
        return true;
      };
      bool ok = wait_bar(q_full, 0, abort_flag, p.err, DEV_ERR_TIMEOUT_MMA) && issue_s(0);
      if (ok && nkv > 1) ok = issue_s(1);
      for (int j = 0; j < nkv && ok; ++j) {
        ok = issue_pv(j);
        if (ok && j + 2 < nkv) ok = issue_s(j + 2);
      }
      tc_commit(drain);
      const uint32_t da = smem_u32(drain);
      const unsigned long long w0 = globaltimer_ns();
      while (!bar_try_wait(da, 0)) {
        if (globaltimer_ns() - w0 > kWaitLimitNs) {
          if (p.err) atomicCAS(p.err, 0, DEV_ERR_TIMEOUT_MMA);
          break;
        }
      }
    }
  } else if (warp >= WARP_FIX) {
    // Every block passes here, so that the two warps follow each phase of the
    // ring; those before jb pass untouched.
    for (int j = 0; j < nkv; ++j) {
      const int s = j % RING;
      const bool good = wait_bar(&v_full[s], (j / RING) & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_PRODUCER);
      if (!__all_sync(0xffffffffu, good)) break;
      if (j < jb) {
        if (lane == 0) bar_arrive(&v_fixed[s]);
        continue;
      }
      const int key0 = (j0 + j) * BKV;
      // one key per thread: row `key` of both halves (the swizzle permutes
      // 16-byte pieces within a 128-byte row only)
      const int r = (warp - WARP_FIX) * 32 + lane;
      uint8_t* at = vs + s * C::KV_BYTES + r * 128;
      if (key0 + r >= kv_len) {
        for (int h = 0; h < C::HALVES; ++h)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<uint4*>(at + h * C::KV_HALF + ((i ^ r) & 7) * 16) = make_uint4(0, 0, 0, 0);
      } else if (key0 + r >= lim_min) {
        for (int h = 0; h < C::HALVES; ++h)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint4* q4 = reinterpret_cast<uint4*>(at + h * C::KV_HALF + ((i ^ r) & 7) * 16);
            uint32_t w[4] = {q4->x, q4->y, q4->z, q4->w};
            bool bad = false;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const bool lo = finite16<kBF16>(w[k]), hi = finite16<kBF16>(w[k] >> 16);
              bad |= !lo || !hi;
              w[k] &= (lo ? 0x0000ffffu : 0u) | (hi ? 0xffff0000u : 0u);
            }
            if (bad) {
              *q4 = make_uint4(w[0], w[1], w[2], w[3]);
              *nonfinite = 1;
            }
          }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) bar_arrive(&v_fixed[s]);
    }
  } else if (warp < active) {
    const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
    const uint32_t o_addr = tmem + lane_base + O_COL;
    const int lim = valid ? keys_seen(tok) : 0;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int j = 0; j < nkv; ++j) {
      const int buf = j & 1;
      const uint32_t s_addr = tmem + lane_base + S_COL + buf * BKV;
      bool good = wait_bar(&s_full[buf], (j >> 1) & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_SOFTMAX);
      if (!__all_sync(0xffffffffu, good)) {
        ok = false;
        break;
      }
      tc_fence_after();
      float s[BKV];
      {
        uint32_t r0[32], r1[32];
        tmem_ld32(s_addr, r0);
        tmem_ld32(s_addr + 32, r1);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          s[i] = __uint_as_float(r0[i]);
          s[32 + i] = __uint_as_float(r1[i]);
        }
      }
      if (j >= jb) {  // a key past the row's limit: whatever it gave, it counts nothing
        const int left = lim - (j0 + j) * BKV;
#pragma unroll
        for (int c = 0; c < BKV; ++c)
          if (c >= left) s[c] = -INFINITY;
      }
      float m8[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) m8[i] = fmaxf(s[i], s[8 + i]);
#pragma unroll
      for (int c = 16; c < BKV; c += 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) m8[i] = fmaxf(m8[i], s[c + i]);
      }
      float mx = fmaxf(fmaxf(fmaxf(m8[0], m8[1]), fmaxf(m8[2], m8[3])),
                       fmaxf(fmaxf(m8[4], m8[5]), fmaxf(m8[6], m8[7])));
      mx *= p.scale_log2;
      float alpha = 1.0f;
      if (mx > m + kRescaleThreshold) {
        alpha = ex2(m - mx);
        m = mx;
      }
      if (j > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
        good = wait_bar(&pv_done[buf ^ 1], ((j - 1) >> 1) & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_SOFTMAX);
        if (!__all_sync(0xffffffffu, good)) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t r[32];
          tmem_ld32(o_addr + c * 32, r);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
          tmem_st32(o_addr + c * 32, r);
        }
      }
      const float mref = m == -INFINITY ? 0.0f : m;  // no key seen yet: every p is 2^-inf = 0
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ch = 0; ch < BKV / 32; ++ch) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float a = ex2(fmaf(s[ch * 32 + 2 * i], p.scale_log2, -mref));
          const float b = ex2(fmaf(s[ch * 32 + 2 * i + 1], p.scale_log2, -mref));
          sum[i & 3] += a + b;
          pk[i] = cvt2<kBF16>(a, b);
        }
        tmem_st16(s_addr + ch * 16, pk);
      }
      l = l * alpha + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(&p_ready[buf]);
    }
    if (ok) {
      const int last = nkv - 1;
      const bool good = wait_bar(&pv_done[last & 1], (last >> 1) & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_SOFTMAX);
      if (__all_sync(0xffffffffu, good)) {
        tc_fence_after();
        const float inv_l = l == 0.0f ? 0.0f : 1.0f / l;  // no key in this range: zeros
        const bool repair = *nonfinite != 0;
        // keys that only some rows see, within this CTA's range
        const int from = max(lim_min, (j0 + jb) * BKV), to = min(lim, (j0 + nkv) * BKV);
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t r[32];
          tmem_ld32(o_addr + c * 32, r);
          tmem_wait_ld();
          if (!valid) continue;
          float o[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __uint_as_float(r[i]) * inv_l;
          if (repair) {
            for (int key = from; key < to; ++key) {
              const uint16_t* src = static_cast<const uint16_t*>(p.v) + (size_t)kvh * p.v_head + c * 32;
              if constexpr (kPaged) {
                const int page = p.table[(size_t)seq * p.table_ld + (key >> p.page_shift)];
                if (page < 0 || page >= p.n_pages) continue;
                src += (size_t)page * p.v_page + (size_t)(key & ((1 << p.page_shift) - 1)) * p.v_token;
              } else {
                src += (size_t)(q_begin + key) * p.v_token;
              }
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!finite16<kBF16>(src[i])) o[i] += to_f32<kBF16>(src[i]);
            }
          }
          if (p.splits > 1) {
            float4* d4 = reinterpret_cast<float4*>(p.part_o + part * HD + c * 32);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              d4[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          } else {
            uint4* d4 = reinterpret_cast<uint4*>(dst + c * 32);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              d4[i] = make_uint4(cvt2<kBF16>(o[8 * i], o[8 * i + 1]), cvt2<kBF16>(o[8 * i + 2], o[8 * i + 3]),
                                 cvt2<kBF16>(o[8 * i + 4], o[8 * i + 5]), cvt2<kBF16>(o[8 * i + 6], o[8 * i + 7]));
          }
        }
        if (valid && p.splits > 1) p.part_lse[part] = l == 0.0f ? -INFINITY : m + log2f(l);
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == WARP_MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// Merges the partial outputs of the key ranges of each (row, head): with
// lse_s = log2 of range s's exponential sum, out = sum_s 2^(lse_s - top) O_s
// / sum_s 2^(lse_s - top).  A range without a key has lse -inf and is not read.
template <int HD, bool kBF16>
__global__ void text_combine_kernel(const float* __restrict__ part_o, const float* __restrict__ part_lse,
                                    int splits, int rows, int n_heads, uint16_t* out,
                                    long long out_token, long long out_head) {
  const long long idx = blockIdx.x * (long long)blockDim.x + threadIdx.x;
  const long long items = (long long)rows * n_heads;
  const long long it = idx / (HD / 8);
  if (it >= items) return;
  const int d8 = (int)(idx % (HD / 8)) * 8;
  float top = -INFINITY;
  for (int s = 0; s < splits; ++s) {
    const float x = part_lse[s * items + it];
    top = x > top || x != x ? x : top;  // a NaN sum stays
  }
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  float total = 0.f;
  for (int s = 0; s < splits; ++s) {
    const float lse = part_lse[s * items + it];
    if (lse == -INFINITY) continue;
    const float w = exp2f(lse - top);
    total += w;
    const float4* src = reinterpret_cast<const float4*>(part_o + (s * items + it) * HD + d8);
    const float4 a = src[0], b = src[1];
    acc[0] += w * a.x; acc[1] += w * a.y; acc[2] += w * a.z; acc[3] += w * a.w;
    acc[4] += w * b.x; acc[5] += w * b.y; acc[6] += w * b.z; acc[7] += w * b.w;
  }
  const float inv = total == 0.f ? 0.f : 1.0f / total;
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = cvt2<kBF16>(acc[2 * i] * inv, acc[2 * i + 1] * inv);
  *reinterpret_cast<uint4*>(out + (it / n_heads) * out_token + (it % n_heads) * out_head + d8) =
      make_uint4(h[0], h[1], h[2], h[3]);
}

// One 16-byte piece per thread: token t of the packed new keys / values goes
// to slot ctx - q_len + i of its sequence.  Pure copies, bound by latency.
__global__ void paged_append_kernel(const uint16_t* __restrict__ k, const uint16_t* __restrict__ v,
                                    long long k_token, long long k_head, long long v_token,
                                    long long v_head, uint16_t* kc, uint16_t* vc, long long kc_page,
                                    long long kc_token, long long kc_head, long long vc_page,
                                    long long vc_token, long long vc_head, int n_pages, int page_shift,
                                    const int* __restrict__ table, long long table_ld, int table_width,
                                    const int* __restrict__ cu, const int* __restrict__ ctx, int n_seqs,
                                    int total, int n_kv, int head_dim) {
  const int pieces = n_kv * (head_dim / 8);
  const long long idx = blockIdx.x * (long long)blockDim.x + threadIdx.x;
  const long long t = idx / pieces;
  if (t >= total) return;
  const int piece = (int)(idx - t * pieces);
  const int h = piece / (head_dim / 8), d = (piece - h * (head_dim / 8)) * 8;
  int lo = 0, hi = n_seqs;  // the last sequence that begins at or before t
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (cu[mid] <= t) lo = mid; else hi = mid;
  }
  if (t < cu[lo] || t >= cu[lo + 1]) return;  // a row of no sequence
  const long long pos = (long long)ctx[lo] - cu[lo + 1] + t;
  if (pos < 0 || (pos >> page_shift) >= table_width) return;
  const int page = table[lo * table_ld + (pos >> page_shift)];
  if (page < 0 || page >= n_pages) return;
  const long long slot = pos & ((1 << page_shift) - 1);
  *reinterpret_cast<uint4*>(kc + page * kc_page + slot * kc_token + h * kc_head + d) =
      *reinterpret_cast<const uint4*>(k + t * k_token + h * k_head + d);
  *reinterpret_cast<uint4*>(vc + page * vc_page + slot * vc_token + h * vc_head + d) =
      *reinterpret_cast<const uint4*>(v + t * v_token + h * v_head + d);
}

// ------------------------------------------------------------------- host
int encode(CUtensorMap* map, void* base, bool bf16, int rank, const long long* dims,
           const long long* strides /* elements, of dims 1.. */, const int* box) {
  auto fn = gemm::get_encode_fn();
  if (!fn) return fail(-5, "cuTensorMapEncodeTiled entry point unavailable");
  cuuint64_t d[5], st[4];
  cuuint32_t b[5], e[5];
  for (int i = 0; i < rank; ++i) {
    d[i] = (cuuint64_t)dims[i];
    b[i] = (cuuint32_t)box[i];
    e[i] = 1;
    // the stride of a dimension of size one is never used, whatever the caller has there
    if (i > 0) st[i - 1] = (cuuint64_t)(dims[i] == 1 ? dims[0] : strides[i - 1]) * 2;
  }
  const CUresult r = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                        (cuuint32_t)rank, base, d, st, b, e, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(-5, "cuTensorMapEncodeTiled (text attention) failed (code " + std::to_string((int)r) + ")");
  return 0;
}

template <int HD, bool kBF16, bool kPaged>
int launch(const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, const Params& p,
           long long ctas, cudaStream_t st) {
  auto kern = text_attention_kernel<HD, kBF16, kPaged>;
  static std::once_flag once[64];
  cudaError_t e = cudaSuccess;
  std::call_once(once[device_slot()], [&] {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<HD>::SMEM_BYTES);
  });
  if (e != cudaSuccess) return cuda_status(e, "text attention set smem attribute");
  kern<<<(unsigned)ctas, NUM_THREADS, Cfg<HD>::SMEM_BYTES, st>>>(qm, km, vm, p);
  int rc = launch_status("text_attention_kernel launch");
  if (rc || p.splits == 1) return rc;
  const long long threads = (long long)p.total_q * p.n_heads * (HD / 8);
  text_combine_kernel<HD, kBF16><<<(unsigned)((threads + 255) / 256), 256, 0, st>>>(
      p.part_o, p.part_lse, p.splits, p.total_q, p.n_heads, static_cast<uint16_t*>(p.out), p.out_token,
      p.out_head);
  return launch_status("text_combine_kernel launch");
}

template <bool kPaged>
int dispatch(const TextAttention& a, const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm,
             const Params& p, long long ctas, cudaStream_t st) {
  if (a.head_dim == 128)
    return a.bf16 ? launch<128, true, kPaged>(qm, km, vm, p, ctas, st)
                  : launch<128, false, kPaged>(qm, km, vm, p, ctas, st);
  return a.bf16 ? launch<64, true, kPaged>(qm, km, vm, p, ctas, st)
                : launch<64, false, kPaged>(qm, km, vm, p, ctas, st);
}

}  // namespace text

int launch_text_attention(const TextAttention& a, cudaStream_t st) {
  using namespace text;
  if (a.total_q == 0 || a.n_seqs == 0) return 0;
  if (a.n_seqs > kMaxSeqs) return fail(-2, "text attention: more than 8192 sequences in one call");
  const int group = a.n_heads / a.n_kv;
  Params p{};
  p.cu = a.cu;
  p.ctx = a.ctx;
  p.table = a.table;
  p.table_ld = a.table_ld;
  p.table_width = a.table_width;
  p.page_shift = a.page_shift;
  p.n_pages = a.n_pages;
  p.n_seqs = a.n_seqs;
  p.total_q = a.total_q;
  p.n_heads = a.n_heads;
  p.n_kv = a.n_kv;
  p.group = group;
  p.tile_tokens = BQ / group;
  p.causal = a.causal;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.out = a.out.data;
  p.out_token = a.out.token;
  p.out_head = a.out.head;
  p.v = a.v.data;
  p.v_page = a.v.page;
  p.v_token = a.v.token;
  p.v_head = a.v.head;
  p.err = device_error_word();
  const bool paged = a.table != nullptr;

  CUtensorMap qm, km, vm;
  {
    const long long dims[3] = {a.head_dim, a.n_heads, a.total_q}, str[2] = {a.q.head, a.q.token};
    const int box[3] = {64, group, p.tile_tokens};
    int rc = encode(&qm, a.q.data, a.bf16, 3, dims, str, box);
    if (rc) return rc;
  }
  for (int i = 0; i < 2; ++i) {
    const TextTensor& t = i ? a.v : a.k;
    CUtensorMap* m = i ? &vm : &km;
    int rc;
    if (paged) {
      const long long dims[4] = {a.head_dim, a.n_kv, 1ll << a.page_shift, a.n_pages};
      const long long str[3] = {t.head, t.token, t.page};
      const int box[4] = {64, 1, std::min(BKV, 1 << a.page_shift), 1};
      rc = encode(m, t.data, a.bf16, 4, dims, str, box);
    } else {
      const long long dims[3] = {a.head_dim, a.n_kv, a.total_q}, str[2] = {t.head, t.token};
      const int box[3] = {64, 1, BKV};
      rc = encode(m, t.data, a.bf16, 3, dims, str, box);
    }
    if (rc) return rc;
  }

  // Tiles: sum_i ceil(q_len_i / T) <= (total + n * (T - 1)) / T; CTAs past the
  // real number of tiles end at once.
  const long long T = p.tile_tokens;
  const long long seqs = std::min<long long>(a.n_seqs, a.total_q);
  const long long units = ((a.total_q + seqs * (T - 1)) / T) * a.n_kv;
  // Key split: where the units leave CTA slots (two per SM) empty, each
  // unit's keys are cut into ranges of at least 4 blocks.
  const long long slots = 2ll * num_sms();
  const long long blocks = ((long long)a.max_ctx + BKV - 1) / BKV;
  long long splits = paged ? std::min(slots / units, blocks / 4) : 1;
  p.splits = (int)std::max(1ll, std::min(splits, 64ll));
  const long long ctas = units * p.splits;
  if (ctas > 0x7fffffffll) return fail(-2, "text attention: too many tiles in one call");

  void* part = nullptr;
  if (p.splits > 1) {
    const size_t items = (size_t)p.splits * a.total_q * a.n_heads;
    const int rc = scratch_alloc(&part, items * (a.head_dim + 1) * sizeof(float), "text attention", st);
    if (rc) return rc;
    p.part_o = static_cast<float*>(part);
    p.part_lse = p.part_o + items * a.head_dim;
  }
  const int rc = paged ? dispatch<true>(a, qm, km, vm, p, ctas, st) : dispatch<false>(a, qm, km, vm, p, ctas, st);
  scratch_free(part, st);
  return rc;
}

int launch_paged_append(const TextTensor& k, const TextTensor& v, const TextTensor& kc, const TextTensor& vc,
                        const int* table, long long table_ld, int table_width, int page_shift, int n_pages,
                        const int* cu, const int* ctx, int n_seqs, int total, int n_kv, int head_dim,
                        cudaStream_t st) {
  if (total == 0 || n_seqs == 0) return 0;
  const long long threads = (long long)total * n_kv * (head_dim / 8);
  const long long blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffffll) return fail(-2, "paged_append: too many values in one call");
  text::paged_append_kernel<<<(unsigned)blocks, 256, 0, st>>>(
      static_cast<const uint16_t*>(k.data), static_cast<const uint16_t*>(v.data), k.token, k.head, v.token,
      v.head, static_cast<uint16_t*>(kc.data), static_cast<uint16_t*>(vc.data), kc.page, kc.token, kc.head,
      vc.page, vc.token, vc.head, n_pages, page_shift, table, table_ld, table_width, cu, ctx, n_seqs, total,
      n_kv, head_dim);
  return launch_status("paged_append_kernel launch");
}

}  // namespace bonsai
