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
// A unit of work = one sequence x one key/value head x one tile of 128 query
// rows, where a row is a (token, head of the group) pair: row r is token r / G,
// head r % G.  Taking the group's heads into the rows reads every key once for
// G heads, makes the causal triangle's diagonal G times narrower, and lets a
// single token fill G rows.  Two persistent CTAs share an SM (one's softmax runs
// beside the other's products and loads); each walks through its units, longest
// first over the whole launch, with the next unit's loads and first products
// under way while the last one's rows are written.
//   warps 0-3   softmax: thread i owns row i (TMEM lane i).  Online softmax
//               in the log2 domain; the running max moves (and O in TMEM is
//               rescaled) only when a block's max exceeds it by more than 8.
//               Warps without a row (a single token has G rows) only pass on.
//   warp 4      issues tcgen05.mma: S(j) = Q K_j^T (SMEM, SMEM),
//               O += P(j) V_j (P from TMEM, V MN-major); S runs two blocks
//               ahead (double-buffered).
//   warp 5      TMA: Q, then K and V blocks of 64 keys (128-byte swizzle,
//               64-dim halves); paged: one box per page and half, issued by
//               one lane each, page indices read 32 at a time.
//   warp 6      blocks that not every row sees whole (a causal diagonal, the
//               end of a sequence inside a block or page): V rows past the
//               sequence's end are zeroed in shared memory before the
//               product, since 0 * NaN would reach every row; V values of
//               keys that only some rows see are zeroed where they are not
//               finite, and the rows that do see them add them at the end.
//               It also finds the units, two ahead.
// Where the units leave CTA slots empty (a few single tokens), each unit's keys
// are split between the CTAs of a cluster, which merge their parts through
// distributed shared memory; a split wider than a cluster goes through global
// memory and a second kernel.
// TMEM (256 columns): S(even) [0, 64) S(odd) [64, 128) O [128, 128 + HD);
// P(j) (16-bit pairs) overwrites the first 32 columns of its S.
//
// Bounds and measurements (B200, 32 / 8 heads of 128, bf16 unless noted; a call
// among others, over several boxes): single tokens by HBM, 4.9-5.1 TB/s for 64
// sequences of 130 to 4000 keys (102-107 us) and 5.4-5.7 TB/s for 4 of 30000 to
// 65536 in f16 (149-158 us); long prompts by the 64-key Q K^T, whose 192 bytes of shared memory per clock are
// more than an SM reads, and by the power limit: 10007 tokens 843-853 us, 962-973
// TFLOP/s; batches of short prompts by the start and end of each unit: 48 of 7
// to 512 tokens 100 us.  128 rows per CTA, two CTAs per SM, because 256 rows
// per CTA (half the reads of K and V) measured the same on long prompts (778
// to 838 us against 760 to 804) and 10 to 20 % slower on batches of short
// ones: 8 x 150 tokens 19.7 against 16.5 us, 48 x 80 40.5 against 33.9.
#include "internal.cuh"
#include "ptx.cuh"

#include <cudaTypedefs.h>

#include <algorithm>

namespace bonsai {
namespace gemm {
PFN_cuTensorMapEncodeTiled_v12000 get_encode_fn();
}
namespace text {

constexpr int BQ = 128;   // query rows per tile
constexpr int BKV = 64;   // keys per block
constexpr int RING = 2;   // K and V slots
constexpr int WARP_MMA = 4, WARP_TMA = 5, WARP_FIX = 6;
constexpr int NUM_THREADS = 224;
constexpr int TMEM_COLS = 256;  // S(even), S(odd) of 64 columns each, O from 128 on
constexpr int O_COL = 128;
constexpr int BAR_BYTES = 512;
constexpr int EC = 32;    // columns that the epilogue takes at a time through a warp's staging rows
constexpr float kRescaleThreshold = 8.0f;
// P is 2^(s - m + kLift): an f16 P reaches 2^15 then, with the threshold, and is
// zero below 2^-32 of the row's maximum, not 2^-25 (65536 keys of 2^-25.4 beside
// one of 1 are 0.15 % of the sum).  The factor is in the row's sum too, and the
// same in every part of a split.
template <bool kBF16>
constexpr float kLift = kBF16 ? 0.0f : 7.0f;
constexpr int kMaxSeqs = 256;     // sequences of one launch (16 bytes each in shared memory)
constexpr int kMaxCluster = 16;   // CTAs that split a unit's keys and merge in shared memory

template <int HD>
struct Cfg {
  static constexpr int HALVES = HD / 64;
  static constexpr int Q_HALF = BQ * 128;         // 128 rows x 64 dims
  static constexpr int Q_BYTES = HALVES * Q_HALF;
  static constexpr int KV_HALF = BKV * 128;
  static constexpr int KV_BYTES = HALVES * KV_HALF;
  // Q and the rings; once a unit's products are done they can hold its O (f32)
  static constexpr int TILES_BYTES = Q_BYTES + 2 * RING * KV_BYTES;
  static_assert(TILES_BYTES >= BQ * HD * 4, "O does not fit the tiles");
  // As much for 64 dims as for 128: a CTA takes half of the tensor memory, and
  // so no less of the shared memory than that leaves to others (see TmemShare).
  static constexpr int SMEM_BYTES = 1024 + 2 * Q_HALF + 2 * RING * 2 * KV_HALF + BAR_BYTES + BQ * 8 + kMaxSeqs * 16 +
                                    4 * 32 * EC * 2;
  static_assert(SMEM_BYTES >= 1024 + TILES_BYTES + BAR_BYTES + BQ * 8 + kMaxSeqs * 16 + 4 * 32 * EC * 2, "layout");
};
static_assert(2 * (Cfg<128>::SMEM_BYTES + kSmemReserved) <= kSmemPerSm, "two CTAs per SM");

struct Params {
  const int* cu;        // [n_seqs + 1] first query row of each sequence
  const int* ctx;       // [n_seqs] keys of each sequence (null: its query rows)
  const int* table;     // [n_seqs][table_ld] page indices (paged)
  long long table_ld;
  int table_width, page_shift, n_pages;
  int n_seqs, total_q, n_heads, n_kv, group, tile_tokens;
  int causal, splits;
  int in_cluster;       // the splits of a unit are one cluster
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
// Non-zero where one of eight values has an exponent of all ones: adding one to
// the exponent field carries into the sign's place then, and nowhere else.
template <bool kBF16>
__device__ __forceinline__ uint32_t nonfinite_bits(uint4 v) {
  constexpr uint32_t e = kBF16 ? 0x7f807f80u : 0x7c007c00u, one = kBF16 ? 0x00800080u : 0x04000400u;
  return (((v.x & e) + one) | ((v.y & e) + one) | ((v.z & e) + one) | ((v.w & e) + one)) & 0x80008000u;
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

// Packed pairs of f32 in one 64-bit register.
__device__ __forceinline__ unsigned long long pack2(float a, float b) {
  unsigned long long d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void unpack2(unsigned long long v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b,
                                                   unsigned long long c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3f(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// What the roles of a CTA need to know of a unit (64 bytes in shared memory).
struct Unit {
  int seq, kvh, q_begin, t0, n_tok;  // tokens t0 .. t0 + n_tok of the sequence
  int first;                         // place of token t0 in the sequence
  int kv_len, lim_min;               // keys; keys that the first token sees
  int j0, nkv;                       // key blocks [j0, j0 + nkv) (nkv < 0: no more units)
  int jb;                            // blocks from jb on hold a key that some row does not see
  int pad[5];
};
static_assert(sizeof(Unit) == 64, "read as four int4");

// Keys [0, n) that token `tok` of a tile sees.
__device__ __forceinline__ int keys_seen(const Unit& u, int causal, int tok) {
  return causal ? max(0, min(u.kv_len, u.first + tok + 1)) : u.kv_len;
}

// What the search for units keeps of a sequence (shared memory).
struct Seq {
  int q_len, before;  // query tokens, keys before them
  int kv_len, tiles;  // keys, query tiles
};
static_assert(sizeof(Seq) == 16, "read as one int4");

// The order of a launch's query tiles: by their key blocks, most first (ties:
// by sequence, then latest tokens first), so that the long ones do not end up
// alone at the end.  One warp, for every unit again, so what it does per
// sequence is kept small: lengths and tile counts are computed once per launch
// (divided out at every look instead, 256 single tokens over 100-900 keys took
// 166 us, not 117, and 250 prompts of 40 tokens 78, not 66), and a launch takes
// at most 256 sequences (with 512, before that, 512 single tokens took 377 us
// against 328, 500 prompts of 40 tokens 177 against 152).
struct Finder {
  const Seq* seqs;
  int n, tile_tokens, causal;
  int c, at_c, above_c;  // tiles of >= c blocks, of > c blocks

  __device__ Seq seq(int i) const {
    Seq s;
    *reinterpret_cast<int4*>(&s) = *reinterpret_cast<const int4*>(seqs + i);
    return s;
  }
  // Tiles of a sequence with at least `blocks` key blocks: the last ones.
  __device__ int tiles(const Seq& s, int blocks) const {
    const int keys = (blocks - 1) * BKV + 1;  // blocks <= 0: any tile
    if (s.kv_len < keys) return blocks > 0 ? 0 : s.tiles;
    if (!causal || s.tiles <= 1 || blocks <= 0) return s.tiles;
    const int toks = keys - s.before;  // tokens up to the first that sees as many
    return toks <= tile_tokens ? s.tiles : s.tiles - ((toks + tile_tokens - 1) / tile_tokens - 1);
  }
  __device__ int total(int blocks) const {
    int v = 0;
    for (int i = (int)lane_id(); i < n; i += 32) v += tiles(seq(i), blocks);
    return __reduce_add_sync(0xffffffffu, v);
  }
  __device__ void init() {
    int most = 0;
    for (int i = (int)lane_id(); i < n; i += 32) most = max(most, seqs[i].kv_len);
    c = (__reduce_max_sync(0xffffffffu, most) + BKV - 1) / BKV + 1;
    at_c = above_c = 0;
  }
  // Tile b (b never falls from call to call): its sequence and its place among
  // the sequence's tiles; false where there are at most b tiles.
  __device__ bool find(int b, int& at, int& level) {
    if (b >= at_c) {
      if (c == 0 || total(0) <= b) return false;
      int lo = 0, hi = c;  // total(lo) = n_lo > b >= n_hi = total(hi)
      int n_lo = -1, n_hi = at_c;
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2, v = total(mid);
        if (v > b) {
          lo = mid;
          n_lo = v;
        } else {
          hi = mid;
          n_hi = v;
        }
      }
      c = lo;
      at_c = n_lo >= 0 ? n_lo : total(lo);
      above_c = n_hi;
    }
    int rank = b - above_c;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + (int)lane_id();
      int more = 0, e = 0, all = 0;
      if (i < n) {
        const Seq s = seq(i);
        more = tiles(s, c + 1);
        e = tiles(s, c) - more;
        all = s.tiles;
      }
      const int here = __reduce_add_sync(0xffffffffu, e);
      if (rank >= here) {
        rank -= here;
        continue;
      }
      int incl = e;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if ((int)lane_id() >= o) incl += v;
      }
      const int l = __ffs(__ballot_sync(0xffffffffu, incl > rank)) - 1;
      at = i0 + l;
      level = __shfl_sync(0xffffffffu, all - 1 - more + incl - e, l) - rank;
      return true;
    }
    return false;
  }
};

// wait_bar for a phase that has usually completed already.
__device__ __forceinline__ bool wait_fast(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err,
                                          int code) {
  return bar_test_wait(smem_u32(bar), parity) || wait_bar(bar, parity, abort_flag, err, code);
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
  Unit* units = reinterpret_cast<Unit*>(vs + RING * C::KV_BYTES);  // [2]
  uint64_t* unit_full = reinterpret_cast<uint64_t*>(units + 2);
  uint64_t* unit_empty = unit_full + 2;
  uint64_t* q_full = unit_empty + 2;
  uint64_t* q_empty = q_full + 1;
  uint64_t* k_full = q_empty + 1;
  uint64_t* k_empty = k_full + RING;
  uint64_t* v_full = k_empty + RING;
  uint64_t* v_empty = v_full + RING;
  uint64_t* v_fixed = v_empty + RING;
  uint64_t* s_full = v_fixed + RING;
  uint64_t* p_ready = s_full + 2;
  uint64_t* pv_done = p_ready + 2;
  uint64_t* o_empty = pv_done + 2;
  uint64_t* drain = o_empty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* nonfinite = abort_flag + 1;  // [2] by unit
  float2* stats = reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(units) + BAR_BYTES);  // [BQ] log2 sum (cluster merge)
  Seq* seqs = reinterpret_cast<Seq*>(stats + BQ);  // [kMaxSeqs]
  uint4* stage = reinterpret_cast<uint4*>(seqs + kMaxSeqs);  // 32 rows of EC columns per softmax warp

  const int warp = threadIdx.x / 32;
  const int lane = (int)lane_id();
  const int split = (int)(blockIdx.x % (unsigned)p.splits);
  const int unit0 = (int)(blockIdx.x / (unsigned)p.splits);
  const int ustep = (int)(gridDim.x / (unsigned)p.splits);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      bar_init(&unit_full[i], 1);
      bar_init(&unit_empty[i], 6);  // softmax warps, MMA, TMA
      nonfinite[i] = 0;
      bar_init(&s_full[i], 1);
      bar_init(&p_ready[i], 4);
      bar_init(&pv_done[i], 1);
    }
    bar_init(q_full, 1);
    bar_init(q_empty, 1);
    for (int s = 0; s < RING; ++s) {
      bar_init(&k_full[s], 1);
      bar_init(&k_empty[s], 1);
      bar_init(&v_full[s], 1);
      bar_init(&v_empty[s], 1);
      bar_init(&v_fixed[s], 1);
    }
    bar_init(o_empty, 4);
    bar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&qmap);
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
  }
  if (warp == WARP_MMA) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  griddep_wait();
  for (int i = threadIdx.x; i < p.n_seqs; i += NUM_THREADS) {
    const int a = max(0, min(p.cu[i], p.total_q)), b = max(a, min(p.cu[i + 1], p.total_q));
    Seq s;
    s.q_len = b - a;
    s.kv_len = b - a;
    s.before = 0;
    if constexpr (kPaged) {  // a length past the table is cut to it
      const int ctx = max(0, p.ctx[i]);
      s.kv_len = (int)min((long long)ctx, (long long)p.table_width << p.page_shift);
      s.before = ctx - s.q_len;
    }
    s.tiles = (s.q_len + p.tile_tokens - 1) / p.tile_tokens;
    *reinterpret_cast<int4*>(seqs + i) = *reinterpret_cast<const int4*>(&s);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_launch();  // after the TMEM allocation: a dependent's could block it, and waits for this grid
  const uint32_t tmem = *tmem_slot;

  // Unit i of this CTA, as every role gets it.
  auto next_unit = [&](int i, Unit& u) -> bool {
    const bool good = wait_bar(&unit_full[i & 1], (i >> 1) & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_PRODUCER);
    if (!good) return false;
    const int4* src = reinterpret_cast<const int4*>(&units[i & 1]);
    int4* dst = reinterpret_cast<int4*>(&u);
#pragma unroll
    for (int k = 0; k < 4; ++k) dst[k] = src[k];
    return u.nkv >= 0;
  };

  if (warp == WARP_TMA) {
    // Paged: a block of 64 keys takes 64 / page boxes (one where a page holds
    // more), and each half of the head dims its own; lane l issues box
    // l / HALVES, half l % HALVES.
    const int box_shift = min(p.page_shift, 6);
    const int box = lane / C::HALVES, half = lane % C::HALVES;
    const bool issues = kPaged ? box < (BKV >> box_shift) : lane < C::HALVES;
    uint32_t kn = 0, vn = 0, qn = 0;  // loads so far
    bool ok = true;
    Unit u;
    for (int i = 0; ok; ++i) {
      if (!__all_sync(0xffffffffu, next_unit(i, u))) break;
      if (lane == 0) bar_arrive(&unit_empty[i & 1]);
      if (u.nkv == 0) continue;
      // 32 page indices each for K and V, which runs behind
      int ent_k = -1, base_k = -1, ent_v = -1, base_v = -1;
      auto load = [&](const void* map, uint8_t* ring, uint64_t* full, uint64_t* empty, uint32_t depth, uint32_t& cnt,
                      int& ent, int& ent_base, int j) -> bool {
        const uint32_t s = cnt % depth;
        const int key0 = (u.j0 + j) * BKV;
        int page = 0;
        if constexpr (kPaged) {
          const int want = (key0 >> p.page_shift) & ~31;
          if (want != ent_base) {  // 64 keys never reach past 32 pages (page >= 8)
            ent_base = want;
            ent = want + lane < p.table_width ? p.table[(size_t)u.seq * p.table_ld + want + lane] : -1;
          }
          page = __shfl_sync(0xffffffffu, ent, (((key0 + (box << box_shift)) >> p.page_shift) - ent_base) & 31);
        }
        const bool good = wait_bar(&empty[s], ((cnt / depth) & 1) ^ 1, abort_flag, p.err, DEV_ERR_TIMEOUT_TMA);
        if (!__all_sync(0xffffffffu, good)) return false;
        if (lane == 0) bar_arrive_expect_tx(&full[s], C::KV_BYTES);
        __syncwarp();
        if (issues) {
          uint8_t* d = ring + s * C::KV_BYTES + half * C::KV_HALF;
          if constexpr (kPaged)
            tma_load_4d(d + (box << box_shift) * 128, map, &full[s], half * 64, u.kvh,
                        (key0 + (box << box_shift)) & ((1 << p.page_shift) - 1), page);
          else
            tma_load_3d(d, map, &full[s], half * 64, u.kvh, u.q_begin + key0);
        }
        ++cnt;
        return true;
      };
      const bool good = wait_bar(q_empty, (qn & 1) ^ 1, abort_flag, p.err, DEV_ERR_TIMEOUT_TMA);
      ok = __all_sync(0xffffffffu, good);
      if (!ok) break;
      if (lane == 0) {
        bar_arrive_expect_tx(q_full, (uint32_t)(p.group * p.tile_tokens * HD * 2));
        for (int h = 0; h < C::HALVES; ++h)
          tma_load_3d(qs + h * C::Q_HALF, &qmap, q_full, h * 64, u.kvh * p.group, u.q_begin + u.t0);
      }
      __syncwarp();
      ++qn;
      // K runs two blocks ahead of V, as S does of P V: each load is asked for
      // as soon as its slot is free, two blocks' time before it is needed.
      ok = load(&kmap, ks, k_full, k_empty, RING, kn, ent_k, base_k, 0) && (u.nkv == 1 || load(&kmap, ks, k_full, k_empty, RING, kn, ent_k, base_k, 1));
      for (int j = 0; j < u.nkv && ok; ++j) {
        ok = load(&vmap, vs, v_full, v_empty, RING, vn, ent_v, base_v, j);
        if (ok && j + 2 < u.nkv) ok = load(&kmap, ks, k_full, k_empty, RING, kn, ent_k, base_k, j + 2);
      }
    }
    if (*abort_flag) {  // let copies in flight land before the shared memory is released
      const unsigned long long w0 = globaltimer_ns();
      while (globaltimer_ns() - w0 < 1000000ull) {
      }
    }
  } else if (warp == WARP_MMA) {
    // The whole warp runs this role, one thread of it issues: see mma_ss_if.
    constexpr uint32_t idesc_s = make_idesc_f16(BQ, BKV, kBF16 ? 1 : 0, 0, 0);
    constexpr uint32_t idesc_o = make_idesc_f16(BQ, HD, kBF16 ? 1 : 0, 0, 1);
    const uint32_t leader = elect_one() ? 1u : 0u;
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t q_desc = make_smem_desc(smem_u32(qs), 16, 1024);
    const uint64_t k_desc = make_smem_desc(smem_u32(ks), 16, 1024);
    const uint64_t v_desc = make_smem_desc(smem_u32(vs), C::KV_HALF, 1024);
    uint32_t nb = 0, un = 0;  // blocks and units so far
    auto wait_all = [&](uint64_t* bar, uint32_t parity) -> bool {
      return __all_sync(0xffffffffu, wait_fast(bar, parity, abort_flag, p.err, DEV_ERR_TIMEOUT_MMA));
    };
    auto issue_s = [&](int j) -> bool {
      const uint32_t n = nb + j, s = n % RING, b = n & 1;
      if (!wait_all(&k_full[s], (n / RING) & 1)) return false;
      tc_fence_after();
#pragma unroll
      for (int k16 = 0; k16 < HD / 16; ++k16)  // descriptors count 16 bytes
        mma_ss_if(leader, tm + b * BKV,
                  q_desc + (uint64_t)(((k16 >> 2) * C::Q_HALF + (k16 & 3) * 32) >> 4),
                  k_desc + (uint64_t)(s * (C::KV_BYTES >> 4) + (((k16 >> 2) * C::KV_HALF + (k16 & 3) * 32) >> 4)),
                  idesc_s, k16 > 0 ? 1u : 0u);
      tc_commit_if(leader, &s_full[b]);
      tc_commit_if(leader, &k_empty[s]);
      return true;
    };
    // P V first, then S: its V slot is free while K may still be on its way
    // (the other way around 118 us instead of 111, 64 sequences of 130 to 4000
    // keys, one token each).
    auto issue_pv = [&](int j) -> bool {
      const uint32_t n = nb + j, s = n % RING, b = n & 1;
      // v_fixed: the fix warp has seen the block's copy complete
      if (!wait_all(&v_fixed[s], (n / RING) & 1) || !wait_all(&p_ready[b], (n >> 1) & 1)) return false;
      tc_fence_after();
#pragma unroll
      for (int k16 = 0; k16 < BKV / 16; ++k16)
        mma_ts_if(leader, tm + O_COL, tm + b * BKV + k16 * 8,
                  v_desc + (uint64_t)(s * (C::KV_BYTES >> 4) + k16 * (16 * 128 >> 4)), idesc_o,
                  (j > 0 || k16 > 0) ? 1u : 0u);
      tc_commit_if(leader, &pv_done[b]);
      tc_commit_if(leader, &v_empty[s]);
      return true;
    };
    Unit u;
    bool ok = true;
    for (int i = 0; ok; ++i) {
      if (!__all_sync(0xffffffffu, next_unit(i, u))) break;
      if (leader) bar_arrive(&unit_empty[i & 1]);
      const int nkv = __shfl_sync(0xffffffffu, u.nkv, 0);
      if (nkv == 0) continue;
      ok = wait_all(q_full, un & 1);
      for (int j = 0; j < min(nkv, 2) && ok; ++j) ok = issue_s(j);
      if (ok && nkv <= 2) tc_commit_if(leader, q_empty);
      // the rows of the unit before have been read out of O
      if (ok) ok = wait_all(o_empty, (un & 1) ^ 1);
      for (int j = 0; j < nkv && ok; ++j) {
        ok = issue_pv(j);
        if (ok && j + 2 < nkv) ok = issue_s(j + 2);
        if (ok && j + 3 == nkv) tc_commit_if(leader, q_empty);
      }
      nb += (uint32_t)nkv;
      ++un;
    }
    tc_commit_if(leader, drain);
    const uint32_t da = smem_u32(drain);
    const unsigned long long w0 = globaltimer_ns();
    while (!bar_try_wait(da, 0)) {
      if (globaltimer_ns() - w0 > kWaitLimitNs) {
        if (p.err) atomicCAS(p.err, 0, DEV_ERR_TIMEOUT_MMA);
        break;
      }
    }
    __syncwarp();
  } else if (warp == WARP_FIX) {
    // The units: two are out at a time, the next one is found and put in the
    // place of one that every role has left.
    Finder f{seqs, p.n_seqs, p.tile_tokens, p.causal};
    f.init();
    auto publish = [&](int i, Unit& u) -> bool {
      // units come longest first: rounds go up and down the CTAs in turn, so
      // that who had the longest of one round has the shortest of the next
      const int unit = i * ustep + (i & 1 ? ustep - 1 - unit0 : unit0);
      u = Unit{};
      u.nkv = -1;
      int seq, level;
      // with splits, one unit per CTA (per cluster)
      if ((p.splits == 1 || i == 0) && f.find(unit / p.n_kv, seq, level)) {
        const Seq s = f.seq(seq);
        u.seq = seq;
        u.kvh = unit % p.n_kv;
        u.q_begin = max(0, min(p.cu[seq], p.total_q));
        u.kv_len = s.kv_len;
        u.t0 = level * p.tile_tokens;
        u.n_tok = min(p.tile_tokens, s.q_len - u.t0);
        u.first = s.before + u.t0;
        u.lim_min = keys_seen(u, p.causal, 0);
        const int blocks = (keys_seen(u, p.causal, u.n_tok - 1) + BKV - 1) / BKV;
        const int chunk = (blocks + p.splits - 1) / p.splits;
        u.j0 = split * chunk;
        u.nkv = max(0, min(blocks - u.j0, chunk));
        u.jb = max(0, u.lim_min / BKV - u.j0);
      }
      const bool good = wait_bar(&unit_empty[i & 1], ((i >> 1) & 1) ^ 1, abort_flag, p.err, DEV_ERR_TIMEOUT_PRODUCER);
      if (!__all_sync(0xffffffffu, good)) return false;
      if (lane == 0) {
        units[i & 1] = u;
        nonfinite[i & 1] = 0;  // the softmax warps are done with unit i - 2
        bar_arrive(&unit_full[i & 1]);
      }
      __syncwarp();
      return true;
    };
    uint32_t vn = 0;
    Unit u, after;
    bool ok = publish(0, u);
    after.nkv = -1;
    if (ok && u.nkv >= 0) ok = publish(1, after);
    for (int i = 0; ok && u.nkv >= 0; ++i) {
      // Every block passes here, so that the warp follows each phase of the
      // ring; those before jb pass untouched.
      for (int j = 0; j < u.nkv; ++j, ++vn) {
        const uint32_t s = vn % RING;
        const bool good = wait_bar(&v_full[s], (vn / RING) & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_PRODUCER);
        ok = __all_sync(0xffffffffu, good);
        if (!ok) break;
        if (j >= u.jb) {
          const int key0 = (u.j0 + j) * BKV;
          // Rows from r0 on (the swizzle permutes 16-byte pieces within a
          // 128-byte row only): to r1 they are checked, past it zeroed.
          const int r0 = max(0, u.lim_min - key0), r1 = max(r0, min(BKV, u.kv_len - key0));
          uint8_t* at = vs + s * C::KV_BYTES;
          uint32_t bad = 0;
          for (int h = 0; h < C::HALVES; ++h) {
#pragma unroll 4
            for (int e = r0 * 8 + lane; e < r1 * 8; e += 32)
              bad |= nonfinite_bits<kBF16>(*reinterpret_cast<const uint4*>(at + h * C::KV_HALF + e * 16));
            for (int e = r1 * 8 + lane; e < BKV * 8; e += 32)
              *reinterpret_cast<uint4*>(at + h * C::KV_HALF + e * 16) = make_uint4(0, 0, 0, 0);
          }
          if (__any_sync(0xffffffffu, bad != 0)) {
            for (int h = 0; h < C::HALVES; ++h)
              for (int e = r0 * 8 + lane; e < r1 * 8; e += 32) {
                uint4* q4 = reinterpret_cast<uint4*>(at + h * C::KV_HALF + e * 16);
                uint32_t w[4] = {q4->x, q4->y, q4->z, q4->w};
#pragma unroll
                for (int m = 0; m < 4; ++m)
                  w[m] &= (finite16<kBF16>(w[m]) ? 0x0000ffffu : 0u) | (finite16<kBF16>(w[m] >> 16) ? 0xffff0000u : 0u);
                *q4 = make_uint4(w[0], w[1], w[2], w[3]);
              }
            if (lane == 0) nonfinite[i & 1] = 1;
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) bar_arrive(&v_fixed[s]);
      }
      u = after;
      if (ok && after.nkv >= 0) ok = publish(i + 2, after);
    }
  } else {
    const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
    const uint32_t o_addr = tmem + lane_base + O_COL;
    const int row = warp * 32 + lane;
    const int tok = row / p.group;
    const unsigned long long sc2 = pack2(p.scale_log2, p.scale_log2);
    uint32_t gn = 0;  // blocks so far
    Unit u;
    bool ok = true;
    for (int i = 0; ok; ++i) {
      if (!__all_sync(0xffffffffu, next_unit(i, u))) break;
      const bool valid = tok < u.n_tok && row < p.tile_tokens * p.group;
      const bool any = __any_sync(0xffffffffu, valid);
      const int head = u.kvh * p.group + row - tok * p.group;
      const size_t q_row = (size_t)(u.q_begin + u.t0 + tok);
      uint16_t* dst = reinterpret_cast<uint16_t*>(p.out) + q_row * p.out_token + (size_t)head * p.out_head;
      const size_t part = ((size_t)split * p.total_q + q_row) * p.n_heads + head;
      if (u.nkv == 0) {  // no key: zeros (or a part of weight zero)
        if (p.in_cluster) {
          if (valid) stats[row] = make_float2(-INFINITY, 0.f);
        } else if (valid && p.splits > 1) {
          p.part_lse[part] = -INFINITY;
        } else if (valid) {
          for (int k = 0; k < HD / 8; ++k) reinterpret_cast<uint4*>(dst)[k] = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
        if (lane == 0) bar_arrive(&unit_empty[i & 1]);
        continue;
      }
      const int lim = valid ? keys_seen(u, p.causal, tok) : 0;
      float m = -INFINITY, l = 0.0f;
      for (int j = 0; j < u.nkv; ++j, ++gn) {
        const uint32_t buf = gn & 1;
        const uint32_t s_addr = tmem + lane_base + buf * BKV;
        bool good = wait_fast(&s_full[buf], (gn >> 1) & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_SOFTMAX);
        ok = __all_sync(0xffffffffu, good);
        if (!ok) break;
        if (!any) {  // no row here: P of these rows is never read out
          if (lane == 0) bar_arrive(&p_ready[buf]);
          continue;
        }
        tc_fence_after();
        float s[BKV];
        {
          uint32_t r0[32], r1[32];
          tmem_ld32(s_addr, r0);
          tmem_ld32(s_addr + 32, r1);
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            s[k] = __uint_as_float(r0[k]);
            s[32 + k] = __uint_as_float(r1[k]);
          }
        }
        if (j >= u.jb) {  // a key past the row's limit: whatever it gave, it counts nothing
          const int left = lim - (u.j0 + j) * BKV;
#pragma unroll
          for (int c = 0; c < BKV; ++c)
            if (c >= left) s[c] = -INFINITY;
        }
        float m8[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) m8[k] = fmaxf(s[k], s[8 + k]);
#pragma unroll
        for (int c = 16; c < BKV; c += 16) {
#pragma unroll
          for (int k = 0; k < 8; ++k) m8[k] = max3f(m8[k], s[c + k], s[c + 8 + k]);
        }
        const float mx = max3f(max3f(m8[0], m8[1], m8[2]), max3f(m8[3], m8[4], m8[5]), fmaxf(m8[6], m8[7])) *
                         p.scale_log2;
        float alpha = 1.0f;
        if (mx > m + kRescaleThreshold) {
          alpha = ex2(m - mx);
          m = mx;
        }
        if (j > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
          good = wait_bar(&pv_done[buf ^ 1], ((gn - 1) >> 1) & 1, abort_flag, p.err, DEV_ERR_TIMEOUT_SOFTMAX);
          ok = __all_sync(0xffffffffu, good);
          if (!ok) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t r[32];
            tmem_ld32(o_addr + c * 32, r);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * alpha);
            tmem_st32(o_addr + c * 32, r);
          }
        }
        // no key seen yet: every p is 2^-inf = 0
        const float mref = (m == -INFINITY ? 0.0f : m) - kLift<kBF16>;
        const unsigned long long nm2 = pack2(-mref, -mref);
        unsigned long long sum2[4] = {0ull, 0ull, 0ull, 0ull};
        // P, and its row sum before the rounding
#pragma unroll
        for (int ch = 0; ch < BKV / 32; ++ch) {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float a, b;
            unpack2(fma2(pack2(s[ch * 32 + 2 * k], s[ch * 32 + 2 * k + 1]), sc2, nm2), a, b);
            a = ex2(a);
            b = ex2(b);
            sum2[k & 3] = add2(sum2[k & 3], pack2(a, b));
            pk[k] = cvt2<kBF16>(a, b);
          }
          tmem_st16(s_addr + ch * 16, pk);
        }
        float a0, a1;
        unpack2(add2(add2(sum2[0], sum2[1]), add2(sum2[2], sum2[3])), a0, a1);
        l = l * alpha + (a0 + a1);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(&p_ready[buf]);
      }
      if (!ok) break;
      const bool good = !any || wait_bar(&pv_done[(gn - 1) & 1], ((gn - 1) >> 1) & 1, abort_flag, p.err,
                                         DEV_ERR_TIMEOUT_SOFTMAX);
      ok = __all_sync(0xffffffffu, good);
      if (!ok) break;
      if (any) {
        tc_fence_after();
        const float inv_l = l == 0.0f ? 0.0f : 1.0f / l;  // no key in this range: zeros
        const bool repair = nonfinite[i & 1] != 0 && valid;
        // keys that only some rows see, within this CTA's range
        const int from = max(u.lim_min, (u.j0 + u.jb) * BKV), to = min(lim, (u.j0 + u.nkv) * BKV);
        if (p.in_cluster && valid) stats[row] = make_float2(l == 0.0f ? -INFINITY : m + log2f(l), 0.f);
        constexpr int PIECES = EC / 8;  // 16-byte pieces of a staged row
        // where the rows that this lane helps to write begin (null: no row)
        uint16_t* rows_at[PIECES];
#pragma unroll
        for (int k = 0; k < PIECES; ++k)
          rows_at[k] = reinterpret_cast<uint16_t*>(__shfl_sync(
              0xffffffffu, valid ? reinterpret_cast<unsigned long long>(dst) : 0ull, (k * 32 + lane) / PIECES));
#pragma unroll 1
        for (int c = 0; c < HD; c += EC) {
          float o[EC];
#pragma unroll
          for (int h = 0; h < EC; h += 32) {
            uint32_t r[32];
            tmem_ld32(o_addr + c + h, r);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[h + k] = __uint_as_float(r[k]) * inv_l;
          }
          if (repair) {
            for (int key = from; key < to; ++key) {
              const uint16_t* src = static_cast<const uint16_t*>(p.v) + (size_t)u.kvh * p.v_head + c;
              if constexpr (kPaged) {
                const int page = p.table[(size_t)u.seq * p.table_ld + (key >> p.page_shift)];
                if (page < 0 || page >= p.n_pages) continue;
                src += (size_t)page * p.v_page + (size_t)(key & ((1 << p.page_shift) - 1)) * p.v_token;
              } else {
                src += (size_t)(u.q_begin + key) * p.v_token;
              }
#pragma unroll
              for (int k = 0; k < EC; ++k)
                if (!finite16<kBF16>(src[k])) o[k] += to_f32<kBF16>(src[k]);
            }
          }
          if (p.splits > 1) {
            // global memory, or this CTA's tiles (every product of the unit is
            // done); there, 16-byte pieces are permuted within a row against conflicts
            float* po = p.in_cluster ? reinterpret_cast<float*>(qs) + row * HD : p.part_o + part * HD;
            const int x = p.in_cluster ? row & 7 : 0;
#pragma unroll
            for (int k = 0; k < EC / 4; ++k)
              if (valid)
                *reinterpret_cast<float4*>(po + ((c / 4 + k) ^ x) * 4) =
                    make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
          } else {
            // Through shared memory, so that neighbouring lanes write
            // neighbouring pieces of a row (a lane writing its own row touches
            // 32 lines per instruction, and the SM takes about 3 clocks for
            // each); pieces are permuted against bank conflicts.
            auto place = [](int row, int piece) {
              return row * PIECES + (piece ^ ((row >> 1) & 3));
            };
            uint4* st = stage + warp * (32 * PIECES);
#pragma unroll
            for (int k = 0; k < PIECES; ++k)
              st[place(lane, k)] =
                  make_uint4(cvt2<kBF16>(o[8 * k], o[8 * k + 1]), cvt2<kBF16>(o[8 * k + 2], o[8 * k + 3]),
                             cvt2<kBF16>(o[8 * k + 4], o[8 * k + 5]), cvt2<kBF16>(o[8 * k + 6], o[8 * k + 7]));
            __syncwarp();
#pragma unroll
            for (int k = 0; k < PIECES; ++k) {
              const uint4 v = st[place((k * 32 + lane) / PIECES, lane % PIECES)];
              if (rows_at[k]) *reinterpret_cast<uint4*>(rows_at[k] + c + lane % PIECES * 8) = v;
            }
            __syncwarp();
          }
        }
        if (valid && p.splits > 1 && !p.in_cluster) p.part_lse[part] = l == 0.0f ? -INFINITY : m + log2f(l);
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) {
        bar_arrive(o_empty);
        bar_arrive(&unit_empty[i & 1]);
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (p.in_cluster) {
    // Merge: row r of the unit by CTA r % splits, HD / 8 threads per row, the
    // parts in the order of their keys.
    cluster_sync_all();
    const Unit& u = units[0];
    if (!*abort_flag && u.nkv >= 0) {
      const int rows = u.n_tok * p.group;
      const int d8 = (int)(threadIdx.x % (HD / 8)) * 2;  // 16-byte pieces d8, d8 + 1
      const uint32_t st0 = smem_u32(stats), o0 = smem_u32(qs);
      for (int r = split + p.splits * (int)(threadIdx.x / (HD / 8)); r < rows;
           r += p.splits * (NUM_THREADS / (HD / 8))) {
        float lse[kMaxCluster];
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < kMaxCluster; ++c)
          if (c < p.splits) {
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(lse[c]) : "r"(mapa_shared(st0 + r * 8u, c)) : "memory");
          }
#pragma unroll
        for (int c = 0; c < kMaxCluster; ++c)
          if (c < p.splits) top = lse[c] > top || lse[c] != lse[c] ? lse[c] : top;  // a NaN sum stays
        float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, total = 0.f;
#pragma unroll
        for (int c = 0; c < kMaxCluster; ++c) {
          if (c >= p.splits || lse[c] == -INFINITY) continue;
          const float w = exp2f(lse[c] - top);
          total += w;
          const uint32_t a = mapa_shared(o0 + (uint32_t)r * (HD * 4u), c);
          float v[8];
#pragma unroll
          for (int k = 0; k < 2; ++k)
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(v[4 * k]), "=f"(v[4 * k + 1]), "=f"(v[4 * k + 2]), "=f"(v[4 * k + 3])
                         : "r"(a + (uint32_t)((d8 + k) ^ (r & 7)) * 16u)
                         : "memory");
#pragma unroll
          for (int k = 0; k < 8; ++k) acc[k] = fmaf(w, v[k], acc[k]);
        }
        const float inv = total == 0.f ? 0.f : 1.0f / total;
        const int tk = r / p.group, head = u.kvh * p.group + r - tk * p.group;
        uint32_t h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = cvt2<kBF16>(acc[2 * k] * inv, acc[2 * k + 1] * inv);
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.out) + (size_t)(u.q_begin + u.t0 + tk) * p.out_token +
                                  (size_t)head * p.out_head + d8 * 4) = make_uint4(h[0], h[1], h[2], h[3]);
      }
    }
    cluster_sync_all();  // no CTA ends while another reads its shared memory
  }
  if (warp == WARP_MMA) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
}

// Merges the partial outputs of the key ranges of one (row, head) per block:
// with lse_s = log2 of range s's exponential sum, out = sum_s 2^(lse_s - top)
// O_s / sum_s 2^(lse_s - top).  A range without a key has lse -inf and is not
// read.  HD / 8 threads take a range's row, the block's groups of them every
// 256 / (HD / 8)-th range, so that the few rows of single tokens do not wait
// for one range after the other (one token over 30000 keys of 8 heads: 36 us against 51); the
// groups' sums meet in a fixed order.  Only the rows of this launch's own
// sequences have parts: the others (of another launch of the call, or of no
// sequence at all) are left alone.
constexpr int kMaxSplits = 64;
template <int HD, bool kBF16>
__global__ void __launch_bounds__(256) text_combine_kernel(const float* __restrict__ part_o,
                                                           const float* __restrict__ part_lse, int splits, int rows,
                                                           int n_heads, const int* __restrict__ cu, int n_seqs,
                                                           uint16_t* out, long long out_token, long long out_head) {
  constexpr int LANES = HD / 8, GROUPS = 256 / LANES;
  __shared__ float lse[kMaxSplits];
  __shared__ float sums[GROUPS][HD + 4];
  const size_t items = (size_t)rows * n_heads, it = blockIdx.x;
  const int grp = threadIdx.x / LANES, d = (threadIdx.x % LANES) * 8;
  griddep_wait();
  const int row = (int)(it / n_heads);
  if (row < cu[0] || row >= cu[n_seqs]) return;
  if (threadIdx.x < splits) lse[threadIdx.x] = __ldcg(part_lse + threadIdx.x * items + it);
  __syncthreads();
  float top = -INFINITY;
  for (int s = 0; s < splits; ++s) top = lse[s] > top || lse[s] != lse[s] ? lse[s] : top;  // a NaN sum stays
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = grp; s < splits; s += GROUPS) {
    if (lse[s] == -INFINITY) continue;
    const float w = exp2f(lse[s] - top);
    const float4* src = reinterpret_cast<const float4*>(part_o + (s * items + it) * HD + d);
    const float4 a = __ldcg(src), b = __ldcg(src + 1);
    acc[0] = fmaf(w, a.x, acc[0]);
    acc[1] = fmaf(w, a.y, acc[1]);
    acc[2] = fmaf(w, a.z, acc[2]);
    acc[3] = fmaf(w, a.w, acc[3]);
    acc[4] = fmaf(w, b.x, acc[4]);
    acc[5] = fmaf(w, b.y, acc[5]);
    acc[6] = fmaf(w, b.z, acc[6]);
    acc[7] = fmaf(w, b.w, acc[7]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[grp][d + i] = acc[i];
  __syncthreads();
  if (threadIdx.x < HD / 2) {
    float total = 0.f;
    for (int s = 0; s < splits; ++s) total += lse[s] == -INFINITY ? 0.f : exp2f(lse[s] - top);
    const float inv = total == 0.f ? 0.f : 1.0f / total;
    float x = 0.f, y = 0.f;
#pragma unroll
    for (int k = 0; k < GROUPS; ++k) {
      x += sums[k][2 * threadIdx.x];
      y += sums[k][2 * threadIdx.x + 1];
    }
    reinterpret_cast<uint32_t*>(out + (size_t)row * out_token + (it % n_heads) * out_head)[threadIdx.x] =
        cvt2<kBF16>(x * inv, y * inv);
  }
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
  if (t >= total) {
    griddep_wait();
    return;
  }
  const int piece = (int)(idx - t * pieces);
  griddep_wait();
  griddep_launch();
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

// Largest number of co-resident clusters of `size` CTAs (a cluster lies within
// one GPC).  The occupancy query counts one CTA per SM for a kernel that
// allocates TMEM; two of these fit (256 of the 512 columns, half the shared
// memory and registers each) and do run.
template <int HD, bool kBF16, bool kPaged>
cudaError_t cluster_slots(int size, int* slots) {
  static DeviceMemo<kMaxCluster + 1> memo;
  return memo.get(size, slots, [&](int* n) {
    auto kern = text_attention_kernel<HD, kBF16, kPaged>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<HD>::SMEM_BYTES);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)size;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)size);
    cfg.blockDim = dim3(NUM_THREADS);
    cfg.dynamicSmemBytes = Cfg<HD>::SMEM_BYTES;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int c = 0;
    e = cudaOccupancyMaxActiveClusters(&c, kern, &cfg);
    *n = std::min(2 * c, 2 * num_sms() / size);
    return e;
  });
}

template <int HD, bool kBF16, bool kPaged>
int launch(const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, Params p, long long units,
           int max_ctx, cudaStream_t st) {
  auto kern = text_attention_kernel<HD, kBF16, kPaged>;
  // CTA slots; the query also prepares the kernel for its shared memory
  int one = 0;
  const cudaError_t e = cluster_slots<HD, kBF16, kPaged>(1, &one);
  if (e != cudaSuccess) return cuda_status(e, "text attention: occupancy query");
  const long long slots = one;
  if (slots < 1) return fail(-3, "text attention: the kernel cannot be scheduled on this device");
  // Key split: where the units leave CTA slots empty, each unit's keys are cut
  // into ranges.  Up to kMaxCluster of them are one cluster, as many as fit
  // the GPU at once, and at least 2 blocks each (901 keys, 8 heads: 13.4 us;
  // 14.8 with 4 blocks, 22 with 8).  More go through global memory and a
  // second kernel, at least 8 blocks each (4000 keys: 17.5 us in 15 ranges of
  // a cluster, 28 in 31 ranges).
  const long long blocks = ((long long)max_ctx + BKV - 1) / BKV;
  long long want = kPaged ? std::max(1ll, std::min(slots / units, blocks / 2)) : 1;
  if (want > kMaxCluster) want = std::max<long long>(kMaxCluster, std::min(slots / units, blocks / 8));
  want = std::min<long long>(want, kMaxSplits);
  p.splits = (int)want;
  if (p.splits > 1 && p.splits <= kMaxCluster) {
    int fit = 0;  // an error counts as none: the split goes through global memory then
    while (p.splits > 1 && (cluster_slots<HD, kBF16, kPaged>(p.splits, &fit) != cudaSuccess || fit < units)) --p.splits;
    // Clusters pack badly where the wanted split is odd (32 units in 9 ranges:
    // 6 fit, 196 us; 9 ranges through global memory, 168 us).
    p.in_cluster = 5 * p.splits >= 4 * want && p.splits > 1;
    if (!p.in_cluster) p.splits = (int)want;
  }
  void* part = nullptr;
  if (p.splits > 1 && !p.in_cluster) {
    const size_t items = (size_t)p.splits * p.total_q * p.n_heads;
    const int rc = scratch_alloc(&part, items * (HD + 1) * sizeof(float), "text attention", st);
    if (rc) return rc;
    p.part_o = static_cast<float*>(part);
    p.part_lse = p.part_o + items * HD;
  }
  const long long ctas = p.splits > 1 ? units * p.splits : std::min(units, slots);
  // Work as far as the host knows it: the lengths are on the device, so the
  // products are not counted, and a cache counts as max_ctx keys per sequence.
  const double keys = kPaged ? (double)p.n_seqs * max_ctx : (double)p.total_q;
  ProfScope prof(kPaged ? "paged_attention" : "prompt_attention", 0.0,
                 2.0 * HD * (2.0 * p.total_q * p.n_heads + 2.0 * keys * p.n_kv), st);
  int rc = launch_after("text_attention_kernel launch", kern, dim3((unsigned)ctas), dim3(NUM_THREADS),
                        Cfg<HD>::SMEM_BYTES, p.in_cluster ? p.splits : 1, st, qm, km, vm, p);
  if (rc == 0 && part) {
    rc = launch_after("text_combine_kernel launch", text_combine_kernel<HD, kBF16>,
                      dim3((unsigned)(p.total_q * p.n_heads)), dim3(256), 0, 1, st, p.part_o, p.part_lse, p.splits,
                      p.total_q, p.n_heads, p.cu, p.n_seqs, static_cast<uint16_t*>(p.out), p.out_token, p.out_head);
  }
  scratch_free(part, st);
  return rc;
}

template <bool kPaged>
int dispatch(const TextAttention& a, const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm,
             const Params& p, long long units, cudaStream_t st) {
  if (a.head_dim == 128)
    return a.bf16 ? launch<128, true, kPaged>(qm, km, vm, p, units, a.max_ctx, st)
                  : launch<128, false, kPaged>(qm, km, vm, p, units, a.max_ctx, st);
  return a.bf16 ? launch<64, true, kPaged>(qm, km, vm, p, units, a.max_ctx, st)
                : launch<64, false, kPaged>(qm, km, vm, p, units, a.max_ctx, st);
}

}  // namespace text

int text_tmem_shares(TmemShare* s) {
  s[0] = {text::Cfg<64>::SMEM_BYTES, text::TMEM_COLS};
  s[1] = {text::Cfg<128>::SMEM_BYTES, text::TMEM_COLS};
  return 2;
}

int launch_text_attention(const TextAttention& a, cudaStream_t st) {
  using namespace text;
  if (a.total_q == 0 || a.n_seqs == 0) return 0;
  const int group = a.n_heads / a.n_kv;
  Params p{};
  p.table_ld = a.table_ld;
  p.table_width = a.table_width;
  p.page_shift = a.page_shift;
  p.n_pages = a.n_pages;
  p.splits = 1;
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

  for (int s0 = 0; s0 < a.n_seqs; s0 += kMaxSeqs) {
    p.n_seqs = std::min(kMaxSeqs, a.n_seqs - s0);
    p.cu = a.cu + s0;
    p.ctx = paged ? a.ctx + s0 : nullptr;
    p.table = paged ? a.table + s0 * a.table_ld : nullptr;
    // Tiles: sum_i ceil(q_len_i / T) <= (total + n * (T - 1)) / T; CTAs past
    // the real number of tiles end at once.
    const long long T = p.tile_tokens, seqs = std::min(p.n_seqs, a.total_q);
    const long long units = (a.total_q + seqs * (T - 1)) / T * a.n_kv;
    if (units > 0x7fffffffll / kMaxSplits) return fail(-2, "text attention: too many tiles in one call");
    const int rc = paged ? dispatch<true>(a, qm, km, vm, p, units, st) : dispatch<false>(a, qm, km, vm, p, units, st);
    if (rc) return rc;
  }
  return 0;
}

int launch_paged_append(const TextTensor& k, const TextTensor& v, const TextTensor& kc, const TextTensor& vc,
                        const int* table, long long table_ld, int table_width, int page_shift, int n_pages,
                        const int* cu, const int* ctx, int n_seqs, int total, int n_kv, int head_dim,
                        cudaStream_t st) {
  if (total == 0 || n_seqs == 0) return 0;
  const long long threads = (long long)total * n_kv * (head_dim / 8);
  const long long blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffffll) return fail(-2, "paged_append: too many values in one call");
  ProfScope prof("paged_append", 0.0, 8.0 * total * n_kv * head_dim, st);
  return launch_after("paged_append_kernel launch", text::paged_append_kernel, dim3((unsigned)blocks), dim3(256), 0, 1,
                      st, static_cast<const uint16_t*>(k.data), static_cast<const uint16_t*>(v.data), k.token, k.head,
                      v.token, v.head, static_cast<uint16_t*>(kc.data), static_cast<uint16_t*>(vc.data), kc.page,
                      kc.token, kc.head, vc.page, vc.token, vc.head, n_pages, page_shift, table, table_ld, table_width,
                      cu, ctx, n_seqs, total, n_kv, head_dim);
}

}  // namespace bonsai
