// Attention of new tokens over a paged cache of 8- or 4-bit codes
// (bonsai_paged_attention_quant; the formats: quant.cuh) for sm_100a.
//
//   O[t, h] = sum_j p_j V[j, h / G],  p = softmax_j(scale * Q[t, h] . K[j, h / G])
//
// over the cached places j that token t sees.  The codes are turned into exact
// 16-bit values on their way to the tensor core; scores, statistics and sums are
// f32.  P goes to its product as two 16-bit values, its rounding and the rounding of what
// that leaves (bf16: within 2^-16 of P, f16: 2^-22), so that the output's rounding is the only
// one to 16 bits (half as many products again: 78 us in place of 74 for 64 single tokens, 90 in
// place of 85 for long contexts).
//
// Few rows (single tokens): the codes decide, every one is read once for all rows
// of a key/value head, and the products are small: 16 keys x 8 rows of mma.sync per
// step, keys as the rows of S^T = K Q^T and the head's dims as those of
// O^T = V^T P^T.  With the keys as rows the fragments of both cache operands are
// made from codes in registers (each lane reads whole pieces of a few keys and the
// order of dims inside a product is free), nothing goes through shared memory twice,
// and maxima, sums and rescaling stay in a lane's own columns.
// Work is cut evenly: the launch's units (sequence x tile of rows x key/value head)
// laid end to end are blocks of 128 keys, and each CTA takes the same number of
// them, so that a unit may be cut anywhere; parts of a unit that more than one CTA
// has are joined by a second kernel.  Inside a CTA the warps take 16 or 32 keys in
// turn, each through its own ring of asynchronous copies and with its own softmax;
// they meet once per unit.
//
// Measured (B200, 32 / 8 heads of 128): 64 tokens over 130 to 4000 keys, bf16, 8 bits 78 us,
// 3.5 TB/s (the same over a 16-bit cache 102); 4 over 30000 to 65536, f16, 4 bits 90 us,
// 2.4 TB/s, and of 8 bits 96, 4.4 TB/s.  Without any arithmetic the same loads take 56,
// 64 and 81 us: 64-byte rows of one head are read 128 bytes at a time (1.6 times the bytes
// of 4 bits; two heads to a CTA read each once and took 98 us).  The rest is what waits for them
// more than instructions, 640 (8 bits) and 440 (4 bits) per 16 keys and warp: without the conversion
// of the codes, 30 and 42 % of all, 71 in place of 74 and 74 in place of 85, without the exponents'
// reading or the softmax (an eighth) 69 (P of one 16-bit value in all of these); and 3 to 5 us
// from one unit to the next.  Tried and not kept: asynchronous copies of 16 bytes in TMA's
// place (91 and 86), three stages unrolled (111 and 101), unequal shares for the two CTAs of an
// SM (79 to 89), two chains of products per score (75 and 87), Q asked for before the warps
// meet (83 and 94).
#include "quant.cuh"
#include "ptx.cuh"

#include <cudaTypedefs.h>

#include <algorithm>
#include <type_traits>

namespace bonsai {
namespace gemm {
PFN_cuTensorMapEncodeTiled_v12000 get_encode_fn();
}
namespace quant {

constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int BLOCK = 128;            // keys: the grain of the cut
constexpr int kMaxSeqs = 512;         // sequences of one launch (24 bytes each in shared memory)
// Rows (tokens x heads of a group) of a sequence that this kernel takes where there are longer ones,
// two tiles of 8: 64 sequences of 16 rows over 1000 keys 83 us, by the other kernel 98, 8 over 8000
// 67 and 91; of 32 rows 134 and 98, 105 and 90.  (A call of one sequence of 32 rows over 900 keys
// would be better off here, 23 and 34.)
constexpr int kFewRows = 16;
constexpr float kRescaleThreshold = 8.0f;
// P is 2^(s - m + kLift): an f16 P uses the type's range (with the threshold it
// reaches 2^15), so that weights down to 2^-32 of the largest count.
template <bool kBF16>
constexpr float kLift = kBF16 ? 0.0f : 7.0f;

struct Params {
  Cache c;
  const int* cu;
  const int* ctx;
  int n_seqs, total_q, n_heads, n_kv, group;
  int max_tokens;  // sequences with more query tokens are another launch's
  float scale_log2;
  const uint8_t* q;
  long long q_token, q_head;  // bytes
  uint8_t* out;
  long long out_token, out_head;  // bytes
  int box;         // keys of a copy: a page's slots, at most a step's
  int* err;
  float* part_o;   // [CTA][2][rows of a tile][HD], sums not divided
  float2* part_s;  // [CTA][2][rows of a tile] maximum (log2), sum of exponentials
  int4* joins;     // [CTA] {sequence, tile, head, last CTA} of the unit that begins in its share and ends in a later one, or {-1}
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <bool kBF16>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (kBF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void copy_box(uint32_t dst, const void* map, uint64_t* bar, int head, int slot, int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(map), "r"(smem_u32(bar)), "r"(0), "r"(head), "r"(slot), "r"(page)
      : "memory");
}
template <int kWords>
__device__ __forceinline__ void load_words(uint32_t (&w)[kWords], uint32_t addr) {
  static_assert(kWords == 1 || kWords == 2 || kWords == 4, "one load");
  if constexpr (kWords == 4)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
  else if constexpr (kWords == 2)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
}

// Where 16-byte piece `piece` of row `row` of a tile of codes is kept: rows fill
// lines of 128 bytes, pieces are permuted within a row as TMA's swizzle of the row's
// width does it, so that the reads (a lane's dims of keys g and g + 8; a lane's dims of
// keys 2t, 2t + 1, 2t + 8, 2t + 9) spread over the banks.
template <int kRow>
__device__ __forceinline__ uint32_t place(int row, int piece) {
  if constexpr (kRow == 128)
    return (uint32_t)(row * 128 + ((piece ^ (row & 7)) << 4));
  else if constexpr (kRow == 64)
    return (uint32_t)(row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
  else
    return (uint32_t)(row * 32 + ((piece ^ ((row >> 2) & 1)) << 4));
}

// The scale of a pair of keys' blocks, and codes times it.
template <int kFmt, bool kBF16, bool kSmall>
struct Scale {
  uint32_t s;
  Offsets off;
  __device__ __forceinline__ Scale(uint32_t ea, uint32_t eb, uint32_t block) {
    s = scale_pair_at<kBF16>(ea, eb, block);
    if constexpr (kSmall) off = expand_offsets<kFmt>(s);
  }
  template <int kJ>
  __device__ __forceinline__ uint32_t pair(uint32_t word) const {
    if constexpr (kSmall)
      return expand_small<kFmt, kJ>(word, s, off);
    else
      return expand<kFmt, kBF16, kJ>(word, s);
  }
};

// Blocks of a unit (one where there is no key).  A place may be up to 2^31 - 2: sums with
// places in them are unsigned.
__device__ __forceinline__ int blocks_of(int keys) { return max(1, (int)(((unsigned)keys + BLOCK - 1) / BLOCK)); }

// A CTA's run of keys inside one unit, and the unit's shape.
struct Unit {
  int seq, tile, kvh;
  int q_begin, rows;  // first packed token; rows (tokens x heads of the group) of the sequence
  int kv_len, first;  // keys; place of the sequence's first new token
  int from, to;       // keys of the run
  int last;           // the CTA that has the unit's last block
  bool ends;          // that is this one
};

template <int HD, int kFmt, bool kBF16, int NT>
struct Cfg {
  static constexpr int ROWS = 8 * NT;                // rows of a tile
  static constexpr int RB = kRowBytes<kFmt>(HD);     // bytes of a row of codes
  // Keys of a step: what is done once per step (places of the copies, maxima,
  // exponents) costs a third of it at 16, so 32 where it is no more bytes.
  static constexpr int STEP = RB == 128 ? 16 : 32;
  static constexpr int SUBS = STEP / 16;
  static constexpr int TILE = STEP * RB;             // K or V of a step
  // 8 KB of a warp's codes asked for ahead, with one CTA on an SM (two tiles of
  // rows do not leave two their registers) twice that
  static constexpr int STAGES = (RB == 32 ? 4 : 2) * NT;
  static constexpr int RING = STAGES * 2 * TILE;     // of a warp
  static constexpr int REGS = 4 * NT * (HD / 16);    // O of a lane
  static constexpr int MERGE = WARPS * REGS * 32 * 4;
  static constexpr int SMEM = 1024 + WARPS * RING + MERGE + 2 * WARPS * ROWS * 4 + WARPS * STAGES * 8 + 16;
};

template <int HD, int kFmt, bool kBF16, int NT>
__global__ void __launch_bounds__(THREADS, NT == 1 ? 2 : 1) quant_decode_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const Params p) {
  using C = Cfg<HD, kFmt, kBF16, NT>;
  constexpr int RB = C::RB, ROWS = C::ROWS, S = C::STAGES, STEP = C::STEP, SUBS = C::SUBS;
  constexpr unsigned STRIDE = WARPS * STEP;  // keys from a warp's step to its next
  constexpr int KW = RB / 16, VW = RB / 32;  // words of a key that a lane takes of K, of V
  constexpr int KL = KW > 4 ? 4 : KW, KN = KW / KL;  // words of a load, loads
  constexpr int MT = HD / 16;                // steps of the contraction over dims, tiles of O's dims
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ long long warp_sums[WARPS];
  __shared__ long long seq_before[kMaxSeqs + 1];  // blocks of a head before each sequence
  __shared__ int4 seq_shape[kMaxSeqs];            // first packed token, tokens, keys, place of the first token
  float* buf = reinterpret_cast<float*>(smem + WARPS * C::RING);  // [WARPS][O register][lane]
  float* stat_m = buf + C::MERGE / 4;                             // [WARPS][ROWS]
  float* stat_l = stat_m + WARPS * ROWS;
  uint64_t* bars = reinterpret_cast<uint64_t*>(stat_l + WARPS * ROWS);  // [WARPS][S]: a step's codes are there
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + WARPS * S);

  const int warp = threadIdx.x / 32, lane = (int)lane_id();
  const int g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * C::RING;
  uint64_t* full = bars + warp * S;
  if (lane == 0) {
    for (int s = 0; s < S; ++s) bar_init(&full[s], 1);
    fence_barrier_init();
    if (warp == 0) {
      *abort_flag = 0;
      tma_prefetch_desc(&kmap);
      tma_prefetch_desc(&vmap);
    }
  }
  uint32_t put = 0, got = 0;     // the stages to be filled and read next
  uint32_t got_phase = 0;

  griddep_wait();
  // Blocks of a head before each sequence (a prefix sum over the sequences).
  {
    long long base = 0;
    for (int s0 = 0; s0 < p.n_seqs; s0 += THREADS) {
      const int s = s0 + (int)threadIdx.x;
      long long v = 0;
      if (s < p.n_seqs) {
        int4 x;
        x.x = max(0, min(p.cu[s], p.total_q));
        x.y = max(x.x, min(p.cu[s + 1], p.total_q)) - x.x;
        const int ctx = max(0, p.ctx[s]);
        x.z = (int)min((long long)ctx, (long long)p.c.table_width << p.c.page_shift);  // cut to the table
        x.w = ctx - x.y;
        seq_shape[s] = x;
        if (x.y <= p.max_tokens)
          v = ((long long)x.y * p.group + ROWS - 1) / ROWS * blocks_of(x.z);
      }
      long long incl = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
      }
      if (lane == 31) warp_sums[warp] = incl;
      __syncthreads();
      long long off = base;
      for (int w = 0; w < warp; ++w) off += warp_sums[w];
      if (s < p.n_seqs) seq_before[s] = off + incl - v;
      for (int w = 0; w < WARPS; ++w) base += warp_sums[w];
      __syncthreads();
    }
    if (threadIdx.x == 0) seq_before[p.n_seqs] = base;
    __syncthreads();
  }
  griddep_launch();
  const long long all = seq_before[p.n_seqs] * p.n_kv;
  // shares: no CTA between two with work is without any
  const long long shares = min((long long)gridDim.x, all);
  const bool busy = blockIdx.x < shares;
  const long long b0 = busy ? all * blockIdx.x / shares : 0, b1 = busy ? all * (blockIdx.x + 1) / shares : 0;
  if (threadIdx.x == 0) p.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);

  // The run of this CTA's blocks from b on that lies in one unit; b moves past it.
  // Blocks are ordered by sequence, tile, head, keys.
  auto take_unit = [&](long long& b) {
    Unit u;
    int lo = 0, hi = p.n_seqs;  // the last sequence that begins at or before b, empty ones passed over
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (seq_before[mid] * p.n_kv <= b) lo = mid; else hi = mid;
    }
    const int4 x = seq_shape[lo];
    u.seq = lo;
    u.q_begin = x.x;
    u.rows = x.y * p.group;
    u.kv_len = x.z;
    u.first = x.w;
    const int blocks = blocks_of(u.kv_len);
    const long long base = seq_before[lo] * p.n_kv;
    const int no = (int)((b - base) / blocks);
    u.tile = no / p.n_kv;
    u.kvh = no - u.tile * p.n_kv;
    const long long begin = base + (long long)no * blocks;
    const int end = (int)min((long long)blocks, b1 - begin);
    u.from = (int)(b - begin) * BLOCK;
    u.to = (int)min((unsigned)u.kv_len, (unsigned)end * BLOCK);
    u.ends = end == blocks;
    u.last = u.ends ? (int)blockIdx.x : (int)(((begin + blocks) * shares - 1) / all);
    b = begin + end;
    return u;
  };

  // ---- what the warp reads: steps of keys first_key + i STRIDE, of the unit in
  // hand or, from its last step on, of the next one
  const int mask = (1 << p.c.page_shift) - 1;
  const int boxes = STEP / p.box, my_box = lane % boxes;  // a step is `boxes` copies of each side; lane l has the page of box l % boxes
  const int e_row = lane % STEP, e_box = e_row / p.box;
  // exponents: STEP 16: lanes 0-15 of K's key `lane`, 16-31 of V's; 32: both of key `lane`
  const bool of_v = STEP == 16 && lane >= 16;
  const long long ke_page = of_v ? p.c.v.s_page : p.c.k.s_page;
  const int ke_token = (int)(of_v ? p.c.v.s_token : p.c.k.s_token);
  unsigned first_key = 0, to = 0;
  int steps = 0, kvh = 0;
  const int* table = nullptr;
  const uint8_t *ke = nullptr, *ve = nullptr;
  auto pages = [&](int i) -> int {
    const unsigned k = first_key + i * STRIDE + my_box * p.box;
    return k < to ? __ldg(table + (k >> p.c.page_shift)) : -1;
  };
  auto read_exps = [&](const uint8_t* src) -> uint32_t {
    if constexpr (HD == 128)
      return __ldg(reinterpret_cast<const uint32_t*>(src));
    else
      return __ldg(reinterpret_cast<const uint16_t*>(src));
  };
  // Asks for the codes of step i.  A page outside the cache reads as zeros.
  auto ask = [&](int i, int page) {
    if (i < steps) {
      const int slot = (int)(first_key + i * STRIDE) & mask;
      const uint32_t dst = ring + put * (2 * C::TILE);
      if (boxes == 1) {  // the page is lane 0's own
        if (lane == 0) {
          bar_arrive_expect_tx(&full[put], 2 * C::TILE);
          copy_box(dst, &kmap, &full[put], kvh, slot, page);
          copy_box(dst + C::TILE, &vmap, &full[put], kvh, slot, page);
        }
      } else {
        if (lane == 0) bar_arrive_expect_tx(&full[put], 2 * C::TILE);
        for (int b = 0; b < boxes; ++b) {
          const int pg = __shfl_sync(0xffffffffu, page, b), at = (slot + b * p.box) & mask;
          if (lane == 0) {
            copy_box(dst + b * p.box * RB, &kmap, &full[put], kvh, at, pg);
            copy_box(dst + C::TILE + b * p.box * RB, &vmap, &full[put], kvh, at, pg);
          }
        }
      }
      put = put + 1 == S ? 0 : put + 1;
    }
  };
  // The lane's exponents of step i (of K, and of V where it has both).
  auto ask_exps = [&](int i, int page, uint32_t& e0, uint32_t& e1) {
    e0 = e1 = 0;
    const unsigned k = first_key + i * STRIDE + e_row;
    const int pg = __shfl_sync(0xffffffffu, page, e_box);
    if (k < to && (unsigned)pg < (unsigned)p.c.n_pages) {
      const int slot = (int)k & mask;
      e0 = read_exps(ke + pg * ke_page + (long long)slot * ke_token);
      if (STEP == 32) e1 = read_exps(ve + pg * p.c.v.s_page + (long long)slot * (int)p.c.v.s_token);
    }
  };
  // Codes are asked for S steps ahead, exponents one, page indices one more than either.
  int page_e = -1, next_page = -1;
  uint32_t ex0 = 0, ex1 = 0;
  auto begin_reading = [&](const Unit& u) {
    first_key = u.from + warp * STEP;
    to = u.to;
    kvh = u.kvh;
    steps = to > first_key ? (int)((to - first_key + STRIDE - 1) / STRIDE) : 0;
    if (__any_sync(0xffffffffu, *abort_flag)) steps = 0;  // a stage may still be on its way: it is not asked for again
    table = p.c.table + (size_t)u.seq * p.c.table_ld;
    ke = of_v ? p.c.v.scales + kvh * p.c.v.s_head : p.c.k.scales + kvh * p.c.k.s_head;
    ve = p.c.v.scales + kvh * p.c.v.s_head;
    int pg[S];
#pragma unroll
    for (int s = 0; s < S; ++s) pg[s] = pages(s);
    next_page = pages(S);
    page_e = pages(1);
#pragma unroll
    for (int s = 0; s < S; ++s) ask(s, pg[s]);
    ask_exps(0, pg[0], ex0, ex1);
  };
  const uint32_t k_block = HD == 128 ? t : t / 2, v_block = HD == 128 ? g / 2 : g / 4;  // of this lane's dims
  // Where the lane's words are in a tile.  Rows 8 apart are permuted alike, and a
  // neighbouring piece is the other of its pair.
  const uint32_t k_at = place<RB>(g, t * (RB / 4) / 16) + (t * (RB / 4) & 15);
  const uint32_t v_at = place<RB>(2 * t, g * (RB / 8) / 16) + (g * (RB / 8) & 15);

  long long b = b0;
  Unit u;
  if (b < b1) {
    u = take_unit(b);
    begin_reading(u);
  }
  for (bool more = b0 < b1; more;) {
    // keys that this lane's columns see: rows 2t, 2t + 1 of each tile of 8
    int lim[NT][2];
    int lim_min = 0x7fffffff;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = u.tile * ROWS + n * 8 + 2 * t + i;
        lim[n][i] = r < u.rows ? max(0, min(u.kv_len, u.first + r / p.group + 1)) : 0;
        lim_min = min(lim_min, r < u.rows ? lim[n][i] : 0x7fffffff);
      }
    lim_min = __reduce_min_sync(0xffffffffu, lim_min);

    // Q as the second operand: column g, this lane's dims [t HD/4, (t + 1) HD/4)
    // in the order in which the codes come out of their words
    uint32_t qf[NT][MT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = u.tile * ROWS + n * 8 + g;
      uint32_t raw[HD / 8];
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        uint4 x = make_uint4(0, 0, 0, 0);
        if (r < u.rows) {
          const int tok = r / p.group, head = u.kvh * p.group + r - tok * p.group;
          x = *reinterpret_cast<const uint4*>(p.q + (long long)(u.q_begin + tok) * p.q_token + head * p.q_head +
                                              t * (HD / 2) + i * 16);
        }
        raw[4 * i] = x.x;
        raw[4 * i + 1] = x.y;
        raw[4 * i + 2] = x.z;
        raw[4 * i + 3] = x.w;
      }
      if constexpr (kFmt == kI8) {  // (0, 2) (1, 3) of four dims
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          qf[n][i][0] = __byte_perm(raw[2 * i], raw[2 * i + 1], 0x5410);
          qf[n][i][1] = __byte_perm(raw[2 * i], raw[2 * i + 1], 0x7632);
        }
      } else {  // (0, 4) (1, 5), (2, 6) (3, 7) of eight dims
#pragma unroll
        for (int i = 0; i < MT / 2; ++i) {
          qf[n][2 * i][0] = __byte_perm(raw[4 * i], raw[4 * i + 2], 0x5410);
          qf[n][2 * i][1] = __byte_perm(raw[4 * i], raw[4 * i + 2], 0x7632);
          qf[n][2 * i + 1][0] = __byte_perm(raw[4 * i + 1], raw[4 * i + 3], 0x5410);
          qf[n][2 * i + 1][1] = __byte_perm(raw[4 * i + 1], raw[4 * i + 3], 0x7632);
        }
      }
    }

    float o[NT][MT][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[n][i][k] = 0.f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }

#pragma unroll 1
    for (int i = 0; i < steps; ++i) {
      {
        const unsigned k0 = first_key + i * STRIDE;
        const uint32_t kt = ring + got * (2 * C::TILE) + k_at, vt = ring + got * (2 * C::TILE) + C::TILE + v_at;
        const uint32_t ek = lift_exponents<kFmt, kBF16>(ex0);
        uint32_t ev = STEP == 32 ? lift_exponents<kFmt, kBF16>(ex1) : ek;
        ask_exps(i + 1, page_e, ex0, ex1);
        page_e = pages(i + 2);
        const bool there = bar_test_wait(smem_u32(&full[got]), got_phase) ||
                           wait_bar(&full[got], got_phase, abort_flag, p.err, DEV_ERR_TIMEOUT_TMA);
        if (!__all_sync(0xffffffffu, there)) break;
        got = got + 1 == S ? 0 : got + 1;
        got_phase ^= got == 0;

        // ---- S^T = K Q^T: keys g and g + 8 of each 16, columns 2t, 2t + 1
        float sc[SUBS][NT][4];
        auto scores = [&](auto small) {
          constexpr bool kSmall = decltype(small)::value;
#pragma unroll
          for (int b = 0; b < SUBS; ++b) {
#pragma unroll
            for (int n = 0; n < NT; ++n) sc[b][n][0] = sc[b][n][1] = sc[b][n][2] = sc[b][n][3] = 0.f;
            const uint32_t ea = __shfl_sync(0xffffffffu, ek, 16 * b + g), eb = __shfl_sync(0xffffffffu, ek, 16 * b + g + 8);
            const Scale<kFmt, kBF16, kSmall> sa(ea, ea, k_block), sb(eb, eb, k_block);
#pragma unroll
            for (int h = 0; h < KN; ++h) {
              uint32_t ka[KL], kb[KL];
              // a lane's bytes of a key: [t RB / 4, (t + 1) RB / 4)
              load_words<KL>(ka, (kt ^ (16u * h)) + 16 * b * RB);
              load_words<KL>(kb, (kt ^ (16u * h)) + (16 * b + 8) * RB);
#pragma unroll
              for (int w = 0; w < KL; ++w) {
                constexpr int PER_WORD = kFmt == kI8 ? 1 : 2;
                const int ks = PER_WORD * (h * KL + w);
                {
                  const uint32_t a0 = sa.template pair<0>(ka[w]), a1 = sb.template pair<0>(kb[w]);
                  const uint32_t a2 = sa.template pair<1>(ka[w]), a3 = sb.template pair<1>(kb[w]);
#pragma unroll
                  for (int n = 0; n < NT; ++n) mma16816<kBF16>(sc[b][n], a0, a1, a2, a3, qf[n][ks][0], qf[n][ks][1]);
                }
                if constexpr (kFmt == kI4) {
                  const uint32_t a0 = sa.template pair<2>(ka[w]), a1 = sb.template pair<2>(kb[w]);
                  const uint32_t a2 = sa.template pair<3>(ka[w]), a3 = sb.template pair<3>(kb[w]);
#pragma unroll
                  for (int n = 0; n < NT; ++n)
                    mma16816<kBF16>(sc[b][n], a0, a1, a2, a3, qf[n][ks + 1][0], qf[n][ks + 1][1]);
                }
              }
            }
          }
        };
        // f16: steps without a large exponent (or one of 255) take the shorter way
        const bool plain = kBF16 || __any_sync(0xffffffffu, large_exponent(ek) || large_exponent(ev));
        if (plain)
          scores(std::false_type{});
        else
          scores(std::bool_constant<!kBF16>{});

        // A key or value that is not a number is rare: one look at all of the step's exponents.
        const bool odd = plain && __any_sync(0xffffffffu, (bytes_of_ones(ek) | (STEP == 32 ? bytes_of_ones(ev) : 0u)) != 0);
        if (kBF16 && odd) {
#pragma unroll
          for (int b = 0; b < SUBS; ++b) {
            const bool na = bytes_of_ones(__shfl_sync(0xffffffffu, ek, 16 * b + g)) != 0;
            const bool nb = bytes_of_ones(__shfl_sync(0xffffffffu, ek, 16 * b + g + 8)) != 0;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (k < 2 ? na : nb) sc[b][n][k] = __int_as_float(0x7fffffff);
          }
        }

        // ---- softmax over the keys: a key past a column's limit counts nothing, whatever it gave
        if (k0 + STEP > (unsigned)lim_min) {
          __syncwarp();  // a branch, not a selection in every step
#pragma unroll
          for (int b = 0; b < SUBS; ++b)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (k0 + 16 * b + g + (k >> 1) * 8 >= (unsigned)lim[n][k & 1]) sc[b][n][k] = -INFINITY;
        }
        float mx[NT][2];
        bool move = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float x = fmaxf(sc[0][n][k], sc[0][n][k + 2]);
#pragma unroll
            for (int b = 1; b < SUBS; ++b) x = fmaxf(x, fmaxf(sc[b][n][k], sc[b][n][k + 2]));
            mx[n][k] = x * p.scale_log2;
            move |= mx[n][k] > m[n][k] + kRescaleThreshold;
          }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              float x = mx[n][k];
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
              if (x > m[n][k]) {
                const float alpha = ex2(m[n][k] - x);
                m[n][k] = x;
                l[n][k] *= alpha;
#pragma unroll
                for (int i2 = 0; i2 < MT; ++i2) {
                  o[n][i2][k] *= alpha;
                  o[n][i2][k + 2] *= alpha;
                }
              }
            }
        }
        uint32_t pb[SUBS][NT][2], pl[SUBS][NT][2];  // P rounded, and what that leaves
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          // no key seen yet: every p is 2^-inf = 0
          const float ref0 = kLift<kBF16> - (m[n][0] == -INFINITY ? 0.f : m[n][0]);
          const float ref1 = kLift<kBF16> - (m[n][1] == -INFINITY ? 0.f : m[n][1]);
#pragma unroll
          for (int b = 0; b < SUBS; ++b) {
            const float p0 = ex2(fmaf(sc[b][n][0], p.scale_log2, ref0)), p1 = ex2(fmaf(sc[b][n][1], p.scale_log2, ref1));
            const float p2 = ex2(fmaf(sc[b][n][2], p.scale_log2, ref0)), p3 = ex2(fmaf(sc[b][n][3], p.scale_log2, ref1));
            l[n][0] += p0 + p2;
            l[n][1] += p1 + p3;
            // P^T: keys 2t, 2t + 1 (+ 8) of column g
            const uint32_t x0 = pack16<kBF16>(p0, p1), x1 = pack16<kBF16>(p2, p3);
            pb[b][n][0] = transpose8x8(x0);
            pb[b][n][1] = transpose8x8(x1);
            pl[b][n][0] = transpose8x8(pack16<kBF16>(p0 - low_f32<kBF16>(x0), p1 - high_f32<kBF16>(x0)));
            pl[b][n][1] = transpose8x8(pack16<kBF16>(p2 - low_f32<kBF16>(x1), p3 - high_f32<kBF16>(x1)));
          }
        }

        // ---- O^T += V^T P^T: this lane's dims are [g HD/8, (g + 1) HD/8)
        // A value that is not a number reaches only the columns that see its key: it
        // is zero to the product, 0 * NaN would reach them all.
        if (odd) {
          for (int k = 0; k < STEP; ++k) {
            const uint32_t e1 = (__shfl_sync(0xffffffffu, ev, STEP == 32 ? k : 16 + k) >> (8 * v_block)) & 255u;
            if (e1 == 255u)
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c)
                  if (k0 + k < (unsigned)lim[n][c])
#pragma unroll
                    for (int i2 = 0; i2 < MT; ++i2) o[n][i2][c] = o[n][i2][c + 2] = __int_as_float(0x7fffffff);
          }
          ev &= ~((bytes_of_ones(ev) >> 7) * 255u);
        }
        auto values = [&](auto small) {
          constexpr bool kSmall = decltype(small)::value;
#pragma unroll
          for (int b = 0; b < SUBS; ++b) {
            uint32_t es[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              es[k] = __shfl_sync(0xffffffffu, ev, (STEP == 32 ? 16 * b : 16) + 2 * t + (k & 1) + (k >> 1) * 8);
            const Scale<kFmt, kBF16, kSmall> sa(es[0], es[1], v_block), sb(es[2], es[3], v_block);
            uint32_t v[4][VW];
#pragma unroll
            for (int k = 0; k < 4; ++k)  // of rows of 128 bytes an odd one is permuted by one more
              load_words<VW>(v[k], (RB == 128 && (k & 1) ? vt ^ 16u : vt) + (16 * b + (k & 1) + (k >> 1) * 8) * RB);
#pragma unroll
            for (int w = 0; w < VW; ++w)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                // two bytes of the first key below two of the second
                const uint32_t za = __byte_perm(v[0][w], v[1][w], h ? 0x7632 : 0x5410);
                const uint32_t zb = __byte_perm(v[2][w], v[3][w], h ? 0x7632 : 0x5410);
                const int mt = kFmt == kI8 ? 2 * w + h : 4 * w + 2 * h;
                {
                  const uint32_t a0 = sa.template pair<0>(za), a1 = sa.template pair<1>(za);
                  const uint32_t a2 = sb.template pair<0>(zb), a3 = sb.template pair<1>(zb);
#pragma unroll
                  for (int n = 0; n < NT; ++n) {
                    mma16816<kBF16>(o[n][mt], a0, a1, a2, a3, pb[b][n][0], pb[b][n][1]);
                    mma16816<kBF16>(o[n][mt], a0, a1, a2, a3, pl[b][n][0], pl[b][n][1]);
                  }
                }
                if constexpr (kFmt == kI4) {
                  const uint32_t a0 = sa.template pair<2>(za), a1 = sa.template pair<3>(za);
                  const uint32_t a2 = sb.template pair<2>(zb), a3 = sb.template pair<3>(zb);
#pragma unroll
                  for (int n = 0; n < NT; ++n) {
                    mma16816<kBF16>(o[n][mt + 1], a0, a1, a2, a3, pb[b][n][0], pb[b][n][1]);
                    mma16816<kBF16>(o[n][mt + 1], a0, a1, a2, a3, pl[b][n][0], pl[b][n][1]);
                  }
                }
              }
          }
        };
        if (plain)
          values(std::false_type{});
        else
          values(std::bool_constant<!kBF16>{});
        __syncwarp();
        ask(i + S, next_page);
        next_page = pages(i + S + 1);
      }
    }

    // ---- the next unit's first steps are on their way while the warps meet
    const Unit done = u;
    more = b < b1;
    if (more) {
      u = take_unit(b);
      begin_reading(u);
    }
    __syncthreads();  // the last unit's sums have been read
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        l[n][k] += __shfl_xor_sync(0xffffffffu, l[n][k], 4);
        l[n][k] += __shfl_xor_sync(0xffffffffu, l[n][k], 8);
        l[n][k] += __shfl_xor_sync(0xffffffffu, l[n][k], 16);
        if (g == 0) {
          stat_m[warp * ROWS + n * 8 + 2 * t + k] = m[n][k];
          stat_l[warp * ROWS + n * 8 + 2 * t + k] = l[n][k];
        }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) buf[(warp * C::REGS + (n * MT + i) * 4 + k) * 32 + lane] = o[n][i][k];
    }
    __syncthreads();
    const bool whole = done.from == 0 && done.ends;
    const int slot = (int)blockIdx.x * 2 + (done.from == 0 ? 1 : 0);
    if (threadIdx.x == 0 && done.from == 0 && !whole) p.joins[blockIdx.x] = make_int4(done.seq, done.tile, done.kvh, done.last);
    for (int e4 = threadIdx.x; e4 < ROWS * HD / 4; e4 += THREADS) {
      const int r = e4 / (HD / 4), d = (e4 % (HD / 4)) * 4;
      const int row = done.tile * ROWS + r;
      if (row >= done.rows) continue;
      float mw[WARPS], top = -INFINITY;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        mw[w] = stat_m[w * ROWS + r];
        top = fmaxf(top, mw[w]);
      }
      // dims d .. d + 3 of row r: lane g = d / (HD / 8), registers of two tiles
      const int gg = d / (HD / 8), mt = (d % (HD / 8)) / 2, ln = gg * 4 + (r & 7) / 2;
      const int reg = ((r >> 3) * MT + mt) * 4 + (r & 1);
      float sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        // without a maximum a warp has seen no key (zeros) or only NaN (which 0 * NaN keeps)
        const float f = mw[w] == -INFINITY ? 0.f : ex2(mw[w] - top);
        const float* src = buf + (w * C::REGS + reg) * 32 + ln;
        sum = fmaf(stat_l[w * ROWS + r], f, sum);
        acc[0] = fmaf(src[0], f, acc[0]);
        acc[1] = fmaf(src[2 * 32], f, acc[1]);
        acc[2] = fmaf(src[4 * 32], f, acc[2]);
        acc[3] = fmaf(src[6 * 32], f, acc[3]);
      }
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.0f / sum;
        const int tok = row / p.group, head = done.kvh * p.group + row - tok * p.group;
        *reinterpret_cast<uint2*>(p.out + (long long)(done.q_begin + tok) * p.out_token + head * p.out_head + d * 2) =
            make_uint2(pack16<kBF16>(acc[0] * inv, acc[1] * inv), pack16<kBF16>(acc[2] * inv, acc[3] * inv));
      } else {
        *reinterpret_cast<float4*>(p.part_o + ((size_t)slot * ROWS + r) * HD + d) =
            make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (d == 0) p.part_s[(size_t)slot * ROWS + r] = make_float2(top, sum);
      }
    }
  }
  if (*abort_flag) {  // let copies in flight land before the shared memory is released
    const unsigned long long w0 = globaltimer_ns();
    while (globaltimer_ns() - w0 < 1000000ull) {
    }
  }
}

// Joins the parts of the units that lie in more than one CTA's share: CTA c of
// this kernel takes the unit that begins in share c and ends in a later one.  Its
// parts are [c][1] and [c + 1 .. last][0], joined in that order:
//   O = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i.
template <int HD, bool kBF16>
__global__ void __launch_bounds__(256) quant_join_kernel(const Params p, int tile_rows) {
  griddep_wait();
  const int4 j = p.joins[blockIdx.x];
  if (j.x < 0) return;
  const int q_begin = max(0, min(p.cu[j.x], p.total_q));
  const int rows = (max(q_begin, min(p.cu[j.x + 1], p.total_q)) - q_begin) * p.group;
  const int c = (int)blockIdx.x, n = j.w - c + 1;
  auto slot = [&](int i) { return (size_t)(i == 0 ? 2 * c + 1 : 2 * (c + i)); };
  for (int e = threadIdx.x; e < tile_rows * (HD / 4); e += 256) {
    const int r = e / (HD / 4), d = (e % (HD / 4)) * 4, row = j.y * tile_rows + r;
    if (row >= rows) continue;
    float top = -INFINITY;
    for (int i = 0; i < n; ++i) top = fmaxf(top, __ldcg(p.part_s + slot(i) * tile_rows + r).x);
    float sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float2 s = __ldcg(p.part_s + slot(i) * tile_rows + r);
      const float4 o = __ldcg(reinterpret_cast<const float4*>(p.part_o + (slot(i) * tile_rows + r) * HD + d));
      // without a maximum the part has seen no key (zeros) or only NaN (which 0 * NaN keeps)
      const float f = s.x == -INFINITY ? 0.f : ex2(s.x - top);
      sum = fmaf(f, s.y, sum);
      acc[0] = fmaf(f, o.x, acc[0]);
      acc[1] = fmaf(f, o.y, acc[1]);
      acc[2] = fmaf(f, o.z, acc[2]);
      acc[3] = fmaf(f, o.w, acc[3]);
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    const int tok = row / p.group, head = j.z * p.group + row - tok * p.group;
    *reinterpret_cast<uint2*>(p.out + (long long)(q_begin + tok) * p.out_token + head * p.out_head + d * 2) =
        make_uint2(pack16<kBF16>(acc[0] * inv, acc[1] * inv), pack16<kBF16>(acc[2] * inv, acc[3] * inv));
  }
}

// ------------------------------------------------------------------- host
// The codes of one side as boxes of rows, `box` keys of one head high.
int encode_codes(CUtensorMap* map, const Pages& t, int row, int n_kv, int page_shift, int n_pages, int box) {
  auto fn = gemm::get_encode_fn();
  if (!fn) return fail(-5, "cuTensorMapEncodeTiled entry point unavailable");
  const cuuint64_t d[4] = {(cuuint64_t)row, (cuuint64_t)n_kv, 1ull << page_shift, (cuuint64_t)n_pages};
  // the stride of a dimension of size one is never used, whatever the caller has there
  const cuuint64_t st[3] = {(cuuint64_t)(n_kv == 1 ? row : t.head), (cuuint64_t)t.token,
                            (cuuint64_t)(n_pages == 1 ? row : t.page)};
  const cuuint32_t b[4] = {(cuuint32_t)row, 1, (cuuint32_t)box, 1}, e[4] = {1, 1, 1, 1};
  const CUtensorMapSwizzle sw = row == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : row == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                                                   : CU_TENSOR_MAP_SWIZZLE_32B;
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, t.codes, d, st, b, e, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
                        CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(-5, "cuTensorMapEncodeTiled (quant attention) failed (code " + std::to_string((int)r) + ")");
  return 0;
}

template <int HD, int kFmt, bool kBF16, int NT>
int launch_decode(Params p, long long blocks, cudaStream_t st) {
  using C = Cfg<HD, kFmt, kBF16, NT>;
  auto kern = quant_decode_kernel<HD, kFmt, kBF16, NT>;
  static DeviceMemo<1> memo;
  int per_sm = 0;
  const cudaError_t e = memo.get(0, &per_sm, [&](int* n) {
    cudaError_t r = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (r == cudaSuccess) r = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (r == cudaSuccess) r = cudaOccupancyMaxActiveBlocksPerMultiprocessor(n, kern, THREADS, C::SMEM);
    return r;
  });
  if (e != cudaSuccess) return cuda_status(e, "quant attention: occupancy query");
  if (per_sm < 1) return fail(-3, "quant attention: the kernel cannot be scheduled on this device");
  const long long ctas = std::max(1ll, std::min<long long>((long long)per_sm * num_sms(), blocks));
  CUtensorMap km, vm;
  p.box = std::min(C::STEP, 1 << p.c.page_shift);
  int rc = encode_codes(&km, p.c.k, C::RB, p.n_kv, p.c.page_shift, p.c.n_pages, p.box);
  if (rc == 0) rc = encode_codes(&vm, p.c.v, C::RB, p.n_kv, p.c.page_shift, p.c.n_pages, p.box);
  if (rc) return rc;
  const size_t parts = (size_t)ctas * 2 * C::ROWS;
  void* scratch = nullptr;
  rc = scratch_alloc(&scratch, parts * (HD * sizeof(float) + sizeof(float2)) + ctas * sizeof(int4), "quant attention", st);
  if (rc) return rc;
  p.part_o = static_cast<float*>(scratch);
  p.joins = reinterpret_cast<int4*>(p.part_o + parts * HD);
  p.part_s = reinterpret_cast<float2*>(p.joins + ctas);
  rc = launch_after("quant_decode_kernel launch", kern, dim3((unsigned)ctas), dim3(THREADS), C::SMEM, 1, st, km, vm, p);
  if (rc == 0 && ctas > 1)
    rc = launch_after("quant_join_kernel launch", quant_join_kernel<HD, kBF16>, dim3((unsigned)ctas), dim3(256), 0, 1, st,
                      p, C::ROWS);
  scratch_free(scratch, st);
  return rc;
}

template <int HD, int kFmt, bool kBF16>
int dispatch(const Params& p, int rows, int max_ctx, cudaStream_t st) {
  auto blocks = [&](int tile) {  // an upper bound, by what the host knows
    return (long long)p.n_seqs * ((rows + tile - 1) / tile) * p.n_kv * std::max(1ll, ((long long)max_ctx + BLOCK - 1) / BLOCK);
  };
  if (rows <= 8) return launch_decode<HD, kFmt, kBF16, 1>(p, blocks(8), st);
  return launch_decode<HD, kFmt, kBF16, 2>(p, blocks(16), st);
}

}  // namespace quant

int launch_quant_attention(const QuantAttention& a, cudaStream_t st) {
  using namespace quant;
  if (a.total_q == 0 || a.n_seqs == 0) return 0;
  Params p{};
  p.c = a.cache;
  p.total_q = a.total_q;
  p.n_heads = a.n_heads;
  p.n_kv = a.n_kv;
  p.group = a.n_heads / a.n_kv;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.q = static_cast<const uint8_t*>(a.q.data);
  p.q_token = a.q.token * 2;
  p.q_head = a.q.head * 2;
  p.out = static_cast<uint8_t*>(a.out.data);
  p.out_token = a.out.token * 2;
  p.out_head = a.out.head * 2;
  p.err = device_error_word();
  const double row = (a.format == kI8 ? a.head_dim : a.head_dim / 2) + a.head_dim / kBlock;
  ProfScope prof("paged_attention_quant", 0.0,
                 2.0 * a.n_kv * a.n_seqs * (double)a.max_ctx * row + 4.0 * a.head_dim * a.total_q * a.n_heads, st);
  // Sequences of up to kFewRows rows (tokens x heads of the group) go to the
  // kernel above; the longer ones, where the caller's bound lets there be any, to
  // the tiles of 128 rows of text_attention.cu.
  const int few = std::max(1, kFewRows / p.group);
  const int max_q = std::max(1, std::min(a.max_q, a.total_q));
  const bool chunks = max_q > few;
  const int rows = (int)std::min<long long>((long long)std::min(max_q, few) * p.group, 1 << 30);
  p.max_tokens = chunks ? few : 0x7fffffff;
  if (chunks) {
    TextAttention t;
    t.q = a.q;
    t.out = a.out;
    t.cu = a.cu;
    t.ctx = a.ctx;
    t.table = a.cache.table;
    t.table_ld = a.cache.table_ld;
    t.table_width = a.cache.table_width;
    t.page_shift = a.cache.page_shift;
    t.n_pages = a.cache.n_pages;
    t.n_seqs = a.n_seqs;
    t.total_q = a.total_q;
    t.max_ctx = a.max_ctx;
    t.n_heads = a.n_heads;
    t.n_kv = a.n_kv;
    t.head_dim = a.head_dim;
    t.bf16 = a.bf16;
    t.scale = a.scale;
    t.quant = &a.cache;
    t.quant_i4 = a.format == kI4;
    t.min_tokens = few + 1;
    const int rc = launch_text_attention(t, st);
    if (rc) return rc;
  }
  for (int s0 = 0; s0 < a.n_seqs; s0 += kMaxSeqs) {
    p.n_seqs = std::min(kMaxSeqs, a.n_seqs - s0);
    p.cu = a.cu + s0;
    p.ctx = a.ctx + s0;
    p.c.table = a.cache.table + s0 * a.cache.table_ld;
    int rc;
    if (a.head_dim == 128) {
      if (a.format == kI8)
        rc = a.bf16 ? dispatch<128, kI8, true>(p, rows, a.max_ctx, st) : dispatch<128, kI8, false>(p, rows, a.max_ctx, st);
      else
        rc = a.bf16 ? dispatch<128, kI4, true>(p, rows, a.max_ctx, st) : dispatch<128, kI4, false>(p, rows, a.max_ctx, st);
    } else {
      if (a.format == kI8)
        rc = a.bf16 ? dispatch<64, kI8, true>(p, rows, a.max_ctx, st) : dispatch<64, kI8, false>(p, rows, a.max_ctx, st);
      else
        rc = a.bf16 ? dispatch<64, kI4, true>(p, rows, a.max_ctx, st) : dispatch<64, kI4, false>(p, rows, a.max_ctx, st);
    }
    if (rc) return rc;
  }
  return 0;
}

}  // namespace bonsai
