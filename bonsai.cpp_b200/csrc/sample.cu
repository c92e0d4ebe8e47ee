// The choice of the next token from logits (bonsai_sample_tokens) for sm_100a:
// temperature, top-k, top-p and min-p, with the random numbers as an input.
//
//   z_i = (l_i - max l) / T,  w_i = e^z_i  (0 below z = -40, for NaN and -inf)
//   order: w falling, the lowest index first among equal logits
//   top-k: the first k;  top-p: those with sum of w before them < p * (sum of the top-k);
//   min-p: w_i >= min_p;  the first of the order always stays
//   token: the first index (in the order of indices) whose sum of kept w up to and
//   with it exceeds u * (sum of kept w)
//
// A choice next to a border goes by sums over the whole row, so weights and sums
// are f64 (e^z by a table of 2^(j/64) and a polynomial of degree 4, relative
// error below 1e-13; f32 weights would move the choice of a flat row of 150000 tokens
// about once in a hundred; pairs of f32 within 1e-9 would by some 6e-5 of a token's weight
// and were no faster, 62 and 67 us in place of 60 and 64 below), and every sum has a fixed
// order: results do not depend on the run.
//
// A cluster of CTAs takes a row, each a range of its tokens, which it reads from
// memory once and keeps in shared memory for the passes that follow where that leaves
// room for a second CTA or none is needed; what a pass finds meets through distributed shared memory.
// Nothing is sorted but the few candidates at a border.  A histogram over l (2048 bins
// between the largest and the smallest logit that counts) gives the bin in which the
// k-th token (by counts, exactly), the mass p (by f32 masses, verified against the f64
// sums) or min-p's border lies.  The usual ways from there:
//   up to 1024 tokens in the bins up to it: they go to one CTA, which puts them in
//   order, cuts, sums and chooses;
//   more, and p alone: the tokens of the border's bins go there, which finds the exact
//   border; then every CTA sums what stays, and the one that has the target chooses.
// The general way takes whatever is left (a large k, thousands of equal logits at a
// border): borders one after the other, bisection where a bin has more than 1024.
//
// Bounds and measurements (B200): one row of 150001, top-k 50 and top-p 0.9, 18 us
// (0.1 us of memory): five meetings of a cluster of 16, four passes over 9400
// tokens a CTA, and code that runs once; 64 rows of 128000 with settings of their own
// 60 us (5 of memory), 256 rows of 32000 45 us (2.5): the instructions of
// the passes; 32 flat rows of 150001 cut by p alone 64 us (1.5): two passes with
// weights.  With every border found in the general way these took 45, 137, 101 and 85 us.
#include "internal.cuh"
#include "ptx.cuh"

#include <algorithm>
#include <cfloat>

namespace bonsai {
namespace sampling {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int NB = 2048;      // bins
constexpr int CAP = 1024;     // candidates that are ranked
constexpr int kMaxCluster = 16;
constexpr double kDepth = 40.0;

enum DType : int { kF16 = 0, kBF16 = 1, kF32 = 2 };

struct Params {
  const uint8_t* logits;
  long long ld;  // bytes
  int vocab, per;  // tokens of a row, of a CTA
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  int* tokens;
  float* probs;
};

// What a CTA shows its cluster; each phase has a place of its own, so one
// barrier per phase is enough.
struct Shown {
  unsigned long long top;   // largest composite (value, then lowest index)
  float low;                // smallest logit above -inf
  int pad;
  unsigned long long c_lo, c_hi;  // smallest and largest composite of a bin
  double mass[2][3];        // sums of weights, two turns in use
  int count[2][2];
  int bin, n_bin;           // a border's bin, its tokens
  long long n_above;        // tokens above it
  int found;
  float bin_mass;           // coarse mass of the CTA's bins
  int bin_count;
  unsigned long long cut;   // result of a ranking
  int verdict;              // -1: the border lies above, +1: below
  double cta_sum;
};

template <int kType>
struct Of;
template <>
struct Of<kF16> {
  using T = uint16_t;
  static __device__ __forceinline__ float f32(uint16_t v) { return __half2float(__ushort_as_half(v)); }
};
template <>
struct Of<kBF16> {
  using T = uint16_t;
  static __device__ __forceinline__ float f32(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
};
template <>
struct Of<kF32> {
  using T = uint32_t;
  static __device__ __forceinline__ float f32(uint32_t v) { return __uint_as_float(v); }
};

// NaN counts as -inf; -0 as 0.
__device__ __forceinline__ float clean(float x) { return x == x ? x + 0.0f : -INFINITY; }
// The order of values as that of unsigned numbers, larger index lower.
__device__ __forceinline__ unsigned long long composite(float x, int index) {
  const uint32_t b = __float_as_uint(x);
  const uint32_t key = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return (unsigned long long)key << 32 | (0xffffffffu - (uint32_t)index);
}
__device__ __forceinline__ float value_of(unsigned long long c) {
  const uint32_t key = (uint32_t)(c >> 32);
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ int index_of(unsigned long long c) { return (int)(0xffffffffu - (uint32_t)c); }

__device__ __forceinline__ double shfl_up(double v, int o) { return __shfl_up_sync(0xffffffffu, v, o); }
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <typename V, typename F>
__device__ __forceinline__ V warp_fold(V v, F f) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Sorts CAP values, of which those past `count` are zeros, the largest first (a
// bitonic network over CAP or half of them).
__device__ __forceinline__ void sort_down(unsigned long long* v, int count) {
  static_assert(CAP == 2 * THREADS, "a pair to a thread");
  const int padded = count <= CAP / 2 ? CAP / 2 : CAP, tid = threadIdx.x;
  for (int size = 2; size <= padded; size *= 2)
    for (int d = size / 2; d; d /= 2) {
      __syncthreads();
      if (2 * tid >= padded) continue;
      const int i = 2 * tid - (tid & (d - 1)), j = i + d;  // falls where bit `size` of the place is clear
      const unsigned long long x = v[i], y = v[j];
      if ((x < y) == ((i & size) == 0)) {
        v[i] = y;
        v[j] = x;
      }
    }
  __syncthreads();
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename V>
__device__ __forceinline__ const V* in_cta(const V* mine, int rank) {
  const V* p;
  asm("mapa.u64 %0, %1, %2;" : "=l"(p) : "l"(mine), "r"(rank));
  return p;
}

template <int kType, bool kKept>
__global__ void __launch_bounds__(THREADS, 2) sample_kernel(const Params p, int ctas) {
  using E = typename Of<kType>::T;
  extern __shared__ __align__(16) uint8_t dyn[];
  __shared__ Shown sh;
  __shared__ double table[64];
  __shared__ double part[WARPS][3];
  __shared__ unsigned long long part_u[WARPS][2];
  __shared__ int part_i[WARPS][2];
  __shared__ int n_list;
  __shared__ int edge[6];
  uint32_t* counts = reinterpret_cast<uint32_t*>(dyn);          // [NB]
  uint32_t* masses = counts + NB;                               // [NB]
  unsigned long long* list = reinterpret_cast<unsigned long long*>(masses + NB);  // [CAP]
  unsigned long long* ranked = list + CAP;                      // [CAP]
  float* sum_m = reinterpret_cast<float*>(ranked + CAP);        // [NB] masses of the cluster
  uint8_t* row_at = reinterpret_cast<uint8_t*>(sum_m + NB);     // this CTA's tokens, 16 bytes' phase as in memory

  const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
  const int rank = ctas > 1 ? (int)cluster_ctarank() : 0;
  const int r = (int)(blockIdx.x / (unsigned)ctas);
  const int begin = min(p.vocab, rank * p.per), n = min(p.vocab, begin + p.per) - begin;
  const uint8_t* src = p.logits + (long long)r * p.ld + (long long)begin * sizeof(E);
  const uint32_t phase = (uint32_t)(reinterpret_cast<uintptr_t>(src) & 15);
  const E* kept = kKept ? reinterpret_cast<const E*>(row_at + phase) : reinterpret_cast<const E*>(src);
  auto at = [&](int i) -> float { return clean(Of<kType>::f32(kKept ? kept[i] : __ldg(kept + i))); };
  auto meet = [&]() {
    if (ctas > 1)
      cluster_sync_all();
    else
      __syncthreads();
  };

  if (tid < 64) table[tid] = exp2((double)tid * 0.015625);
  for (int i = tid; i < 2 * NB; i += THREADS) counts[i] = 0;
  griddep_wait();
  griddep_launch();
  const float temp = p.temperature ? p.temperature[r] : 1.0f;
  const int top_k = p.top_k ? p.top_k[r] : 0;
  const float top_p = p.top_p ? p.top_p[r] : 1.0f;
  const float min_p = p.min_p ? p.min_p[r] : 0.0f;
  const float u_in = p.u ? p.u[r] : 0.0f;
  const bool greedy = !(temp > 0.0f);
  const double t64 = (double)temp, inv_t = 1.0 / t64, deepest = fmax(-kDepth * t64, -1.7e308);
  const double per_step = inv_t * 92.332482616893656877;  // 64 / ln 2

  // This CTA's tokens: 16 bytes at a time from `head` on, the few before and after
  // them one by one.  f(logit, token of the range), several tokens of a thread at once.
  constexpr int PER16 = 16 / sizeof(E);
  const int head = min(n, (int)(((16 - phase) & 15) / sizeof(E))), mid = (n - head) / PER16, tail = n - head - mid * PER16;
  auto of_16 = [&](const uint4& v, int j) -> float {
    const uint32_t w = (&v.x)[sizeof(E) == 4 ? j : j / 2];
    return clean(Of<kType>::f32((E)(sizeof(E) == 4 ? w : j & 1 ? w >> 16 : w & 0xffffu)));
  };
  auto for_each = [&](auto f) {
    if (tid < head) f(at(tid), tid);
    if (tid >= 32 && tid - 32 < tail) f(at(n - tail + tid - 32), n - tail + tid - 32);
    const uint4* from = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(kept) + head * sizeof(E));
    for (int i = tid; i < mid; i += THREADS) {
      const uint4 v = kKept ? from[i] : __ldg(from + i);
#pragma unroll
      for (int j = 0; j < PER16; ++j) f(of_16(v, j), head + i * PER16 + j);
    }
  };

  // ---- the row's top and bottom, on its way into shared memory
  float best_x = -INFINITY, low = INFINITY;
  int best_i = 0;
  auto take = [&](float x, int i) {  // i rises, so the first of equals stays
    if (x > best_x) {
      best_x = x;
      best_i = i;
    }
    if (x > -INFINITY) low = fminf(low, x);
  };
  if constexpr (kKept) {
    E* to = reinterpret_cast<E*>(row_at + phase);
    if (tid < head) {
      to[tid] = reinterpret_cast<const E*>(src)[tid];
      take(at(tid), tid);
    }
    const uint4* from16 = reinterpret_cast<const uint4*>(src + head * sizeof(E));
    uint4* to16 = reinterpret_cast<uint4*>(row_at + phase + head * sizeof(E));
    for (int i0 = tid; i0 < mid; i0 += 4 * THREADS) {
      uint4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i0 + k * THREADS < mid) v[k] = __ldcs(from16 + i0 + k * THREADS);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i0 + k * THREADS < mid) {
          to16[i0 + k * THREADS] = v[k];
#pragma unroll
          for (int j = 0; j < PER16; ++j) take(of_16(v[k], j), head + (i0 + k * THREADS) * PER16 + j);
        }
    }
    if (tid >= 32 && tid - 32 < tail) {
      const int i = n - tail + tid - 32;
      to[i] = reinterpret_cast<const E*>(src)[i];
      take(at(i), i);
    }
  } else {
    if (tid < head) take(at(tid), tid);
    const uint4* from16 = reinterpret_cast<const uint4*>(src + head * sizeof(E));
    for (int i0 = tid; i0 < mid; i0 += 4 * THREADS) {
      uint4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i0 + k * THREADS < mid) v[k] = __ldg(from16 + i0 + k * THREADS);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i0 + k * THREADS < mid)
#pragma unroll
          for (int j = 0; j < PER16; ++j) take(of_16(v[k], j), head + (i0 + k * THREADS) * PER16 + j);
    }
    if (tid >= 32 && tid - 32 < tail) take(at(n - tail + tid - 32), n - tail + tid - 32);
  }
  unsigned long long best = best_x > -INFINITY ? composite(best_x, begin + best_i) : 0ull;
  best = warp_fold(best, [](unsigned long long a, unsigned long long b) { return max(a, b); });
  low = warp_fold(low, [](float a, float b) { return fminf(a, b); });
  if (lane == 0) {
    part_u[warp][0] = best;
    part[warp][0] = low;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < WARPS; ++w) {
      best = max(best, part_u[w][0]);
      low = fminf(low, (float)part[w][0]);
    }
    sh.top = best;
    sh.low = low;
    n_list = 0;
  }
  meet();  // 1
  for (int c = 0; c < ctas; ++c) {
    const Shown* s = in_cta(&sh, c);
    best = c == 0 ? s->top : max(best, s->top);
    low = c == 0 ? s->low : fminf(low, s->low);
  }
  const float top = value_of(best);
  if (best == 0 || greedy) {
    if (rank == 0 && tid == 0) {
      p.tokens[r] = best == 0 ? -1 : index_of(best);
      if (p.probs) p.probs[r] = best == 0 ? 0.0f : 1.0f;
    }
    meet();  // no CTA ends while another reads what it shows
    return;
  }

  // ---- weights
  // The smallest f32 that counts: l - max l >= -40 T, decided in f64.  Near the
  // rounded sum as a rule; where that is next to zero, very many f32 give the same
  // difference in f64, and bisection over all of them finds it.
  float least_x = top;
  if (top < INFINITY) {
    auto in = [&](unsigned long long c) { return (double)value_of(c) - (double)top >= deepest; };
    constexpr unsigned long long kNext = 1ull << 32;
    const unsigned long long bottom = composite(-FLT_MAX, 0);
    unsigned long long c = composite(fmaxf((float)((double)top + deepest), -FLT_MAX), 0);
    if (!in(c)) c += kNext;
    if (c > bottom && in(c - kNext)) {
      c -= kNext;
      unsigned long long lo = bottom >> 32, hi = c >> 32;  // hi is in; the first that is lies in [lo, hi]
      if (c > bottom && in(c - kNext)) {
        while (lo < hi) {
          const unsigned long long half = (lo + hi) / 2;
          if (in(half << 32))
            hi = half;
          else
            lo = half + 1;
        }
        c = hi << 32;
      }
    }
    least_x = value_of(c);
  }
  auto weight = [&](float x) -> double {  // of a logit that counts; without a branch, so that several are under way
    const double d = (double)x - (double)top;
    // 2^(k / 64) e^r, |r| <= ln 2 / 128; the sum with 1.5 * 2^52 rounds to a whole number
    const double tk = fma(d, per_step, 6755399441055744.0);
    const int k = __double2loint(tk);
    const double kf = tk - 6755399441055744.0;
    const double rr = fma(kf, -0.010830424696249145, d * inv_t);
    const double q = fma(fma(fma(rr, 1.0 / 24, 1.0 / 6), rr, 0.5), rr, 1.0) * rr;
    const double s = table[k & 63];
    const double sc = __hiloint2double(__double2hiint(s) + ((k >> 6) << 20), __double2loint(s));
    return x == top ? 1.0 : fma(sc, q, sc);
  };
  // bins from the top down; the last one also takes what rounding puts past it
  const float span = fminf(top - low, (float)(kDepth * t64));
  const float per_unit = span > 0.0f && top < INFINITY ? fminf((float)NB / span, 1e37f) : 0.0f;
  auto bin_of = [&](float x) { return x == top ? 0 : min(NB - 1, (int)((top - x) * per_unit)); };
  // a bin's f32 mass: weights relative to the bin's upper end, in whole numbers
  const float unit = fminf(65536.0f, 2147483648.0f / (float)p.per);
  const float log2_t = fminf(1.4426950408889634f * (float)inv_t, 1e37f);
  const float bin_log2 = per_unit > 0.0f ? log2_t / per_unit : 0.0f;

  const bool k_cuts = top_k > 0 && top_k < p.vocab;
  const bool p_cuts = top_p < 1.0f;
  unsigned long long cut = 0;  // tokens with a composite from here on are in,
  int bin_cut = NB - 1;        // in bins up to this one
  bool decided = false;        // cut is

  // Sum of up to three values and two counts over the cluster, in the order of
  // threads and CTAs; every CTA gets them.
  int turn = 0;
  auto add_up = [&](double (&m)[3], int (&c)[2]) {
#pragma unroll
    for (int i = 0; i < 3; ++i) m[i] = warp_sum(m[i]);
    c[0] = __reduce_add_sync(0xffffffffu, c[0]);
    c[1] = __reduce_add_sync(0xffffffffu, c[1]);
    if (lane == 0) {
      for (int i = 0; i < 3; ++i) part[warp][i] = m[i];
      part_i[warp][0] = c[0];
      part_i[warp][1] = c[1];
    }
    __syncthreads();
    if (warp == 0) {
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const double s = warp_sum(lane < WARPS ? part[lane][i] : 0.0);
        if (lane == 0) sh.mass[turn][i] = s;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int s = __reduce_add_sync(0xffffffffu, lane < WARPS ? part_i[lane][i] : 0);
        if (lane == 0) sh.count[turn][i] = s;
      }
    }
    meet();
    m[0] = m[1] = m[2] = 0.0;
    c[0] = c[1] = 0;
    for (int q = 0; q < ctas; ++q) {
      const Shown* s = in_cta(&sh, q);
      for (int i = 0; i < 3; ++i) m[i] += s->mass[turn][i];
      c[0] += s->count[turn][0];
      c[1] += s->count[turn][1];
    }
    turn ^= 1;
  };

  const double least = (double)min_p;
  const bool m_cuts = least > 0.0;
  // f32 masses are needed where the mass alone says where the border lies
  const bool mass_bins = p_cuts && !k_cuts;
  auto histogram = [&](bool with_counts, bool with_masses) {
    for_each([&](float x, int) {
      if (x >= least_x) {
        const int b = bin_of(x);
        if (with_counts) atomicAdd(&counts[b], 1u);
        if (with_masses) {
          const float w = x == top ? 1.0f : ex2((x - top) * log2_t + (float)b * bin_log2);
          atomicAdd(&masses[b], (uint32_t)(fminf(w, 1.0f) * unit));
        }
      }
    });
  };
  if (k_cuts || p_cuts || m_cuts) {
    histogram(true, mass_bins);
    meet();  // 2: every CTA's bins
    // Every CTA adds up all the bins of the cluster, thread t bins t * each and on.
    constexpr int each_bins = NB / THREADS;
    uint32_t cn[each_bins];
    float ma[each_bins];
#pragma unroll
    for (int k = 0; k < each_bins; ++k) {
      cn[k] = 0;
      ma[k] = 0.0f;
    }
    static_assert(each_bins == 4, "one load");
    auto add_bins = [&](int at, uint32_t (&c)[4], float (&m)[4]) {  // four bins from `at` on, of every CTA
      for (int c0 = 0; c0 < ctas; c0 += 4) {  // four CTAs' loads under way
        uint4 v[4], w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v[k] = w[k] = make_uint4(0, 0, 0, 0);
          if (c0 + k < ctas) {
            v[k] = *reinterpret_cast<const uint4*>(in_cta(counts, c0 + k) + at);
            if (mass_bins) w[k] = *reinterpret_cast<const uint4*>(in_cta(masses, c0 + k) + at);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          c[0] += v[k].x;
          c[1] += v[k].y;
          c[2] += v[k].z;
          c[3] += v[k].w;
          m[0] += (float)w[k].x;
          m[1] += (float)w[k].y;
          m[2] += (float)w[k].z;
          m[3] += (float)w[k].w;
        }
      }
    };
    if (ctas <= 4) {
      add_bins(tid * each_bins, cn, ma);
    } else {
      // every CTA adds up its share of the bins and gives the sums to all (with
      // sixteen, all of them reading all the bins takes 6 us, this 2)
      // (not in the candidates' list: another CTA may begin to fill it before this one has read)
      uint32_t* sum_c = reinterpret_cast<uint32_t*>(ranked);
      static_assert(CAP * 8 >= NB * 4, "sums take the ranked candidates' place");
      const int share = NB / ctas;
      if (tid * 4 < share) {
        uint32_t c[4] = {0, 0, 0, 0};
        float m[4] = {0.f, 0.f, 0.f, 0.f};
        add_bins(rank * share + tid * 4, c, m);
        for (int k = 0; k < ctas; ++k) {
          *reinterpret_cast<uint4*>(const_cast<uint32_t*>(in_cta(sum_c, k)) + rank * share + tid * 4) =
              make_uint4(c[0], c[1], c[2], c[3]);
          if (mass_bins)
            *reinterpret_cast<float4*>(const_cast<float*>(in_cta(sum_m, k)) + rank * share + tid * 4) =
                make_float4(m[0], m[1], m[2], m[3]);
        }
      }
      meet();
#pragma unroll
      for (int k = 0; k < each_bins; ++k) {
        cn[k] = sum_c[tid * each_bins + k];
        if (mass_bins) ma[k] = sum_m[tid * each_bins + k];
      }
    }
    uint32_t c_in = 0;
    float m_in = 0.0f;
#pragma unroll
    for (int k = 0; k < each_bins; ++k) {
      if (mass_bins) ma[k] *= exp2f(-(float)(tid * each_bins + k) * bin_log2) / unit;
      c_in += cn[k];
      m_in += ma[k];
    }
    uint32_t c_upto = c_in;
    float m_upto = m_in;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t cc = __shfl_up_sync(0xffffffffu, c_upto, o);
      const float mm = __shfl_up_sync(0xffffffffu, m_upto, o);
      if (lane >= o) {
        c_upto += cc;
        m_upto += mm;
      }
    }
    if (lane == 31) {
      part_i[warp][0] = (int)c_upto;
      part[warp][0] = (double)m_upto;
    }
    // k bin; p bin, and bins that its border may lie in (f32 sums); tokens up to the last bin in, before the first in
    if (tid < 6) edge[tid] = tid < 3 ? NB - 1 : 0;
    __syncthreads();
    uint32_t c_at = c_upto - c_in, c_total = 0;
    float m_at = m_upto - m_in, m_total = 0.0f;
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) {
        c_at += (uint32_t)part_i[w][0];
        m_at += (float)part[w][0];
      }
      c_total += (uint32_t)part_i[w][0];
      m_total += (float)part[w][0];
    }
    // the bin of the k-th token, and that of the mass
    const float want32 = top_p * m_total;
    {
      uint32_t c = c_at;
      float m = m_at;
#pragma unroll
      for (int k = 0; k < each_bins; ++k) {
        // (the lowest of several, should rounding make there be any: every CTA has to find the same)
        if (k_cuts && c < (uint32_t)top_k && c + cn[k] >= (uint32_t)top_k) atomicMin(&edge[0], tid * each_bins + k);
        // A border this near to a bin's end may lie in the next one by the f64 sums: a bin's mass
        // falls short by up to a unit for each of its tokens, which are 0.97 of `unit` units
        // or more each, on both sides of the comparison, and f32 adds 2^-16 of it at most.
        const float near = m_total * fminf(1.0f, 8.0f / unit);
        if (mass_bins && cn[k] && m + ma[k] >= want32 - near) atomicMin(&edge[1], tid * each_bins + k);
        if (mass_bins && cn[k] && m + ma[k] >= want32 + near) atomicMin(&edge[2], tid * each_bins + k);
        c += cn[k];
        m += ma[k];
      }
    }
    __syncthreads();
    // The last bin that can hold a token that stays: the k-th token's; else the
    // mass's; min-p's.
    int m_bin = NB - 1;
    if (m_cuts && least > 1.0) {
      m_bin = 0;
    } else if (m_cuts && top < INFINITY && span > 0.0f) {
      // a logit below every one that min-p keeps
      m_bin = bin_of(value_of(composite(fmaxf(__double2float_rd((double)top + log(least) * t64), -FLT_MAX), 0) - (1ull << 32)));
    }
    // (top-p's share is of all that top-k leaves, min-p or not)
    int last_bin = k_cuts && p_cuts ? NB - 1 : m_bin;
    if (k_cuts) last_bin = min(last_bin, edge[0]);
    if (mass_bins) last_bin = min(last_bin, edge[2]);
    auto count_upto = [&](int b) {  // tokens in bins up to b, by the thread that has b
      uint32_t c = c_at;
#pragma unroll
      for (int k = 0; k < each_bins; ++k) {
        c += cn[k];
        if (tid * each_bins + k == b) return (int)c;
      }
      return -1;
    };
    if (tid == last_bin / each_bins) edge[4] = count_upto(last_bin);
    // p alone: only the bins around the border are looked at, if those before it are too many
    const int first_bin = mass_bins ? edge[1] : 0;
    if (tid == max(first_bin - 1, 0) / each_bins) edge[5] = first_bin > 0 ? count_upto(first_bin - 1) : 0;
    __syncthreads();
    const int upto = edge[4], before_first = edge[5];
    // min-p cuts before the mass does: the mass cuts nothing
    const bool by_m = mass_bins && m_bin < first_bin;
    const bool few = upto <= CAP, around = !few && mass_bins && !by_m && upto - before_first <= CAP;
    decided = !few && !k_cuts && (by_m || !p_cuts);
    if (few || around) {
      // ---- candidates to CTA 0, with the f64 sums of what is above and below them
      const int lo_bin = few ? 0 : first_bin;
      unsigned long long* to = const_cast<unsigned long long*>(in_cta(list, 0));
      int* counter = const_cast<int*>(in_cta(&n_list, 0));
      double m[3] = {0.0, 0.0, 0.0};
      int c[2] = {0, 0};
      if (mass_bins)
        for_each([&](float x, int i) {
          const bool in = x >= least_x;
          const int b = in ? bin_of(x) : NB;
          const bool taken = b >= lo_bin && b <= last_bin;
          if (taken) to[atomicAdd(counter, 1)] = composite(x, begin + i);
          const double w = weight(fmaxf(x, least_x));
          m[0] += b < lo_bin ? w : 0.0;
          m[1] += in && b > last_bin ? w : 0.0;
        });
      else
        for_each([&](float x, int i) {
          if (x >= least_x && bin_of(x) <= last_bin) to[atomicAdd(counter, 1)] = composite(x, begin + i);
        });
      if (mass_bins)
        add_up(m, c);
      else
        meet();
      if (rank == 0) {
        // ---- in order: few by counting the larger ones, with as many lanes as there are
        // threads for a candidate; more by a bitonic network
        const int nl = n_list;
        if (nl <= 256) {
          int lanes = 2;
          while (lanes < 32 && nl * lanes * 2 <= THREADS) lanes *= 2;
          const int i = tid / lanes;
          const unsigned long long key = i < nl ? list[i] : 0;
          int place = 0;
          for (int j = tid % lanes; j < nl; j += lanes) place += list[j] > key;
          for (int o = 1; o < lanes; o <<= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
          if (i < nl && tid % lanes == 0) ranked[place] = key;
        } else {
          for (int i = tid; i < CAP; i += THREADS) ranked[i] = i < nl ? list[i] : 0;
          sort_down(ranked, nl);
        }
        __syncthreads();
        // ---- weights, and the sums before them
        constexpr int E = CAP / THREADS;
        const int nk = k_cuts ? min(nl, top_k) : nl;
        double w[E], upto_w[E], sum = 0.0;
#pragma unroll
        for (int k = 0; k < E; ++k) {
          const int i = tid * E + k;
          w[k] = i < nk ? weight(value_of(ranked[i])) : 0.0;
          sum += w[k];
          upto_w[k] = sum;
        }
        double incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double v = shfl_up(incl, o);
          if (lane >= o) incl += v;
        }
        if (lane == 31) part[warp][0] = incl;
        if (tid == 0) edge[0] = 0;
        __syncthreads();
        double off = incl - sum, whole = 0.0;
        for (int v = 0; v < WARPS; ++v) {
          if (v < warp) off += part[v][0];
          whole += part[v][0];
        }
        const double want = (double)top_p * (m[0] + whole + m[1]);
        int stay = 0;
#pragma unroll
        for (int k = 0; k < E; ++k) {
          const int i = tid * E + k;
          const double before = m[0] + off + upto_w[k] - w[k];
          // (around the mass's border min-p is left to what follows)
          const bool in = i < nk && ((!p_cuts || before < want) && (!few || !(w[k] < least)) || (i == 0 && lo_bin == 0));
          stay += in;
        }
        stay = __reduce_add_sync(0xffffffffu, stay);  // those that stay come first
        if (lane == 0) atomicAdd(&edge[0], stay);
        __syncthreads();
        stay = edge[0];
        // The mass's border has to be among the candidates by the f64 sums, too (behind
        // the last bin min-p keeps nothing, and of all bins p next to 1 may leave all).
        const bool outside = mass_bins && ((last_bin < m_bin && m[0] + whole < want) || (lo_bin > 0 && !(m[0] < want)));
        if (tid == 0) {
          sh.verdict = outside ? 1 : 0;
          sh.cut = stay > 0 ? ranked[stay - 1] : 0;
        }
        if (few && !outside) {
          // ---- the token: those that stay, by their index
          double* by_index = reinterpret_cast<double*>(masses);
          uint32_t* index = reinterpret_cast<uint32_t*>(counts);
          static_assert(CAP * 8 <= NB * 4, "weights take the masses' place");
          if (stay <= 256) {
            int lanes2 = 2;
            while (lanes2 < 32 && stay * lanes2 * 2 <= THREADS) lanes2 *= 2;
            const int i = tid / lanes2;
            const unsigned long long key = i < stay ? ranked[i] : 0;
            int place = 0;  // the low half falls with the index
            for (int j = tid % lanes2; j < stay; j += lanes2) place += (uint32_t)ranked[j] > (uint32_t)key;
            for (int o = 1; o < lanes2; o <<= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
            if (i < stay && tid % lanes2 == 0) {
              by_index[place] = weight(value_of(key));
              index[place] = (uint32_t)index_of(key);
            }
          } else {
            for (int i = tid; i < CAP; i += THREADS)
              list[i] = i < stay ? (unsigned long long)(uint32_t)ranked[i] << 32 | (uint32_t)i : 0ull;
            sort_down(list, stay);
            for (int i = tid; i < stay; i += THREADS) {
              const unsigned long long key = ranked[(uint32_t)list[i]];
              by_index[i] = weight(value_of(key));
              index[i] = (uint32_t)index_of(key);
            }
          }
          __syncthreads();
          double s2 = 0.0, up[E];
#pragma unroll
          for (int k = 0; k < E; ++k) {
            const int i = tid * E + k;
            s2 += i < stay ? by_index[i] : 0.0;
            up[k] = s2;
          }
          double in2 = s2;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double v = shfl_up(in2, o);
            if (lane >= o) in2 += v;
          }
          if (lane == 31) part[warp][1] = in2;
          if (tid == 0) edge[1] = stay - 1;
          __syncthreads();
          double o2 = in2 - s2, total = 0.0;
          for (int v = 0; v < WARPS; ++v) {
            if (v < warp) o2 += part[v][1];
            total += part[v][1];
          }
          const double target = (u_in > 0.0f ? fmin((double)u_in, 1.0) : 0.0) * total;
#pragma unroll
          for (int k = E - 1; k >= 0; --k) {
            const int i = tid * E + k;
            if (i < stay && o2 + up[k] > target) atomicMin(&edge[1], i);
          }
          __syncthreads();
          if (tid == 0) {
            p.tokens[r] = (int)index[edge[1]];
            if (p.probs) p.probs[r] = (float)(by_index[edge[1]] / total);
          }
        }
      }
      meet();  // the verdict
      const Shown* s = in_cta(&sh, 0);
      const int verdict = s->verdict;
      const unsigned long long found = s->cut;
      meet();  // no CTA ends, or writes it again, while another reads it
      if (verdict == 0) {
        if (few) return;
        cut = found;
      }
      if (tid == 0) n_list = 0;
      __syncthreads();
      if (verdict == 0) decided = true;
    }
  }
  // ---- the general way: borders one after the other, whatever lies at them
  if ((k_cuts || p_cuts) && !decided) {
    if (p_cuts && !mass_bins) histogram(false, true);
    meet();
    // Each CTA adds up a range of the bins over the cluster.
    const int mine = NB / ctas, b0 = rank * mine;
    uint32_t cnt[NB / THREADS];
    float mas[NB / THREADS];
    // thread t of a CTA takes bins b0 + t * each ...
    const int each = (mine + THREADS - 1) / THREADS;
    uint32_t c_sum = 0;
    float m_sum = 0.0f;
#pragma unroll
    for (int k = 0; k < NB / THREADS; ++k) {
      cnt[k] = 0;
      mas[k] = 0.0f;
      const int b = b0 + tid * each + k;
      if (k < each && tid * each + k < mine) {
        for (int c = 0; c < ctas; ++c) {
          cnt[k] += in_cta(counts, c)[b];
          if (p_cuts) mas[k] += (float)in_cta(masses, c)[b];
        }
        mas[k] *= exp2f(-(float)b * bin_log2) / unit;
        c_sum += cnt[k];
        m_sum += mas[k];
      }
    }
    // sums before this thread's bins, within the CTA
    uint32_t c_incl = c_sum;
    float m_incl = m_sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t cc = __shfl_up_sync(0xffffffffu, c_incl, o);
      const float mm = __shfl_up_sync(0xffffffffu, m_incl, o);
      if (lane >= o) {
        c_incl += cc;
        m_incl += mm;
      }
    }
    if (lane == 31) {
      part_i[warp][0] = (int)c_incl;
      part[warp][0] = (double)m_incl;
    }
    __syncthreads();
    uint32_t c_before = c_incl - c_sum;
    float m_before = m_incl - m_sum;
    uint32_t c_cta = 0;
    float m_cta = 0.0f;
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) {
        c_before += (uint32_t)part_i[w][0];
        m_before += (float)part[w][0];
      }
      c_cta += (uint32_t)part_i[w][0];
      m_cta += (float)part[w][0];
    }
    if (tid == 0) {
      sh.bin_count = (int)c_cta;
      sh.bin_mass = m_cta;
      sh.found = 0;
    }
    meet();  // 3
    uint32_t c_all = 0;
    float m_all = 0.0f;
    for (int c = 0; c < ctas; ++c) {
      const Shown* s = in_cta(&sh, c);
      if (c < rank) {
        c_before += (uint32_t)s->bin_count;
        m_before += s->bin_mass;
      }
      c_all += (uint32_t)s->bin_count;
      m_all += s->bin_mass;
    }

    // Finds the exact border inside bin `b`, of which n_bin tokens come after
    // n_above others: by_mass false: the top_k-th token; true: the first with a
    // mass before it of at least top_p times that of all tokens in.  Sets cut; -1
    // or 1 where the border is not in this bin but above or below.
    auto border = [&](int b, int n_bin, long long n_above, bool by_mass) -> int {
      // composites of the bin between lo and hi (inclusive), n_bin of them; bisection
      unsigned long long lo = 0, hi = ~0ull;
      long long above = n_above;  // tokens above hi
      double total = 0.0;
      bool have_total = false;
      if (n_bin > CAP) {
        unsigned long long mn = ~0ull, mx = 0;
        for (int i = tid; i < n; i += THREADS) {
          const float x = at(i);
          if (x >= least_x && bin_of(x) == b) {
            const unsigned long long c = composite(x, begin + i);
            mn = min(mn, c);
            mx = max(mx, c);
          }
        }
        mn = warp_fold(mn, [](unsigned long long a, unsigned long long c) { return min(a, c); });
        mx = warp_fold(mx, [](unsigned long long a, unsigned long long c) { return max(a, c); });
        if (lane == 0) {
          part_u[warp][0] = mn;
          part_u[warp][1] = mx;
        }
        __syncthreads();
        if (tid == 0) {
          for (int w = 1; w < WARPS; ++w) {
            mn = min(mn, part_u[w][0]);
            mx = max(mx, part_u[w][1]);
          }
          sh.c_lo = mn;
          sh.c_hi = mx;
        }
        meet();
        lo = ~0ull;
        hi = 0;
        for (int c = 0; c < ctas; ++c) {
          const Shown* s = in_cta(&sh, c);
          lo = min(lo, s->c_lo);
          hi = max(hi, s->c_hi);
        }
        while (n_bin > CAP) {
          // tokens in [mid, hi], above hi
          const unsigned long long mid = lo + ((hi - lo) >> 1) + 1;
          double m[3] = {0.0, 0.0, 0.0};  // in [mid, hi] and above; all that are in
          int c[2] = {0, 0};
          for (int i = tid; i < n; i += THREADS) {
            const float x = at(i);
            if (!(x >= least_x)) continue;
            const unsigned long long k = composite(x, begin + i);
            if (k >= mid && k <= hi) ++c[0];
            if (by_mass && k >= cut) {
              const double w = weight(x);
              m[1] += w;
              if (k >= mid) m[0] += w;
            }
          }
          add_up(m, c);
          if (by_mass && !have_total) {
            total = m[1];
            have_total = true;
          }
          // the border is at or below mid's tokens where they do not hold all that is wanted
          const bool in_upper = by_mass ? !(m[0] < (double)top_p * total) : above + c[0] >= top_k;
          if (in_upper) {
            lo = mid;
            n_bin = c[0];
          } else {
            hi = mid - 1;
            above += c[0];
            n_bin -= c[0];
          }
          if (lo >= hi) break;
        }
      }
      // the candidates, to CTA 0; mass above them, mass of all that are in
      double m[3] = {0.0, 0.0, 0.0};
      int c[2] = {0, 0};
      unsigned long long* to = const_cast<unsigned long long*>(in_cta(list, 0));
      int* counter = const_cast<int*>(in_cta(&n_list, 0));
      for (int i = tid; i < n; i += THREADS) {
        const float x = at(i);
        if (!(x >= least_x)) continue;
        const unsigned long long k = composite(x, begin + i);
        const int bb = bin_of(x);
        const bool inside = bb == b && k >= lo && k <= hi && k >= cut;
        if (inside) {
          const int slot = atomicAdd(counter, 1);
          if (slot < CAP) to[slot] = k;
        }
        if (by_mass && k >= cut) {
          const double w = weight(x);
          m[1] += w;
          if (!inside && (bb < b || (bb == b && k > hi))) m[0] += w;
        }
      }
      add_up(m, c);
      if (rank == 0) {
        const int nl = min(n_list, CAP);
        for (int i = tid; i < nl; i += THREADS) {
          const unsigned long long k = list[i];
          int place = 0;
          for (int j = 0; j < nl; ++j) place += list[j] > k;
          ranked[place] = k;
        }
        __syncthreads();
        if (warp == 0) {
          int keep = 0, verdict = 0;
          if (!by_mass) {
            keep = (int)min((long long)nl, (long long)top_k - above);
          } else {
            const double want = (double)top_p * m[1];
            double before = m[0];
            // the first token is always in: its border cannot lie above the top
            if (!(before < want) && before > 0.0) verdict = -1;
            for (int j0 = 0; j0 < nl && verdict == 0; j0 += 32) {
              const double w = j0 + lane < nl ? weight(value_of(ranked[j0 + lane])) : 0.0;
              double incl = w;
#pragma unroll
              for (int o = 1; o < 32; o <<= 1) {
                const double v = shfl_up(incl, o);
                if (lane >= o) incl += v;
              }
              double prev = shfl_up(incl, 1);
              if (lane == 0) prev = 0.0;
              const bool in = j0 + lane < nl && (before + prev < want || (before == 0.0 && j0 + lane == 0));
              const unsigned ins = __ballot_sync(0xffffffffu, in);
              keep += __popc(ins);
              before += __shfl_sync(0xffffffffu, incl, 31);
              if (ins != 0xffffffffu) break;
            }
            if (verdict == 0 && keep == nl && before < want) verdict = 1;
          }
          if (lane == 0) {
            sh.verdict = verdict;
            sh.cut = keep > 0 ? ranked[keep - 1] : nl > 0 ? ranked[0] + 1 : 0;
            n_list = 0;
          }
        }
      }
      meet();
      const Shown* s = in_cta(&sh, 0);
      const int verdict = s->verdict;
      const unsigned long long found = s->cut;
      meet();  // before CTA 0 writes them again
      if (verdict == 0) cut = max(cut, found);
      return verdict;
    };

    // The bin that holds a border: shown by the CTA (of its range of bins) that has it.
    auto locate = [&](bool by_mass, float want, int& b, int& n_bin, long long& n_above) {
      uint32_t cb = c_before;
      float mb = m_before;
#pragma unroll
      for (int k = 0; k < NB / THREADS; ++k) {
        const int bb = b0 + tid * each + k;
        if (k < each && tid * each + k < mine && cnt[k]) {
          const bool here = by_mass ? mb < want && mb + mas[k] >= want : cb < (uint32_t)top_k && cb + cnt[k] >= (uint32_t)top_k;
          if (here) {
            sh.bin = bb;
            sh.n_bin = (int)cnt[k];
            sh.n_above = cb;
            sh.found = 1;
          }
        }
        cb += cnt[k];
        mb += mas[k];
      }
      meet();
      b = -1;
      for (int c = 0; c < ctas; ++c) {
        const Shown* s = in_cta(&sh, c);
        if (s->found && b < 0) {
          b = s->bin;
          n_bin = s->n_bin;
          n_above = s->n_above;
        }
      }
      meet();
      if (tid == 0) sh.found = 0;
      __syncthreads();
    };

    float k_mass = m_all;  // f32 mass of what the top-k leaves
    if (k_cuts && c_all > (uint32_t)top_k) {
      int b, n_bin;
      long long n_above;
      locate(false, 0.0f, b, n_bin, n_above);
      if (b >= 0) {
        border(b, n_bin, n_above, false);
        // for the mass that follows: the masses above the bin, a share of the bin's own
        if (p_cuts) {
          float mb = m_before, got = 0.0f;
          bool has = false;
#pragma unroll
          for (int k = 0; k < NB / THREADS; ++k) {
            if (k < each && tid * each + k < mine && b0 + tid * each + k == b) {
              got = mb + mas[k] * (float)(top_k - n_above) / (float)n_bin;
              has = true;
            }
            mb += mas[k];
          }
          if (has) {
            sh.bin_mass = got;
            sh.found = 1;
          }
          meet();
          for (int c = 0; c < ctas; ++c) {
            const Shown* s = in_cta(&sh, c);
            if (s->found) k_mass = s->bin_mass;
          }
          meet();
          if (tid == 0) sh.found = 0;
          __syncthreads();
        }
      }
    }
    if (p_cuts) {
      int b = 0, n_bin = 0;
      long long n_above = 0;
      const float want = fmaxf(top_p, 0.0f) * k_mass;
      if (want > 0.0f) locate(true, want, b, n_bin, n_above);
      if (b < 0) b = NB - 1;
      // By f64 sums the border may lie in another bin: steps that double, then
      // halves.  Where two neighbours send it to each other, it is between them.
      // (Where no bin is below the last, everything stays.)
      int above = -1, below = NB, step = 1;  // the border is below bin `above`, above bin `below`
      for (;;) {
        int nb = 0;
        for (int c = 0; c < ctas; ++c) nb += (int)in_cta(counts, c)[b];
        const int verdict = border(b, nb, 0, true);
        if (verdict == 0) break;
        if (verdict > 0)
          above = b;
        else
          below = b;
        if (below - above <= 1) {
          bin_cut = above;
          break;
        }
        b = above >= 0 && below < NB ? (above + below) / 2 : verdict > 0 ? min(NB - 1, b + step) : max(0, b - step);
        step *= 2;
      }
    }
  }

  // ---- the sum of what stays, and the token
  const float cut_x = cut ? value_of(cut) : -INFINITY;  // the last that is in, and its place
  const int cut_i = cut ? index_of(cut) - begin : 0;
  auto stays = [&](float x, int i, double& w) {
    bool in = x >= least_x && (x > cut_x || (x == cut_x && i <= cut_i));
    if (bin_cut < NB - 1) in = in && bin_of(x) <= bin_cut;
    w = weight(fmaxf(x, least_x));
    in = in && (!(w < least) || (x == top && begin + i == index_of(best)));
    w = in ? w : 0.0;
    return in;
  };
  // Tokens [i0, i1) of this CTA's, 32 neighbours at a time: the sum of their weights.
  auto mass_of = [&](int i0, int i1) {
    double a[4] = {0.0, 0.0, 0.0, 0.0};
    for (int i = i0 + lane; i < i1; i += 128) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        double w;
        stays(i + 32 * k < i1 ? at(i + 32 * k) : -INFINITY, i + 32 * k, w);
        a[k] += w;
      }
    }
    return warp_sum((a[0] + a[1]) + (a[2] + a[3]));
  };
  // The first of WARPS parts in which the sum passes the target (from `from` on, which
  // moves to the part's beginning); the last with any where rounding lets none: its last token.
  const auto part_of = [&](int column, double target, double& from) {
    double s = from;
    int own = -1, last_any = -1;
    for (int w = 0; w < WARPS; ++w) {
      const double m = part[w][column];
      if (m > 0.0) {
        last_any = w;
        if (own < 0 && s + m > target) {
          own = w;
          from = s;
        }
      }
      s += m;
    }
    if (own < 0) from = -INFINITY;
    return own < 0 ? last_any : own;
  };
  const int run = ((n + WARPS - 1) / WARPS + 31) & ~31;
  {
    const double mass = mass_of(min(n, warp * run), min(n, warp * run + run));
    if (lane == 0) part[warp][2] = mass;
  }
  __syncthreads();
  if (tid == 0) {
    double s = 0.0;
    for (int w = 0; w < WARPS; ++w) s += part[w][2];
    sh.cta_sum = s;
  }
  meet();
  double total = 0.0, before = 0.0;
  int last = -1;
  for (int c = 0; c < ctas; ++c) {
    const double s = in_cta(&sh, c)->cta_sum;
    if (c < rank) before += s;
    total += s;
    if (s > 0.0) last = c;
  }
  const double uu = u_in > 0.0f ? fmin((double)u_in, 1.0) : 0.0;
  const double target = uu * total;
  // the CTA in whose range the sum passes the target; the last with any where rounding lets none
  double acc = 0.0;
  int owner = -1;
  for (int c = 0; c < ctas && owner < 0; ++c) {
    acc += in_cta(&sh, c)->cta_sum;
    if (acc > target) owner = c;
  }
  if (owner < 0) owner = last;
  double before_own = before;
  if (rank == owner) {
    // the warp's run likewise, and of that run's sixteen parts the one
    const int w_own = part_of(2, target, before);
    const int r0 = min(n, w_own * run), r1 = min(n, r0 + run), sub = (run / WARPS + 31) & ~31;
    {
      const double mass = mass_of(min(r1, r0 + warp * sub), min(r1, r0 + warp * sub + sub));
      if (lane == 0) part[warp][0] = mass;
    }
    __syncthreads();
  }
  if (rank == owner && warp == 0) {
    const int r0 = min(n, part_of(2, target, before_own) * run), r1 = min(n, r0 + run), sub = (run / WARPS + 31) & ~31;
    double w_before = before_own;
    const int s_own = part_of(0, target, w_before);
    const int i0 = min(r1, r0 + s_own * sub), i1 = min(r1, i0 + sub);
    int pick = -1;
    double pick_w = 0.0;
    for (int i = i0; i < i1; i += 32) {
      double w = 0.0;
      const bool in = i + lane < i1 && stays(at(i + lane), i + lane, w);
      if (!in) w = 0.0;
      double incl = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double v = shfl_up(incl, o);
        if (lane >= o) incl += v;
      }
      const unsigned ins = __ballot_sync(0xffffffffu, in), over = __ballot_sync(0xffffffffu, in && w_before + incl > target);
      if (over) {
        const int l = __ffs(over) - 1;
        pick = i + l;
        pick_w = __shfl_sync(0xffffffffu, w, l);
        break;
      }
      if (ins) {  // the last so far
        const int l = 31 - __clz(ins);
        pick = i + l;
        pick_w = __shfl_sync(0xffffffffu, w, l);
      }
      w_before += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) {
      p.tokens[r] = pick < 0 ? -1 : begin + pick;
      if (p.probs) p.probs[r] = pick < 0 ? 0.0f : (float)(pick_w / total);
    }
  }
  meet();  // no CTA ends while another reads what it shows
}

// ------------------------------------------------------------------- host
constexpr int FIXED = NB * 12 + CAP * 16;        // bins and candidates
constexpr int kMaxKept = kSmemMax - FIXED - 8192;  // bytes of a row that a CTA can keep (the rest: static)

template <int kType, bool kKept>
int launch(const Params& p, int rows, int ctas, size_t smem, cudaStream_t st) {
  auto kern = sample_kernel<kType, kKept>;
  static DeviceMemo<kMaxCluster + 1> memo;  // clusters of a size that fit the GPU, with all the shared memory
  int fit = 0;
  const cudaError_t e = memo.get(ctas, &fit, [&](int* n) {
    cudaError_t r = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, FIXED + kMaxKept);
    if (r == cudaSuccess) r = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (r != cudaSuccess) return r;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = FIXED + kMaxKept;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaOccupancyMaxActiveClusters(n, kern, &cfg);
  });
  if (e != cudaSuccess) return cuda_status(e, "sample_tokens: occupancy query");
  if (fit < 1) return fail(-3, "sample_tokens: the kernel cannot be scheduled on this device");
  return launch_after("sample_kernel launch", kern, dim3((unsigned)(rows * ctas)), dim3(THREADS), smem, ctas, st, p, ctas);
}

}  // namespace sampling

int launch_sample_tokens(const Sampling& a, cudaStream_t st) {
  using namespace sampling;
  const int width = a.dtype == kF32 ? 4 : 2;
  Params p{};
  p.logits = static_cast<const uint8_t*>(a.logits);
  p.ld = a.ld * width;
  p.vocab = a.vocab;
  p.temperature = a.temperature;
  p.top_k = a.top_k;
  p.top_p = a.top_p;
  p.min_p = a.min_p;
  p.u = a.u;
  p.tokens = a.tokens;
  p.probs = a.probs;
  // CTAs of a row: two per SM while they have 1024 tokens each, more where the row
  // needs their shared memory.
  int ctas = 1;
  auto share = [&](int c) { return ((a.vocab + c - 1) / c + 31) / 32 * 32; };
  while (ctas < kMaxCluster && ((long long)a.rows * ctas * 2 <= 2 * num_sms() && a.vocab / (2 * ctas) >= 1024)) ctas *= 2;
  while (ctas < kMaxCluster && (long long)share(ctas) * width + 32 > kMaxKept) ctas *= 2;
  p.per = share(ctas);
  // Rows stay in shared memory where that leaves an SM room for two CTAs, or each CTA has an SM
  // to itself: one row of 150001 (top-k 40, top-p 0.9 / p alone) 22.5 / 43 us, read from L2 again for
  // every pass 24.6 / 47; 400 of 32000, f16, 49.1 / 113 and 49.2 / 115.  Where the row takes the
  // second CTA's room, the other way around: 64 rows of 128000 53 / 113 kept and 41 / 90 not, 400 of
  // 50000, f16, 80 / 199 and 68 / 168, 1000 of 32000 148 / 322 and 117 / 252.
  const long long bytes = (long long)p.per * width + 32, all = (long long)a.rows * ctas;
  const bool two = 2 * (FIXED + bytes + 4096) <= kSmemPerSm;
  const bool kept = bytes <= kMaxKept && (two || all <= num_sms());
  const size_t smem = FIXED + (kept ? (size_t)bytes : 0);
  ProfScope prof("sample_tokens", 0.0, (double)a.rows * a.vocab * width, st);
  if (a.rows > 0x7fffffff / kMaxCluster) return fail(-2, "sample_tokens: too many rows in one call");
  if (a.dtype == kF32) return kept ? launch<kF32, true>(p, a.rows, ctas, smem, st) : launch<kF32, false>(p, a.rows, ctas, smem, st);
  if (a.dtype == kBF16)
    return kept ? launch<kBF16, true>(p, a.rows, ctas, smem, st) : launch<kBF16, false>(p, a.rows, ctas, smem, st);
  return kept ? launch<kF16, true>(p, a.rows, ctas, smem, st) : launch<kF16, false>(p, a.rows, ctas, smem, st);
}

}  // namespace bonsai
