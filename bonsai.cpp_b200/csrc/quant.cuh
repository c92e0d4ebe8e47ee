// The cache formats of 8 and 4 bits.  A row of head_dim values is blocks of 32:
// whole numbers n, and one exponent byte e per block; the values are
// n * 2^(e - 127).
//
//   8 bits: byte n + 128, |n| <= 127, e = (biased f32 exponent of the block's largest magnitude) - 6
//   4 bits: nibble n + 8, |n| <= 7 (the even dimension in the low half), e = the same - 2
//
// n = x * 2^(127 - e) rounded to the nearest (ties to even) and cut to the
// largest, so a value is off by at most half of 2^(e - 127), the block's largest
// by less than one.  e is at least 1, for f16 at least 103: a step of 2^-24, f16's
// own.  A block of zeros has e = 0 (memory of zeros therefore reads as zeros),
// one that holds a NaN or an infinity e = 255 and n = 0; it reads as NaN, whatever n.
// A power of two as the scale, because n * 2^k is then exact in f16 and bf16: what
// a code stands for is the same number in a product of f16, of bf16, or in f32.
#pragma once
#include "internal.cuh"

namespace bonsai {
namespace quant {

enum Format : int { kI8 = 0, kI4 = 1 };
constexpr int kBlock = 32;
template <int kFmt>
constexpr int kRowBytes(int head_dim) { return kFmt == kI8 ? head_dim : head_dim / 2; }
template <int kFmt>
constexpr int kLower = kFmt == kI8 ? 6 : 2;
template <int kFmt>
constexpr uint32_t kZeroCodes = kFmt == kI8 ? 0x80808080u : 0x88888888u;
constexpr int kLowestF16 = 103, kLowestBF16 = 1;

template <bool kBF16>
__device__ __forceinline__ float low_f32(uint32_t pair) {
  if constexpr (kBF16)
    return __uint_as_float(pair << 16);
  else
    return __half2float(__ushort_as_half((unsigned short)(pair & 0xffffu)));
}
template <bool kBF16>
__device__ __forceinline__ float high_f32(uint32_t pair) {
  if constexpr (kBF16)
    return __uint_as_float(pair & 0xffff0000u);
  else
    return __half2float(__ushort_as_half((unsigned short)(pair >> 16)));
}
template <bool kBF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t y;
  if constexpr (kBF16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}

// The bytes of a word that are 255, as 0x80 each.
__device__ __forceinline__ uint32_t bytes_of_ones(uint32_t e4) {
  return ((e4 & 0x7f7f7f7fu) + 0x01010101u) & e4 & 0x80808080u;
}
// Exponent bytes as expand() below takes them: f16 as they are; bf16 six (I8) or
// two (I4) more, since it works with n / 64 or n / 4; zero and 255 are kept (the
// writer's are at most 248 and 252).
template <int kFmt, bool kBF16>
__device__ __forceinline__ uint32_t lift_exponents(uint32_t e4) {
  if constexpr (!kBF16) return e4;
  const uint32_t some = (((e4 & 0x7f7f7f7fu) + 0x7f7f7f7fu) | e4) & 0x80808080u & ~bytes_of_ones(e4);
  return e4 + (some >> 7) * (kFmt == kI8 ? 6u : 2u);
}
// The scales of two (lifted) exponents as a pair of 16-bit values; 0 gives zero, 255
// NaN: in f16 by the lowest bit of the f32, which the rounding of a number takes off.
template <bool kBF16>
__device__ __forceinline__ uint32_t scale_pair(uint32_t ea, uint32_t eb) {
  if constexpr (kBF16)
    return (ea == 255u ? 0x7fc0u : ea << 7) | (eb == 255u ? 0x7fc00000u : eb << 23);
  else
    return pack16<false>(__uint_as_float(ea << 23 | 1u), __uint_as_float(eb << 23 | 1u));
}
// The same from byte `at` of two words, but infinity for 255 in bf16.
template <bool kBF16>
__device__ __forceinline__ uint32_t scale_pair_at(uint32_t wa, uint32_t wb, uint32_t at) {
  if constexpr (kBF16) {
    return (__byte_perm(wa, wb, 0x0400u + at * 0x0101u) & 0x00ff00ffu) << 7;
  } else {
    const uint32_t top = at * 0x1000u + 0x0554u;  // the byte at the top, zeros below and the lowest bit
    return pack16<false>(__uint_as_float(__byte_perm(wa, 2u, top) >> 1), __uint_as_float(__byte_perm(wb, 2u, top) >> 1));
  }
}

__device__ __forceinline__ uint32_t add_f16x2(uint32_t a, uint32_t b) {
  uint32_t y;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t y;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(a), "r"(b), "r"(c));
  return y;
}
template <bool kBF16>
__device__ __forceinline__ uint32_t mul16x2(uint32_t a, uint32_t b) {
  uint32_t y;
  if constexpr (kBF16)
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  else
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b));
  return y;
}

// The pair number kJ of a word of codes, times `scale`: the codes whose low bits
// are at 8 kJ (4 kJ for 4 bits) of each half of the word.  Every step is exact.
// f16: the code is set into the mantissa of 1024 (of 64, four bits higher), and
// what is too much is taken off.  bf16 has 7 bits of mantissa, an 8-bit code does
// not fit; but as the low bits of a bf16 the code c is c * 2^-133, so c * 2^-6 - 2 is
// one multiply-add, and the exponents are lifted by six (4 bits: c / 4 - 2).  One
// logic operation per pair, of the pipe that is busiest (two and a half in bf16
// before: 105 us for 64 single tokens, 83 so; chunks 446 and 367).
template <int kFmt, bool kBF16, int kJ>
__device__ __forceinline__ uint32_t expand(uint32_t word, uint32_t scale) {
  uint32_t n;
  if constexpr (kFmt == kI8) {
    static_assert(kJ < 2, "two codes to a half word");
    if constexpr (kBF16)
      n = fma_bf16x2(kJ == 0 ? word & 0x00ff00ffu : __byte_perm(word, 0u, 0x4341), 0x7f007f00u, 0xc000c000u);  // 2^127, - 2
    else
      n = add_f16x2(kJ == 0 ? (word & 0x00ff00ffu) | 0x64006400u : __byte_perm(word, 0x64646464u, 0x4341),
                    0xe480e480u);  // - 1152
  } else {
    static_assert(kJ < 4, "four codes to a half word");
    const uint32_t w = kJ < 2 ? word : word >> 8;
    if constexpr (kBF16) {
      if constexpr ((kJ & 1) == 0)
        n = fma_bf16x2((w & 0x000f000fu) | 0x43004300u, 0x3e803e80u, 0xc208c208u);  // (128 + c) / 4 - 34
      else
        n = fma_bf16x2(w & 0x00f000f0u, 0x7f007f00u, 0xc000c000u);  // 16 c 2^-133 2^127 - 2
    } else if constexpr ((kJ & 1) == 0) {
      n = add_f16x2((w & 0x000f000fu) | 0x64006400u, 0xe408e408u);  // - 1032
    } else {
      n = add_f16x2((w & 0x00f000f0u) | 0x54005400u, 0xd480d480u);  // - 72
    }
  }
  return mul16x2<kBF16>(n, scale);
}

// expand() with what is taken off times the scale at hand (`off`, of expand_offsets), in
// one multiply-add of f16: for scales up to 2^5 (exponents below kSmallExponent),
// beyond which the product of 1152 and the scale is no f16.
constexpr uint32_t kSmallExponent = 133;
// Whether a byte is kSmallExponent or more.
__device__ __forceinline__ bool large_exponent(uint32_t e4) {
  return (((e4 & 0x7f7f7f7fu) + 0x7b7b7b7bu) & e4 & 0x80808080u) != 0;
}
struct Offsets {
  uint32_t even, odd;
};
template <int kFmt>
__device__ __forceinline__ Offsets expand_offsets(uint32_t scale) {
  if constexpr (kFmt == kI8) {
    const uint32_t o = mul16x2<false>(scale, 0xe480e480u);  // - 1152
    return {o, o};
  } else {
    return {mul16x2<false>(scale, 0xe408e408u), mul16x2<false>(scale, 0xd480d480u)};  // - 1032, - 72
  }
}
template <int kFmt, int kJ>
__device__ __forceinline__ uint32_t expand_small(uint32_t word, uint32_t scale, const Offsets& off) {
  uint32_t c;
  if constexpr (kFmt == kI8) {
    c = kJ == 0 ? (word & 0x00ff00ffu) | 0x64006400u : __byte_perm(word, 0x64646464u, 0x4341);
  } else {
    const uint32_t w = kJ < 2 ? word : word >> 8;
    c = (kJ & 1) == 0 ? (w & 0x000f000fu) | 0x64006400u : (w & 0x00f000f0u) | 0x54005400u;
  }
  uint32_t y;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(y) : "r"(c), "r"(scale), "r"((kJ & 1) == 0 ? off.even : off.odd));
  return y;
}

// One side of a cache as the kernels address it (bytes).
struct Pages {
  uint8_t* codes = nullptr;
  long long page = 0, token = 0, head = 0;
  uint8_t* scales = nullptr;
  long long s_page = 0, s_token = 0, s_head = 0;
};
// The cache and its page table.
struct Cache {
  Pages k, v;
  const int* table = nullptr;
  long long table_ld = 0;
  int table_width = 0, page_shift = 0, n_pages = 0;
};

}  // namespace quant

struct QuantAttention {
  TextTensor q, out;
  quant::Cache cache;
  const int* cu = nullptr;
  const int* ctx = nullptr;
  int n_seqs = 0, total_q = 0, max_q = 0, max_ctx = 0;
  int n_heads = 0, n_kv = 0, head_dim = 0, format = 0;
  bool bf16 = false;
  float scale = 0.f;
};
int launch_quant_attention(const QuantAttention& a, cudaStream_t st);
int launch_quant_append(const TextTensor& k, const TextTensor& v, const quant::Cache& c, const int* cu, const int* ctx,
                        int n_seqs, int total, int n_kv, int head_dim, int format, bool bf16, cudaStream_t st);
// first: place of each sequence's first row (null: 0)
int launch_quant_read(const quant::Cache& c, const int* cu, const int* first, int n_seqs, int total, int n_kv,
                      int head_dim, int format, bool bf16, const TextTensor& k, const TextTensor& v, cudaStream_t st);

}  // namespace bonsai
