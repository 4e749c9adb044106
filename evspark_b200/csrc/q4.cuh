// The 4-bit format of the low-bit decode path (q4_linear.cu, q4_cache.cu, q4_attention.cu).
//
// A group of values shares a scale s; a code c in 1..15 stands for (c - 8) s.
//   s = absmax / 7 rounded to five significant bits (nearest, ties to even), stored as bf16;
//   c = 8 + round(x / s) (ties to even, at most 7 steps from 8);
//   absmax / 7 < 2^-120: s = 0, every code 8;
//   a NaN, an infinity or absmax / 7 > 2^120 in the group: s = NaN (the group reads back as NaN).
// Why five bits: |c - 8| has three significant bits, so (c - 8) s has at most eight, a bf16's. The
// decoded bf16 operands of a tensor-core product are then the held values themselves, with no
// rounding between the codes and the product. A scale off by at most 1/32 costs less than the
// codes' own rounding (absmax / s <= 7 (1 + 1/32) < 7.22, reached just below and at the tie 1 + 1/32, and holding
// such a value at 7 moves it by at most 0.22 s).
//
// Decoding two codes costs three instructions: a shift and a bitwise (w & mask) | 1.0 put the code
// into the top mantissa bits of 1.0 (1 + c / 16), and one bf16x2 fma gives
// (1 + c / 16) 16 s - 24 s = (c - 8) s. 16 s and 24 s (3 s 8: seven bits) are exact, and so is the
// fma's one rounding.
#pragma once

#include "common.cuh"

constexpr float Q4_TINY = 7.52316384526264e-37f;  // 2^-120
constexpr float Q4_HUGE = 1.329227995784916e36f;  // 2^120
constexpr int Q4_KV_GROUP = 32;                   // values per scale of the KV cache (along head_dim)
constexpr int Q4_KBLOCK = 128;                    // weights: input features are padded to a multiple of this

// Weights, codes, scales, page ids and partial results may be written by a kernel that still runs when their reader
// starts (programmatic launches): readers load them by ordinary loads behind pdl_wait(), never by the read-only path,
// which asks for data that nothing writes while the kernel lives.  So no __ldg, and no restrict on such inputs.
template <typename V>
__device__ __forceinline__ V q4_ld(const void* p) {
  return *reinterpret_cast<const V*>(p);
}

// fma of bf16 pairs
__device__ __forceinline__ uint32_t q4_fma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t q4_mul2(uint32_t a, uint32_t b) {
  return q4_fma2(a, b, 0x80008000u);  // + (-0): the product itself
}

// scale pair -> the two constants of the decoding fma: 16 s and -24 s
struct Q4Scale {
  uint32_t mul, add;
};
__device__ __forceinline__ Q4Scale q4_scale(uint32_t s2) {
  return {q4_mul2(s2, 0x41804180u), q4_mul2(s2, 0xC1C0C1C0u)};
}

// codes at bits 3 .. 6 of both halves of t -> the pair of values
__device__ __forceinline__ uint32_t q4_value(uint32_t t, const Q4Scale& s) {
  uint32_t m;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(m) : "r"(t), "r"(0x00780078u), "r"(0x3F803F80u));  // (t & mask) | 1.0
  return q4_fma2(m, s.mul, s.add);
}
// eight codes of one word -> value pairs (0,4) (1,5) (2,6) (3,7)
__device__ __forceinline__ void q4_word(uint32_t w, const Q4Scale& s, uint32_t (&v)[4]) {
  v[0] = q4_value(w << 3, s);
  v[1] = q4_value(w >> 1, s);
  v[2] = q4_value(w >> 5, s);
  v[3] = q4_value(w >> 9, s);
}

// d += a b, one m16n8k16 tensor-core product (bf16 operands, fp32 sums)
__device__ __forceinline__ void q4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A float as three bf16 parts that add up to it: truncated at eight bits, what is left truncated
// again, and the last eight bits. A product with an exact bf16 operand summed over the parts has
// fp32's accuracy. Infinities and NaN stay in the first part.
__device__ __forceinline__ void q4_parts(float x, uint32_t (&p)[3]) {
  const uint32_t h = __float_as_uint(x) & 0xFFFF0000u;
  p[0] = h >> 16;
  if ((h & 0x7F800000u) == 0x7F800000u) {
    if (x != x) p[0] = 0x7FC0u;
    p[1] = p[2] = 0u;
    return;
  }
  const float r = x - __uint_as_float(h);
  const uint32_t m = __float_as_uint(r) & 0xFFFF0000u;
  p[1] = m >> 16;
  p[2] = __float_as_uint(r - __uint_as_float(m)) >> 16;
}

// the scale of a group from its largest magnitude, as bf16 bits (t = absmax / 7)
__device__ __forceinline__ uint32_t q4_scale_bits(double absmax) {
  const double t = absmax / 7.0;
  if (!(t <= static_cast<double>(Q4_HUGE))) return 0x7FC0u;
  if (t < static_cast<double>(Q4_TINY)) return 0u;
  // five significant bits of a double: the implicit one and four of the 52 mantissa bits
  unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(t));
  b += 0x7FFFFFFFFFFFull + ((b >> 48) & 1ull);
  b &= ~0xFFFFFFFFFFFFull;
  const float s = static_cast<float>(__longlong_as_double(static_cast<long long>(b)));
  return __float_as_uint(s) >> 16;
}
// code of x under scale s (bf16 bits)
__device__ __forceinline__ uint32_t q4_code(double x, uint32_t scale_bits) {
  const float s = __uint_as_float(scale_bits << 16);
  if (!(s > 0.f)) return 8u;  // a group of zeros, or one that reads back as NaN
  const double q = rint(x / static_cast<double>(s));
  return static_cast<uint32_t>(8 + static_cast<int>(fmin(fmax(q, -7.0), 7.0)));
}
