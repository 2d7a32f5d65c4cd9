// Weight levels from bit planes to 16-bit float operands.
//
// `gather_fields` turns the words of the planes (32 elements, element k in bit 31 - k) into words of fields, each field one
// element's level: masked merges, log2(planes) stages of them.  `level_pair` takes the same field of the two halves of such
// a word to a pair of 16-bit floats level - zero: a field at bit `pos` inside the mantissa, under the exponent that gives this bit
// the weight 1, is 2^(mantissa bits - pos) + level, so one LOP3 sets the exponent and one addition takes away 2^(..) + zero.
// Both are exact: zero is a multiple of 1/2 up to 15 and 2^(..) + zero keeps its half for pos >= 1; a field at bit 0 takes two
// additions.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace apnn {

// (a & b) | c and (a & b) | (c & ~b), one instruction each whatever the compiler makes of the constants
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t select_bits(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xE2;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

template <int WB>
struct Fields {
  static constexpr int WORDS = WB == 1 ? 1 : WB == 2 ? 2 : 4;       // three planes count as four
  static constexpr int WIDTH = WB == 1 ? 1 : WB == 2 ? 2 : 4;       // bits of a field
  static constexpr int PER_HALF = 16 / WIDTH;
};

// Word i of the result holds, in field j, the element at bit WIDTH * j + i of the planes.
template <int WB>
__device__ __forceinline__ void gather_fields(const uint32_t (&p)[WB], uint32_t (&f)[Fields<WB>::WORDS]) {
  if constexpr (WB == 1) {
    f[0] = p[0];
  } else {
    const uint32_t a0 = select_bits(p[0], 0x55555555u, p[1] << 1), a1 = select_bits(p[0] >> 1, 0x55555555u, p[1]);
    if constexpr (WB == 2) {
      f[0] = a0;
      f[1] = a1;
    } else {
      uint32_t c0, c1;
      if constexpr (WB == 3) {
        c0 = p[2] & 0x55555555u;
        c1 = (p[2] >> 1) & 0x55555555u;
      } else {
        c0 = select_bits(p[2], 0x55555555u, p[3] << 1);
        c1 = select_bits(p[2] >> 1, 0x55555555u, p[3]);
      }
      f[0] = select_bits(a0, 0x33333333u, c0 << 2);
      f[1] = select_bits(a1, 0x33333333u, c1 << 2);
      f[2] = select_bits(a0 >> 2, 0x33333333u, c0);
      f[3] = select_bits(a1 >> 2, 0x33333333u, c1);
    }
  }
}

// How far a half word is shifted before field `j` is taken: few different shifts, the field inside the mantissa, not at bit 0.
template <int WIDTH, bool BF16>
__host__ __device__ constexpr int field_shift(int j) {
  if (WIDTH == 4) return j == 0 ? 0 : BF16 ? 4 * j - 3 : 4 * (j - 1);
  if (WIDTH == 2) return BF16 ? (j < 3 ? 0 : j < 5 ? 4 : j < 7 ? 8 : 10) : (j < 5 ? 0 : 8);
  return BF16 ? (j < 7 ? 0 : j < 13 ? 6 : 12) : (j < 10 ? 0 : 8);
}

// -(2^(mantissa bits - pos) + zero), twice; pos 0: -2^(mantissa bits) alone, `zero` itself in `none`.
template <bool BF16>
struct ZeroPoint {
  uint32_t at[10], none;
  __device__ __forceinline__ explicit ZeroPoint(float zero) {
#pragma unroll
    for (int p = 0; p < 10; p++) at[p] = both(-((float)(1 << ((BF16 ? 7 : 10) - (p < (BF16 ? 7 : 10) ? p : 0))) + (p == 0 ? 0.0f : zero)));
    none = both(-zero);
  }
  __device__ __forceinline__ static uint32_t both(float x) {
    if (BF16) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(x, x);
      return *reinterpret_cast<const uint32_t*>(&v);
    }
    const __half2 v = __floats2half2_rn(x, x);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
};

template <bool BF16>
__device__ __forceinline__ uint32_t add16x2(uint32_t a, uint32_t b) {
  if (BF16) {
    const __nv_bfloat162 v = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __hadd2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Field j of both halves of w (STRIDE * j bits up, BITS wide) as level - zero.
template <int STRIDE, bool BF16, int BITS = STRIDE>
__device__ __forceinline__ uint32_t level_pair(uint32_t w, int j, const ZeroPoint<BF16>& z) {
  constexpr int MANTISSA = BF16 ? 7 : 10;
  const int shift = field_shift<STRIDE, BF16>(j), pos = STRIDE * j - shift;
  const uint32_t mask = (((1u << BITS) - 1u) << pos) * 0x00010001u;
  const uint32_t exponent = (uint32_t)(((BF16 ? 127 : 15) + MANTISSA - pos) << MANTISSA) * 0x00010001u;
  const uint32_t v = add16x2<BF16>(and_or(w >> shift, mask, exponent), z.at[pos]);
  return pos == 0 ? add16x2<BF16>(v, z.none) : v;
}

// The 32 elements of a word of each plane as 16 pairs in order, pair j = elements 2 j (low half) and 2 j + 1.
template <int WB, bool BF16>
__device__ __forceinline__ void spread_in_order(const uint32_t (&p)[WB], const ZeroPoint<BF16>& z, uint32_t (&out)[16]) {
  if constexpr (WB <= 2) {
    uint32_t even, odd;      // field i: elements 30 - 2 i, 31 - 2 i
    if constexpr (WB == 1) {
      even = p[0] >> 1;
      odd = p[0];
    } else {
      uint32_t f[2];
      gather_fields<2>(p, f);
      even = f[1];
      odd = f[0];
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const uint32_t x = __byte_perm(even, odd, h ? 0x7632 : 0x5410);
#pragma unroll
      for (int i = 0; i < 8; i++) out[15 - 8 * h - i] = level_pair<2, BF16, WB>(x, i, z);
    }
  } else {
    uint32_t f[4];           // field i of f[q]: element 31 - 4 i - q
    gather_fields<WB>(p, f);
#pragma unroll
    for (int q = 0; q < 4; q += 2)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint32_t x = __byte_perm(f[q + 1], f[q], h ? 0x7632 : 0x5410);
#pragma unroll
        for (int i = 0; i < 4; i++) out[15 - q / 2 - 2 * (4 * h + i)] = level_pair<4, BF16>(x, i, z);
      }
  }
}

}  // namespace apnn
