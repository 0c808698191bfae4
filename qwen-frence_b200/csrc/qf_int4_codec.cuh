// The 4-bit paged KV cache: layout of a tile and the codec of a group.
//
// A tile holds 16 tokens of one KV head, K and V together, in 20 * D bytes (D = 64 or 128):
// one contiguous block, which a warp fetches whole, 16 bytes a lane side by side.
// Every 32 consecutive channels of a row are a group with a step and a floor in the element
// type T of the queries; a channel is a code n in 0..15 and stands for n * step + floor:
//     floor = min(x),  step = T((max(x) - min(x)) / 15),  n = rint((x - floor) / step)
// 5 bits a channel in all.  For normal values a group of 32 is off by 0.08 of their standard
// deviation, a group of 64 by 0.09, a row of 128 by 0.11, and a channel with a large offset
// (K has them after a projection with bias) coarsens its own group alone; 64 would save a
// tenth of the bytes.  A step below 2^-60 (bf16 only) is held as 0: its quotients could
// overflow, and the group is then its floor to within 15 * 2^-60.  A group with an infinity
// or a NaN in it is NaN as a whole.
//
// Bytes of a tile, W = D / 32 groups a row:
//     [0, 8D)     K codes [16 tokens][4 t][W][4]: word (t, w) holds channels 32w + 8t + j, j in
//                 bits 4j..4j+3.  A lane of an m16n8k16 A fragment (rows = tokens) reads its
//                 4W bytes of a token with one load.
//     [8D, 16D)   V codes [8 pairs][8 g][W][4]: word (g, w) holds channels 32w + 4g + j of token
//                 2 * pair in bits 4j..4j+3 and of token 2 * pair + 1 in bits 16 + 4j..: the two
//                 halves of an A fragment register (rows = channels, columns = tokens).
//     [16D, 20D)  K steps [16][W], K floors [16][W], V steps [16][W], V floors [16][W], type T
#pragma once

#include "qf_common.cuh"

namespace qf {

constexpr int kInt4Tile = 16;    // tokens of a tile
constexpr int kInt4Group = 32;   // channels of a group
constexpr float kInt4MinStep = 8.673617379884035e-19f;  // 2^-60

__host__ __device__ constexpr int int4_tile_bytes(int head_dim) { return 20 * head_dim; }

struct Int4Group {
  float step, low;  // values of type T, NaN where the group is not finite
};

// Minimum and maximum that keep a NaN, of three.
__device__ __forceinline__ float min_nan(float a, float b, float c) {
  float r;
  asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Correctly rounded x / d from y, the correctly rounded 1 / d: q = x y, and the exact remainder
// x - q d times y added to it (Markstein, "Computation of elementary functions on the IBM RISC
// System/6000", 1990; a d of 11 bits or fewer is never the all-ones mantissa it excludes).
__device__ __forceinline__ float divide_by(float x, float d, float y) {
  const float q = __fmul_rn(x, y);
  return __fmaf_rn(__fmaf_rn(-q, d, x), y, q);
}

// step and floor of a group from its extremes (values of T, NaN if the group holds one), rounded
// to T as they are held.
template <typename T>
__device__ __forceinline__ Int4Group int4_group(float low, float high) {
  Int4Group g;
  const float range = __fsub_rn(high, low);
  const float step = to_float(from_float<T>(divide_by(range, 15.f, 1.f / 15.f)));
  const bool finite = range <= 3.402823466e38f;
  g.step = finite ? (step < kInt4MinStep ? 0.f : step) : __int_as_float(0x7fc00000);
  g.low = finite ? low : __int_as_float(0x7fc00000);
  return g;
}

// Eight codes as one word, the first in the low bits.  T's coarse grid puts many quotients exactly
// between two codes, and the product with a rounded reciprocal alone would tip those either way:
// the quotients are correctly rounded.  Adding 1.5 * 2^23 rounds to an integer, ties to even; four
// codes are summed as one number below 2^16 and read off the mantissa of 2^23.
__device__ __forceinline__ uint32_t int4_word(const float (&x)[8], const Int4Group& g) {
  if (!(g.step > 0.f)) return 0u;
  const float inverse = __frcp_rn(g.step);
  uint32_t half[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float sum = 0.f;
#pragma unroll
    for (int j = 3; j >= 0; --j) {
      const float n = fminf(divide_by(__fsub_rn(x[4 * k + j], g.low), g.step, inverse), 15.f);
      sum = __fmaf_rn(sum, 16.f, __fsub_rn(__fadd_rn(n, 12582912.f), 12582912.f));
    }
    half[k] = __float_as_uint(__fadd_rn(sum, 8388608.f));
  }
  return __byte_perm(half[0], half[1], 0x5410);
}

__device__ __forceinline__ uint64_t pair32(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair32(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
// Two products, sums, or products and sums in one instruction, each rounded once.
__device__ __forceinline__ uint64_t mul32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// The values of eight codes.  Four codes laid into the mantissa of 2^23 are n, 16 n, 256 n and
// 4096 n above it; with step / 1, 16, 256 and 4096 their products are those of n and step, exact in
// fp32 (4 + 11 bits), so each value is one rounding.
__device__ __forceinline__ void int4_values(uint32_t word, float step, float low, float (&x)[8]) {
  const uint64_t steps[2] = {pair32(step, step * 0.0625f), pair32(step * 0.00390625f, step * 0.000244140625f)};
  const uint64_t lows = pair32(low, low), minus = pair32(-8388608.f, -8388608.f);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t half = word >> (16 * k);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint64_t n = add32x2(pair32(__uint_as_float((half & (15u << (8 * j))) | 0x4b000000u),
                                        __uint_as_float((half & (240u << (8 * j))) | 0x4b000000u)), minus);
      const float2 two = unpair32(fma32x2(n, steps[j], lows));
      x[4 * k + 2 * j] = two.x, x[4 * k + 2 * j + 1] = two.y;
    }
  }
}

// n / d and n % d for n < 2^31 by a product: with 2^(s - 1) < d <= 2^s and m = ceil(2^(31 + s) / d),
// floor(n m / 2^(31 + s)) is the quotient (Granlund and Montgomery, "Division by invariant
// integers using multiplication", 1994).
struct Divisor {
  uint32_t d, m;
  int shift;
};
inline Divisor make_divisor(uint32_t d) {
  Divisor r{d, 0, 0};
  if (d > 1) {
    int s = 1;
    while ((1ull << s) < d) ++s;
    r.m = static_cast<uint32_t>(((1ull << (31 + s)) + d - 1) / d);
    r.shift = s - 1;
  }
  return r;
}
__device__ __forceinline__ uint32_t quotient(uint32_t n, const Divisor& d) {
  return d.d == 1 ? n : __umulhi(n, d.m) >> d.shift;
}

}  // namespace qf
