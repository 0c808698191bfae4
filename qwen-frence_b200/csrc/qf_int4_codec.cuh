// The 4-bit paged KV cache: layout of a tile and the codec of a group.
//
// A tile holds 16 tokens of one KV head, K and V together, in 20 * D bytes (D = 64 or 128):
// one contiguous block, so one bulk copy brings everything a warp needs for 16 tokens.
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
  float step, low;  // values of type T
  bool finite;
};

// step and floor of a group from its extremes (values of T), rounded to T as they are held.
template <typename T>
__device__ __forceinline__ Int4Group int4_group(float low, float high, bool finite) {
  Int4Group g;
  const float step = to_float(from_float<T>(__fdiv_rn(__fsub_rn(high, low), 15.f)));
  g.step = finite ? (step < kInt4MinStep ? 0.f : step) : __int_as_float(0x7fc00000);
  g.low = finite ? low : __int_as_float(0x7fc00000);
  g.finite = finite;
  return g;
}

// rint(x / step) as the nearest integers of correctly rounded quotients: T's coarse grid puts
// many quotients exactly between two codes, and the product with a rounded reciprocal alone
// would tip those either way.  With y the correctly rounded 1 / step, q = x y and the exact
// remainder x - q step, q + remainder * y is the correctly rounded quotient (Markstein, "Computation
// of elementary functions on the IBM RISC System/6000", 1990; steps of 11 bits at most are never
// the all-ones mantissa it excludes).  Adding 1.5 * 2^23 rounds to an integer, ties to even.
__device__ __forceinline__ float int4_code(float x, const Int4Group& g, float inverse) {
  const float t = __fsub_rn(x, g.low);
  const float q = __fmul_rn(t, inverse);
  const float n = __fmaf_rn(__fmaf_rn(-q, g.step, t), inverse, q);
  return __fsub_rn(__fadd_rn(fminf(n, 15.f), 12582912.f), 12582912.f);
}

// Eight codes as one word, the first in the low bits.  The sums are whole numbers below 2^16.
__device__ __forceinline__ uint32_t int4_word(const float (&x)[8], const Int4Group& g) {
  if (!g.finite || g.step == 0.f) return 0u;
  const float inverse = __frcp_rn(g.step);
  float half[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    half[k] = int4_code(x[4 * k + 3], g, inverse);
#pragma unroll
    for (int j = 2; j >= 0; --j) half[k] = __fmaf_rn(half[k], 16.f, int4_code(x[4 * k + j], g, inverse));
  }
  return static_cast<uint32_t>(half[0]) | static_cast<uint32_t>(half[1]) << 16;
}

// Four codes (bits 0..15 of `word`) as floats n, 16 n, 256 n, 4096 n: the bits laid into the
// mantissa of 2^23.  Products with step / 1, 16, 256, 4096 are those of n and step.
__device__ __forceinline__ void int4_scaled(uint32_t word, float (&n)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) n[j] = __fsub_rn(__uint_as_float((word & (15u << (4 * j))) | 0x4b000000u), 8388608.f);
}

// The values of eight codes.  n * step is exact in fp32 (4 + 11 bits), so each is one rounding.
__device__ __forceinline__ void int4_values(uint32_t word, float step, float low, float (&x)[8]) {
  const float steps[4] = {step, step * 0.0625f, step * 0.00390625f, step * 0.000244140625f};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float n[4];
    int4_scaled(word >> (16 * k), n);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[4 * k + j] = __fmaf_rn(n[j], steps[j], low);
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
