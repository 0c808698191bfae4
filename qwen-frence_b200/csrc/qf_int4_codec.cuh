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

// A true division: T's coarse grid puts many quotients exactly between two codes, and the
// product with a rounded reciprocal would tip those either way.
__device__ __forceinline__ uint32_t int4_code(float x, const Int4Group& g) {
  if (!g.finite || g.step == 0.f) return 0u;
  const float n = rintf(__fdiv_rn(__fsub_rn(x, g.low), g.step));
  return static_cast<uint32_t>(fminf(fmaxf(n, 0.f), 15.f));
}

// n * step is exact in fp32 (4 + 11 bits), so this is one rounding of the value.
__device__ __forceinline__ float int4_value(uint32_t n, float step, float low) {
  return __fmaf_rn(static_cast<float>(n), step, low);
}

}  // namespace qf
