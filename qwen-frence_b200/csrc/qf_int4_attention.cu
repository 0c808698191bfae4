// GQA decode attention over the 4-bit paged KV cache (layout: qf_int4_codec.cuh): one query
// token a sequence, a block table a sequence or one a (sequence, KV head).
//
// Mathematics.  A row is a (sequence, KV head) with up to 16 query heads.  For a tile of 16
// tokens, with K codes n, steps a and floors b of 32-channel groups w,
//     s[t, h] = sum_w a[t, w] * (sum_{d in w} n[t, d] q[d, h]) + sum_w b[t, w] * (sum_{d in w} q[d, h])
// so the codes go into the tensor cores as they are: a code in the low bits of an fp16 is the
// subnormal n * 2^-24, which m16n8k16 multiplies exactly; four bits higher it is n * 2^-20, and
// q carries the 1/16.  One AND makes two matrix elements.  Steps meet the fp32 sums of a group,
// floors are one more product.  With p = exp2(s - offset) and V codes m, steps c, floors e,
//     o[d, h] = sum_t (p[t, h] c[t, w(d)]) m[t, d] + sum_t p[t, h] e[t, w(d)]
// where p c is rounded to fp16 (2^-11 of a weight; the products and sums are fp32).  The offset
// is the running maximum of s plus that of log2(c) less 10, so p c stays between 2^-14 and 2^15
// for all weights down to 2^-24 of the largest, whatever the magnitude of V; it is raised, and the
// sums rescaled, only when a score or a step exceeds what the last offset allows by 2^4.
//
// Work.  Rows are laid end to end as tiles and every CTA takes an equal share of them, every warp
// of the CTA an equal share of that, whatever rows it covers.  A warp streams its tiles, 20 * D
// contiguous bytes each, through a ring of bulk copies of its own; warps share nothing until
// their tiles are done.  A row that one warp holds whole is written from its registers; what the
// warps of a CTA hold of one row is summed at the CTA's end, and rows that span CTAs by a second
// kernel, in the order of the tiles: the same call gives the same bits.
#include "qf_int4_paged.cuh"

namespace qf {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr uint32_t kBadTile = 0xffffffffu;
constexpr float kLog2e = 1.4426950408889634f;

// Bytes of shared memory of a warp's ring, and tiles in it.
template <int D, int NT>
struct Shape {
  static constexpr int kTileBytes = 20 * D;
  static constexpr int kStages = (NT == 1 ? 12800 : 25600) / kTileBytes;  // D 128: 5 or 10, D 64: 10 or 20
  static constexpr int kRing = kStages * kTileBytes;
  static constexpr int kHeads = 8 * NT;        // query heads a row has room for
  static constexpr int kStride = D + 4;        // floats between heads of a piece: its float4 stores miss no bank
  static constexpr int kPiece = kHeads * kStride + 2 * kHeads;  // floats: o, then offset and sum of every head
  static constexpr int kCtasPerSm = NT == 1 ? 2 : 1;
  static constexpr int kSmem = kWarps * kRing;
  static_assert(kPiece * 4 <= kRing, "a piece fits its warp's ring");
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ void mma_t(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_t<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  mma_f16(c, a0, a1, a2, a3, b0, b1);
}
template <>
__device__ __forceinline__ void mma_t<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                     uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8 x 8 transpose of 16-bit elements across the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float pow2i(int e) {  // 2^e, e in [-126, 127]
  return __int_as_float((e + 127) << 23);
}

__device__ __forceinline__ bool wait_stage(uint32_t bar, uint32_t parity) {
  for (int spin = 0; spin < (1 << 20); ++spin) {
    uint32_t done;
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(done)
                 : "r"(bar), "r"(parity)
                 : "memory");
    if (done) return true;
  }
  return false;
}

// What a call shares out: tiles of all rows, tiles of a CTA.
struct Plan {
  int64_t units;
  int64_t share;
};

// Thread-chunk prefix sums of the rows' tiles: s_prefix[i] = tiles before thread i's rows.
__device__ __forceinline__ Plan make_plan(const PagedInt4& p, int64_t* s_prefix, int64_t* s_warp, int chunk, int ctas) {
  const int rows = p.batch * p.kv_heads;
  const int first = threadIdx.x * chunk;
  int64_t mine = 0;
  for (int r = first; r < first + chunk && r < rows; ++r) mine += (row_tokens(p, r / p.kv_heads, r % p.kv_heads) + kInt4Tile - 1) / kInt4Tile;
  int64_t sum = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, sum, off);
    if ((threadIdx.x & 31) >= off) sum += up;
  }
  if ((threadIdx.x & 31) == 31) s_warp[threadIdx.x >> 5] = sum;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < (threadIdx.x >> 5)) before += s_warp[w];
    total += s_warp[w];
  }
  s_prefix[threadIdx.x] = before + sum - mine;
  __syncthreads();
  Plan plan;
  plan.units = total;
  plan.share = (total + ctas - 1) / ctas;
  if (plan.share < kWarps) plan.share = kWarps;  // a tile a warp at least: fewer pieces for the second kernel
  return plan;
}

// Tiles of 32 units ahead: lane i holds the tile, the tokens in it and the row of unit i.
struct Batch {
  uint32_t tile;
  int meta;  // tokens 1..16, kRowStart, kRowEnd
  int row;
};
constexpr int kRowStart = 32, kRowEnd = 64;

struct Walk {
  int row;    // next unit's row and tile in the row
  int tile;
  int left;   // units not described yet
  int base;   // row of lane 0's length
  int length; // tokens of row base + lane
};

__device__ __forceinline__ void load_lengths(const PagedInt4& p, Walk& w, int lane) {
  const int rows = p.batch * p.kv_heads;
  w.base = w.row;
  const int r = w.row + lane;
  w.length = r < rows ? static_cast<int>(row_tokens(p, r / p.kv_heads, r % p.kv_heads)) : 0;
}

__device__ __forceinline__ void next_batch(const PagedInt4& p, Walk& w, Batch& b, int lane) {
  const int per_page = p.page_size / kInt4Tile;
  int filled = 0, mine = -1, tokens = 0;
  b.row = 0;
  while (filled < 32 && w.left > 0 && w.row < p.batch * p.kv_heads) {
    if (w.row - w.base >= 32) load_lengths(p, w, lane);
    const int length = __shfl_sync(0xffffffffu, w.length, w.row - w.base);
    const int tiles = (length + kInt4Tile - 1) / kInt4Tile;
    const int n = min(min(32 - filled, tiles - w.tile), w.left);
    if (lane >= filled && lane < filled + n) {
      mine = w.tile + lane - filled;
      tokens = length;
      b.row = w.row;
    }
    filled += n, w.left -= n, w.tile += n;
    if (w.tile == tiles) ++w.row, w.tile = 0;
  }
  b.tile = kBadTile;
  b.meta = 0;
  if (mine >= 0) {
    const int h = b.row % p.kv_heads;
    const int64_t page = page_id(p, b.row / p.kv_heads, h, mine / per_page);
    if (page >= 0 && page < p.num_pages) {
      b.tile = static_cast<uint32_t>((page * p.kv_heads + h) * per_page + mine % per_page);
    } else {
      atomicMax(p.status, kStatusBadPageId);
    }
    b.meta = min(tokens - mine * kInt4Tile, kInt4Tile) | (mine == 0 ? kRowStart : 0) | ((mine + 1) * kInt4Tile >= tokens ? kRowEnd : 0);
  }
}

template <typename T, int D, int NT>
struct Row {
  static constexpr int W = D / kInt4Group;
  uint32_t q[NT][2 * W][2];   // B fragments of the codes' product, two k-steps a group
  uint32_t qs[NT][2];         // and of the floors' product
  float c[NT][2];             // log2 units per unit of the products, heads 2t and 2t + 1 of an n-tile
  float o[NT][2 * W][4];
  float z[NT][W][2];          // this lane's tokens' p * floor
  float l[NT][2];             // and p
  float m[NT][2];             // offset = m + e - 10
  int e;

  // Query rows as fp16 with the largest element in [2^9, 2^10): a power of two, so exact but for
  // elements 2^-20 below the largest.
  __device__ __forceinline__ void start(const PagedInt4& p, int row, int group, int lane) {
    const int b = row / p.kv_heads, h = row % p.kv_heads;
    const int g = lane >> 2, t = lane & 3;
    const T* src = static_cast<const T*>(p.q) + b * p.q_sb + static_cast<int64_t>(h) * group * p.q_sh;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int head = 8 * i + g;
      uint4 raw[W];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        raw[w] = make_uint4(0, 0, 0, 0);
        if (head < group) raw[w] = *reinterpret_cast<const uint4*>(src + head * p.q_sh + 32 * w + 8 * t);
      }
      float top = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 x = unpack2<T>((&raw[w].x)[j]);
          top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
        }
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int exponent = top > 0.f ? max(-100, min(100, 136 - (__float_as_int(top) >> 23))) : 0;
      const float up = pow2i(exponent);
      float sums[W];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 y = unpack2<T>((&raw[w].x)[j]);
          x[2 * j] = y.x * up, x[2 * j + 1] = y.y * up;
        }
        q[i][2 * w][0] = pack2<__half>(x[0], x[4]);
        q[i][2 * w][1] = pack2<__half>(x[1] * 0.0625f, x[5] * 0.0625f);
        q[i][2 * w + 1][0] = pack2<__half>(x[2], x[6]);
        q[i][2 * w + 1][1] = pack2<__half>(x[3] * 0.0625f, x[7] * 0.0625f);
        float s = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        sums[w] = s;
      }
      // The sums as terms of T that add up to them (fp16 two, bf16 three): the k index of the
      // floors' product is (term, pair of groups), W / 2 lanes a term.
      float pair[2];
      pair[0] = W == 2 || (t & 1) == 0 ? sums[0] : sums[W - 2];
      pair[1] = W == 2 || (t & 1) == 0 ? sums[1] : sums[W - 1];
      const int term = t / (W / 2);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float part[2] = {0.f, 0.f};
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          float rest = pair[y];
          const int which = term + k * (8 / W);
#pragma unroll
          for (int n = 0; n < 3; ++n) {
            const float piece = to_float(from_float<T>(rest));
            if (n == which) part[y] = piece;
            rest -= piece;
          }
        }
        qs[i][k] = pack2<T>(part[0], part[1]);
      }
      const float scale = p.scale * kLog2e * pow2i(-exponent);
      c[i][0] = __shfl_sync(0xffffffffu, scale, 8 * t);
      c[i][1] = __shfl_sync(0xffffffffu, scale, 8 * t + 4);
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        l[i][y] = 0.f, m[i][y] = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; ++w) z[i][w][y] = 0.f;
      }
#pragma unroll
      for (int w = 0; w < 2 * W; ++w) o[i][w][0] = o[i][w][1] = o[i][w][2] = o[i][w][3] = 0.f;
    }
    e = -60;
  }

  static __device__ __forceinline__ void unpack_params(const uint8_t* at, uint32_t (&x)[W / 2]) {
    if constexpr (W == 4) {
      const uint2 y = *reinterpret_cast<const uint2*>(at);
      x[0] = y.x, x[1] = y.y;
    } else {
      x[0] = *reinterpret_cast<const uint32_t*>(at);
    }
  }
  static __device__ __forceinline__ void unpack_words(const uint8_t* at, uint32_t (&x)[W]) {
    if constexpr (W == 4) {
      const uint4 y = *reinterpret_cast<const uint4*>(at);
      x[0] = y.x, x[1] = y.y, x[2] = y.z, x[3] = y.w;
    } else {
      const uint2 y = *reinterpret_cast<const uint2*>(at);
      x[0] = y.x, x[1] = y.y;
    }
  }

  // Raise the offset to this tile's largest scores and steps.
  __device__ __forceinline__ void raise(const float (&s)[NT][4], float magnitude) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) magnitude = fmaxf(magnitude, __shfl_xor_sync(0xffffffffu, magnitude, off));
    const int above = max(-60, (__float_as_int(magnitude) >> 23) - 126);  // magnitude < 2^above
    const int next = max(e, min(above, 100));
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float top = fmaxf(s[i][y], s[i][2 + y]);
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        top = fmaxf(top, m[i][y]);
        const float keep = fast_exp2((m[i][y] - top) + static_cast<float>(e - next));
        m[i][y] = top;
        l[i][y] *= keep;
#pragma unroll
        for (int w = 0; w < W; ++w) z[i][w][y] *= keep;
#pragma unroll
        for (int w = 0; w < 2 * W; ++w) o[i][w][y] *= keep, o[i][w][2 + y] *= keep;
      }
    }
    e = next;
  }

  __device__ __forceinline__ void tile(const uint8_t* smem, int tokens, int lane) {
    const int g = lane >> 2, t = lane & 3;
    // scores
    float s[NT][4];
    {
      float x[NT][4], y[NT][4];
      uint32_t k0[W], k1[W], a0[W / 2], a1[W / 2];
      unpack_words(smem + g * (D / 2) + t * 4 * W, k0);
      unpack_words(smem + (g + 8) * (D / 2) + t * 4 * W, k1);
      const uint8_t* params = smem + 16 * D;
      unpack_params(params + g * 2 * W, a0);
      unpack_params(params + (g + 8) * 2 * W, a1);
      const int pair = W == 4 ? (t & 1) * 4 : 0;
      const uint32_t f0 = *reinterpret_cast<const uint32_t*>(params + D + g * 2 * W + pair);
      const uint32_t f1 = *reinterpret_cast<const uint32_t*>(params + D + (g + 8) * 2 * W + pair);
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        y[i][0] = y[i][1] = y[i][2] = y[i][3] = 0.f;
        mma_t<T>(y[i], f0, f1, f0, f1, qs[i][0], qs[i][1]);
        x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const uint32_t u0 = k0[w] >> 8, u1 = k1[w] >> 8;
        const float2 step0 = unpack2<T>(a0[w / 2]), step1 = unpack2<T>(a1[w / 2]);
        const float st0 = w % 2 ? step0.y : step0.x, st1 = w % 2 ? step1.y : step1.x;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
          mma_f16(d, k0[w] & 0x000f000fu, k1[w] & 0x000f000fu, k0[w] & 0x00f000f0u, k1[w] & 0x00f000f0u, q[i][2 * w][0], q[i][2 * w][1]);
          mma_f16(d, u0 & 0x000f000fu, u1 & 0x000f000fu, u0 & 0x00f000f0u, u1 & 0x00f000f0u, q[i][2 * w + 1][0], q[i][2 * w + 1][1]);
          x[i][0] = fmaf(st0, d[0], x[i][0]), x[i][1] = fmaf(st0, d[1], x[i][1]);
          x[i][2] = fmaf(st1, d[2], x[i][2]), x[i][3] = fmaf(st1, d[3], x[i][3]);
        }
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = fmaf(x[i][j], 16777216.f, y[i][j]) * c[i][j & 1];
      }
    }
    // values' steps and floors; what lies behind the last token may be anything
    uint32_t c0[W / 2], c1[W / 2], e0[W / 2], e1[W / 2];
    {
      const uint8_t* params = smem + 18 * D;
      unpack_params(params + g * 2 * W, c0);
      unpack_params(params + (g + 8) * 2 * W, c1);
      unpack_params(params + D + g * 2 * W, e0);
      unpack_params(params + D + (g + 8) * 2 * W, e1);
    }
    if (tokens < kInt4Tile) {
#pragma unroll
      for (int j = 0; j < W / 2; ++j) {
        if (g >= tokens) c0[j] = e0[j] = 0u;
        if (g + 8 >= tokens) c1[j] = e1[j] = 0u;
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        if (g >= tokens) s[i][0] = s[i][1] = -INFINITY;
        if (g + 8 >= tokens) s[i][2] = s[i][3] = -INFINITY;
      }
    }
    float vc0[W], vc1[W], ve0[W], ve1[W];
    float magnitude = 0.f;
#pragma unroll
    for (int j = 0; j < W / 2; ++j) {
      const float2 w0 = unpack2<T>(c0[j]), w1 = unpack2<T>(c1[j]), w2 = unpack2<T>(e0[j]), w3 = unpack2<T>(e1[j]);
      vc0[2 * j] = w0.x, vc0[2 * j + 1] = w0.y, vc1[2 * j] = w1.x, vc1[2 * j + 1] = w1.y;
      ve0[2 * j] = w2.x, ve0[2 * j + 1] = w2.y, ve1[2 * j] = w3.x, ve1[2 * j + 1] = w3.y;
    }
#pragma unroll
    for (int w = 0; w < W; ++w) {
      magnitude = fmaxf(magnitude, fmaxf(vc0[w], vc1[w]));
      magnitude = fmaxf(magnitude, 0.015625f * fmaxf(fabsf(ve0[w]), fabsf(ve1[w])));
    }
    bool over = magnitude > pow2i(e);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) over = over || s[i][j] > m[i][j & 1] + 4.f;
    }
    if (__any_sync(0xffffffffu, over)) raise(s, magnitude);
    uint32_t v0[W], v1[W];
    unpack_words(smem + 8 * D + t * D + g * 4 * W, v0);
    unpack_words(smem + 8 * D + (t + 4) * D + g * 4 * W, v1);
    uint32_t pb[NT][W][2];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      float pr[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) pr[j] = fast_exp2(s[i][j] - (m[i][j & 1] + static_cast<float>(e - 10)));
      l[i][0] += pr[0] + pr[2];
      l[i][1] += pr[1] + pr[3];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        z[i][w][0] = fmaf(pr[0], ve0[w], fmaf(pr[2], ve1[w], z[i][w][0]));
        z[i][w][1] = fmaf(pr[1], ve0[w], fmaf(pr[3], ve1[w], z[i][w][1]));
        pb[i][w][0] = transpose8(pack2<__half>(pr[0] * vc0[w], pr[1] * vc0[w]));
        pb[i][w][1] = transpose8(pack2<__half>(pr[2] * vc1[w], pr[3] * vc1[w]));
      }
    }
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const uint32_t u0 = v0[w] >> 8, u1 = v1[w] >> 8;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        mma_f16(o[i][2 * w], v0[w] & 0x000f000fu, v0[w] & 0x00f000f0u, v1[w] & 0x000f000fu, v1[w] & 0x00f000f0u, pb[i][w][0], pb[i][w][1]);
        mma_f16(o[i][2 * w + 1], u0 & 0x000f000fu, u0 & 0x00f000f0u, u1 & 0x000f000fu, u1 & 0x00f000f0u, pb[i][w][0], pb[i][w][1]);
      }
    }
  }

  // Sum the lanes' tokens: every lane then holds l and o (heads 2t, 2t + 1, channels 32w + 4g + 0..3).
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[i][y] += __shfl_xor_sync(0xffffffffu, l[i][y], off);
#pragma unroll
        for (int w = 0; w < W; ++w) {
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) z[i][w][y] += __shfl_xor_sync(0xffffffffu, z[i][w][y], off);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            o[i][2 * w + k][y] = fmaf(o[i][2 * w + k][y], 16777216.f, z[i][w][y]);
            o[i][2 * w + k][2 + y] = fmaf(o[i][2 * w + k][2 + y], 1048576.f, z[i][w][y]);
          }
        }
      }
    }
  }

  __device__ __forceinline__ void write_out(const PagedInt4& p, int row, int group, int lane) const {
    const int b = row / p.kv_heads, h = row % p.kv_heads, g = lane >> 2, t = lane & 3;
    T* dst = static_cast<T*>(p.out) + b * p.o_sb + static_cast<int64_t>(h) * group * p.o_sh + 4 * g;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int head = 8 * i + 2 * t + y;
        if (head >= group) continue;
        const float inv = __fdividef(1.f, l[i][y]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
          uint2 x;
          x.x = pack2<T>(o[i][2 * w][y] * inv, o[i][2 * w][2 + y] * inv);
          x.y = pack2<T>(o[i][2 * w + 1][y] * inv, o[i][2 * w + 1][2 + y] * inv);
          *reinterpret_cast<uint2*>(dst + head * p.o_sh + 32 * w) = x;
        }
      }
    }
  }

  __device__ __forceinline__ void deposit(float* piece, int lane) const {
    using S = Shape<D, NT>;
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int head = 8 * i + 2 * t + y;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          *reinterpret_cast<float4*>(piece + head * S::kStride + 32 * w + 4 * g) =
              make_float4(o[i][2 * w][y], o[i][2 * w][2 + y], o[i][2 * w + 1][y], o[i][2 * w + 1][2 + y]);
        }
        if (g == 0) {
          *reinterpret_cast<float2*>(piece + S::kHeads * S::kStride + 2 * head) =
              make_float2(m[i][y] + static_cast<float>(e - 10), l[i][y]);
        }
      }
    }
  }
};

// Running sum of pieces of one (row, head); a lane holds D / 32 channels from channel
// lane * D / 32.  A piece's offset is finite, or NaN where its scores are.
template <int D>
struct Merge {
  static constexpr int C = D / 32;
  float o[C], offset, sum;
  __device__ __forceinline__ void clear() {
    offset = -INFINITY, sum = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = 0.f;
  }
  __device__ __forceinline__ void add(const float (&x)[C], float off, float l) {
    const float top = fmaxf(offset, off);
    const float a = sum == 0.f ? 0.f : fast_exp2(offset - top), b = fast_exp2(off - top);
    sum = sum * a + l * b;
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = o[c] * a + x[c] * b;
    offset = top;
  }
  static __device__ __forceinline__ void load(const float* at, float (&x)[C]) {
    if constexpr (C == 4) {
      const float4 v = *reinterpret_cast<const float4*>(at);
      x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else {
      const float2 v = *reinterpret_cast<const float2*>(at);
      x[0] = v.x, x[1] = v.y;
    }
  }
  template <typename T>
  __device__ __forceinline__ void write_out(const PagedInt4& p, int row, int group, int head, int lane) const {
    const int b = row / p.kv_heads, h = row % p.kv_heads;
    T* dst = static_cast<T*>(p.out) + b * p.o_sb + (static_cast<int64_t>(h) * group + head) * p.o_sh + lane * C;
    const float inv = __fdividef(1.f, sum);
    if constexpr (C == 4) {
      uint2 x;
      x.x = pack2<T>(o[0] * inv, o[1] * inv), x.y = pack2<T>(o[2] * inv, o[3] * inv);
      *reinterpret_cast<uint2*>(dst) = x;
    } else {
      *reinterpret_cast<uint32_t*>(dst) = pack2<T>(o[0] * inv, o[1] * inv);
    }
  }
};

// Scratch: two pieces a CTA for the second kernel (the row it shares with the CTAs before it, the
// row it starts and shares with those behind), one a warp for the row a warp shares with the warps
// before it, and the first and last CTA of every row.
struct Scratch {
  float* cta_pieces;
  float* warp_pieces;
  int2* spans;
};
template <int D, int NT>
__host__ __device__ Scratch carve(void* workspace, int ctas) {
  Scratch s;
  s.cta_pieces = static_cast<float*>(workspace);
  s.warp_pieces = s.cta_pieces + static_cast<int64_t>(2 * ctas) * Shape<D, NT>::kPiece;
  s.spans = reinterpret_cast<int2*>(s.warp_pieces + static_cast<int64_t>(kWarps * ctas) * Shape<D, NT>::kPiece);
  return s;
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, Shape<D, NT>::kCtasPerSm) int4_attention_kernel(const PagedInt4 p, int chunk) {
  using S = Shape<D, NT>;
  extern __shared__ __align__(128) uint8_t s_ring[];
  __shared__ __align__(8) uint64_t s_bar[kWarps][S::kStages];
  __shared__ int64_t s_prefix[kThreads];
  __shared__ int64_t s_warp[kWarps];
  __shared__ int s_row[2 * kWarps];    // rows of the pieces left to merge, warp by warp (first, last), -1: none
  __shared__ int s_flags[2 * kWarps];  // kRowStart / kRowEnd of those pieces

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ctas = gridDim.x, cta = blockIdx.x;
  const int group = p.q_heads / p.kv_heads;
  const Scratch scratch = carve<D, NT>(p.workspace, ctas);
  uint8_t* ring = s_ring + warp * S::kRing;
  const uint32_t ring_at = smem_u32(ring), bar_at = smem_u32(&s_bar[warp][0]);
  if (lane < S::kStages) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar_at + 8 * lane));
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  if (threadIdx.x < 2 * kWarps) s_row[threadIdx.x] = -1;
  release_dependents();
  dependency_wait();
  const Plan plan = make_plan(p, s_prefix, s_warp, chunk, ctas);

  // this warp's units
  const int64_t cta_first = min(plan.share * cta, plan.units);
  const int64_t cta_units = min(plan.share, plan.units - cta_first);
  const int64_t first = cta_first + cta_units * warp / kWarps;
  const int units = static_cast<int>(cta_first + cta_units * (warp + 1) / kWarps - first);

  if (units > 0) {
    Walk walk;
    {
      int lo = 0;
#pragma unroll
      for (int step = kThreads / 2; step > 0; step >>= 1) {
        if (s_prefix[lo + step] <= first) lo += step;
      }
      walk.row = lo * chunk;
      int64_t before = first - s_prefix[lo];
      load_lengths(p, walk, lane);
      const int rows = p.batch * p.kv_heads;
      while (walk.row < rows) {
        if (walk.row - walk.base >= 32) load_lengths(p, walk, lane);
        const int tiles = (__shfl_sync(0xffffffffu, walk.length, walk.row - walk.base) + kInt4Tile - 1) / kInt4Tile;
        if (before < tiles) break;
        before -= tiles;
        ++walk.row;
      }
      walk.tile = static_cast<int>(before);
      walk.left = units;
    }
    Batch now, next;
    next_batch(p, walk, now, lane);
    next.tile = kBadTile, next.meta = 0, next.row = 0;

    auto request = [&](int unit, const Batch& b) {
      const uint32_t tile = __shfl_sync(0xffffffffu, b.tile, unit & 31);
      const int stage = unit % S::kStages;
      if (tile != kBadTile) {
        if (lane == 0) {
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar_at + 8 * stage), "r"(S::kTileBytes) : "memory");
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                           ring_at + stage * S::kTileBytes),
                       "l"(p.pool + static_cast<int64_t>(tile) * S::kTileBytes), "r"(S::kTileBytes), "r"(bar_at + 8 * stage)
                       : "memory");
        }
      } else {  // a page outside the pool: zeros
        for (int i = lane; i < S::kTileBytes / 16; i += 32) {
          *reinterpret_cast<uint4*>(ring + stage * S::kTileBytes + 16 * i) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar_at + 8 * stage) : "memory");
      }
    };
    for (int u = 0; u < S::kStages && u < units; ++u) request(u, now);

    Row<T, D, NT> row;
    bool starts = false, in_row = false;
    int pieces = 0;
    for (int u = 0; u < units; ++u) {
      if ((u & 31) == 0) {
        if (u > 0) now = next;
        if (walk.left > 0) next_batch(p, walk, next, lane);
      }
      const int meta = __shfl_sync(0xffffffffu, now.meta, u & 31);
      const int id = __shfl_sync(0xffffffffu, now.row, u & 31);
      if (!in_row) {
        row.start(p, id, group, lane);
        starts = (meta & kRowStart) != 0;
        in_row = true;
        if (starts && lane == 0) {
          // the CTAs that hold the row: this one and those its last tile reaches
          const int tiles = static_cast<int>((row_tokens(p, id / p.kv_heads, id % p.kv_heads) + kInt4Tile - 1) / kInt4Tile);
          scratch.spans[id] = make_int2(cta, static_cast<int>((first + u + tiles - 1) / plan.share));
        }
      }
      const int stage = u % S::kStages;
      if (!wait_stage(bar_at + 8 * stage, (u / S::kStages) & 1) && lane == 0) atomicMax(p.status, kStatusPipelineTimeout);
      row.tile(ring + stage * S::kTileBytes, meta & 31, lane);
      __syncwarp();
      const int ahead = u + S::kStages;
      if (ahead < units) request(ahead, (ahead ^ u) < 32 ? now : next);
      if ((meta & kRowEnd) || u == units - 1) {
        const bool ends = (meta & kRowEnd) != 0;
        row.finish();
        if (starts && ends) {
          row.write_out(p, id, group, lane);
        } else {
          const bool last = u == units - 1;
          row.deposit(last ? reinterpret_cast<float*>(ring) : scratch.warp_pieces + static_cast<int64_t>(cta * kWarps + warp) * S::kPiece, lane);
          if (lane == 0) {
            s_row[2 * warp + (last ? 1 : 0)] = id;
            s_flags[2 * warp + (last ? 1 : 0)] = (starts ? kRowStart : 0) | (ends ? kRowEnd : 0);
          }
        }
        in_row = false;
        ++pieces;
      }
    }
  }
  __syncthreads();

  // Rows that several warps, or several CTAs, hold: a warp takes the heads with its number.
  for (int i = 0; i < 2 * kWarps;) {
    const int id = s_row[i];
    if (id < 0) {
      ++i;
      continue;
    }
    int end = i, last = i;
    for (; end < 2 * kWarps && (s_row[end] == id || s_row[end] < 0); ++end) last = s_row[end] == id ? end : last;
    const bool starts = (s_flags[i] & kRowStart) != 0, ends = (s_flags[last] & kRowEnd) != 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int head = 8 * nt + warp;
      if (head >= group) break;
      Merge<D> sum;
      sum.clear();
      for (int k = i; k <= last; ++k) {
        if (s_row[k] < 0) continue;
        const float* piece = (k & 1) ? reinterpret_cast<const float*>(s_ring + (k >> 1) * S::kRing)
                                     : scratch.warp_pieces + static_cast<int64_t>(cta * kWarps + (k >> 1)) * S::kPiece;
        float x[Merge<D>::C];
        Merge<D>::load(piece + head * S::kStride + lane * Merge<D>::C, x);
        const float2 ml = *reinterpret_cast<const float2*>(piece + S::kHeads * S::kStride + 2 * head);
        sum.add(x, ml.x, ml.y);
      }
      if (starts && ends) {
        sum.template write_out<T>(p, id, group, head, lane);
      } else {
        float* piece = scratch.cta_pieces + static_cast<int64_t>(2 * cta + (starts ? 1 : 0)) * S::kPiece;
#pragma unroll
        for (int c = 0; c < Merge<D>::C; ++c) piece[head * S::kStride + lane * Merge<D>::C + c] = sum.o[c];
        if (lane == 0) *reinterpret_cast<float2*>(piece + S::kHeads * S::kStride + 2 * head) = make_float2(sum.offset, sum.sum);
      }
    }
    i = end;
  }
}

// Rows that span CTAs, and zeros for rows without tokens: one CTA of four warps a (row, head),
// the pieces dealt out to the warps in turn.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(128) int4_combine_kernel(const PagedInt4 p, int ctas) {
  using S = Shape<D, NT>;
  constexpr int C = Merge<D>::C;
  __shared__ float s_o[4][D];
  __shared__ float2 s_ml[4];
  release_dependents();
  dependency_wait();
  const int group = p.q_heads / p.kv_heads;
  const int row = blockIdx.x / group, head = blockIdx.x % group;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = row / p.kv_heads, h = row % p.kv_heads;
  if (row_tokens(p, b, h) == 0) {
    T* dst = static_cast<T*>(p.out) + b * p.o_sb + (static_cast<int64_t>(h) * group + head) * p.o_sh;
    for (int d = threadIdx.x; d < D; d += 128) dst[d] = from_float<T>(0.f);
    return;
  }
  const Scratch scratch = carve<D, NT>(p.workspace, ctas);
  const int2 span = scratch.spans[row];
  if (span.x == span.y) return;
  Merge<D> sum;
  sum.clear();
#pragma unroll 4
  for (int c = span.x + warp; c <= span.y; c += 4) {
    const float* piece = scratch.cta_pieces + static_cast<int64_t>(2 * c + (c == span.x ? 1 : 0)) * S::kPiece;
    float x[C];
    Merge<D>::load(piece + head * S::kStride + lane * C, x);
    const float2 ml = *reinterpret_cast<const float2*>(piece + S::kHeads * S::kStride + 2 * head);
    sum.add(x, ml.x, ml.y);
  }
#pragma unroll
  for (int c = 0; c < C; ++c) s_o[warp][lane * C + c] = sum.o[c];
  if (lane == 0) s_ml[warp] = make_float2(sum.offset, sum.sum);
  __syncthreads();
  if (warp != 0) return;
  for (int w = 1; w < 4 && span.x + w <= span.y; ++w) {
    float x[C];
    Merge<D>::load(&s_o[w][lane * C], x);
    sum.add(x, s_ml[w].x, s_ml[w].y);
  }
  sum.template write_out<T>(p, row, group, head, lane);
}

int sm_count() {
  int device = 0, count = 0;
  if (cudaGetDevice(&device) != cudaSuccess ||
      cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
    (void)cudaGetLastError();
    return 148;
  }
  return count;
}

template <int D, int NT>
int64_t scratch_bytes(int64_t rows, int ctas) {
  const int64_t pieces = static_cast<int64_t>(2 + kWarps) * ctas * Shape<D, NT>::kPiece * 4;
  return (pieces + rows * 8 + 15) / 16 * 16;
}

template <typename T, int D, int NT>
int launch(const PagedInt4& p, cudaStream_t stream) {
  using S = Shape<D, NT>;
  const int64_t rows = static_cast<int64_t>(p.batch) * p.kv_heads;
  const int ctas = sm_count() * S::kCtasPerSm;
  const int64_t need = scratch_bytes<D, NT>(rows, ctas);
  QF_REQUIRE(p.workspace != nullptr && p.workspace_bytes >= need, "the workspace holds %lld bytes, %lld are needed",
             static_cast<long long>(p.workspace_bytes), static_cast<long long>(need));
  QF_REQUIRE(rows * (p.q_heads / p.kv_heads) < (1LL << 31), "too many rows");
  static thread_local int ready = -1;  // device whose kernel attribute this thread has set
  int device = 0;
  QF_CUDA(cudaGetDevice(&device));
  if (ready != device) {
    QF_CUDA(cudaFuncSetAttribute(int4_attention_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
    ready = device;
  }
  const int chunk = static_cast<int>((rows + kThreads - 1) / kThreads);
  QF_CUDA(launch_chained(int4_attention_kernel<T, D, NT>, dim3(ctas), dim3(kThreads), static_cast<size_t>(S::kSmem), stream, p, chunk));
  QF_CUDA(launch_chained(int4_combine_kernel<T, D, NT>, dim3(static_cast<unsigned>(rows * (p.q_heads / p.kv_heads))), dim3(128),
                         static_cast<size_t>(0), stream, p, ctas));
  QF_CUDA(cudaGetLastError());
  return QF_OK;
}

template <typename T>
int launch_for(const PagedInt4& p, int head_dim, cudaStream_t stream) {
  const bool two = p.q_heads / p.kv_heads > 8;
  if (head_dim == 128) return two ? launch<T, 128, 2>(p, stream) : launch<T, 128, 1>(p, stream);
  return two ? launch<T, 64, 2>(p, stream) : launch<T, 64, 1>(p, stream);
}

}  // namespace

int64_t int4_attention_bytes(const PagedInt4& p, int head_dim) {
  const int64_t rows = static_cast<int64_t>(p.batch) * p.kv_heads;
  const bool two = p.q_heads / p.kv_heads > 8;
  const int sms = sm_count();
  if (head_dim == 128) {
    return two ? scratch_bytes<128, 2>(rows, sms * Shape<128, 2>::kCtasPerSm) : scratch_bytes<128, 1>(rows, sms * Shape<128, 1>::kCtasPerSm);
  }
  return two ? scratch_bytes<64, 2>(rows, sms * Shape<64, 2>::kCtasPerSm) : scratch_bytes<64, 1>(rows, sms * Shape<64, 1>::kCtasPerSm);
}

int launch_int4_attention(const PagedInt4& p, int head_dim, int dtype, cudaStream_t stream) {
  return dtype == QF_DTYPE_F16 ? launch_for<__half>(p, head_dim, stream) : launch_for<__nv_bfloat16>(p, head_dim, stream);
}

}  // namespace qf

extern "C" int qf_int4_decode_attention(const qf_paged_int4_args* args, void* stream) {
  qf::PagedInt4 p;
  if (const int rc = qf::fill_paged_int4(args, qf::kNeedsQuery | qf::kNeedsPool | qf::kNeedsOut, &p)) return rc;
  if (p.batch == 0) return QF_OK;
  return qf::launch_int4_attention(p, args->head_dim, args->dtype, static_cast<cudaStream_t>(stream));
}
