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
// where p c is rounded to fp16 (2^-11 of a weight at most; products and sums are fp32).  The offset is
// the running maximum of s, plus the exponent of the largest c (or of |e| / 64 where that is larger), less
// 10, so that p c stays below 2^15; it is raised, and the sums rescaled, only when a score or a step exceeds
// what the last offset allows by 2^4.  One exponent serves all groups of the tokens that a warp has seen of
// a row: in a group whose steps are 2^-k of the largest, p c keeps fp16's precision down to 2^-(24 - k) of
// the largest weight; below that it is off by at most 2^-25, where the largest p c is 2^10.
//
// Work.  Rows are laid end to end as units of two tiles and every CTA, one an SM, takes an equal share
// of them, every warp of the CTA an equal share of that, whatever rows it covers.  A warp streams its
// units, 2 x 20 * D contiguous bytes each, through a ring of its own with cp.async (as bulk copies with
// a barrier a stage, the same ring took 125 instructions more a unit and 7 % more time at D = 64); warps
// share nothing until their units are done.  A row that one warp holds whole is written from its
// registers; what the warps of a CTA hold of one row is summed at the CTA's end, and rows that span
// CTAs by a second kernel, in the order of the tiles: the same call gives the same bits.  Where tables
// are so short that it ends sooner, a row is one CTA's alone or one cluster's, whose CTAs join their sums
// behind a barrier, without a second kernel (row_parts).  Table and lengths are read while the kernel in
// front drains, unless it writes them.
//
// Bound.  The cache's 5 bits a channel come in at the memory's rate only if the SM spends no more than
// 110 cycles on a tile of D = 128 (55 at D = 64); it issues about 250 (200) instructions a tile, a third
// of them the masks and shifts that take codes apart, on four schedulers of which each issues in 47 (D
// 64: 63) cycles of a hundred.  With all tiles in one page, that is with no memory to wait for, calls take 7 % less
// time, so issue and dependences bound it, and for short calls the way to the first tile (lengths, table,
// tile: 3 us) and the launches.  64 sequences of 129..4097 tokens, 12 heads on 2 of 128: 18.5 us, 42 MB,
// 2.3 TB/s; 256 of 64..4096, 16 on 4 of 64: 45.6 us, 172 MB, 3.8 TB/s; one of 513: 7.0 us (all in graphs).
// Warps an SM, measured before rows counted a place of their own, D = 128: 8 take 22 us for the
// first, 10 22.3, 12 20.0, 14 20.9, 16 21.2 (from 13 on the registers no longer hold a row: 168 against 128 a
// thread); D = 64: 12 take 54 us, 16 52, 20 54.
// Taking the next unit's scores beside this one's values gives the schedulers two chains to choose from
// and cost 3 to 5 %; V words rotated so that no two lanes meet in a bank changed nothing.
#include <algorithm>
#include <atomic>

#include "qf_int4_paged.cuh"

namespace qf {
namespace {

constexpr int kUnit = 2 * kInt4Tile;  // tokens a warp takes at a time: two tiles, for the distance between dependent steps
constexpr uint32_t kNoTile = 0xffffffffu;
constexpr int kRowStart = 1, kRowEnd = 2;
constexpr float kLog2e = 1.4426950408889634f;

template <int D, int NT>
struct Shape {
  static constexpr int kWarps = NT == 2 ? 8 : D == 128 ? 12 : 16;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kTileBytes = 20 * D;
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kStages = 204 * 1024 / kWarps / kStageBytes;  // of a warp's ring, one less in flight: D 128 3 or 5, D 64 5 or 10
  static constexpr int kRing = kStages * kStageBytes;
  static constexpr int kHeads = 8 * NT;        // query heads a row has room for
  static constexpr int kStride = D + 4;        // floats between heads of a piece: its float4 stores miss no bank
  static constexpr int kPiece = kHeads * kStride + 2 * kHeads;  // floats: o, then offset and sum of every head
  static constexpr int kSmem = kWarps * kRing;
  static_assert(kPiece * 4 <= kRing, "a piece fits its warp's ring");
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8 x 8 transpose of 16-bit elements across the warp.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Largest value of the warp, NaNs left out.
__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float pow2i(int e) {  // 2^e, e in [-126, 127]
  return __int_as_float((e + 127) << 23);
}

// 16 bytes to shared memory, or zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_close() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A row costs its units and one more: its queries' way to the registers and its result's way out
// take about as long as a unit.  A place in a row counts that one first, so unit u is at place u + 1.
// Shares are runs of places: without the extra one the CTAs with the most short rows of 256 sequences of
// 64..4096 tokens ended at 50 us and half of them before 42.5.
__device__ __forceinline__ int row_units(int tokens) { return (tokens + kUnit - 1) / kUnit; }
__device__ __forceinline__ int row_places(int tokens) { return tokens > 0 ? row_units(tokens) + 1 : 0; }

// What a call shares out: places of all rows (fewer than 2^31), places of a CTA.
struct Plan {
  int places;
  int share;
};

// First unit of CTA `rank` of the `parts` that a row is split over.
__device__ __forceinline__ int part_first(int units, int rank, int parts) { return static_cast<int>(static_cast<uint32_t>(units) * rank / parts); }

__device__ __forceinline__ int row_tokens_at(const PagedInt4& p, int row) {
  const int2 at = row_place(p, row);
  return static_cast<int>(row_tokens(p, at.x, at.y));
}

// Shared by a CTA's warps: prefix sums of the rows' places, thread by thread (`chunk` rows each),
// and the lengths of the first rows.
constexpr int kRowsKept = 2048;
template <int kWarps>
struct Shares {
  int prefix[32 * kWarps];
  int warp[kWarps];
  int tokens[kRowsKept];
};

template <int kWarps>
__device__ __forceinline__ Plan make_plan(const PagedInt4& p, Shares<kWarps>& s, int chunk, int ctas) {
  const int rows = p.batch * p.kv_heads;
  const int first = threadIdx.x * chunk, lane = threadIdx.x & 31;
  int mine = 0;
  for (int r = first; r < first + chunk && r < rows; ++r) {
    const int tokens = row_tokens_at(p, r);
    mine += row_places(tokens);
    if (r < kRowsKept) s.tokens[r] = tokens;
  }
  int sum = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, sum, off);
    if (lane >= off) sum += up;
  }
  if (lane == 31) s.warp[threadIdx.x >> 5] = sum;
  s.prefix[threadIdx.x] = sum - mine;  // within the warp's rows
  __syncthreads();
  Plan plan;
  plan.places = __reduce_add_sync(0xffffffffu, lane < kWarps ? s.warp[lane] : 0);
  plan.share = (plan.places + ctas - 1) / ctas;
  if (plan.share < kWarps) plan.share = kWarps;  // a place a warp at least: fewer pieces for the second kernel
  return plan;
}

// The thread whose rows hold place `first`, and the places before those rows.
template <int kWarps>
__device__ __forceinline__ int2 find_rows(const Shares<kWarps>& s, int first, int lane) {
  const int mine = lane < kWarps ? s.warp[lane] : 0;
  int sum = mine;
#pragma unroll
  for (int off = 1; off < kWarps; off <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, sum, off);
    if (lane >= off) sum += up;
  }
  const int warp = __popc(__ballot_sync(0xffffffffu, lane < kWarps && sum <= first));  // warps that end before it
  const int before = __shfl_sync(0xffffffffu, sum - mine, warp);
  const int start = before + s.prefix[32 * warp + lane];
  const int thread = __popc(__ballot_sync(0xffffffffu, start <= first)) - 1;
  return make_int2(32 * warp + thread, __shfl_sync(0xffffffffu, start, thread));
}

template <int kWarps>
__device__ __forceinline__ int tokens_of(const PagedInt4& p, const Shares<kWarps>& s, int row) {
  return row < kRowsKept ? s.tokens[row] : row_tokens_at(p, row);
}

// The next units to request, 32 or fewer: lane i holds the two tiles of unit i, kNoTile for one
// behind the row's end or in a page outside the pool.
struct Requests {
  int row, place;  // the next one
  int left;        // places
  int count, next; // units held, and the first of them not requested yet
  uint32_t tile[2];

  template <int kWarps>
  __device__ __forceinline__ void refill(const PagedInt4& p, const Shares<kWarps>& s, int lane) {
    int mine = -1, mine_row = 0, mine_tokens = 0;
    count = next = 0;
    while (count < 32 && left > 0 && row < p.batch * p.kv_heads) {
      const int tokens = tokens_of(p, s, row), places = row_places(tokens);
      if (place == 0 && places > 0) place = 1, --left;
      const int n = min(min(32 - count, places - place), left);
      if (lane >= count && lane < count + n) mine = place - 1 + lane - count, mine_row = row, mine_tokens = tokens;
      count += n, left -= n, place += n;
      if (place >= places) ++row, place = 0;
    }
    tile[0] = tile[1] = kNoTile;
    if (mine < 0) return;
    const int2 at = row_place(p, mine_row);
    const int first = 2 * mine, second = (first + 1) * kInt4Tile < mine_tokens ? first + 1 : first;
    const int page0 = quotient(first, p.by_tiles), page1 = quotient(second, p.by_tiles);
    const int64_t id0 = page_id(p, at.x, at.y, page0), id1 = page_id(p, at.x, at.y, page1);
    const bool ok0 = id0 >= 0 && id0 < p.num_pages, ok1 = id1 >= 0 && id1 < p.num_pages;
    if (!ok0 || !ok1) atomicMax(p.status, kStatusBadPageId);
    if (ok0) tile[0] = (static_cast<uint32_t>(id0) * p.kv_heads + at.y - page0) * p.by_tiles.d + first;
    if (ok1 && second != first) tile[1] = (static_cast<uint32_t>(id1) * p.kv_heads + at.y - page1) * p.by_tiles.d + second;
  }
};

template <typename T>
struct Pair;
template <>
struct Pair<__half> {
  using type = __half2;
  static constexpr bool kFine = true;
  static __device__ __forceinline__ __half2 of(uint32_t x) { return *reinterpret_cast<__half2*>(&x); }
};
template <>
struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static constexpr bool kFine = false;
  static __device__ __forceinline__ __nv_bfloat162 of(uint32_t x) { return *reinterpret_cast<__nv_bfloat162*>(&x); }
};

template <typename T, int D, int NT>
struct Row {
  static constexpr int W = D / kInt4Group;
  // A rounded weight is off by 2^-12 of itself on average, times a code of 7.5 on average.  For fp16
  // results the codes count from 7.5: sum_t (p c) m = sum_t fl(p c) (m - 7.5) + 7.5 sum_t p c but for the
  // rounding of fl, now times |m - 7.5|.  bf16 results are rounded coarser than either: they differ from an
  // fp32 attention's by 1.3e-4 to 2.4e-4 of their norm, a last place here and there, and are as far from the exact
  // ones as those (1.5e-3); centred codes would make that 0.9e-4 to 1.9e-4 and 256 sequences of 64..4096 tokens
  // (D 64) 49.6 us instead of 45.8, weights as two fp16 terms 0.3e-4 to 1.6e-4 and 51.3 us.
  static constexpr bool kCentred = Pair<T>::kFine;
  uint32_t q[NT][2 * W][2];   // B fragments of the codes' product, two k-steps a group
  uint32_t qs[NT][2];         // and of the floors' product
  float c[NT][2];             // log2 units per unit of the products, heads 2t and 2t + 1 of an n-tile
  float o[NT][2 * W][4];
  uint64_t z[NT][W / 2][2];   // this lane's tokens' p * floor: pairs of groups, head 2t or 2t + 1
  float l[NT][2];             // and p
  float h[NT][4];             // fp16: 7.5 times the rounded weights of group g, heads 2t and 2t + 1 (half of the lanes')
  float off[NT][2];           // largest score so far (of the last raise) + e - 10
  int e;

  // Query rows as fp16 with the largest element in [2^9, 2^10), of bf16 rows below 2^-117 less: a power
  // of two, so exact but for elements 2^-20 below the largest.
  static __device__ __forceinline__ void load(const PagedInt4& p, int row, int group, int lane, uint4 (&raw)[NT][W]) {
    const int2 at = row_place(p, row);
    const T* src = static_cast<const T*>(p.q) + at.x * p.q_sb + static_cast<int64_t>(at.y) * group * p.q_sh + 8 * (lane & 3);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const int head = 8 * i + (lane >> 2);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        raw[i][w] = make_uint4(0, 0, 0, 0);
        if (head < group) raw[i][w] = *reinterpret_cast<const uint4*>(src + head * p.q_sh + 32 * w);
      }
    }
  }
  __device__ __forceinline__ void start(const PagedInt4& p, const uint4 (&all)[NT][W], int lane) {
    const int t = lane & 3;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const uint4(&raw)[W] = all[i];
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
      const int exponent = top > 0.f ? min(126, 136 - (__float_as_int(top) >> 23)) : 0;  // -119 for NaN and infinity
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
        l[i][y] = 0.f, off[i][y] = -INFINITY, h[i][y] = h[i][2 + y] = 0.f;
#pragma unroll
        for (int w = 0; w < W / 2; ++w) z[i][w][y] = 0u;
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

  // exp2 arguments of the scores x, those behind the row's end -inf
  __device__ __forceinline__ void arguments(const float (&x)[NT][8], float (&a)[NT][8], int left, int g) const {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) a[i][j] = fmaf(x[i][j], c[i][j & 1], -off[i][j & 1]);
    }
    if (__any_sync(0xffffffffu, left < kUnit)) {  // a vote: the compiler then knows the branch is the warp's
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) a[i][j] = g + 8 * (j >> 1) < left ? a[i][j] : -INFINITY;
      }
    }
  }

  // Raise the offset to this unit's largest scores and steps.
  __device__ __forceinline__ void raise(const float (&x)[NT][8], float magnitude, int left, int g) {
    magnitude = warp_max(magnitude);
    const int above = max(-60, (__float_as_int(magnitude) >> 23) - 126);  // magnitude < 2^above
    const int next = max(e, min(above, 127));
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) top = fmaxf(top, g + 8 * j < left ? x[i][2 * j + y] * c[i][y] : -INFINITY);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float raised = fmaxf(top, off[i][y] - static_cast<float>(e - 10)) + static_cast<float>(next - 10);
        const float keep = fast_exp2(off[i][y] - raised);
        off[i][y] = raised;
        l[i][y] *= keep;
        h[i][y] *= keep;
#pragma unroll
        for (int w = 0; w < W / 2; ++w) z[i][w][y] = mul32x2(z[i][w][y], pair32(keep, keep));
#pragma unroll
        for (int w = 0; w < 2 * W; ++w) o[i][w][y] *= keep, o[i][w][2 + y] *= keep;
      }
    }
    e = next;
  }

  // Scores of one tile, in units of c: x[.][0..3] are (token g, heads 2t, 2t + 1), (token g + 8, ..).
  __device__ __forceinline__ void scores(const uint8_t* smem, float (&x)[NT][8], int at, int lane) const {
    const int g = lane >> 2, t = lane & 3;
    uint32_t k0[W], k1[W], a0[W / 2], a1[W / 2];
    unpack_words(smem + g * (D / 2) + t * 4 * W, k0);
    unpack_words(smem + (g + 8) * (D / 2) + t * 4 * W, k1);
    const uint8_t* params = smem + 16 * D;
    unpack_params(params + g * 2 * W, a0);
    unpack_params(params + (g + 8) * 2 * W, a1);
    const int pair = W == 4 ? (t & 1) * 4 : 0;
    const uint32_t f0 = *reinterpret_cast<const uint32_t*>(params + D + g * 2 * W + pair);
    const uint32_t f1 = *reinterpret_cast<const uint32_t*>(params + D + (g + 8) * 2 * W + pair);
    float sum[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) sum[i][0] = sum[i][1] = sum[i][2] = sum[i][3] = 0.f;
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
        sum[i][0] = fmaf(st0, d[0], sum[i][0]), sum[i][1] = fmaf(st0, d[1], sum[i][1]);
        sum[i][2] = fmaf(st1, d[2], sum[i][2]), sum[i][3] = fmaf(st1, d[3], sum[i][3]);
      }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      float y[4] = {0.f, 0.f, 0.f, 0.f};
      mma_t<T>(y, f0, f1, f0, f1, qs[i][0], qs[i][1]);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[i][at + j] = fmaf(sum[i][j], 16777216.f, y[j]);
    }
  }

  // A NaN step as a step of 0 and a NaN floor: the sums of the weights, one product for all groups, stay
  // finite, and the group is NaN by its floors' sum alone.  Returns the magnitude of what is left.
  static __device__ __forceinline__ float keep_nans_apart(uint32_t (&vc)[4][W / 2], uint32_t (&ve)[4][W / 2], float largest_floor) {
    float magnitude = fmaxf(largest_floor, 0.f);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int j = 0; j < W / 2; ++j) {
        const float2 step = unpack2<T>(vc[k][j]), floor = unpack2<T>(ve[k][j]);
        ve[k][j] = pack2<T>(step.x == step.x ? floor.x : step.x, step.y == step.y ? floor.y : step.y);
        vc[k][j] = pack2<T>(step.x == step.x ? step.x : 0.f, step.y == step.y ? step.y : 0.f);
        magnitude = fmaxf(magnitude, fmaxf(step.x, step.y));
      }
    }
    return magnitude;
  }

  // Two tiles, `left` tokens of the row from their first on.
  __device__ __forceinline__ void unit(const uint8_t* smem, int left, int lane) {
    using V2 = typename Pair<T>::type;
    const int g = lane >> 2, t = lane & 3;
    float x[NT][8];
    scores(smem, x, 0, lane);
    scores(smem + 20 * D, x, 4, lane);
    // values' steps and floors; what lies behind the last token may be anything
    uint32_t vc[4][W / 2], ve[4][W / 2];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint8_t* params = smem + (k >> 1) * 20 * D + 18 * D + (g + 8 * (k & 1)) * 2 * W;
      unpack_params(params, vc[k]);
      unpack_params(params + D, ve[k]);
    }
    if (__any_sync(0xffffffffu, left < kUnit)) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
#pragma unroll
        for (int j = 0; j < W / 2; ++j) {
          vc[k][j] = g + 8 * k < left ? vc[k][j] : 0u;
          ve[k][j] = g + 8 * k < left ? ve[k][j] : 0u;
        }
      }
    }
    V2 steps = Pair<T>::of(vc[0][0]), floors = __habs2(Pair<T>::of(ve[0][0]));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
#pragma unroll
      for (int j = 0; j < W / 2; ++j) {
        // a NaN step is kept where it must be seen: it takes the rare branch below
        steps = kCentred ? __hmax2_nan(steps, Pair<T>::of(vc[k][j])) : __hmax2(steps, Pair<T>::of(vc[k][j]));
        floors = __hmax2(floors, __habs2(Pair<T>::of(ve[k][j])));
      }
    }
    const float largest_floor = 0.015625f * fmaxf(to_float(floors.x), to_float(floors.y));
    float magnitude = kCentred ? max_nan(to_float(steps.x), to_float(steps.y), largest_floor) : fmaxf(fmaxf(to_float(steps.x), to_float(steps.y)), largest_floor);
    float a[NT][8];
    arguments(x, a, left, g);
    float top = a[0][0];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, a[i][j]);
    }
    if (__any_sync(0xffffffffu, (top > static_cast<float>(14 - e)) | (kCentred ? !(magnitude <= pow2i(e)) : magnitude > pow2i(e)))) {
      if constexpr (kCentred) {
        if (__any_sync(0xffffffffu, magnitude != magnitude)) magnitude = keep_nans_apart(vc, ve, largest_floor);
      }
      raise(x, magnitude, left, g);
      arguments(x, a, left, g);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t v0[W], v1[W];
      unpack_words(smem + k * 20 * D + 8 * D + t * D + g * 4 * W, v0);
      unpack_words(smem + k * 20 * D + 8 * D + (t + 4) * D + g * 4 * W, v1);
      uint32_t pb[NT][W][2];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        float pr[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) pr[j] = fast_exp2(a[i][4 * k + j]);
        l[i][0] += pr[0] + pr[2];
        l[i][1] += pr[1] + pr[3];
        uint64_t twice[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) twice[j] = pair32(pr[j], pr[j]);
#pragma unroll
        for (int w = 0; w < W / 2; ++w) {
          const float2 s0 = unpack2<T>(vc[2 * k][w]), s1 = unpack2<T>(vc[2 * k + 1][w]);
          const float2 f0 = unpack2<T>(ve[2 * k][w]), f1 = unpack2<T>(ve[2 * k + 1][w]);
          const uint64_t c0 = pair32(s0.x, s0.y), c1 = pair32(s1.x, s1.y);
          uint64_t e0 = pair32(f0.x, f0.y), e1 = pair32(f1.x, f1.y);
          if constexpr (kCentred) e0 = fma32x2(c0, pair32(7.5f, 7.5f), e0), e1 = fma32x2(c1, pair32(7.5f, 7.5f), e1);
          z[i][w][0] = fma32x2(twice[0], e0, fma32x2(twice[2], e1, z[i][w][0]));
          z[i][w][1] = fma32x2(twice[1], e0, fma32x2(twice[3], e1, z[i][w][1]));
          const float2 p0 = unpair32(mul32x2(twice[0], c0)), p1 = unpair32(mul32x2(twice[1], c0));
          const float2 p2 = unpair32(mul32x2(twice[2], c1)), p3 = unpair32(mul32x2(twice[3], c1));
          pb[i][2 * w][0] = transpose8(pack2<__half>(p0.x, p1.x));
          pb[i][2 * w + 1][0] = transpose8(pack2<__half>(p0.y, p1.y));
          pb[i][2 * w][1] = transpose8(pack2<__half>(p2.x, p3.x));
          pb[i][2 * w + 1][1] = transpose8(pack2<__half>(p2.y, p3.y));
        }
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        // rows g of a product are codes 2 k, rows g + 8 the bytes with codes 2 k (low) and 2 k + 1
        const uint32_t u0 = __byte_perm(v0[w], 0u, 0x4341u), u1 = __byte_perm(v1[w], 0u, 0x4341u);
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          if constexpr (kCentred) {  // 7.5 in row w of an A that is zero elsewhere: one sum for all groups
            const uint32_t ones = g == w ? 0x47804780u : 0u;
            mma_f16(h[i], ones, 0u, ones, 0u, pb[i][w][0], pb[i][w][1]);
          }
          mma_f16(o[i][2 * w], v0[w] & 0x000f000fu, v0[w] & 0x00ff00ffu, v1[w] & 0x000f000fu, v1[w] & 0x00ff00ffu, pb[i][w][0], pb[i][w][1]);
          mma_f16(o[i][2 * w + 1], u0 & 0x000f000fu, u0, u1 & 0x000f000fu, u1, pb[i][w][0], pb[i][w][1]);
        }
      }
    }
  }

  // Sum the lanes' tokens: every lane then holds l and o (heads 2t, 2t + 1, channels 32w + 4g + 0..3).
  __device__ __forceinline__ void finish(int lane) {
    const int t = lane & 3;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) l[i][y] += __shfl_xor_sync(0xffffffffu, l[i][y], off);
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float2 both = unpair32(z[i][w / 2][y]);
          float sum = w % 2 ? both.y : both.x;
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
          if constexpr (kCentred) sum -= __shfl_sync(0xffffffffu, h[i][y], 4 * w + t);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            // rows g + 8 are code + 16 * next code
            const float next = o[i][2 * w + k][2 + y] - o[i][2 * w + k][y];
            o[i][2 * w + k][y] = fmaf(o[i][2 * w + k][y], 16777216.f, sum);
            o[i][2 * w + k][2 + y] = fmaf(next, 1048576.f, sum);
          }
        }
      }
    }
  }

  __device__ __forceinline__ void write_out(const PagedInt4& p, int row, int group, int lane) const {
    const int2 at = row_place(p, row);
    const int b = at.x, h = at.y, g = lane >> 2, t = lane & 3;
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
              make_float2(off[i][y], l[i][y]);
        }
      }
    }
  }
};

// The channels of one (row, head) that a lane sums over pieces: D / 32 from channel lane * D / 32.
template <int D>
struct Merge {
  static constexpr int C = D / 32;
  float o[C];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = 0.f;
  }
  __device__ __forceinline__ void add(const float (&x)[C], float weight) {
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = fmaf(x[c], weight, o[c]);
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
  static __device__ __forceinline__ void store(float* at, const float (&x)[C]) {
    if constexpr (C == 4) {
      *reinterpret_cast<float4*>(at) = make_float4(x[0], x[1], x[2], x[3]);
    } else {
      *reinterpret_cast<float2*>(at) = make_float2(x[0], x[1]);
    }
  }
  template <typename T>
  __device__ __forceinline__ void write_out(const PagedInt4& p, int row, int group, int head, int lane, float sum) const {
    const int2 at = row_place(p, row);
    const int b = at.x, h = at.y;
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

// The weighted sum of the pieces of `chain`, whose lanes hold the weights; at(k): piece k's channels of this lane.
template <int D, typename At>
__device__ __forceinline__ Merge<D> merged(unsigned chain, float weight, At at) {
  Merge<D> merge;
  merge.clear();
  const int i = __ffs(chain) - 1;
  for (unsigned left = chain; left != 0u;) {
    float x[4][Merge<D>::C], scale[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {  // four pieces in flight; the first one again, weightless, where fewer are left
      const int k = left != 0u ? __ffs(left) - 1 : i;
      scale[n] = __shfl_sync(0xffffffffu, weight, k);
      if (left == 0u) scale[n] = 0.f;
      left &= left - 1;
      Merge<D>::load(at(k), x[n]);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) merge.add(x[n], scale[n]);
  }
  return merge;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
  return x;
}

// Scratch: two pieces a CTA for the second kernel (the row it shares with the CTAs before it, the
// row it starts and shares with those behind), one a warp for the row a warp shares with the warps
// before it, and for every CTA the row that it starts and shares (-1: none) and the last CTA of it.
struct Scratch {
  float* cta_pieces;
  float* warp_pieces;
  int2* shared_rows;
};
template <int D, int NT>
__host__ __device__ Scratch carve(void* workspace, int ctas) {
  Scratch s;
  s.cta_pieces = static_cast<float*>(workspace);
  s.warp_pieces = s.cta_pieces + static_cast<int64_t>(2 * ctas) * Shape<D, NT>::kPiece;
  s.shared_rows = reinterpret_cast<int2*>(s.warp_pieces + static_cast<int64_t>(Shape<D, NT>::kWarps * ctas) * Shape<D, NT>::kPiece);
  return s;
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(Shape<D, NT>::kThreads, 1) int4_attention_kernel(const PagedInt4 p, int chunk, int parts) {
  using S = Shape<D, NT>;
  constexpr int kWarps = S::kWarps;
  extern __shared__ __align__(128) uint8_t s_ring[];
  __shared__ Shares<kWarps> s_shares;
  __shared__ int s_row[2 * kWarps];    // rows of the pieces left to merge, warp by warp (first, last), -1: none
  __shared__ int s_flags[2 * kWarps];  // kRowStart / kRowEnd of those pieces
  __shared__ int2 s_shared_row;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ctas = gridDim.x, cta = blockIdx.x;
  const int group = p.q_heads / p.kv_heads;
  const Scratch scratch = carve<D, NT>(p.workspace, ctas);
  uint8_t* ring = s_ring + warp * S::kRing;
  if (threadIdx.x < 2 * kWarps) s_row[threadIdx.x] = -1;
  if (threadIdx.x == 0) s_shared_row = make_int2(-1, -1);
  if (!p.early) dependency_wait();
  // this warp's places, of all rows or (parts > 0) of this cluster's row
  Plan plan;
  int cta_first, cta_places, first, end, units = 0;
  const int rank = parts > 0 ? cta % parts : 0;
  Requests ahead{};
  if (parts > 0) {
    ahead.row = cta / parts;
    const int tokens = row_tokens_at(p, ahead.row);
    if (threadIdx.x == 0) s_shares.tokens[ahead.row] = tokens;
    __syncthreads();
    units = row_units(tokens);
    plan.places = units + 1, plan.share = units + 1;
    cta_first = 1 + part_first(units, rank, parts), cta_places = 1 + part_first(units, rank + 1, parts) - cta_first;
  } else {
    plan = make_plan(p, s_shares, chunk, ctas);
    cta_first = static_cast<int>(min(static_cast<int64_t>(plan.share) * cta, static_cast<int64_t>(plan.places)));
    cta_places = min(plan.share, plan.places - cta_first);
  }
  first = cta_first + static_cast<int>(static_cast<int64_t>(cta_places) * warp / kWarps);
  end = cta_first + static_cast<int>(static_cast<int64_t>(cta_places) * (warp + 1) / kWarps);
  if (first < end) {
    int before = first;
    if (parts == 0) {
      const int2 found = find_rows(s_shares, first, lane);
      before -= found.y;
      for (ahead.row = found.x * chunk; ahead.row < p.batch * p.kv_heads; ++ahead.row) {
        const int places = row_places(tokens_of(p, s_shares, ahead.row));
        if (before < places) break;
        before -= places;
      }
    }
    ahead.place = before;
    ahead.left = end - first;
  }
  int id = ahead.row, place = ahead.place;  // of the unit at hand
  if (first < end) ahead.refill(p, s_shares, lane);
  if (p.early) dependency_wait();

  if (ahead.count > 0) {  // a unit, not the first place of a row alone
    Row<T, D, NT> row;
    uint4 queries[NT][D / kInt4Group];
    bool loaded = place > 0 || row_places(tokens_of(p, s_shares, id)) > 0;  // else a row without tokens stands here
    if (loaded) row.load(p, id, group, lane, queries);

    uint32_t request_at = smem_u32(ring) + 16 * lane;  // where this lane's part of the next goes
    const uint32_t ring_end = request_at + S::kRing;
    const uint8_t* pool = p.pool + 16 * lane;
    // One group of copies a call, an empty one behind the last unit.
    auto request = [&]() {
      if (ahead.next == ahead.count && ahead.left > 0) ahead.refill(p, s_shares, lane);
      if (ahead.next < ahead.count) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t tile = __shfl_sync(0xffffffffu, ahead.tile[k], ahead.next);
          const bool real = tile != kNoTile;
          const uint8_t* src = pool + (real ? static_cast<int64_t>(tile) * S::kTileBytes : 0);
#pragma unroll
          for (int n = 0; n < S::kTileBytes / 512; ++n) copy16(request_at + k * S::kTileBytes + 512 * n, src + 512 * n, real);
          if (S::kTileBytes % 512 != 0 && lane < S::kTileBytes % 512 / 16) {
            constexpr int kDone = S::kTileBytes / 512 * 512;
            copy16(request_at + k * S::kTileBytes + kDone, src + kDone, real);
          }
        }
        ++ahead.next;
        request_at = request_at + S::kStageBytes == ring_end ? request_at + S::kStageBytes - S::kRing : request_at + S::kStageBytes;
      }
      copies_close();
    };
#pragma unroll
    for (int k = 0; k < S::kStages - 1; ++k) request();

    int now = first;  // place, of all rows
    const uint8_t* at = ring;
    while (now < end) {
      int tokens = 0;
      for (; id < p.batch * p.kv_heads; ++id, place = 0, loaded = false) {
        tokens = tokens_of(p, s_shares, id);
        if (place < row_places(tokens)) break;
      }
      if (id >= p.batch * p.kv_heads) break;  // lengths that change under a call must not lead it out of the batch
      if (place == 0) {
        place = 1;
        if (++now == end) break;
      }
      const int in_all = row_units(tokens), in_row = place - 1;
      const int n = min(in_all - in_row, end - now);
      if (!loaded) row.load(p, id, group, lane, queries);
      row.start(p, queries, lane);
      const bool starts = in_row == 0, ends = in_row + n >= in_all;
      if (starts && lane == 0) {
        const int beyond = now + in_all - cta_first;  // places of the row's end from this CTA's first on
        if (beyond > cta_places) s_shared_row = make_int2(id, cta + (beyond - 1) / plan.share);
      }
      int left = tokens - in_row * kUnit;
      for (int k = 0; k < n; ++k, left -= kUnit) {
        copies_wait<S::kStages - 2>();
        __syncwarp();  // this unit is here, and every lane is done with the one before
        request();     // into that one's place
        row.unit(at, left, lane);
        at = at + S::kStageBytes == ring + S::kRing ? ring : at + S::kStageBytes;
      }
      now += n, place += n;
      row.finish(lane);
      if (starts && ends) {
        row.write_out(p, id, group, lane);
      } else {
        const bool last = end - now <= 1;  // one more place is the next row's first
        __syncwarp();
        row.deposit(last ? reinterpret_cast<float*>(ring) : scratch.warp_pieces + static_cast<int64_t>(cta * kWarps + warp) * S::kPiece, lane);
        if (lane == 0) {
          s_row[2 * warp + (last ? 1 : 0)] = id;
          s_flags[2 * warp + (last ? 1 : 0)] = (starts ? kRowStart : 0) | (ends ? kRowEnd : 0);
        }
      }
      loaded = false;
    }
    copies_wait<0>();
  }
  __syncthreads();

  // Only now: CTAs of the kernel behind, standing by from the start, cost 1 to 4 % of a long call.
  release_dependents();
  if (threadIdx.x == 0 && parts == 0) scratch.shared_rows[cta] = s_shared_row;
  // rows without tokens
  for (int r = parts == 0 ? cta : rank == 0 ? cta / parts : p.batch * p.kv_heads; r < p.batch * p.kv_heads; r += ctas) {
    if (tokens_of(p, s_shares, r) != 0) continue;
    const int2 at = row_place(p, r);
    for (int i = threadIdx.x; i < group * (D / 8); i += S::kThreads) {
      const int head = at.y * group + i / (D / 8), d = i % (D / 8) * 8;
      *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + at.x * p.o_sb + head * p.o_sh + d) = make_uint4(0, 0, 0, 0);
    }
  }

  // Rows that several warps, or several CTAs, hold: a warp takes a head, a lane the offset and the
  // sum of one piece.
  const int my_row = lane < 2 * kWarps ? s_row[lane] : -1;
  const int my_flags = my_row >= 0 ? s_flags[lane] : 0;
  const float* warp_pieces = scratch.warp_pieces + static_cast<int64_t>(cta) * kWarps * S::kPiece;
  auto piece_of = [&](int k) {
    return (k & 1) ? reinterpret_cast<const float*>(s_ring + (k >> 1) * S::kRing) : warp_pieces + (k >> 1) * S::kPiece;
  };
  int item = 0;  // (chain, head) pairs are dealt out to the warps in turn
  for (unsigned rest = __ballot_sync(0xffffffffu, my_row >= 0); rest != 0u;) {
    const int i = __ffs(rest) - 1;
    const int id = __shfl_sync(0xffffffffu, my_row, i);
    const unsigned chain = __ballot_sync(0xffffffffu, my_row == id);
    rest &= ~chain;
    const bool starts = (__shfl_sync(0xffffffffu, my_flags, i) & kRowStart) != 0;
    const bool ends = (__shfl_sync(0xffffffffu, my_flags, 31 - __clz(chain)) & kRowEnd) != 0;
    int head = warp - item + (warp < item ? kWarps : 0);
    item = (item + group) % kWarps;
    for (; head < group; head += kWarps) {
      float2 ml = make_float2(-INFINITY, 0.f);
      if (my_row == id) ml = *reinterpret_cast<const float2*>(piece_of(lane) + S::kHeads * S::kStride + 2 * head);
      const float top = warp_max(ml.x);
      const float weight = my_row == id ? fast_exp2(ml.x - top) : 0.f;
      const Merge<D> merge = merged<D>(chain, weight, [&](int k) { return piece_of(k) + head * S::kStride + lane * Merge<D>::C; });
      const float sum = warp_sum(ml.y * weight);
      if (starts && ends) {
        merge.template write_out<T>(p, id, group, head, lane, sum);
      } else {
        float* piece = scratch.cta_pieces + static_cast<int64_t>(2 * cta + (starts ? 1 : 0)) * S::kPiece;
        Merge<D>::store(piece + head * S::kStride + lane * Merge<D>::C, merge.o);
        if (lane == 0) *reinterpret_cast<float2*>(piece + S::kHeads * S::kStride + 2 * head) = make_float2(top, sum);
      }
    }
  }

  // the row of a cluster: its CTAs' pieces, a warp a head as before
  if (parts > 1) {
    cluster_sync();
    const int from = lane < parts ? part_first(units, lane, parts) : 0, to = lane < parts ? part_first(units, lane + 1, parts) : 0;
    const unsigned chain = __ballot_sync(0xffffffffu, from < to);
    if (chain & (chain - 1)) {  // one CTA alone has written its row
      const int first_cta = cta - rank, id = cta / parts;
      auto cta_piece = [&](int k) { return scratch.cta_pieces + static_cast<int64_t>(2 * (first_cta + k) + (part_first(units, k, parts) == 0 ? 1 : 0)) * S::kPiece; };
      for (int head = warp * parts + rank; head < group; head += kWarps * parts) {
        float2 ml = make_float2(-INFINITY, 0.f);
        if (from < to) ml = *reinterpret_cast<const float2*>(cta_piece(lane) + S::kHeads * S::kStride + 2 * head);
        const float top = warp_max(ml.x);
        const float weight = from < to ? fast_exp2(ml.x - top) : 0.f;
        const Merge<D> merge = merged<D>(chain, weight, [&](int k) { return cta_piece(k) + head * S::kStride + lane * Merge<D>::C; });
        merge.template write_out<T>(p, id, group, head, lane, warp_sum(ml.y * weight));
      }
    }
  }
}

// Rows that span CTAs: one CTA a CTA of the first kernel, for the row that starts there and goes on,
// `each` warps a query head, the pieces dealt out to those in turn.  Bound by latency: two dependent
// loads and a barrier; about 2 us, most of it the launch.  With 32 registers a thread, so that a CTA
// could stand by beside the first kernel's, its loads are no longer in flight together: 3 us more.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(1024) int4_combine_kernel(const PagedInt4 p, int ctas, int each) {
  using S = Shape<D, NT>;
  constexpr int C = Merge<D>::C;
  __shared__ float s_o[32][D];
  __shared__ float s_top[32], s_sum[32];
  release_dependents();
  dependency_wait();
  const Scratch scratch = carve<D, NT>(p.workspace, ctas);
  const int2 shared = scratch.shared_rows[blockIdx.x];
  const int row = shared.x, from = blockIdx.x, to = shared.y;
  if (row < 0) return;
  const int group = p.q_heads / p.kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = warp / each, part = warp % each;
  auto piece_of = [&](int c) { return scratch.cta_pieces + static_cast<int64_t>(2 * c + (c == from ? 1 : 0)) * S::kPiece; };
  float top = -INFINITY, sum = 0.f;
  Merge<D> merge;
  merge.clear();
  // offset and sum of 32 pieces of this warp at a time, a lane each
  for (int first = from + part; first <= to; first += 32 * each) {
    const int n = min(32, (to - first) / each + 1);
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < n) ml = *reinterpret_cast<const float2*>(piece_of(first + each * lane) + S::kHeads * S::kStride + 2 * head);
    float x[4][C];
#pragma unroll
    for (int y = 0; y < 4; ++y) Merge<D>::load(piece_of(first + each * min(y, n - 1)) + head * S::kStride + lane * C, x[y]);
    const float now = fmaxf(top, warp_max(ml.x));
    const float keep = sum == 0.f ? 0.f : fast_exp2(top - now);
    const float weight = lane < n ? fast_exp2(ml.x - now) : 0.f;
    top = now;
    sum = sum * keep + warp_sum(ml.y * weight);
#pragma unroll
    for (int c = 0; c < C; ++c) merge.o[c] *= keep;
    for (int k = 0; k < n; k += 4) {
      float next[4][C];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        if (k + 4 < n) Merge<D>::load(piece_of(first + each * min(k + 4 + y, n - 1)) + head * S::kStride + lane * C, next[y]);
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float scale = __shfl_sync(0xffffffffu, weight, (k + y) & 31);
        if (k + y < n) merge.add(x[y], scale);
#pragma unroll
        for (int c = 0; c < C; ++c) x[y][c] = next[y][c];
      }
    }
  }
  Merge<D>::store(&s_o[warp][lane * C], merge.o);
  if (lane == 0) s_top[warp] = top, s_sum[warp] = sum;
  __syncthreads();
  if (part != 0) return;
  const int parts = min(each, to - from + 1);
  float all = top;
  for (int w = 1; w < parts; ++w) all = fmaxf(all, s_top[warp + w]);
  sum = 0.f;
  merge.clear();
  for (int w = 0; w < parts; ++w) {
    const float weight = fast_exp2(s_top[warp + w] - all);
    float x[C];
    Merge<D>::load(&s_o[warp + w][lane * C], x);
    merge.add(x, weight);
    sum = fmaf(s_sum[warp + w], weight, sum);
  }
  merge.template write_out<T>(p, row, group, head, lane, sum);
}

int64_t units_of_table(const PagedInt4& p) { return (p.table_width * p.page_size + kUnit - 1) / kUnit; }

// None where row_parts() says one CTA a row for every smaller batch too: two units a warp at most.  (A
// call that needs none is 2 us shorter on the host: nothing is allocated for it.)
template <int D, int NT>
int64_t scratch_bytes(const PagedInt4& p) {
  const int ctas = sm_count();
  if (static_cast<int64_t>(p.batch) * p.kv_heads <= ctas && units_of_table(p) <= 2 * Shape<D, NT>::kWarps) return 0;
  const int64_t pieces = static_cast<int64_t>(2 + Shape<D, NT>::kWarps) * ctas * Shape<D, NT>::kPiece * 4;
  return (pieces + 8 * ctas + 15) / 16 * 16;
}

// CTAs, a cluster, that hold a row each alone; 0: all CTAs share the places of all rows and the second
// kernel joins rows that span some.  In units of a warp times two (0.85 us), of what rows as long as the
// table take: a row's CTA starts and ends in about 3.2 us and those of a cluster in 5.5, with 1.7 for
// every unit of a warp; the shares with the second kernel take 8.1 us and more.  Two sequences' rows (2 x
// 128, 12 warps) of 128 tokens: 4.5 us on one CTA, 6.8 by shares; 513: 6.9, 8.1; 1024: 8.6, on four 7.2,
// 8.2; 2048: on eight 7.5, 8.6; 4096: on eight 9.4, 9.0.  Lengths are not known here, so a row has its
// own CTAs only where the longest possible rows take less than the shortest shares, unless the rows are
// known to be about equally long.  More clusters of eight than 112 CTAs do not run at once, of four 128.
// Other shapes have other times and the same order, rows as long as the table, alone and by shares: 8 of 512
// tokens, 4 x 64 (16 warps) 5.8 and 7.9 us, 16 heads on 1 x 128 (8 warps) 9.4 and 11.3, 16 on 1 x 64 7.3 and 9.6;
// 8 of 2048, 7.4 (four CTAs) and 7.8, 10.6 (eight) and 13.0, 8.9 (eight) and 11.0.  Of 30 sizes a shape, 128..8192
// tokens in 2..64 rows, the worst choice of CTAs was 8.7 us against 8.4 by shares (32 of 2048, 4 x 64); where the
// shares are kept for want of the lengths, full rows would be up to 23 % sooner alone (64 of 1024, 16 on 1 x 64).
int row_parts(int64_t rows, int64_t row_units, int warps, int ctas, bool even) {
  auto warp_units = [&](int64_t units) { return (units + warps - 1) / warps; };
  int64_t best = even ? 5 + 2 * warp_units((rows * (row_units + 1) + ctas - 1) / ctas) : 7;
  int parts = 0;
  for (int n = 1; n <= 8; n *= 2) {
    if (rows * n > (n == 8 ? ctas * 3 / 4 : n > 1 ? ctas * 7 / 8 : ctas)) break;
    const int64_t time = 2 * warp_units((row_units + n - 1) / n) + (n > 1 ? 3 : 0);
    if (time < best) best = time, parts = n;
  }
  return parts;
}

template <typename T, int D, int NT>
int launch(const PagedInt4& p, cudaStream_t stream) {
  using S = Shape<D, NT>;
  const int64_t rows = static_cast<int64_t>(p.batch) * p.kv_heads;
  const int ctas = sm_count();
  const int64_t need = scratch_bytes<D, NT>(p);
  QF_REQUIRE((p.workspace != nullptr || need == 0) && p.workspace_bytes >= need, "the workspace holds %lld bytes, %lld are needed",
             static_cast<long long>(p.workspace_bytes), static_cast<long long>(need));
  static thread_local int ready = -1;  // device whose kernel attribute this thread has set
  int device = 0;
  QF_CUDA(cudaGetDevice(&device));
  if (ready != device) {
    QF_CUDA(cudaFuncSetAttribute(int4_attention_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
    ready = device;
  }
  const int64_t row_units = units_of_table(p);
  if (const int parts = row_parts(rows, row_units, S::kWarps, ctas, p.even); parts > 0) {
    const dim3 grid(static_cast<unsigned>(rows * parts)), block(S::kThreads);
    if (parts == 1) {
      QF_CUDA(launch_chained(int4_attention_kernel<T, D, NT>, grid, block, static_cast<size_t>(S::kSmem), stream, p, 0, parts));
    } else {
      QF_CUDA(launch_chained(int4_attention_kernel<T, D, NT>, grid, block, static_cast<size_t>(S::kSmem), stream,
                             ClusterShape{static_cast<unsigned>(parts), 1, 1}, p, 0, parts));
    }
    return QF_OK;
  }
  const int chunk = static_cast<int>((rows + S::kThreads - 1) / S::kThreads);
  QF_CUDA(launch_chained(int4_attention_kernel<T, D, NT>, dim3(ctas), dim3(S::kThreads), static_cast<size_t>(S::kSmem), stream, p, chunk, 0));
  // warps a head in the second kernel, four pieces each or more: a row is on all CTAs' share of the
  // rows at most, and on as many CTAs as its table has room for
  const int group = p.q_heads / p.kv_heads;
  const int64_t row_ctas = std::min<int64_t>(ctas / rows, row_units / S::kWarps) / 4;
  const int each = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(row_ctas, group <= 8 ? 4 : 2)));
  QF_CUDA(launch_chained(int4_combine_kernel<T, D, NT>, dim3(ctas), dim3(32 * group * each), static_cast<size_t>(0), stream, p, ctas, each));
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

int sm_count() {
  static std::atomic<int> counts[64];  // 0: not asked yet; the answer never changes
  int device = 0, count = 0;
  if (cudaGetDevice(&device) != cudaSuccess) {
    (void)cudaGetLastError();
    return 148;
  }
  if (device < 64 && (count = counts[device].load(std::memory_order_relaxed)) != 0) return count;
  if (cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) {
    (void)cudaGetLastError();
    return 148;
  }
  if (device < 64) counts[device].store(count, std::memory_order_relaxed);
  return count;
}

int64_t int4_attention_bytes(const PagedInt4& p, int head_dim) {
  const bool two = p.q_heads / p.kv_heads > 8;
  if (head_dim == 128) return two ? scratch_bytes<128, 2>(p) : scratch_bytes<128, 1>(p);
  return two ? scratch_bytes<64, 2>(p) : scratch_bytes<64, 1>(p);
}

int launch_int4_attention(const PagedInt4& p, int head_dim, int dtype, cudaStream_t stream) {
  return dtype == QF_DTYPE_F16 ? launch_for<__half>(p, head_dim, stream) : launch_for<__nv_bfloat16>(p, head_dim, stream);
}

}  // namespace qf

extern "C" int qf_int4_decode_attention(const qf_paged_int4_args* args, void* stream) {
  qf::PagedInt4 p;
  if (const int rc = qf::fill_paged_int4(args, qf::kNeedsQuery | qf::kNeedsPool | qf::kNeedsOut, &p)) return rc;
  if (p.batch == 0) return QF_OK;
  // a table a KV head is what a choice of pages wrote: read behind the wait, whatever was launched since
  p.early = p.t_sh == 0 && p.l_sh == 0;
  return qf::launch_int4_attention(p, args->head_dim, args->dtype, static_cast<cudaStream_t>(stream));
}
