// Choosing the pages a query attends.  Bounds: the smallest and the largest key of every page
// and channel, as the 4-bit cache reads back.  No key k of a page scores above
//     sum_d max(q_d low_d, q_d high_d)  >=  q . k
// so a page's score is the largest of that over the query heads of its KV head, and a row
// (sequence, KV head) takes its newest page and the take - 1 others that score highest, ties
// to the lower page.  The products are exact in fp32 and are added pairwise, neighbours first,
// whatever the kernel's layout: the same inputs choose the same pages everywhere.
#include <algorithm>

#include "qf_int4_paged.cuh"

namespace qf {

int fill_paged_int4(const qf_paged_int4_args* a, int needs, PagedInt4* p) {
  QF_REQUIRE(a != nullptr, "args must not be null");
  QF_REQUIRE(a->dtype == QF_DTYPE_F16 || a->dtype == QF_DTYPE_BF16, "q must be float16 or bfloat16");
  QF_REQUIRE(a->head_dim == 64 || a->head_dim == 128, "head dimension must be 64 or 128");
  QF_REQUIRE(a->page_size >= kInt4Tile && a->page_size % kInt4Tile == 0, "page size must be a multiple of 16");
  QF_REQUIRE(a->batch >= 0 && a->kv_heads >= 1, "batch and head counts must be positive");
  QF_REQUIRE(static_cast<int64_t>(a->batch) * a->kv_heads < (1LL << 31), "too many rows");
  QF_REQUIRE(a->num_pages >= 0 && a->num_pages < (1LL << 31) && a->table_width >= 0, "invalid pool or table size");
  // tiles of the pool are counted in 32 bits
  QF_REQUIRE(a->num_pages <= 0xfffffffeLL / a->kv_heads / (a->page_size / kInt4Tile), "invalid pool or table size");
  // tokens of a row, and tiles of all rows, are counted in 31 bits
  QF_REQUIRE(a->table_width < (1LL << 30) / a->page_size, "a block table row holds 2^30 tokens or more");
  QF_REQUIRE(static_cast<int64_t>(a->batch) * a->kv_heads * a->table_width < (1LL << 30) / (a->page_size / kInt4Tile),
             "the block tables of a call hold 2^30 tiles of 16 tokens or more");
  if (needs & kNeedsQuery) {
    QF_REQUIRE(a->q_heads >= 1 && a->q_heads % a->kv_heads == 0, "query heads must be divisible by KV heads");
    QF_REQUIRE(a->q_heads / a->kv_heads <= 16, "at most 16 query heads share a KV head");
  }
  QF_REQUIRE(a->table_dtype == QF_INDEX_I32 || a->table_dtype == QF_INDEX_I64, "page table must use an integer dtype");
  QF_REQUIRE(a->lens_dtype == QF_INDEX_I32 || a->lens_dtype == QF_INDEX_I64, "lengths must use an integer dtype");
  auto aligned = [](const void* x) { return on_boundary(x, 16); };
  if (a->batch > 0) {
    QF_REQUIRE(a->seq_lens && (a->block_table || a->table_width == 0), "block table and lengths must not be null");
    QF_REQUIRE(index_aligned(a->block_table, a->table_dtype) && index_aligned(a->seq_lens, a->lens_dtype),
               "block table and lengths must be aligned to their elements");
    if (needs & kNeedsQuery) {
      QF_REQUIRE(aligned(a->workspace), "the workspace must be 16-byte aligned");
      QF_REQUIRE(a->q && aligned(a->q) && a->q_stride_b % 8 == 0 && a->q_stride_h % 8 == 0,
                 "q must be 16-byte aligned with strides of a multiple of 8 elements");
    }
    if (needs & kNeedsPool) QF_REQUIRE((a->pool || a->num_pages == 0) && aligned(a->pool), "the pool must be 16-byte aligned");
    if (needs & kNeedsOut) {
      QF_REQUIRE(a->out && aligned(a->out) && a->o_stride_b % 8 == 0 && a->o_stride_h % 8 == 0,
                 "out must be 16-byte aligned with strides of a multiple of 8 elements");
    }
    if (needs & kNeedsBounds) {
      QF_REQUIRE((a->key_bounds || a->num_pages == 0) && aligned(a->key_bounds), "key bounds must be 16-byte aligned");
    }
    if (needs & kNeedsSelection) {
      QF_REQUIRE(a->take >= 1, "at least one page must be taken");
      QF_REQUIRE(a->take < (1LL << 30) / a->page_size, "the pages taken hold 2^30 tokens or more");
      QF_REQUIRE(static_cast<int64_t>(a->batch) * a->kv_heads * a->take < (1LL << 30) / (a->page_size / kInt4Tile),
                 "the pages taken hold 2^30 tiles of 16 tokens or more");
      QF_REQUIRE(a->page_table && a->page_lens, "page_table and page_lens must not be null");
      QF_REQUIRE(index_aligned(a->page_table, QF_INDEX_I32) && index_aligned(a->page_lens, QF_INDEX_I32),
                 "page_table and page_lens must be aligned to their elements");
    }
  }
  PagedInt4 r{};
  r.q = a->q, r.out = a->out, r.pool = static_cast<const uint8_t*>(a->pool), r.bounds = a->key_bounds;
  r.table = a->block_table, r.lens = a->seq_lens, r.workspace = a->workspace, r.workspace_bytes = a->workspace_bytes;
  r.page_table = a->page_table, r.page_lens = a->page_lens;
  r.q_sb = a->q_stride_b, r.q_sh = a->q_stride_h, r.o_sb = a->o_stride_b, r.o_sh = a->o_stride_h;
  r.t_sb = a->table_stride_b, r.t_sh = a->table_stride_h, r.t_sp = a->table_stride_p;
  r.l_sb = a->lens_stride_b, r.l_sh = a->lens_stride_h;
  r.num_pages = a->num_pages, r.table_width = a->table_width;
  r.scale = a->scale;
  r.batch = a->batch, r.q_heads = a->q_heads, r.kv_heads = a->kv_heads, r.page_size = a->page_size;
  r.table_dtype = a->table_dtype, r.lens_dtype = a->lens_dtype;
  r.new_tokens = a->new_tokens, r.take = a->take;
  r.even = false;
  r.early = true;
  r.by_heads = make_divisor(a->kv_heads), r.by_page = make_divisor(a->page_size);
  r.by_tiles = make_divisor(a->page_size / kInt4Tile);
  if (a->batch > 0) {
    r.status = device_status_word();
    QF_REQUIRE(r.status != nullptr, "no device status word");
  }
  *p = r;
  return QF_OK;
}

namespace {

// Extremes and scores keep a NaN: a page that holds one must not look harmless.
__device__ __forceinline__ float max2_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// A warp takes a page, or four warps a page of kManyTiles and more, or two or four where pages are few;
// a lane holds eight channels of
// 16 / (32 / (D / 8)) tokens of a tile, all loaded at once, and two tokens a step of the
// three-operand minimum and maximum.  Rounding to T is monotone and comes once, after the warps of a
// page have met.  Bound by issue, 25 instructions an eight codes: 16 prompts of 4096..8192 tokens
// (2 x 128, pages of 64, 16 MB) take 10.7 us, a step's newest pages of 64 sequences 2.3 us.  Four warps
// a page against one, the same prompts: pages of 64 tokens 14.8 and 10.7 us, of 128 12.0 and 15.5, of
// 256 11.1 and 22.7; the newest page of each of 32 sequences ahead of their sparse attention, pages of
// 64: 37.2 us in all and 40.0.
constexpr int kBoundWarps = 4, kManyTiles = 8;
template <typename T, int D>
__global__ void __launch_bounds__(32 * kBoundWarps) key_bounds_kernel(const PagedInt4 p, const Divisor by_each, int warps_each) {
  constexpr int W = D / kInt4Group, kWords = D / 8, kStep = 32 / kWords, kTokens = kInt4Tile / kStep;
  __shared__ float s_low[kBoundWarps][8][kWords], s_high[kBoundWarps][8][kWords];
  dependency_wait();
  release_dependents();  // behind the wait: scores and attention read lengths and tables before theirs
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int part = warp % warps_each;  // of the page's warps
  const uint32_t unit = blockIdx.x * (kBoundWarps / warps_each) + warp / warps_each;
  const uint32_t row = quotient(unit, by_each);
  const int2 at = row_place(p, row);
  const int i = unit - row * by_each.d, h = at.y;
  int64_t page = -1;
  int live = 0;
  if (at.x < p.batch) {
    const int tokens = static_cast<int>(row_tokens(p, at.x, 0));
    const int before = tokens > p.new_tokens ? tokens - p.new_tokens : 0;
    const int n = quotient(before, p.by_page) + i;
    const int left = tokens - n * p.page_size;
    if (n < p.table_width && left > 0) {
      page = page_id(p, at.x, 0, n);
      if (page >= 0 && page < p.num_pages) {
        live = min(left, p.page_size);
      } else if (lane == 0 && part == 0) {
        atomicMax(p.status, kStatusBadPageId);
      }
    }
  }
  const int word = lane % kWords, t = word / W, w = word % W, first = lane / kWords;
  float low[8], high[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) low[j] = INFINITY, high[j] = -INFINITY;
  const uint8_t* tile = p.pool + ((page * p.kv_heads + h) * (p.page_size / kInt4Tile) + part) * int4_tile_bytes(D);
  for (int begin = part * kInt4Tile; begin < live; begin += warps_each * kInt4Tile, tile += warps_each * int4_tile_bytes(D)) {
    uint32_t codes[kTokens];
    T steps[kTokens], floors[kTokens];
    auto load = [&](int k, int r) {
      codes[k] = *reinterpret_cast<const uint32_t*>(tile + r * (D / 2) + 4 * word);
      const T* params = reinterpret_cast<const T*>(tile + 16 * D) + r * W + w;
      steps[k] = params[0], floors[k] = params[D / 2];
    };
    if (begin + kInt4Tile <= live) {
#pragma unroll
      for (int k = 0; k < kTokens; ++k) load(k, first + kStep * k);
    } else {  // behind the last token: the first one of the tile again, which every tile here has
#pragma unroll
      for (int k = 0; k < kTokens; ++k) load(k, begin + first + kStep * k < live ? first + kStep * k : 0);
    }
#pragma unroll
    for (int k = 0; k < kTokens; k += 2) {
      float x[8], y[8];
      int4_values(codes[k], to_float(steps[k]), to_float(floors[k]), x);
      int4_values(codes[k + 1], to_float(steps[k + 1]), to_float(floors[k + 1]), y);
#pragma unroll
      for (int j = 0; j < 8; ++j) low[j] = min_nan(low[j], x[j], y[j]), high[j] = max_nan(high[j], x[j], y[j]);
    }
  }
#pragma unroll
  for (int off = kWords; off < 32; off <<= 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = __shfl_xor_sync(0xffffffffu, low[j], off), z = __shfl_xor_sync(0xffffffffu, high[j], off);
      low[j] = min_nan(low[j], a, a), high[j] = max_nan(high[j], z, z);
    }
  }
  if (warps_each > 1) {
    if (lane < kWords) {
#pragma unroll
      for (int j = 0; j < 8; ++j) s_low[warp][j][lane] = low[j], s_high[warp][j][lane] = high[j];
    }
    __syncthreads();
    if (part != 0) return;
    for (int k = 1; k < warps_each; ++k) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float a = s_low[warp + k][j][word], z = s_high[warp + k][j][word];
        low[j] = min_nan(low[j], a, a), high[j] = max_nan(high[j], z, z);
      }
    }
  }
  if (live > 0 && lane < kWords) {
    T* dst = static_cast<T*>(p.bounds) + (page * p.kv_heads + h) * 2 * D + 32 * w + 8 * t;
    *reinterpret_cast<uint4*>(dst) =
        make_uint4(pack2<T>(low[0], low[1]), pack2<T>(low[2], low[3]), pack2<T>(low[4], low[5]), pack2<T>(low[6], low[7]));
    *reinterpret_cast<uint4*>(dst + D) =
        make_uint4(pack2<T>(high[0], high[1]), pack2<T>(high[2], high[3]), pack2<T>(high[4], high[5]), pack2<T>(high[6], high[7]));
  }
}

// Scores as unsigned keys that order like the scores, NaN above all; 0 is below every score.
__device__ __forceinline__ uint32_t score_key(float s) {
  if (!(s == s)) return 0xffffffffu;
  const uint32_t u = __float_as_uint(__fadd_rn(s, 0.f));  // -0 and 0 tie
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// keys[row][n], row = b * kv_heads + h: D / 8 lanes a page, eight channels each, two pages a lane,
// whose products and sums are the two halves of packed instructions; the row's queries lie in
// shared memory, every element twice for that.  Bound by issue, about 80 instructions a page pair and
// query head, and by lengths -> table -> bounds: 10 300 pages of 32 sequences (2 x 128, 6 heads each,
// 10.5 MB) take 8 us, 2048 pages of one 4 us.
template <typename T, int D>
__global__ void __launch_bounds__(128) page_score_kernel(const PagedInt4 p, uint32_t* keys) {
  constexpr int kLanes = D / 8, kPages = 32 / kLanes, kMaxGroup = 16, kCtaPages = 4 * 2 * kPages;
  __shared__ __align__(16) float4 s_q[kMaxGroup][4][kLanes];  // two channels of a lane: neighbouring lanes, neighbouring banks
  if (!p.early) dependency_wait();
  const int row = blockIdx.y;
  const int2 at = row_place(p, row);
  const int b = at.x, h = at.y;
  const int lane = threadIdx.x % 32, l = lane % kLanes;
  const int group = p.q_heads / p.kv_heads;
  const int tokens = static_cast<int>(row_tokens(p, b, 0));
  const int count = quotient(tokens + p.page_size - 1, p.by_page);
  const bool idle = count <= p.take || static_cast<int>(blockIdx.x) * kCtaPages >= count - 1;  // every page is taken, or none is left
  const int step = gridDim.x * kCtaPages;
  int first = blockIdx.x * kCtaPages + threadIdx.x / 32 * 2 * kPages;
  int64_t page[2];  // of this turn
  auto find = [&](int from) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int n = from + k * kPages + lane / kLanes;
      page[k] = n < count - 1 ? page_id(p, b, 0, n) : -1;
      if (n < count - 1 && (page[k] < 0 || page[k] >= p.num_pages)) {
        page[k] = -1;
        if (l == 0) atomicMax(p.status, kStatusBadPageId);
      }
    }
  };
  if (!idle) find(first);
  if (p.early) dependency_wait();
  if (idle) return;
  uint4 lo[2], hi[2];
  bool ok[2];
  auto fetch = [&]() {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      ok[k] = page[k] >= 0;
      lo[k] = hi[k] = make_uint4(0, 0, 0, 0);
      if (ok[k]) {
        const T* src = static_cast<const T*>(p.bounds) + (page[k] * p.kv_heads + h) * 2 * D + 8 * l;
        lo[k] = *reinterpret_cast<const uint4*>(src), hi[k] = *reinterpret_cast<const uint4*>(src + D);
      }
    }
  };
  fetch();
  for (int i = threadIdx.x; i < group * (D / 8); i += 128) {
    const int g = i / (D / 8), d = i % (D / 8) * 8;
    const uint4 raw = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + b * p.q_sb + static_cast<int64_t>(h * group + g) * p.q_sh + d);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 x = unpack2<T>((&raw.x)[j]);
      s_q[g][j][d / 8] = make_float4(x.x, x.x, x.y, x.y);
    }
  }
  __syncthreads();
  release_dependents();  // not from the start: kernels standing by cost this one 2 to 4 us, and to release at the end 1 us in front of one sequence
  for (; first < count - 1; first += step) {
    uint64_t low[8], high[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 a = unpack2<T>((&lo[0].x)[j]), c = unpack2<T>((&lo[1].x)[j]), y = unpack2<T>((&hi[0].x)[j]), z = unpack2<T>((&hi[1].x)[j]);
      low[2 * j] = pair32(a.x, c.x), low[2 * j + 1] = pair32(a.y, c.y);
      high[2 * j] = pair32(y.x, z.x), high[2 * j + 1] = pair32(y.y, z.y);
    }
    const bool now[2] = {ok[0], ok[1]};
    if (first + step < count - 1) {  // the next turn's bounds come in meanwhile
      find(first + step);
      fetch();
    }
    float best[2] = {-INFINITY, -INFINITY};
    for (int g = 0; g < group; ++g) {
      uint64_t term[8];
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const ulonglong2 q = *reinterpret_cast<const ulonglong2*>(&s_q[g][j / 2][l]);
        const float2 a = unpair32(mul32x2(q.x, low[j])), c = unpair32(mul32x2(q.x, high[j]));
        const float2 y = unpair32(mul32x2(q.y, low[j + 1])), z = unpair32(mul32x2(q.y, high[j + 1]));
        term[j] = pair32(max2_nan(a.x, c.x), max2_nan(a.y, c.y));
        term[j + 1] = pair32(max2_nan(y.x, z.x), max2_nan(y.y, z.y));
      }
      uint64_t s = add32x2(add32x2(add32x2(term[0], term[1]), add32x2(term[2], term[3])),
                           add32x2(add32x2(term[4], term[5]), add32x2(term[6], term[7])));
#pragma unroll
      for (int off = 1; off < kLanes; off <<= 1) s = add32x2(s, __shfl_xor_sync(0xffffffffu, s, off));
      const float2 both = unpair32(s);
      best[0] = max2_nan(best[0], both.x), best[1] = max2_nan(best[1], both.y);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int n = first + k * kPages + lane / kLanes;
      if (l == 0 && n < count - 1) keys[static_cast<int64_t>(row) * p.table_width + n] = now[k] ? score_key(best[k]) : 0u;
    }
  }
}

// A page id as the choice holds it: an id that 32 bits do not hold is no page either way.
__device__ __forceinline__ int32_t chosen_id(int64_t id) { return id < 0 || id > 0x7fffffff ? -1 : static_cast<int32_t>(id); }

constexpr int kPickThreads = 512;

// One CTA a row.  The take - 1 largest keys of the pages before the newest: the smallest of them eight
// bits at a time from the highest bit in which keys differ, by counting the keys that agree so far over
// their next bits; it ends with a bin that is taken whole, mostly the second.  Then the pages in order,
// those that tie with the smallest as long as there is room.  A thread holds a run of kHeld neighbouring
// keys and their pages in registers; longer rows are read again from the second level cache every time.
// Bound by latency, loads and barriers: 2048 pages of one sequence take 6.7 us by themselves with the
// launch; two bits at a time, counted in registers, took 10.6.  `last`: the choice ends a call.  Kernels
// behind may read table and lengths before they wait, so they start only when those are written; the
// attention of a sparse call waits first and may stand by from the start.
template <int kHeld>
__global__ void __launch_bounds__(kPickThreads) page_pick_kernel(const PagedInt4 p, const uint32_t* keys, bool last) {
  constexpr int kBins = 256, kPasses = 4;
  __shared__ __align__(16) int s_bins[kPasses][kBins];
  __shared__ uint32_t s_low[kPickThreads / 32], s_high[kPickThreads / 32];
  __shared__ int2 s_scan[kPickThreads / 32];
  if (!last) release_dependents();
  const int row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  for (int i = tid; i < kPasses * kBins; i += kPickThreads) (&s_bins[0][0])[i] = 0;
  if (!p.early) dependency_wait();
  const int2 at = row_place(p, row);
  const int b = at.x;
  const int tokens = static_cast<int>(row_tokens(p, b, 0));
  const int count = quotient(tokens + p.page_size - 1, p.by_page);
  int32_t* out = p.page_table + static_cast<int64_t>(row) * p.take;
  const int others = count - 1, want = p.take - 1;
  const int run = kHeld > 0 ? kHeld : (others + kPickThreads - 1) / kPickThreads;
  const int first = min(tid * run, others), end = min(first + run, others);
  const bool all = count <= p.take;
  uint32_t held[kHeld > 0 ? kHeld : 1];
  int32_t pages[kHeld > 0 ? kHeld : 1];
  if constexpr (kHeld > 0) {
#pragma unroll
    for (int k = 0; k < kHeld; ++k) pages[k] = !all && first + k < end ? chosen_id(page_id(p, b, 0, first + k)) : -1;
  }
  if (p.early) dependency_wait();
  if (tid == 0) p.page_lens[row] = tokens - (all ? 0 : (count - p.take) * p.page_size);
  if (all) {
    for (int n = tid; n < p.take; n += kPickThreads) out[n] = n < count ? chosen_id(page_id(p, b, 0, n)) : -1;
    return;
  }
  const uint32_t* mine = keys + static_cast<int64_t>(row) * p.table_width;
  if constexpr (kHeld > 0) {
#pragma unroll
    for (int k = 0; k < kHeld; ++k) held[k] = first + k < end ? mine[first + k] : 0u;
  }
  // `visit` sees this thread's keys, those of places behind the last too
  auto visit = [&](auto&& f) {
    if constexpr (kHeld > 0) {
#pragma unroll
      for (int k = 0; k < kHeld; ++k) f(first + k, held[k], pages[k]);
    } else {
      for (int n = first; n < end; ++n) f(n, mine[n], -1);
    }
  };
  auto id_of = [&](int n, int32_t page) { return kHeld > 0 ? page : chosen_id(page_id(p, b, 0, n)); };
  // the bits that all keys share
  uint32_t low = 0xffffffffu, high = 0u;
  visit([&](int n, uint32_t key, int32_t) {
    if (n < end) low = min(low, key), high = max(high, key);
  });
  low = __reduce_min_sync(0xffffffffu, low), high = __reduce_max_sync(0xffffffffu, high);
  if (lane == 0) s_low[warp] = low, s_high[warp] = high;
  __syncthreads();
  low = __reduce_min_sync(0xffffffffu, lane < kPickThreads / 32 ? s_low[lane] : 0xffffffffu);
  high = __reduce_max_sync(0xffffffffu, lane < kPickThreads / 32 ? s_high[lane] : 0u);
  // `least`: the largest value that at least `want` keys reach, its bits from `shift` on so far
  uint32_t least = low;
  if (low != high) {
    int shift = max(24 - __clz(low ^ high), 0), left = want;
    uint32_t bins = kBins;  // of the pass: keys that agree so far are less than so many steps off
    least = shift == 24 ? 0u : high >> (shift + 8) << (shift + 8);
    for (int pass = 0;; ++pass) {
      visit([&](int n, uint32_t key, int32_t) {
        const uint32_t bin = (key ^ least) >> shift;
        if (n < end && bin < bins) atomicAdd(&s_bins[pass][bin], 1);
      });
      __syncthreads();
      // every warp for itself: eight bins a lane, the lanes' sums from the top, and the bin in which the
      // count passes `left`
      const int4 x = reinterpret_cast<const int4*>(s_bins[pass])[2 * lane], y = reinterpret_cast<const int4*>(s_bins[pass])[2 * lane + 1];
      const int n8[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
      const int mine8 = (x.x + x.y) + (x.z + x.w) + ((y.x + y.y) + (y.z + y.w));
      int from = mine8;  // of this lane and those above
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int z = __shfl_down_sync(0xffffffffu, from, off);
        if (lane + off < 32) from += z;
      }
      int over = from - mine8, bin = 0, size = 0;  // keys in the bins above, the bin, its keys
      bool found = false;
#pragma unroll
      for (int k = 7; k >= 0; --k) {
        if (!found) {
          bin = 8 * lane + k, size = n8[k];
          found = over + size >= left;
          if (!found) over += size;
        }
      }
      const int lane_of = 31 - __clz(__ballot_sync(0xffffffffu, from >= left));  // the highest such lane holds the bin
      over = __shfl_sync(0xffffffffu, over, lane_of), bin = __shfl_sync(0xffffffffu, bin, lane_of), size = __shfl_sync(0xffffffffu, size, lane_of);
      least |= static_cast<uint32_t>(bin) << shift;
      left -= over;
      if (size == left || shift == 0) break;
      bins = min(1u << shift, static_cast<uint32_t>(kBins));
      shift = max(shift - 8, 0);
    }
  }
  int above = 0, equal = 0;
  visit([&](int n, uint32_t key, int32_t) { above += n < end && key > least, equal += n < end && key == least; });
  // exclusive sums of both over the threads before this one
  int2 sum = make_int2(above, equal);
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, sum.x, off), y = __shfl_up_sync(0xffffffffu, sum.y, off);
    if (lane >= off) sum.x += x, sum.y += y;
  }
  if (lane == 31) s_scan[warp] = sum;
  __syncthreads();
  int before_above = sum.x - above, before_equal = sum.y - equal, all_above = 0;
#pragma unroll
  for (int w = 0; w < kPickThreads / 32; ++w) {
    const int2 x = s_scan[w];
    if (w < warp) before_above += x.x, before_equal += x.y;
    all_above += x.x;
  }
  const int ties = want - all_above;  // the first so many of the keys equal to `least`
  visit([&](int n, uint32_t key, int32_t page) {
    if (n >= end) return;
    if (key > least) {
      out[before_above + min(before_equal, ties)] = id_of(n, page);
      ++before_above;
    } else if (key == least) {
      if (before_equal < ties) out[before_above + before_equal] = id_of(n, page);
      ++before_equal;
    }
  });
  if (tid == 0) out[p.take - 1] = chosen_id(page_id(p, b, 0, count - 1));
}

// Bytes of the keys, a multiple of 16.
int64_t select_bytes(const PagedInt4& p) {
  return (static_cast<int64_t>(p.batch) * p.kv_heads * p.table_width * 4 + 15) / 16 * 16;
}

// Attention over the selection: its table and lengths, and the scratch behind the keys.
PagedInt4 over_selection(PagedInt4 p) {
  p.table = p.page_table, p.table_dtype = QF_INDEX_I32, p.table_width = p.take;
  p.t_sb = static_cast<int64_t>(p.kv_heads) * p.take, p.t_sh = p.take, p.t_sp = 1;
  p.lens = p.page_lens, p.lens_dtype = QF_INDEX_I32;
  p.l_sb = p.kv_heads, p.l_sh = 1;
  p.early = false;  // the kernel in front writes both
  p.even = true;
  return p;
}

int launch_select(const PagedInt4& p, int head_dim, int dtype, bool last, cudaStream_t stream) {
  QF_REQUIRE((p.workspace != nullptr || select_bytes(p) == 0) && p.workspace_bytes >= select_bytes(p), "the workspace holds %lld bytes, %lld are needed",
             static_cast<long long>(p.workspace_bytes), static_cast<long long>(select_bytes(p)));
  const int rows = p.batch * p.kv_heads;
  QF_REQUIRE(rows <= 65535, "at most 65535 (sequence, KV head) rows choose pages in one call");
  uint32_t* keys = static_cast<uint32_t*>(p.workspace);
  // A CTA takes 16 pages (D 128) or 32 at a time: all of them at once while that is one wave of
  // about 900 CTAs, in turns beyond it.
  const int64_t pages = head_dim == 128 ? 16 : 32;
  const int64_t blocks = (p.table_width + pages - 1) / pages, most = std::max<int64_t>(1, 900 / rows);
  const dim3 grid(static_cast<unsigned>(std::max<int64_t>(1, std::min(blocks, most))), rows);
  cudaError_t err = cudaSuccess;
  if (dtype == QF_DTYPE_F16) {
    err = head_dim == 128 ? launch_chained(page_score_kernel<__half, 128>, grid, dim3(128), 0, stream, p, keys)
                          : launch_chained(page_score_kernel<__half, 64>, grid, dim3(128), 0, stream, p, keys);
  } else {
    err = head_dim == 128 ? launch_chained(page_score_kernel<__nv_bfloat16, 128>, grid, dim3(128), 0, stream, p, keys)
                          : launch_chained(page_score_kernel<__nv_bfloat16, 64>, grid, dim3(128), 0, stream, p, keys);
  }
  QF_CUDA(err);
  const uint32_t* scored = keys;
  // As few keys a thread as the table needs: bounds and sparse attention of 32 sequences with tables of 512 pages
  // take 29.6 us with two a thread, 30.2 with five, 32.8 with sixteen; of one with 2049 pages, the 32768 tokens of a
  // full context and the next, 17.3 with five and 20.0 with sixteen (four would hold 2048).
  if (p.table_width <= 2 * kPickThreads) {
    err = launch_chained(page_pick_kernel<2>, dim3(rows), dim3(kPickThreads), 0, stream, p, scored, last);
  } else if (p.table_width <= 5 * kPickThreads) {
    err = launch_chained(page_pick_kernel<5>, dim3(rows), dim3(kPickThreads), 0, stream, p, scored, last);
  } else if (p.table_width <= 16 * kPickThreads) {
    err = launch_chained(page_pick_kernel<16>, dim3(rows), dim3(kPickThreads), 0, stream, p, scored, last);
  } else {
    err = launch_chained(page_pick_kernel<0>, dim3(rows), dim3(kPickThreads), 0, stream, p, scored, last);
  }
  QF_CUDA(err);
  QF_CUDA(cudaGetLastError());
  return QF_OK;
}

}  // namespace
}  // namespace qf

extern "C" {

int qf_int4_key_bounds(const qf_paged_int4_args* args, void* stream) {
  using namespace qf;
  PagedInt4 p;
  if (const int rc = fill_paged_int4(args, kNeedsPool | kNeedsBounds, &p)) return rc;
  QF_REQUIRE(p.new_tokens >= 0, "new_tokens must not be negative");
  if (p.batch == 0 || p.new_tokens == 0 || p.table_width == 0) return QF_OK;
  // a row's new tokens start anywhere in a page
  const int64_t spanned = (static_cast<int64_t>(p.new_tokens) + p.page_size - 2) / p.page_size + 1;
  const int pages_each = static_cast<int>(spanned < p.table_width ? spanned : p.table_width);
  const int64_t units = static_cast<int64_t>(p.batch) * p.kv_heads * pages_each;
  QF_REQUIRE(units < (1LL << 31) - 4, "too many pages in one call");
  const int tiles = p.page_size / kInt4Tile;
  const bool few = units <= 4LL * sm_count();  // of them a warp each would leave schedulers idle
  const int warps_each = tiles >= (few ? 4 : kManyTiles) ? 4 : tiles >= 2 && few ? 2 : 1;
  const int pages_a_cta = kBoundWarps / warps_each;
  const dim3 grid(static_cast<unsigned>((units + pages_a_cta - 1) / pages_a_cta));
  const Divisor by_each = make_divisor(pages_each);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t err = cudaSuccess;
  if (args->dtype == QF_DTYPE_F16) {
    err = args->head_dim == 128 ? launch_chained(key_bounds_kernel<__half, 128>, grid, dim3(32 * kBoundWarps), 0, s, p, by_each, warps_each)
                                : launch_chained(key_bounds_kernel<__half, 64>, grid, dim3(32 * kBoundWarps), 0, s, p, by_each, warps_each);
  } else {
    err = args->head_dim == 128 ? launch_chained(key_bounds_kernel<__nv_bfloat16, 128>, grid, dim3(32 * kBoundWarps), 0, s, p, by_each, warps_each)
                                : launch_chained(key_bounds_kernel<__nv_bfloat16, 64>, grid, dim3(32 * kBoundWarps), 0, s, p, by_each, warps_each);
  }
  QF_CUDA(err);
  QF_CUDA(cudaGetLastError());
  return QF_OK;
}

int qf_select_kv_pages(const qf_paged_int4_args* args, void* stream) {
  qf::PagedInt4 p;
  if (const int rc = qf::fill_paged_int4(args, qf::kNeedsQuery | qf::kNeedsBounds | qf::kNeedsSelection, &p)) return rc;
  if (p.batch == 0) return QF_OK;
  if (const int rc = qf::launch_select(p, args->head_dim, args->dtype, true, static_cast<cudaStream_t>(stream))) return rc;
  qf::request_ordered_launch();  // the selection is step metadata written by a kernel
  return QF_OK;
}

int qf_int4_sparse_decode_attention(const qf_paged_int4_args* args, void* stream) {
  using namespace qf;
  PagedInt4 p;
  QF_REQUIRE(args == nullptr || !(args->scale < 0.f), "scale must not be negative: pages are chosen by their largest scores");
  if (const int rc = fill_paged_int4(args, kNeedsQuery | kNeedsPool | kNeedsOut | kNeedsBounds | kNeedsSelection, &p)) return rc;
  if (p.batch == 0) return QF_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  PagedInt4 next = over_selection(p);
  const int64_t keys = select_bytes(p);
  const int64_t more = int4_attention_bytes(next, args->head_dim);
  QF_REQUIRE((p.workspace != nullptr || keys + more == 0) && p.workspace_bytes >= keys + more, "the workspace holds %lld bytes, %lld are needed",
             static_cast<long long>(p.workspace_bytes), static_cast<long long>(keys + more));
  if (const int rc = launch_select(p, args->head_dim, args->dtype, false, s)) return rc;
  next.workspace = static_cast<uint8_t*>(p.workspace) + keys;
  next.workspace_bytes = p.workspace_bytes - keys;
  return launch_int4_attention(next, args->head_dim, args->dtype, s);
}

int qf_paged_int4_workspace(const qf_paged_int4_args* args, int32_t call, int64_t* bytes) {
  using namespace qf;
  QF_REQUIRE(args != nullptr && bytes != nullptr, "args and bytes must not be null");
  QF_REQUIRE(call == QF_INT4_ATTENTION || call == QF_INT4_SELECT || call == QF_INT4_SPARSE, "unknown call %d", call);
  PagedInt4 p{};
  p.batch = args->batch, p.q_heads = args->q_heads, p.kv_heads = args->kv_heads, p.page_size = args->page_size;
  p.table_width = args->table_width, p.take = args->take;
  QF_REQUIRE(p.batch >= 0 && p.kv_heads >= 1 && p.q_heads >= 0 && p.table_width >= 0 && p.page_size >= 1, "invalid sizes");
  *bytes = 0;
  if (call != QF_INT4_ATTENTION) *bytes += select_bytes(p);
  if (call != QF_INT4_SELECT) *bytes += int4_attention_bytes(call == QF_INT4_SPARSE ? over_selection(p) : p, args->head_dim);
  return QF_OK;
}

}  // extern "C"
