// The 4-bit paged KV cache: RoPE + quantising write, read-back of rows, and the smallest and
// largest key of a page.  Layout and codec: qf_int4_codec.cuh.  Compiled without fast-math:
// the rotation is separate fp32 multiplies and adds and every division is IEEE, so a cache
// written here equals, byte for byte, one computed with the same fp32 operations elsewhere.
#include <cmath>

#include "qf_int4_paged.cuh"
#include "qf_rope_math.cuh"

namespace qf {
namespace {

struct WriteParams {
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  int64_t q_sr, q_sh, q_sd;
  int64_t k_sr, k_sh, k_sd;
  int64_t v_sr, v_sh, v_sd;
  int64_t o_sr, o_sh, o_sd;
  const void* positions;  // null: no rotation
  int64_t pos_stride;
  const void* slots;      // null: slot = row
  int64_t slot_stride;
  const float2* table;    // null: cosf / sinf
  uint8_t* pool;
  int64_t num_slots;
  const int32_t* valid_tokens;
  int* status;
  Divisor items, page_size;
  int rows, q_heads, kv_heads, table_positions;
  int pos_dtype, slot_dtype;
  bool one_wave;  // the grid is resident at once
};

constexpr int kWriteThreads = 128;

// Where the angles of a call come from.
enum : int { kNoRope, kTable, kAngles };
constexpr int write_ctas(int rope) { return rope == kAngles ? 12 : 16; }  // an SM

// Rows and their segments (heads) are laid end to end: a segment takes D / 16 threads, each with
// the eight channels at d0 and the eight they rotate with at d0 + D / 2, so a CTA of 128 covers a row
// of 12 + 2 + 2 heads and no thread idles.  A group of 32 channels is four neighbouring threads, whose
// extremes meet in two shuffles.  A thread fetches its cosines and sines from the table itself (a
// row's 14 rotated heads hit the first level cache; passing them through shared memory instead costs
// a barrier behind two dependent loads, 28 -> 22 us for 8192 rows); without a table the CTA computes
// each once and shares it.  Bound by the latency of position -> table -> row and by issue: 8192 rows of
// 12 + 2 + 2 x 128 take 15.6 us, 64 MB at 4.1 TB/s; of 17 us, CTAs of 256 made 20, of 512 23, and 12
// CTAs an SM (40 registers) instead of 16 (32) 18.
template <typename T, int D, bool VEC, int ROPE>
__global__ void __launch_bounds__(kWriteThreads, write_ctas(ROPE)) int4_write_kernel(const WriteParams p, const __grid_constant__ InvFreqTable freq) {
  constexpr int kHalf = D / 2, kLanes = D / 16, W = D / kInt4Group;
  dependency_wait();
  // Behind the wait: attention reads lengths and tables before its own, and what the kernel in front of
  // this one wrote is complete only now.
  // The kernel behind may stand by early where this one leaves the SMs at once (64 rows, then attention
  // of 64 sequences: 24.5 us, else 24.6), but not beside the CTAs of a long grid (8192 rows written and read
  // back 20.9 us, else 21.6).
  if (p.one_wave) release_dependents();
  const uint32_t first = blockIdx.x * kWriteThreads;
  const int index = first + threadIdx.x;
  const int row = quotient(index, p.items);
  const bool on = row < p.rows;
  const int item = index - row * p.items.d;
  const int live_rows = p.valid_tokens ? min(*p.valid_tokens, p.rows) : p.rows;
  const bool live = row < live_rows;
  const int segment = item / kLanes, d0 = (item % kLanes) * 8;
  const bool is_q = segment < p.q_heads;
  const bool is_k = !is_q && segment < p.q_heads + p.kv_heads;
  const int head = is_q ? segment : is_k ? segment - p.q_heads : segment - p.q_heads - p.kv_heads;
  int64_t position = 0;
  if (ROPE == kTable && live) position = load_index(p.positions, p.pos_dtype, row * p.pos_stride);
  int64_t slot = -1;
  if (live && !is_q) slot = p.slots != nullptr ? load_index(p.slots, p.slot_dtype, row * p.slot_stride) : row;
  const bool slot_ok = slot >= 0 && slot < p.num_slots;
  // eight channels and the eight they rotate with, two to a register
  uint32_t x[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  if (live) {
    const T* src;
    int64_t sd;
    if (is_q) {
      src = static_cast<const T*>(p.q) + row * p.q_sr + head * p.q_sh, sd = p.q_sd;
    } else if (is_k) {
      src = static_cast<const T*>(p.k) + row * p.k_sr + head * p.k_sh, sd = p.k_sd;
    } else {
      src = static_cast<const T*>(p.v) + row * p.v_sr + head * p.v_sh, sd = p.v_sd;
    }
    if constexpr (VEC) {
      *reinterpret_cast<uint4*>(x[0]) = *reinterpret_cast<const uint4*>(src + d0);
      *reinterpret_cast<uint4*>(x[1]) = *reinterpret_cast<const uint4*>(src + d0 + kHalf);
    } else {
      const uint16_t* bits = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j / 4][j % 4] = bits[(d0 + j / 4 * kHalf + 2 * (j % 4)) * sd] |
                          static_cast<uint32_t>(bits[(d0 + j / 4 * kHalf + 2 * (j % 4) + 1) * sd]) << 16;
      }
    }
  }

  if constexpr (ROPE != kNoRope) {
    const bool turns = live && (is_q || is_k);
    float4 cs[4];  // (cos, sin) of channels d0 + 2 j and d0 + 2 j + 1
    if constexpr (ROPE == kTable) {
      if (turns) {
        if (position < 0 || position >= p.table_positions) {
          position = position < 0 ? 0 : p.table_positions - 1;
          atomicMax(p.status, kStatusPositionPastTable);
        }
        const float4* at = reinterpret_cast<const float4*>(p.table + position * kHalf + d0);
#pragma unroll
        for (int j = 0; j < 4; ++j) cs[j] = at[j];
      }
    } else {
      constexpr int kRows = kWriteThreads / (2 * kLanes) + 1;  // one KV head and no query heads: the most rows a CTA meets
      __shared__ __align__(16) float2 s_rope[kRows][kHalf];
      const int first_row = quotient(first, p.items);
      const int last_row = min(static_cast<int>(quotient(first + kWriteThreads - 1, p.items)), live_rows - 1);
      for (int i = threadIdx.x; i < (last_row - first_row + 1) * kHalf; i += kWriteThreads) {
        const int r = i / kHalf, f = i % kHalf;
        const float angle = __fmul_rn(load_position(p.positions, p.pos_dtype, (first_row + r) * p.pos_stride), freq.v[f]);
        s_rope[r][f] = make_float2(cosf(angle), sinf(angle));
      }
      __syncthreads();
      if (turns) {
#pragma unroll
        for (int j = 0; j < 4; ++j) cs[j] = *reinterpret_cast<const float4*>(&s_rope[row - first_row][d0 + 2 * j]);
      }
    }
    if (turns) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 a = unpack2<T>(x[0][j]), b = unpack2<T>(x[1][j]);
        x[0][j] = pack2<T>(__fsub_rn(__fmul_rn(a.x, cs[j].x), __fmul_rn(b.x, cs[j].y)), __fsub_rn(__fmul_rn(a.y, cs[j].z), __fmul_rn(b.y, cs[j].w)));
        x[1][j] = pack2<T>(__fadd_rn(__fmul_rn(b.x, cs[j].x), __fmul_rn(a.x, cs[j].y)), __fadd_rn(__fmul_rn(b.y, cs[j].z), __fmul_rn(a.y, cs[j].w)));
      }
    }
  }
  if (on && is_q) {
    T* dst = static_cast<T*>(p.q_out) + row * p.o_sr + head * p.o_sh;
    if constexpr (VEC) {
      *reinterpret_cast<uint4*>(dst + d0) = *reinterpret_cast<uint4*>(x[0]);
      *reinterpret_cast<uint4*>(dst + d0 + kHalf) = *reinterpret_cast<uint4*>(x[1]);
    } else {
      uint16_t* bits = reinterpret_cast<uint16_t*>(dst);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        bits[(d0 + j / 4 * kHalf + 2 * (j % 4)) * p.o_sd] = static_cast<uint16_t>(x[j / 4][j % 4]);
        bits[(d0 + j / 4 * kHalf + 2 * (j % 4) + 1) * p.o_sd] = static_cast<uint16_t>(x[j / 4][j % 4] >> 16);
      }
    }
  }
  if (__all_sync(0xffffffffu, is_q || !slot_ok)) return;

  const uint32_t page = slot_ok ? quotient(static_cast<uint32_t>(slot), p.page_size) : 0u;
  const int in_page = slot_ok ? static_cast<int>(static_cast<uint32_t>(slot) - page * p.page_size.d) : 0;
  const int token = in_page % kInt4Tile;
  uint8_t* tile = p.pool + ((static_cast<int64_t>(page) * p.kv_heads + head) * (p.page_size.d / kInt4Tile) + in_page / kInt4Tile) *
                               int4_tile_bytes(D);
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 two = unpack2<T>(x[side][j]);
      f[2 * j] = two.x, f[2 * j + 1] = two.y;
    }
    float low = min_nan(min_nan(f[0], f[1], f[2]), min_nan(f[3], f[4], f[5]), min_nan(f[6], f[7], f[7]));
    float high = max_nan(max_nan(f[0], f[1], f[2]), max_nan(f[3], f[4], f[5]), max_nan(f[6], f[7], f[7]));
#pragma unroll
    for (int off = 1; off <= 2; off <<= 1) {
      const float a = __shfl_xor_sync(0xffffffffu, low, off), z = __shfl_xor_sync(0xffffffffu, high, off);
      low = min_nan(low, a, a), high = max_nan(high, z, z);
    }
    if (is_q || !slot_ok) continue;
    const Int4Group g = int4_group<T>(low, high);
    const uint32_t word = int4_word(f, g);
    const int channel = d0 + side * kHalf;
    const int w = channel / kInt4Group, t = channel % kInt4Group / 8;
    uint8_t* params = tile + 16 * D + (is_k ? 0 : 2 * D) + token * 2 * W + 2 * w;
    if (t == 0) {
      *reinterpret_cast<T*>(params) = from_float<T>(g.step);
      *reinterpret_cast<T*>(params + D) = from_float<T>(g.low);
    }
    if (is_k) {
      *reinterpret_cast<uint32_t*>(tile + token * (D / 2) + t * 4 * W + 4 * w) = word;
    } else {
      uint8_t* v = tile + 8 * D + token / 2 * D + 2 * t * 4 * W + 4 * w + token % 2 * 2;
      *reinterpret_cast<uint16_t*>(v) = static_cast<uint16_t>(word);
      *reinterpret_cast<uint16_t*>(v + 4 * W) = static_cast<uint16_t>(word >> 16);
    }
  }
}

// W 32-bit words, W 16-bit elements.
template <int W>
__device__ __forceinline__ void load_words(const uint8_t* at, uint32_t (&x)[W]) {
  if constexpr (W == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(at);
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(at);
    x[0] = v.x, x[1] = v.y;
  }
}
template <typename T, int W>
__device__ __forceinline__ void load_elements(const uint8_t* at, float (&x)[W]) {
  uint32_t bits[W / 2];
  if constexpr (W == 4) {
    const uint2 v = *reinterpret_cast<const uint2*>(at);
    bits[0] = v.x, bits[1] = v.y;
  } else {
    bits[0] = *reinterpret_cast<const uint32_t*>(at);
  }
#pragma unroll
  for (int j = 0; j < W / 2; ++j) {
    const float2 two = unpack2<T>(bits[j]);
    x[2 * j] = two.x, x[2 * j + 1] = two.y;
  }
}

// Rows at a list of slots as 16-bit K and V.  Four threads a row and head, eight channels of every
// group each: seven loads bring a thread's D / 2 values, and its stores are 16 bytes beside its
// neighbours' (16 threads a row, each with its own slot and addresses, were bound by those: 40 us for
// 131072 rows of 2 x 128).  Bound by the stores: the 177 MB take 32.6 us, 5.4 TB/s.  A slot outside the
// pool gives a row of zeros.  Pool and slots may be written by the kernel in front: no __restrict__.
template <typename T, int D>
__global__ void __launch_bounds__(128) int4_read_kernel(const uint8_t* pool, const void* slots,
                                                        int slot_dtype, int64_t slot_stride, int rows, int64_t num_slots,
                                                        const Divisor kv_heads, const Divisor page_size,
                                                        T* k_out, T* v_out) {
  constexpr int W = D / kInt4Group;
  dependency_wait();
  release_dependents();  // behind the wait, as in the write
  const uint32_t segment = blockIdx.x * 32 + threadIdx.x / 4;
  const int t = threadIdx.x % 4;
  const int row = quotient(segment, kv_heads);
  const int head = segment - row * kv_heads.d;
  if (row >= rows) return;
  const int64_t slot = slots != nullptr ? load_index(slots, slot_dtype, row * slot_stride) : row;
  T* k_at = k_out + static_cast<int64_t>(segment) * D + 8 * t;
  T* v_at = v_out + static_cast<int64_t>(segment) * D + 8 * t;
  if (slot < 0 || slot >= num_slots) {
#pragma unroll
    for (int w = 0; w < W; ++w) {
      *reinterpret_cast<uint4*>(k_at + 32 * w) = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(v_at + 32 * w) = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const uint32_t page = quotient(static_cast<uint32_t>(slot), page_size);
  const int in_page = static_cast<int>(static_cast<uint32_t>(slot) - page * page_size.d), token = in_page % kInt4Tile;
  const uint8_t* tile = pool + ((static_cast<int64_t>(page) * kv_heads.d + head) * (page_size.d / kInt4Tile) + in_page / kInt4Tile) *
                                   int4_tile_bytes(D);
  uint32_t k[W], even[W], odd[W];  // K words, V words of channels 8t..8t + 3 and 8t + 4..8t + 7 of every group
  load_words<W>(tile + token * (D / 2) + t * 4 * W, k);
  load_words<W>(tile + 8 * D + token / 2 * D + 2 * t * 4 * W, even);
  load_words<W>(tile + 8 * D + token / 2 * D + (2 * t + 1) * 4 * W, odd);
  float steps[2][W], floors[2][W];
  const uint8_t* params = tile + 16 * D + token * 2 * W;
  load_elements<T, W>(params, steps[0]);
  load_elements<T, W>(params + D, floors[0]);
  load_elements<T, W>(params + 2 * D, steps[1]);
  load_elements<T, W>(params + 3 * D, floors[1]);
  const uint32_t which = token % 2 ? 0x7632u : 0x5410u;  // the halves of the pair's words that are this token's
#pragma unroll
  for (int w = 0; w < W; ++w) {
    float x[8];
    int4_values(k[w], steps[0][w], floors[0][w], x);
    *reinterpret_cast<uint4*>(k_at + 32 * w) =
        make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
    int4_values(__byte_perm(even[w], odd[w], which), steps[1][w], floors[1][w], x);
    *reinterpret_cast<uint4*>(v_at + 32 * w) =
        make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
  }
}

bool aligned16(const void* p) { return on_boundary(p, 16); }

bool good_geometry(int head_dim, int page_size) {
  return (head_dim == 64 || head_dim == 128) && page_size >= kInt4Tile && page_size % kInt4Tile == 0;
}

int launch_write(const qf_int4_write_args* a, cudaStream_t stream) {
  QF_REQUIRE(a != nullptr, "args must not be null");
  QF_REQUIRE(a->rows >= 0, "rows must be non-negative");
  QF_REQUIRE(a->dtype == QF_DTYPE_F16 || a->dtype == QF_DTYPE_BF16, "q, k, and v must use float16 or bfloat16");
  QF_REQUIRE(good_geometry(a->head_dim, a->page_size),
             "a 4-bit cache has head dimension 64 or 128 and pages of a multiple of 16 tokens");
  QF_REQUIRE(a->kv_heads >= 1 && a->q_heads >= 0, "head counts must be positive");
  QF_REQUIRE(a->num_pages >= 0 && a->num_pages < (1LL << 31) / a->page_size, "a pool holds fewer than 2^31 slots");
  if (a->rows == 0) return QF_OK;
  const int items = (a->q_heads + 2 * a->kv_heads) * (a->head_dim / 16);
  QF_REQUIRE(a->q_heads < (1 << 20) && a->kv_heads < (1 << 20) && static_cast<int64_t>(a->rows) * items < (1LL << 31) - kWriteThreads,
             "too many rows in one call");
  QF_REQUIRE(a->k && a->v && (a->pool || a->num_pages == 0), "k, v and the pool must not be null");
  QF_REQUIRE(a->q_heads == 0 || (a->q && a->q_out), "q and q_out are required with query heads");
  QF_REQUIRE(aligned16(a->pool), "the pool must be 16-byte aligned");
  if (a->positions != nullptr) {
    QF_REQUIRE(a->positions_dtype == QF_INDEX_I32 || a->positions_dtype == QF_INDEX_I64 ||
                   (a->positions_dtype == QF_INDEX_F32 && a->rope_table == nullptr),
               "positions must be int32, int64, or (without a table) float32");
    QF_REQUIRE(a->rope_table != nullptr || a->base > 0.0, "rope base must be positive");
    QF_REQUIRE(a->rope_table == nullptr || a->table_positions >= 1, "the RoPE table is empty");
    QF_REQUIRE(aligned16(a->rope_table), "the RoPE table must be 16-byte aligned");
  }
  QF_REQUIRE(a->slot_mapping == nullptr || a->slot_dtype == QF_INDEX_I32 || a->slot_dtype == QF_INDEX_I64,
             "slot mapping must use an integer dtype");
  QF_REQUIRE(on_boundary(a->q, 2) && on_boundary(a->k, 2) && on_boundary(a->v, 2) && on_boundary(a->q_out, 2) &&
                 index_aligned(a->positions, a->positions_dtype) && index_aligned(a->slot_mapping, a->slot_dtype) &&
                 on_boundary(a->valid_tokens, 4),
             "inputs must be aligned to their elements");

  WriteParams p{};
  p.q = a->q, p.k = a->k, p.v = a->v, p.q_out = a->q_out;
  p.q_sr = a->q_stride_row, p.q_sh = a->q_stride_head, p.q_sd = a->q_stride_d;
  p.k_sr = a->k_stride_row, p.k_sh = a->k_stride_head, p.k_sd = a->k_stride_d;
  p.v_sr = a->v_stride_row, p.v_sh = a->v_stride_head, p.v_sd = a->v_stride_d;
  p.o_sr = a->o_stride_row, p.o_sh = a->o_stride_head, p.o_sd = a->o_stride_d;
  p.positions = a->positions, p.pos_stride = a->positions_stride, p.pos_dtype = a->positions_dtype;
  p.slots = a->slot_mapping, p.slot_stride = a->slot_stride, p.slot_dtype = a->slot_dtype;
  p.table = reinterpret_cast<const float2*>(a->rope_table), p.table_positions = a->table_positions;
  p.pool = static_cast<uint8_t*>(a->pool), p.num_slots = a->num_pages * a->page_size;
  p.valid_tokens = a->valid_tokens;
  p.rows = a->rows, p.q_heads = a->q_heads, p.kv_heads = a->kv_heads;
  p.items = make_divisor(items), p.page_size = make_divisor(a->page_size);
  p.status = device_status_word();
  QF_REQUIRE(p.status != nullptr, "no device status word");
  InvFreqTable freq{};
  if (a->positions != nullptr && a->rope_table == nullptr) freq = make_inv_freq(a->base, a->head_dim / 2);

  auto mult8 = [](int64_t s) { return (s & 7) == 0; };
  bool vec = a->k_stride_d == 1 && a->v_stride_d == 1 && aligned16(a->k) && aligned16(a->v) && mult8(a->k_stride_row) &&
             mult8(a->k_stride_head) && mult8(a->v_stride_row) && mult8(a->v_stride_head);
  if (a->q_heads > 0) {
    vec = vec && a->q_stride_d == 1 && a->o_stride_d == 1 && aligned16(a->q) && aligned16(a->q_out) &&
          mult8(a->q_stride_row) && mult8(a->q_stride_head) && mult8(a->o_stride_row) && mult8(a->o_stride_head);
  }
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(a->rows) * items + kWriteThreads - 1) / kWriteThreads));
  p.one_wave = grid.x <= static_cast<unsigned>(sm_count() * write_ctas(a->positions == nullptr ? kNoRope : a->rope_table != nullptr ? kTable : kAngles));
  cudaError_t err = cudaSuccess;
#define QF_LAUNCH_WRITE_AS(T, D, ROPE)                                                                              \
  err = vec ? launch_chained(int4_write_kernel<T, D, true, ROPE>, grid, dim3(kWriteThreads), 0, stream, p, freq)     \
            : launch_chained(int4_write_kernel<T, D, false, ROPE>, grid, dim3(kWriteThreads), 0, stream, p, freq)
#define QF_LAUNCH_WRITE(T, D)                     \
  do {                                            \
    if (a->positions == nullptr) {                \
      QF_LAUNCH_WRITE_AS(T, D, kNoRope);          \
    } else if (a->rope_table != nullptr) {        \
      QF_LAUNCH_WRITE_AS(T, D, kTable);           \
    } else {                                      \
      QF_LAUNCH_WRITE_AS(T, D, kAngles);          \
    }                                             \
  } while (0)
  if (a->dtype == QF_DTYPE_F16) {
    if (a->head_dim == 128) QF_LAUNCH_WRITE(__half, 128); else QF_LAUNCH_WRITE(__half, 64);
  } else {
    if (a->head_dim == 128) QF_LAUNCH_WRITE(__nv_bfloat16, 128); else QF_LAUNCH_WRITE(__nv_bfloat16, 64);
  }
#undef QF_LAUNCH_WRITE
#undef QF_LAUNCH_WRITE_AS
  QF_CUDA(err);
  QF_CUDA(cudaGetLastError());
  return QF_OK;
}

}  // namespace
}  // namespace qf

extern "C" {

int qf_int4_rope_kv_write(const qf_int4_write_args* args, void* stream) {
  return qf::launch_write(args, static_cast<cudaStream_t>(stream));
}

int qf_int4_read_rows(const void* pool, int64_t num_pages, int32_t page_size, int32_t kv_heads, int32_t head_dim,
                      int32_t dtype, const void* slots, int32_t slot_dtype, int64_t slot_stride, int64_t rows,
                      void* k_out, void* v_out, void* stream) {
  using namespace qf;
  QF_REQUIRE(dtype == QF_DTYPE_F16 || dtype == QF_DTYPE_BF16, "rows are read as float16 or bfloat16");
  QF_REQUIRE(good_geometry(head_dim, page_size),
             "a 4-bit cache has head dimension 64 or 128 and pages of a multiple of 16 tokens");
  QF_REQUIRE(kv_heads >= 1 && rows >= 0 && num_pages >= 0 && num_pages < (1LL << 31) / page_size, "invalid pool geometry");
  QF_REQUIRE(slots == nullptr || slot_dtype == QF_INDEX_I32 || slot_dtype == QF_INDEX_I64,
             "slot mapping must use an integer dtype");
  if (rows == 0) return QF_OK;
  QF_REQUIRE((pool || num_pages == 0) && k_out && v_out, "pool, k_out and v_out must not be null");
  QF_REQUIRE(aligned16(pool) && aligned16(k_out) && aligned16(v_out), "pool and outputs must be 16-byte aligned");
  QF_REQUIRE(index_aligned(slots, slot_dtype), "slots must be aligned to their elements");
  QF_REQUIRE(rows < (1LL << 31) / kv_heads - 256, "too many rows in one call");
  const dim3 grid(static_cast<unsigned>((rows * kv_heads + 31) / 32));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uint8_t* bytes = static_cast<const uint8_t*>(pool);
  cudaError_t err = cudaSuccess;
#define QF_LAUNCH_READ(T, D)                                                                                       \
  err = launch_chained(int4_read_kernel<T, D>, grid, dim3(128), 0, s, bytes, slots, static_cast<int>(slot_dtype),  \
                       slot_stride, static_cast<int>(rows), num_pages * page_size, make_divisor(kv_heads),         \
                       make_divisor(page_size), static_cast<T*>(k_out), static_cast<T*>(v_out))
  if (dtype == QF_DTYPE_F16) {
    if (head_dim == 128) QF_LAUNCH_READ(__half, 128); else QF_LAUNCH_READ(__half, 64);
  } else {
    if (head_dim == 128) QF_LAUNCH_READ(__nv_bfloat16, 128); else QF_LAUNCH_READ(__nv_bfloat16, 64);
  }
#undef QF_LAUNCH_READ
  QF_CUDA(err);
  QF_CUDA(cudaGetLastError());
  return QF_OK;
}

}  // extern "C"
