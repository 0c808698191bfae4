// The 4-bit paged KV cache: RoPE + quantising write, read-back of rows, and the smallest and
// largest key of a page.  Layout and codec: qf_int4_codec.cuh.  Compiled without fast-math:
// the rotation is separate fp32 multiplies and adds and every division is IEEE, so a cache
// written here equals, byte for byte, one computed with the same fp32 operations elsewhere.
#include <cmath>

#include "qf_int4_codec.cuh"
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
};

constexpr int kWriteThreads = 256;

__device__ __forceinline__ bool finite32(float x) { return fabsf(x) <= 3.402823466e38f; }

// Rows and their segments (heads) are laid end to end: a segment takes D / 16 threads, each with
// the eight channels at d0 and the eight they rotate with at d0 + D / 2, so a CTA of 256 covers
// two rows of 12 + 2 + 2 heads and no thread idles.  A group of 32 channels is four neighbouring
// threads, whose extremes meet in two shuffles.  The CTA's cosines and sines go through shared
// memory: 14 heads of a row use each.
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(kWriteThreads) int4_write_kernel(const WriteParams p, const __grid_constant__ InvFreqTable freq) {
  constexpr int kHalf = D / 2, kLanes = D / 16, W = D / kInt4Group;
  constexpr int kRows = kWriteThreads / (2 * kLanes) + 1;  // one KV head and no query heads: the most rows a CTA meets
  __shared__ float2 s_rope[kRows][kHalf];
  release_dependents();
  dependency_wait();
  const uint32_t first = blockIdx.x * kWriteThreads;
  const int first_row = quotient(first, p.items);
  const int index = first + threadIdx.x;
  const int row = quotient(index, p.items);
  const bool on = row < p.rows;
  const int item = index - row * p.items.d;
  const int live_rows = p.valid_tokens ? min(*p.valid_tokens, p.rows) : p.rows;
  const bool live = row < live_rows;
  int64_t slot = -1;
  if (live) slot = p.slots != nullptr ? load_index(p.slots, p.slot_dtype, row * p.slot_stride) : row;
  const bool slot_ok = slot >= 0 && slot < p.num_slots;
  const int segment = item / kLanes, d0 = (item % kLanes) * 8;
  const bool is_q = segment < p.q_heads;
  const bool is_k = !is_q && segment < p.q_heads + p.kv_heads;
  const int head = is_q ? segment : is_k ? segment - p.q_heads : segment - p.q_heads - p.kv_heads;
  const T* src;
  int64_t sd;
  if (is_q) {
    src = static_cast<const T*>(p.q) + row * p.q_sr + head * p.q_sh, sd = p.q_sd;
  } else if (is_k) {
    src = static_cast<const T*>(p.k) + row * p.k_sr + head * p.k_sh, sd = p.k_sd;
  } else {
    src = static_cast<const T*>(p.v) + row * p.v_sr + head * p.v_sh, sd = p.v_sd;
  }
  alignas(16) T x[16];
  if (live && (is_q || slot_ok)) {
    if constexpr (VEC) {
      *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(src + d0);
      *reinterpret_cast<uint4*>(x + 8) = *reinterpret_cast<const uint4*>(src + d0 + kHalf);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = src[(d0 + j) * sd], x[8 + j] = src[(d0 + kHalf + j) * sd];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) x[j] = from_float<T>(0.f);
  }

  if (p.positions != nullptr) {
    const int last_row = min(static_cast<int>(quotient(first + kWriteThreads - 1, p.items)), live_rows - 1);
    for (int i = threadIdx.x; i < (last_row - first_row + 1) * kHalf; i += kWriteThreads) {
      const int r = i / kHalf, f = i % kHalf;
      if (p.table != nullptr) {
        int64_t position = load_index(p.positions, p.pos_dtype, (first_row + r) * p.pos_stride);
        if (position < 0 || position >= p.table_positions) {
          position = position < 0 ? 0 : p.table_positions - 1;
          if (f == 0) atomicMax(p.status, kStatusPositionPastTable);
        }
        s_rope[r][f] = p.table[position * kHalf + f];
      } else {
        const float angle = __fmul_rn(load_position(p.positions, p.pos_dtype, (first_row + r) * p.pos_stride), freq.v[f]);
        s_rope[r][f] = make_float2(cosf(angle), sinf(angle));
      }
    }
    __syncthreads();
    if (live && (is_q || is_k)) {
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float4 cs = *reinterpret_cast<const float4*>(&s_rope[row - first_row][d0 + j]);
        const float a0 = to_float(x[j]), b0 = to_float(x[8 + j]), a1 = to_float(x[j + 1]), b1 = to_float(x[9 + j]);
        x[j] = from_float<T>(__fsub_rn(__fmul_rn(a0, cs.x), __fmul_rn(b0, cs.y)));
        x[8 + j] = from_float<T>(__fadd_rn(__fmul_rn(b0, cs.x), __fmul_rn(a0, cs.y)));
        x[j + 1] = from_float<T>(__fsub_rn(__fmul_rn(a1, cs.z), __fmul_rn(b1, cs.w)));
        x[9 + j] = from_float<T>(__fadd_rn(__fmul_rn(b1, cs.z), __fmul_rn(a1, cs.w)));
      }
    }
  }
  if (on && is_q) {
    T* dst = static_cast<T*>(p.q_out) + row * p.o_sr + head * p.o_sh;
    if constexpr (VEC) {
      *reinterpret_cast<uint4*>(dst + d0) = *reinterpret_cast<uint4*>(x);
      *reinterpret_cast<uint4*>(dst + d0 + kHalf) = *reinterpret_cast<uint4*>(x + 8);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) dst[(d0 + j) * p.o_sd] = x[j], dst[(d0 + kHalf + j) * p.o_sd] = x[8 + j];
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
    float low, high;
    bool finite = true;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      f[j] = to_float(x[8 * side + j]);
      low = j == 0 ? f[j] : fminf(low, f[j]);
      high = j == 0 ? f[j] : fmaxf(high, f[j]);
      finite = finite && finite32(f[j]);
    }
#pragma unroll
    for (int off = 1; off <= 2; off <<= 1) {
      low = fminf(low, __shfl_xor_sync(0xffffffffu, low, off));
      high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, off));
      finite = __shfl_xor_sync(0xffffffffu, finite ? 1 : 0, off) != 0 && finite;
    }
    if (is_q || !slot_ok) continue;
    const Int4Group g = int4_group<T>(low, high, finite);
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

// Rows at a list of slots as 16-bit K and V.  A thread takes eight channels of one row of K
// and of V: 16-byte stores side by side.  A slot outside the pool gives a row of zeros.
template <typename T, int D>
__global__ void __launch_bounds__(256) int4_read_kernel(const uint8_t* __restrict__ pool, const void* __restrict__ slots,
                                                        int slot_dtype, int64_t slot_stride, int rows, int64_t num_slots,
                                                        const Divisor kv_heads, const Divisor page_size,
                                                        T* __restrict__ k_out, T* __restrict__ v_out) {
  constexpr int kLanes = D / 8, W = D / kInt4Group;
  release_dependents();
  dependency_wait();
  const uint32_t segment = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  const int lane = threadIdx.x % kLanes;
  const int row = quotient(segment, kv_heads);
  const int head = segment - row * kv_heads.d;
  if (row >= rows) return;
  const int64_t slot = slots != nullptr ? load_index(slots, slot_dtype, row * slot_stride) : row;
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  if (slot >= 0 && slot < num_slots) {
    const uint32_t page = quotient(static_cast<uint32_t>(slot), page_size);
    const int in_page = static_cast<int>(static_cast<uint32_t>(slot) - page * page_size.d), token = in_page % kInt4Tile;
    const uint8_t* tile = pool + ((static_cast<int64_t>(page) * kv_heads.d + head) * (page_size.d / kInt4Tile) + in_page / kInt4Tile) *
                                     int4_tile_bytes(D);
    const int w = lane / 4, t = lane % 4;
    const T* params = reinterpret_cast<const T*>(tile + 16 * D) + token * W + w;
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(tile + token * (D / 2) + t * 4 * W + 4 * w);
    const uint8_t* vp = tile + 8 * D + token / 2 * D + 2 * t * 4 * W + 4 * w + token % 2 * 2;
    const uint32_t vw = *reinterpret_cast<const uint16_t*>(vp) |
                        static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(vp + 4 * W)) << 16;
    float x[8];
    int4_values(kw, to_float(params[0]), to_float(params[D / 2]), x);
    k = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
    int4_values(vw, to_float(params[D]), to_float(params[3 * D / 2]), x);
    v = make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
  }
  const int64_t at = static_cast<int64_t>(segment) * D + lane * 8;
  *reinterpret_cast<uint4*>(k_out + at) = k;
  *reinterpret_cast<uint4*>(v_out + at) = v;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

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
  QF_REQUIRE(a->k && a->v && a->pool, "k, v and the pool must not be null");
  QF_REQUIRE(a->q_heads == 0 || (a->q && a->q_out), "q and q_out are required with query heads");
  QF_REQUIRE(aligned16(a->pool), "the pool must be 16-byte aligned");
  if (a->positions != nullptr) {
    QF_REQUIRE(a->positions_dtype == QF_INDEX_I32 || a->positions_dtype == QF_INDEX_I64 ||
                   (a->positions_dtype == QF_INDEX_F32 && a->rope_table == nullptr),
               "positions must be int32, int64, or (without a table) float32");
    QF_REQUIRE(a->rope_table != nullptr || a->base > 0.0, "rope base must be positive");
    QF_REQUIRE(a->rope_table == nullptr || a->table_positions >= 1, "the RoPE table is empty");
  }
  QF_REQUIRE(a->slot_mapping == nullptr || a->slot_dtype == QF_INDEX_I32 || a->slot_dtype == QF_INDEX_I64,
             "slot mapping must use an integer dtype");

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
  cudaError_t err = cudaSuccess;
#define QF_LAUNCH_WRITE(T, D)                                                                             \
  err = vec ? launch_chained(int4_write_kernel<T, D, true>, grid, dim3(kWriteThreads), 0, stream, p, freq) \
            : launch_chained(int4_write_kernel<T, D, false>, grid, dim3(kWriteThreads), 0, stream, p, freq)
  if (a->dtype == QF_DTYPE_F16) {
    if (a->head_dim == 128) QF_LAUNCH_WRITE(__half, 128); else QF_LAUNCH_WRITE(__half, 64);
  } else {
    if (a->head_dim == 128) QF_LAUNCH_WRITE(__nv_bfloat16, 128); else QF_LAUNCH_WRITE(__nv_bfloat16, 64);
  }
#undef QF_LAUNCH_WRITE
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
  QF_REQUIRE(pool && k_out && v_out, "pool, k_out and v_out must not be null");
  QF_REQUIRE(aligned16(pool) && aligned16(k_out) && aligned16(v_out), "pool and outputs must be 16-byte aligned");
  QF_REQUIRE(rows < (1LL << 31) / kv_heads - 256, "too many rows in one call");
  const int64_t items = rows * kv_heads * (head_dim / 8);
  const dim3 grid(static_cast<unsigned>((items + 255) / 256));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uint8_t* bytes = static_cast<const uint8_t*>(pool);
  cudaError_t err = cudaSuccess;
#define QF_LAUNCH_READ(T, D)                                                                                       \
  err = launch_chained(int4_read_kernel<T, D>, grid, dim3(256), 0, s, bytes, slots, static_cast<int>(slot_dtype),  \
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
