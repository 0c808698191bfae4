// Choosing the pages a query attends.  Bounds: the smallest and the largest key of every page
// and channel, as the 4-bit cache reads back.  No key k of a page scores above
//     sum_d max(q_d low_d, q_d high_d)  >=  q . k
// so a page's score is the largest of that over the query heads of its KV head, and a row
// (sequence, KV head) takes its newest page and the take - 1 others that score highest, ties
// to the lower page.  The products are exact in fp32 and are added pairwise, neighbours first,
// whatever the kernel's layout: the same inputs choose the same pages everywhere.
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
  // tokens of a row are counted in 32 bits
  QF_REQUIRE(a->table_width <= ((1LL << 31) - 1) / a->page_size, "a block table row holds 2^31 tokens or more");
  if (needs & kNeedsQuery) {
    QF_REQUIRE(a->q_heads >= 1 && a->q_heads % a->kv_heads == 0, "query heads must be divisible by KV heads");
    QF_REQUIRE(a->q_heads / a->kv_heads <= 16, "at most 16 query heads share a KV head");
  }
  QF_REQUIRE(a->table_dtype == QF_INDEX_I32 || a->table_dtype == QF_INDEX_I64, "page table must use an integer dtype");
  QF_REQUIRE(a->lens_dtype == QF_INDEX_I32 || a->lens_dtype == QF_INDEX_I64, "lengths must use an integer dtype");
  auto aligned = [](const void* x) { return (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
  if (a->batch > 0) {
    QF_REQUIRE(a->seq_lens && (a->block_table || a->table_width == 0), "block table and lengths must not be null");
    if (needs & kNeedsQuery) {
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
      QF_REQUIRE(a->page_table && a->page_lens, "page_table and page_lens must not be null");
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
  if (a->batch > 0) {
    r.status = device_status_word();
    QF_REQUIRE(r.status != nullptr, "no device status word");
  }
  *p = r;
  return QF_OK;
}

namespace {

// The extremes of a page keep a NaN: a page that holds one must not look harmless.
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// One warp a (sequence, page, KV head).  A lane reads one word (eight channels) of a token's
// codes, so 32 / (D / 8) tokens at a time; rounding to T is monotone and comes once, at the end.
template <typename T, int D>
__global__ void __launch_bounds__(128) key_bounds_kernel(const PagedInt4 p, int pages_each) {
  constexpr int W = D / kInt4Group, kWords = D / 8, kTokens = 32 / kWords;
  release_dependents();
  dependency_wait();
  const int lane = threadIdx.x % 32;
  const int64_t unit = blockIdx.x * static_cast<int64_t>(blockDim.x / 32) + threadIdx.x / 32;
  const int h = static_cast<int>(unit % p.kv_heads);
  const int64_t rest = unit / p.kv_heads;
  const int i = static_cast<int>(rest % pages_each);
  const int64_t b = rest / pages_each;
  if (b >= p.batch) return;
  const int64_t tokens = row_tokens(p, static_cast<int>(b), 0);
  const int64_t before = tokens > p.new_tokens ? tokens - p.new_tokens : 0;
  const int64_t n = before / p.page_size + i;
  if (n * p.page_size >= tokens) return;
  const int64_t page = page_id(p, static_cast<int>(b), 0, n);
  if (page < 0 || page >= p.num_pages) {
    if (lane == 0) atomicMax(p.status, kStatusBadPageId);
    return;
  }
  const int64_t left = tokens - n * p.page_size;
  const int live = left < p.page_size ? static_cast<int>(left) : p.page_size;
  const int word = lane % kWords, t = word / W, w = word % W;
  float low[8], high[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) low[j] = INFINITY, high[j] = -INFINITY;
  for (int token = lane / kWords; token < live; token += kTokens) {
    const uint8_t* tile = p.pool + ((page * p.kv_heads + h) * (p.page_size / kInt4Tile) + token / kInt4Tile) * int4_tile_bytes(D);
    const int r = token % kInt4Tile;
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(tile + r * (D / 2) + 4 * word);
    const T* params = reinterpret_cast<const T*>(tile + 16 * D) + r * W + w;
    const float step = to_float(params[0]), floor = to_float(params[D / 2]);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = int4_value((codes >> (4 * j)) & 15u, step, floor);
      low[j] = min_nan(low[j], x), high[j] = max_nan(high[j], x);
    }
  }
#pragma unroll
  for (int off = kWords; off < 32; off <<= 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      low[j] = min_nan(low[j], __shfl_xor_sync(0xffffffffu, low[j], off));
      high[j] = max_nan(high[j], __shfl_xor_sync(0xffffffffu, high[j], off));
    }
  }
  if (lane < kWords) {
    T* dst = static_cast<T*>(p.bounds) + (page * p.kv_heads + h) * 2 * D + 32 * w + 8 * t;
    uint4 a, z;
    a.x = pack2<T>(low[0], low[1]), a.y = pack2<T>(low[2], low[3]), a.z = pack2<T>(low[4], low[5]), a.w = pack2<T>(low[6], low[7]);
    z.x = pack2<T>(high[0], high[1]), z.y = pack2<T>(high[2], high[3]), z.z = pack2<T>(high[4], high[5]), z.w = pack2<T>(high[6], high[7]);
    *reinterpret_cast<uint4*>(dst) = a;
    *reinterpret_cast<uint4*>(dst + D) = z;
  }
}

// Scores as unsigned keys that order like the scores, NaN above all; 0 is below every score.
__device__ __forceinline__ uint32_t score_key(float s) {
  if (!(s == s)) return 0xffffffffu;
  const uint32_t u = __float_as_uint(__fadd_rn(s, 0.f));  // -0 and 0 tie
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// keys[row][n], row = b * kv_heads + h: D / 8 lanes a page, eight channels each.
template <typename T, int D>
__global__ void __launch_bounds__(256) page_score_kernel(const PagedInt4 p, uint32_t* keys) {
  constexpr int kLanes = D / 8, kPages = 32 / kLanes;
  release_dependents();
  dependency_wait();
  const int row = blockIdx.y, b = row / p.kv_heads, h = row % p.kv_heads;
  const int lane = threadIdx.x % 32, l = lane % kLanes;
  const int64_t tokens = row_tokens(p, b, 0);
  const int count = static_cast<int>((tokens + p.page_size - 1) / p.page_size);
  if (count <= p.take) return;  // every page is taken
  const int group = p.q_heads / p.kv_heads;
  const int step = gridDim.x * (blockDim.x / 32) * kPages;
  for (int first = (blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32) * kPages; first < count - 1; first += step) {
    const int n = first + lane / kLanes;
    const int64_t page = n < count - 1 ? page_id(p, b, 0, n) : 0;
    const bool ok = n < count - 1 && page >= 0 && page < p.num_pages;
    if (!ok && n < count - 1 && l == 0) atomicMax(p.status, kStatusBadPageId);
    uint4 low = make_uint4(0, 0, 0, 0), high = low;
    if (ok) {
      const T* src = static_cast<const T*>(p.bounds) + (page * p.kv_heads + h) * 2 * D + 8 * l;
      low = *reinterpret_cast<const uint4*>(src), high = *reinterpret_cast<const uint4*>(src + D);
    }
    float best = -INFINITY;
    for (int g = 0; g < group; ++g) {
      const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + b * p.q_sb + (h * group + g) * p.q_sh + 8 * l);
      float sum[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = unpack2<T>((&q.x)[j]), lo = unpack2<T>((&low.x)[j]), hi = unpack2<T>((&high.x)[j]);
        sum[j] = __fadd_rn(max_nan(__fmul_rn(x.x, lo.x), __fmul_rn(x.x, hi.x)), max_nan(__fmul_rn(x.y, lo.y), __fmul_rn(x.y, hi.y)));
      }
      float s = __fadd_rn(__fadd_rn(sum[0], sum[1]), __fadd_rn(sum[2], sum[3]));
#pragma unroll
      for (int off = 1; off < kLanes; off <<= 1) s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, off));
      best = max_nan(best, s);
    }
    if (l == 0 && n < count - 1) keys[static_cast<int64_t>(row) * p.table_width + n] = ok ? score_key(best) : 0u;
  }
}

// One CTA a row.  The take - 1 largest keys of the pages before the newest: their smallest key
// by radix, eight bits a pass, then the pages in order, those that tie with it as long as there
// is room.
__global__ void __launch_bounds__(1024) page_pick_kernel(const PagedInt4 p, const uint32_t* keys) {
  __shared__ int s_count[256];
  __shared__ int s_warp[2][32];
  __shared__ uint32_t s_key;
  __shared__ int s_left;
  release_dependents();
  dependency_wait();
  const int row = blockIdx.x, b = row / p.kv_heads, h = row % p.kv_heads;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int64_t tokens = row_tokens(p, b, 0);
  const int count = static_cast<int>((tokens + p.page_size - 1) / p.page_size);
  int32_t* out = p.page_table + static_cast<int64_t>(row) * p.take;
  if (tid == 0) {
    const int64_t left_out = count > p.take ? static_cast<int64_t>(count - p.take) * p.page_size : 0;
    p.page_lens[row] = static_cast<int32_t>(tokens - left_out);
  }
  if (count <= p.take) {
    for (int n = tid; n < p.take; n += blockDim.x) out[n] = n < count ? static_cast<int32_t>(page_id(p, b, h, n)) : -1;
    return;
  }
  const uint32_t* mine = keys + static_cast<int64_t>(row) * p.table_width;
  const int others = count - 1;
  if (tid == 0) s_key = 0, s_left = p.take - 1;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (tid < 256) s_count[tid] = 0;
    __syncthreads();
    const uint32_t prefix = s_key;
    const int left = s_left;
    for (int n = tid; n < others; n += blockDim.x) {
      const uint32_t key = mine[n];
      if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&s_count[(key >> shift) & 255u], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int above = 0, digit = 255;
      for (; digit > 0 && above + s_count[digit] < left; --digit) above += s_count[digit];
      s_key = prefix | static_cast<uint32_t>(digit) << shift;
      s_left = left - above;
    }
  }
  __syncthreads();
  const uint32_t least = s_key;  // the smallest key taken; s_left pages that have it are
  const int ties = s_left;
  int written = 0, equal = 0;
  for (int first = 0; first < others; first += blockDim.x) {
    const int n = first + tid;
    const uint32_t key = n < others ? mine[n] : 0u;
    const bool is_equal = n < others && key == least;
    const unsigned equal_mask = __ballot_sync(0xffffffffu, is_equal);
    __syncthreads();
    if (lane == 0) s_warp[0][warp] = __popc(equal_mask);
    __syncthreads();
    int rank = equal;
    for (int w = 0; w < 32; ++w) rank += w < warp ? s_warp[0][w] : 0, equal += s_warp[0][w];
    rank += __popc(equal_mask & ((1u << lane) - 1));
    const bool taken = n < others && (key > least || (is_equal && rank < ties));
    const unsigned mask = __ballot_sync(0xffffffffu, taken);
    if (lane == 0) s_warp[1][warp] = __popc(mask);
    __syncthreads();
    int at = written;
    for (int w = 0; w < 32; ++w) at += w < warp ? s_warp[1][w] : 0, written += s_warp[1][w];
    at += __popc(mask & ((1u << lane) - 1));
    if (taken) out[at] = static_cast<int32_t>(page_id(p, b, h, n));
  }
  if (tid == 0) out[p.take - 1] = static_cast<int32_t>(page_id(p, b, h, count - 1));
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
  return p;
}

int launch_select(const PagedInt4& p, int head_dim, int dtype, cudaStream_t stream) {
  QF_REQUIRE(p.workspace != nullptr && p.workspace_bytes >= select_bytes(p), "the workspace holds %lld bytes, %lld are needed",
             static_cast<long long>(p.workspace_bytes), static_cast<long long>(select_bytes(p)));
  const int rows = p.batch * p.kv_heads;
  QF_REQUIRE(rows <= 65535, "at most 65535 (sequence, KV head) rows choose pages in one call");
  uint32_t* keys = static_cast<uint32_t*>(p.workspace);
  const int64_t blocks = (p.table_width + 63) / 64;
  const dim3 grid(static_cast<unsigned>(blocks < 1 ? 1 : blocks > 256 ? 256 : blocks), rows);
  cudaError_t err = cudaSuccess;
  if (dtype == QF_DTYPE_F16) {
    err = head_dim == 128 ? launch_chained(page_score_kernel<__half, 128>, grid, dim3(256), 0, stream, p, keys)
                          : launch_chained(page_score_kernel<__half, 64>, grid, dim3(256), 0, stream, p, keys);
  } else {
    err = head_dim == 128 ? launch_chained(page_score_kernel<__nv_bfloat16, 128>, grid, dim3(256), 0, stream, p, keys)
                          : launch_chained(page_score_kernel<__nv_bfloat16, 64>, grid, dim3(256), 0, stream, p, keys);
  }
  QF_CUDA(err);
  QF_CUDA(launch_chained(page_pick_kernel, dim3(rows), dim3(1024), 0, stream, p, static_cast<const uint32_t*>(keys)));
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
  QF_REQUIRE((units + 3) / 4 < (1LL << 31), "too many pages in one call");
  const dim3 grid(static_cast<unsigned>((units + 3) / 4));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t err = cudaSuccess;
  if (args->dtype == QF_DTYPE_F16) {
    err = args->head_dim == 128 ? launch_chained(key_bounds_kernel<__half, 128>, grid, dim3(128), 0, s, p, pages_each)
                                : launch_chained(key_bounds_kernel<__half, 64>, grid, dim3(128), 0, s, p, pages_each);
  } else {
    err = args->head_dim == 128 ? launch_chained(key_bounds_kernel<__nv_bfloat16, 128>, grid, dim3(128), 0, s, p, pages_each)
                                : launch_chained(key_bounds_kernel<__nv_bfloat16, 64>, grid, dim3(128), 0, s, p, pages_each);
  }
  QF_CUDA(err);
  QF_CUDA(cudaGetLastError());
  return QF_OK;
}

int qf_select_kv_pages(const qf_paged_int4_args* args, void* stream) {
  qf::PagedInt4 p;
  if (const int rc = qf::fill_paged_int4(args, qf::kNeedsQuery | qf::kNeedsBounds | qf::kNeedsSelection, &p)) return rc;
  if (p.batch == 0) return QF_OK;
  if (const int rc = qf::launch_select(p, args->head_dim, args->dtype, static_cast<cudaStream_t>(stream))) return rc;
  qf::request_ordered_launch();  // the selection is step metadata written by a kernel
  return QF_OK;
}

int qf_int4_sparse_decode_attention(const qf_paged_int4_args* args, void* stream) {
  using namespace qf;
  PagedInt4 p;
  if (const int rc = fill_paged_int4(args, kNeedsQuery | kNeedsPool | kNeedsOut | kNeedsBounds | kNeedsSelection, &p)) return rc;
  QF_REQUIRE(static_cast<int64_t>(p.take) * p.page_size < (1LL << 31), "the pages taken hold 2^31 tokens or more");
  if (p.batch == 0) return QF_OK;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  PagedInt4 next = over_selection(p);
  const int64_t keys = select_bytes(p);
  const int64_t more = int4_attention_bytes(next, args->head_dim);
  QF_REQUIRE(p.workspace != nullptr && p.workspace_bytes >= keys + more, "the workspace holds %lld bytes, %lld are needed",
             static_cast<long long>(p.workspace_bytes), static_cast<long long>(keys + more));
  if (const int rc = launch_select(p, args->head_dim, args->dtype, s)) return rc;
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
