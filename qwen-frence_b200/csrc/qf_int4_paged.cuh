// Arguments shared by the kernels that walk a 4-bit paged cache or its key bounds: checked once
// on the host (fill_paged_int4), then handed to a kernel by value.
#pragma once

#include <cmath>

#include "qf_int4_codec.cuh"

namespace qf {

struct PagedInt4 {
  const void* q;
  void* out;
  const uint8_t* pool;
  void* bounds;
  const void* table;
  const void* lens;
  void* workspace;
  int32_t* page_table;
  int32_t* page_lens;
  int* status;
  int64_t q_sb, q_sh, o_sb, o_sh;
  int64_t t_sb, t_sh, t_sp, l_sb, l_sh;
  int64_t num_pages, table_width, workspace_bytes;
  float scale;
  int batch, q_heads, kv_heads, page_size;
  int table_dtype, lens_dtype;
  int new_tokens, take;
  Divisor by_heads, by_page, by_tiles;  // kv_heads, page_size, tiles of a page
  bool even;   // rows are about equally long, most of them as long as the table
  bool early;  // table and lengths are step metadata: read before the kernel in front has finished; not those of a choice
};

enum : int { kNeedsQuery = 1, kNeedsPool = 2, kNeedsOut = 4, kNeedsBounds = 8, kNeedsSelection = 16 };

int fill_paged_int4(const qf_paged_int4_args* args, int needs, PagedInt4* p);
inline bool on_boundary(const void* at, int bytes) { return (reinterpret_cast<uintptr_t>(at) & (bytes - 1)) == 0; }
inline bool index_aligned(const void* at, int dtype) { return on_boundary(at, dtype == QF_INDEX_I64 ? 8 : 4); }
// Multiprocessors of the current device, 148 where there is none.
int sm_count();
int64_t int4_attention_bytes(const PagedInt4& p, int head_dim);  // scratch of launch_int4_attention
int launch_int4_attention(const PagedInt4& p, int head_dim, int dtype, cudaStream_t stream);

// (sequence, KV head) of a row.
__device__ __forceinline__ int2 row_place(const PagedInt4& p, int row) {
  const int b = quotient(row, p.by_heads);
  return make_int2(b, row - b * p.kv_heads);
}

// Tokens of row (b, h): never negative, never more than its table row can hold.
__device__ __forceinline__ int64_t row_tokens(const PagedInt4& p, int b, int h) {
  const int64_t n = load_index(p.lens, p.lens_dtype, b * p.l_sb + h * p.l_sh);
  const int64_t most = p.table_width * p.page_size;
  return n < 0 ? 0 : n > most ? most : n;
}

__device__ __forceinline__ int64_t page_id(const PagedInt4& p, int b, int h, int64_t n) {
  return load_index(p.table, p.table_dtype, b * p.t_sb + h * p.t_sh + n * p.t_sp);
}

}  // namespace qf
