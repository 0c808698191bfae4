// GQA decode attention over the 4-bit paged KV cache (layout: qf_int4_codec.cuh): one query
// token a sequence, a block table a sequence or one a (sequence, KV head).
#include "qf_int4_paged.cuh"

namespace qf {
namespace {

// One CTA a (sequence, KV head); its eight warps take tiles in turn, a lane D / 32 channels.
template <typename T, int D>
__global__ void __launch_bounds__(256) int4_attention_kernel(const PagedInt4 p) {
  constexpr int C = D / 32;  // channels of a lane: 32 c + lane
  constexpr int kWarps = 8, kMaxGroup = 16;
  __shared__ float s_o[kWarps][D];
  __shared__ float s_m[kWarps], s_l[kWarps];
  dependency_wait();
  const int b = blockIdx.x / p.kv_heads, h = blockIdx.x % p.kv_heads;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int group = p.q_heads / p.kv_heads;
  const int64_t tokens = row_tokens(p, b, h);
  for (int g = 0; g < group; ++g) {
    const int head = h * group + g;
    float q[C], o[C], m = -INFINITY, l = 0.f;
    for (int c = 0; c < C; ++c) {
      q[c] = to_float(static_cast<const T*>(p.q)[b * p.q_sb + head * p.q_sh + 32 * c + lane]) * p.scale;
      o[c] = 0.f;
    }
    for (int64_t tile = warp; tile * kInt4Tile < tokens; tile += kWarps) {
      const uint8_t* base = tile_address<D>(p, b, h, tile);
      if (base == nullptr && lane == 0) atomicMax(p.status, kStatusBadPageId);
      for (int token = 0; token < kInt4Tile && tile * kInt4Tile + token < tokens; ++token) {
        float k[C], v[C], s = 0.f;
        for (int c = 0; c < C; ++c) {
          k[c] = v[c] = 0.f;
          if (base != nullptr) {
            const T* params = reinterpret_cast<const T*>(base + 16 * D) + token * C + c;
            const int kb = base[token * (D / 2) + lane / 8 * 4 * C + 4 * c + lane % 8 / 2];
            const int vb = base[8 * D + token / 2 * D + lane / 4 * 4 * C + 4 * c + token % 2 * 2 + lane % 4 / 2];
            k[c] = int4_value((kb >> (lane % 2 * 4)) & 15, to_float(params[0]), to_float(params[D / 2]));
            v[c] = int4_value((vb >> (lane % 2 * 4)) & 15, to_float(params[D]), to_float(params[3 * D / 2]));
          }
          s += q[c] * k[c];
        }
        for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
        const float top = fmaxf(m, s);
        const float keep = m == top ? 1.f : expf(m - top), e = expf(s - top);
        l = l * keep + e;
        for (int c = 0; c < C; ++c) o[c] = o[c] * keep + e * v[c];
        m = top;
      }
    }
    __syncthreads();
    for (int c = 0; c < C; ++c) s_o[warp][32 * c + lane] = o[c];
    if (lane == 0) s_m[warp] = m, s_l[warp] = l;
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += blockDim.x) {
      float top = -INFINITY, sum = 0.f, acc = 0.f;
      for (int w = 0; w < kWarps; ++w) top = s_l[w] != 0.f ? fmaxf(top, s_m[w]) : top;
      for (int w = 0; w < kWarps; ++w) {
        if (s_l[w] == 0.f) continue;
        const float f = expf(s_m[w] - top);
        sum += f * s_l[w], acc += f * s_o[w][d];
      }
      static_cast<T*>(p.out)[b * p.o_sb + head * p.o_sh + d] = from_float<T>(sum == 0.f ? 0.f : acc / sum);
    }
  }
}

}  // namespace

int64_t int4_attention_bytes(const PagedInt4&) { return 0; }

int launch_int4_attention(const PagedInt4& p, int head_dim, int dtype, cudaStream_t stream) {
  const dim3 grid(p.batch * p.kv_heads);
  cudaError_t err = cudaSuccess;
  if (dtype == QF_DTYPE_F16) {
    err = head_dim == 128 ? launch_chained(int4_attention_kernel<__half, 128>, grid, dim3(256), 0, stream, p)
                          : launch_chained(int4_attention_kernel<__half, 64>, grid, dim3(256), 0, stream, p);
  } else {
    err = head_dim == 128 ? launch_chained(int4_attention_kernel<__nv_bfloat16, 128>, grid, dim3(256), 0, stream, p)
                          : launch_chained(int4_attention_kernel<__nv_bfloat16, 64>, grid, dim3(256), 0, stream, p);
  }
  QF_CUDA(err);
  QF_CUDA(cudaGetLastError());
  return QF_OK;
}

}  // namespace qf

extern "C" int qf_int4_decode_attention(const qf_paged_int4_args* args, void* stream) {
  qf::PagedInt4 p;
  if (const int rc = qf::fill_paged_int4(args, qf::kNeedsQuery | qf::kNeedsPool | qf::kNeedsOut, &p)) return rc;
  if (p.batch == 0) return QF_OK;
  return qf::launch_int4_attention(p, args->head_dim, args->dtype, static_cast<cudaStream_t>(stream));
}
