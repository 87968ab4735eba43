// Decode attention over a paged cache held in 4 bits (the format: quant_kv.cuh).
#include "launch.cuh"
#include "ptx.cuh"
#include "quant_kv.cuh"
#include "scalar.cuh"

namespace blitz {

struct DecodeQuantParams {
  const void* q;
  int64_t q_stride;
  const uint8_t* pool;
  const int32_t *indices, *indptr, *last_page_len;
  void* out;
  int64_t out_stride;
  int batch, q_heads, kv_heads, page_size, max_pages;
  float scale;
  int window, keep_first;
  float softcap;
  const void* sink;
  int* status;
};

// A block per (sequence, query head): its warps take every fourth key, a lane D / 32 dimensions.
template <typename T, int D, int GROUP>
__global__ void __launch_bounds__(128) attn_decode_quant_kernel(const DecodeQuantParams p) {
  constexpr QuantKv F = quant_kv(D, GROUP);
  constexpr int N = D / 32;
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int b = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = h / (p.q_heads / p.kv_heads);
  const int pg0 = p.indptr[b], npages = p.indptr[b + 1] - pg0;
  const int len = npages > 0 ? (npages - 1) * p.page_size + p.last_page_len[b] : 0;
  const int lo = p.window > 0 ? max(0, len - p.window) : 0;
  float q[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    q[i] = ldf<T>(reinterpret_cast<const T*>(p.q) + b * p.q_stride + h * D + lane + 32 * i);
    o[i] = 0.f;
  }
  for (int j = warp; j < len; j += 4) {
    if (j < lo && j >= p.keep_first) continue;
    int page = p.indices[pg0 + j / p.page_size];
    if (page < 0 || page >= p.max_pages) {
      if (p.status && lane == 0) atomicCAS(p.status, 0, kStatusBadIndex);
      page = 0;
    }
    const int off = j % p.page_size, tok = off & 15;
    const uint8_t* block = p.pool + ((static_cast<int64_t>(page) * p.kv_heads + kvh) * (p.page_size >> 4) + (off >> 4)) * F.block;
    const __nv_bfloat16* kw = reinterpret_cast<const __nv_bfloat16*>(block + F.codes) + tok * 2 * F.groups;
    const __nv_bfloat16* vw = reinterpret_cast<const __nv_bfloat16*>(block + F.part + F.codes) + tok * 2 * F.groups;
    float dot = 0.f, v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = lane + 32 * i, g = d / GROUP;
      const uint32_t word = reinterpret_cast<const uint32_t*>(block + tok * (D / 2))[((d >> 3) & 3) * (D / 32) + (d >> 5)];
      dot += q[i] * fmaf(__bfloat162float(kw[g]), static_cast<float>((word >> (4 * (d & 7))) & 15u), __bfloat162float(kw[F.groups + g]));
      const uint32_t byte = block[F.part + quant_kv_value_byte(tok, d)];
      v[i] = fmaf(__bfloat162float(vw[g]), static_cast<float>((byte >> (4 * ((d >> 3) & 1))) & 15u), __bfloat162float(vw[F.groups + g]));
    }
    float s = warp_sum(dot) * p.scale;
    if (p.softcap > 0.f) s = p.softcap * tanhf(s / p.softcap);
    const float top = fmaxf(m, s), a = expf(m - top), w = expf(s - top);
    l = l * a + w;
    m = top;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * a + w * v[i];
  }
  __shared__ float so[4][D], sm[4], sl[4];
#pragma unroll
  for (int i = 0; i < N; ++i) so[warp][lane + 32 * i] = o[i];
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
  __syncthreads();
  const float snk = p.sink ? ldf<T>(reinterpret_cast<const T*>(p.sink) + h) : -INFINITY;
  const float top = fmaxf(fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), snk);
  for (int d = threadIdx.x; d < D; d += 128) {
    float acc = 0.f, sum = p.sink ? expf(snk - top) : 0.f;
    for (int w = 0; w < 4; ++w) {
      const float a = sl[w] != 0.f ? expf(sm[w] - top) : 0.f;
      acc += a * so[w][d];
      sum += a * sl[w];
    }
    stf(reinterpret_cast<T*>(p.out) + b * p.out_stride + h * D + d, sum != 0.f ? acc / sum : 0.f);
  }
}

struct DecodeQuantLaunch {
  const DecodeQuantParams& p;
  cudaStream_t stream;
  template <typename T, int D, int GROUP>
  int operator()() const {
    return (int)launch_pdl(attn_decode_quant_kernel<T, D, GROUP>, dim3(p.batch, p.q_heads), dim3(128), 0, stream, p);
  }
};

}  // namespace blitz

extern "C" {
using namespace blitz;

// q: [batch] rows with the query heads in their first q_heads * dim columns.  A sequence without keys has an output of zeros.
int blitz_attn_decode_quant(const void* q, int64_t q_stride, const void* pool, const int32_t* indices, const int32_t* indptr,
                            const int32_t* last_page_len, void* out, int64_t out_stride, int batch, int q_heads, int kv_heads, int dim, int group,
                            int page_size, int max_pages, float sm_scale, int window, int keep_first, float softcap, const void* sink,
                            int* status, int dtype, cudaStream_t stream) {
  if (batch <= 0) return 0;
  if (!quant_kv_supported(dim, group, page_size) || kv_heads < 1 || q_heads % kv_heads || window < 0 || keep_first < 0 || softcap < 0.f) return -1;
  DecodeQuantParams p{q, q_stride, (const uint8_t*)pool, indices, indptr, last_page_len, out, out_stride, batch, q_heads, kv_heads, page_size, max_pages, sm_scale, window, keep_first, softcap, sink, status};
  return quant_kv_dispatch(dtype, dim, group, DecodeQuantLaunch{p, stream});
}

}  // extern "C"
