// Decode attention of beams: one query token per row, rows in groups (the beams of a request) whose first pages are the same.
//
// out = softmax(q K^T scale) V per head over the row's pages [page][K|V][token][kv_head][dim].
#include "launch.cuh"
#include "ptx.cuh"
#include "tmap.cuh"
#include "common.cuh"
#include "mma.cuh"
#include "scalar.cuh"

namespace blitz {

struct BeamAttnParams {
  const void* q;
  int64_t q_stride;
  const void* kv;
  const int32_t *indices, *indptr, *last_page_len, *shared;
  void* out;
  int64_t out_stride;
  int rows, beams, q_heads, kv_heads, page, max_pages;
  float scale, cap;
  const void* sink;
  int* status;
};

// A warp per row and query head.
template <typename T, int HD>
__global__ void __launch_bounds__(128) attn_beams_kernel(const BeamAttnParams p) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  constexpr int N = HD / 32;
  const int lane = threadIdx.x & 31, item = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= p.rows * p.q_heads) return;
  const int row = item / p.q_heads, head = item % p.q_heads, h = head / (p.q_heads / p.kv_heads);
  const T* q = reinterpret_cast<const T*>(p.q) + row * p.q_stride + head * HD + lane * N;
  const int first = p.indptr[row], pages = p.indptr[row + 1] - first;
  const int length = pages > 0 ? (pages - 1) * p.page + p.last_page_len[row] : 0;
  float x[N], o[N] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = ldf(q + i);
  if (p.sink) {
    m = ldf(reinterpret_cast<const T*>(p.sink) + head);
    l = 1.f;
  }
  const int64_t pitch = static_cast<int64_t>(p.kv_heads) * HD;
  for (int t = 0; t < length; ++t) {
    int page = p.indices[first + t / p.page];
    if (page < 0 || page >= p.max_pages) {
      if (p.status && lane == 0) atomicCAS(p.status, 0, kStatusBadIndex);
      page = 0;
    }
    const T* k = reinterpret_cast<const T*>(p.kv) + (static_cast<int64_t>(page) * 2 * p.page + t % p.page) * pitch + h * HD + lane * N;
    const T* v = k + p.page * pitch;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s += x[i] * ldf(k + i);
    s = warp_sum(s) * p.scale;
    if (p.cap > 0.f) s = p.cap * tanhf(s / p.cap);
    const float top = fmaxf(m, s), keep = expf(m - top), w = expf(s - top);
    l = l * keep + w;
    m = top;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * keep + w * ldf(v + i);
  }
  T* out = reinterpret_cast<T*>(p.out) + row * p.out_stride + head * HD + lane * N;
#pragma unroll
  for (int i = 0; i < N; ++i) stf(out + i, l > 0.f ? o[i] / l : 0.f);
}

}  // namespace blitz

extern "C" {
using namespace blitz;

int64_t blitz_attn_beams_workspace_bytes(int rows, int beams, int q_heads, int kv_heads, int head_dim) { return 256; }

int blitz_attn_beams(const void* q, int64_t q_stride, const void* kv, const int32_t* indices, const int32_t* indptr, const int32_t* last_page_len,
                     const int32_t* shared, void* out, int64_t out_stride, void* workspace, int64_t workspace_bytes, int rows, int beams, int q_heads,
                     int kv_heads, int head_dim, int page, int max_pages, float scale, float cap, const void* sink, int static_table, int* status, int dtype,
                     cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (beams < 1 || rows % beams || kv_heads < 1 || q_heads % kv_heads || (head_dim != 64 && head_dim != 128) || page < 1 || max_pages < 1 ||
      workspace_bytes < blitz_attn_beams_workspace_bytes(rows, beams, q_heads, kv_heads, head_dim))
    return -1;
  BeamAttnParams p{q, q_stride, kv, indices, indptr, last_page_len, shared, out, out_stride, rows, beams, q_heads, kv_heads, page, max_pages, scale, cap, sink, status};
  cudaError_t e = cudaSuccess;
  const dim3 grid((rows * q_heads + 3) / 4);
  BLITZ_DISPATCH_DTYPE(dtype, (e = launch_pdl(head_dim == 64 ? attn_beams_kernel<T, 64> : attn_beams_kernel<T, 128>, grid, dim3(128), 0, stream, p)));
  return (int)e;
}

}  // extern "C"
