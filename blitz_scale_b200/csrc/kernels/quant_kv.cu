// Writing rows of keys and values into a 4-bit cache, and reading them back in 16 bits (the format: quant_kv.cuh).
#include "launch.cuh"
#include "ptx.cuh"
#include "quant_kv.cuh"
#include "scalar.cuh"

namespace blitz {

struct QuantStoreParams {
  const void *k, *v;  // [tokens][kv_heads * dim], pitches in elements
  int64_t k_row, v_row;
  const int32_t* slot;
  uint8_t* pool;
  int64_t items;  // tokens * 2 * kv_heads * dim / 8
  int kv_heads, page_size, max_pages;
  int* status;
};

// Eight dimensions of a token a thread: the lanes of a group find its smallest and largest number together.
template <typename T, int D, int GROUP>
__global__ void __launch_bounds__(256) quant_kv_store_kernel(const QuantStoreParams p) {
  constexpr QuantKv F = quant_kv(D, GROUP);
  constexpr int LANES = D / 8;
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int64_t it = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const bool real = it < p.items;
  const int l = static_cast<int>(it % LANES);
  const int64_t rest = it / LANES;
  const int head = static_cast<int>(rest % p.kv_heads);
  const bool value = (rest / p.kv_heads) & 1;
  const int64_t t = rest / (2 * p.kv_heads);
  int s = real ? p.slot[t] : -1;
  if (s >= 0 && s / p.page_size >= p.max_pages) {
    if (p.status) atomicCAS(p.status, 0, kStatusBadIndex);
    s = -1;
  }
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = 0.f;
  if (s >= 0)
    ldf8<T>(reinterpret_cast<const T*>(value ? p.v : p.k) + t * (value ? p.v_row : p.k_row) + static_cast<int64_t>(head) * D + l * 8, x);
  float lo = x[0], hi = x[0], bad = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    bad += x[i] * 0.f;  // NaN where a number is not finite
  }
#pragma unroll
  for (int d = 1; d < GROUP / 8; d <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, d));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, d));
    bad += __shfl_xor_sync(0xffffffffu, bad, d);
  }
  __nv_bfloat16 z16 = __float2bfloat16_rd(lo);
  const float z = __bfloat162float(z16), range = hi - z + bad;
  __nv_bfloat16 s16 = __float2bfloat16_ru(__fdiv_rn(range, 15.f));
  if (!(range <= 3.4e38f)) {
    z16 = __ushort_as_bfloat16(0x7fff);
    s16 = __ushort_as_bfloat16(0);
  }
  const float sc = __bfloat162float(s16);
  uint32_t word = 0;
  if (sc > 0.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = fminf(fmaxf(rintf(__fdiv_rn(x[i] - z, sc)), 0.f), 15.f);
      word |= static_cast<uint32_t>(c) << (4 * i);
    }
  }
  const uint32_t other = __shfl_xor_sync(0xffffffffu, word, 1);  // the eight dimensions beside these of a tile of 16
  if (s < 0) return;
  const int off = s % p.page_size, tok = off & 15;
  uint8_t* block = p.pool + ((static_cast<int64_t>(s / p.page_size) * p.kv_heads + head) * (p.page_size >> 4) + (off >> 4)) * F.block;
  if (value) block += F.part;
  if (!value) {
    reinterpret_cast<uint32_t*>(block + tok * (D / 2))[(l & 3) * (D / 32) + (l >> 2)] = word;
  } else {
    // nibble i of this half of the tile beside nibble i of the other: even lanes write the first four such bytes, odd ones the rest
    const uint32_t low = l & 1 ? other : word, high = l & 1 ? word : other;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int g = (l & 1) * 4 + i;
      block[quant_kv_value_byte(tok, (l >> 1) * 16 + g)] = static_cast<uint8_t>(((low >> (4 * g)) & 15u) | (((high >> (4 * g)) & 15u) << 4));
    }
  }
  if (l % (GROUP / 8) == 0) {
    __nv_bfloat16* w = reinterpret_cast<__nv_bfloat16*>(block + F.codes) + tok * 2 * F.groups + l / (GROUP / 8);
    w[0] = s16;
    w[F.groups] = z16;
  }
}

struct QuantLoadParams {
  const uint8_t* pool;
  const int32_t* at;  // a slot per row, or a page per page_size rows
  void *k, *v;        // row r of page n of the output at n * page_rows + r (slots: rows back to back)
  int64_t items;      // rows * 2 * kv_heads * dim / 8
  int kv_heads, page_size, page_rows, max_pages, whole_pages;
  int* status;
};

template <typename T>
__device__ __forceinline__ float quant_kv_value(float z, float s, uint32_t c) {
  // (a scale that was rounded up can carry the largest number of a group past the type's)
  constexpr float most = std::is_same<T, __half>::value ? 65504.f : 3.3895313892515355e38f;
  const float x = fmaf(s, static_cast<float>(c), z);
  return fabsf(x) > most ? copysignf(most, x) : x;
}

template <typename T, int D, int GROUP>
__global__ void __launch_bounds__(256) quant_kv_load_kernel(const QuantLoadParams p) {
  constexpr QuantKv F = quant_kv(D, GROUP);
  constexpr int LANES = D / 8;
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int64_t it = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (it >= p.items) return;
  const int l = static_cast<int>(it % LANES);
  const int64_t rest = it / LANES;
  const int head = static_cast<int>(rest % p.kv_heads);
  const bool value = (rest / p.kv_heads) & 1;
  const int64_t r = rest / (2 * p.kv_heads);
  int64_t page, to = r;
  int off;
  if (p.whole_pages) {
    off = static_cast<int>(r % p.page_size);
    page = p.at[r / p.page_size];
    to = r / p.page_size * p.page_rows + off;
  } else {
    const int s = p.at[r];
    if (s < 0) return;
    page = s / p.page_size;
    off = s % p.page_size;
  }
  if (page < 0 || page >= p.max_pages) {
    if (p.status) atomicCAS(p.status, 0, kStatusBadIndex);
    return;
  }
  const int tok = off & 15;
  const uint8_t* block = p.pool + ((page * p.kv_heads + head) * (p.page_size >> 4) + (off >> 4)) * F.block;
  if (value) block += F.part;
  const __nv_bfloat16* w = reinterpret_cast<const __nv_bfloat16*>(block + F.codes) + tok * 2 * F.groups + l / (GROUP / 8);
  const float s = __bfloat162float(w[0]), z = __bfloat162float(w[F.groups]);
  float x[8];
  if (!value) {
    const uint32_t word = reinterpret_cast<const uint32_t*>(block + tok * (D / 2))[(l & 3) * (D / 32) + (l >> 2)];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = quant_kv_value<T>(z, s, (word >> (4 * i)) & 15u);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x[i] = quant_kv_value<T>(z, s, (static_cast<uint32_t>(block[quant_kv_value_byte(tok, (l >> 1) * 16 + i)]) >> (4 * (l & 1))) & 15u);
  }
  stf8<T>(reinterpret_cast<T*>(value ? p.v : p.k) + (to * p.kv_heads + head) * D + l * 8, x);
}

struct StoreLaunch {
  const QuantStoreParams& p;
  cudaStream_t stream;
  template <typename T, int D, int GROUP>
  int operator()() const {
    return (int)launch_pdl(quant_kv_store_kernel<T, D, GROUP>, dim3((unsigned)((p.items + 255) / 256)), dim3(256), 0, stream, p);
  }
};
struct LoadLaunch {
  const QuantLoadParams& p;
  cudaStream_t stream;
  template <typename T, int D, int GROUP>
  int operator()() const {
    return (int)launch_pdl(quant_kv_load_kernel<T, D, GROUP>, dim3((unsigned)((p.items + 255) / 256)), dim3(256), 0, stream, p);
  }
};

}  // namespace blitz

extern "C" {
using namespace blitz;

// k, v: [num_tokens] rows of kv_heads * dim elements, pitches k_row and v_row (multiples of 8, 16-byte aligned).  slot[t] = page *
// page_size + offset, negative: the row is not written.  The same slot twice: either row's bytes.
int blitz_quant_kv_store(const void* k, int64_t k_row, const void* v, int64_t v_row, const int32_t* slot, void* pool, int num_tokens,
                         int kv_heads, int dim, int group, int page_size, int max_pages, int* status, int dtype, cudaStream_t stream) {
  if (num_tokens <= 0) return 0;
  if (!quant_kv_supported(dim, group, page_size) || kv_heads < 1 || ((k_row | v_row) & 7)) return -1;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(pool)) & 15) return -1;
  QuantStoreParams p{k, v, k_row, v_row, slot, (uint8_t*)pool, (int64_t)num_tokens * 2 * kv_heads * (dim / 8), kv_heads, page_size, max_pages, status};
  if (p.items > (int64_t)256 * 0x7fffffff) return -1;
  return quant_kv_dispatch(dtype, dim, group, StoreLaunch{p, stream});
}

// Rows back in 16 bits.  whole_pages = 0: at[r] is a slot (negative: row r is left as it is), row r goes to row r of k and v; else at[n] is a
// page, whose tokens go to rows n * page_rows .. of k and v.  `count`: entries of at.
int blitz_quant_kv_load(const void* pool, const int32_t* at, int64_t count, int whole_pages, void* k, void* v, int kv_heads, int dim, int group,
                        int page_size, int page_rows, int max_pages, int* status, int dtype, cudaStream_t stream) {
  if (count <= 0) return 0;
  if (!quant_kv_supported(dim, group, page_size) || kv_heads < 1) return -1;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(pool)) & 15) return -1;
  QuantLoadParams p{(const uint8_t*)pool, at, k, v, count * (whole_pages ? page_size : 1) * 2 * kv_heads * (dim / 8), kv_heads, page_size, page_rows, max_pages, whole_pages, status};
  if (p.items > (int64_t)256 * 0x7fffffff) return -1;
  return quant_kv_dispatch(dtype, dim, group, LoadLaunch{p, stream});
}

}  // extern "C"
