// Writing rows of keys and values into a 4-bit cache, and reading them back in 16 bits (the format: quant_kv.cuh).
#include "launch.cuh"
#include "ptx.cuh"
#include "quant_kv.cuh"
#include "scalar.cuh"
#include "tmap.cuh"

namespace blitz {

// The smaller, or larger, of two pairs of numbers (NaN where there is one).
template <typename T>
using QuantPair = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
template <typename T>
__device__ __forceinline__ uint32_t quant_kv_least(uint32_t a, uint32_t b) {
  const QuantPair<T> m = __hmin2_nan(*reinterpret_cast<QuantPair<T>*>(&a), *reinterpret_cast<QuantPair<T>*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
template <typename T>
__device__ __forceinline__ uint32_t quant_kv_largest(uint32_t a, uint32_t b) {
  const QuantPair<T> m = __hmax2_nan(*reinterpret_cast<QuantPair<T>*>(&a), *reinterpret_cast<QuantPair<T>*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
// A lane's numbers, eight in each of N words of four registers, of a group that LANES lanes share: codes, and the group's scale and offset.
template <typename T, int N, int LANES>
__device__ __forceinline__ void quant_kv_group(const uint4 (&u)[N], uint32_t (&word)[N], __nv_bfloat16& s16, __nv_bfloat16& z16) {
  // the smallest number and the negative of the largest, as a pair (NaN where there is one)
  uint32_t lo2[N], hi2[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    lo2[i] = quant_kv_least<T>(quant_kv_least<T>(u[i].x, u[i].y), quant_kv_least<T>(u[i].z, u[i].w));
    hi2[i] = quant_kv_largest<T>(quant_kv_largest<T>(u[i].x, u[i].y), quant_kv_largest<T>(u[i].z, u[i].w));
  }
#pragma unroll
  for (int d = N / 2; d > 0; d >>= 1)
#pragma unroll
    for (int i = 0; i < d; ++i) {
      lo2[i] = quant_kv_least<T>(lo2[i], lo2[i + d]);
      hi2[i] = quant_kv_largest<T>(hi2[i], hi2[i + d]);
    }
  hi2[0] ^= 0x80008000u;
  uint32_t ends = quant_kv_least<T>(__byte_perm(lo2[0], hi2[0], 0x5410), __byte_perm(lo2[0], hi2[0], 0x7632));
#pragma unroll
  for (int d = 1; d < LANES; d <<= 1) ends = quant_kv_least<T>(ends, __shfl_xor_sync(0xffffffffu, ends, d));
  const float2 end = cvt2<T>(ends);
  z16 = __float2bfloat16_rd(end.x);
  const float z = __bfloat162float(z16), range = -end.y - z;
  // the smallest scale whose 15 steps cover the range: near range / 15, and then by what its product says
  uint32_t sb = __bfloat16_as_ushort(__float2bfloat16_ru(range * (1.f / 15.f)));
  if (fmaf(__uint_as_float(sb << 16), 15.f, -range) < 0.f) ++sb;
  else if (sb > 0 && fmaf(__uint_as_float((sb - 1) << 16), 15.f, -range) >= 0.f) --sb;
  if (!(range <= 3.4e38f)) {
    z16 = __ushort_as_bfloat16(0x7fff);
    sb = 0;
  }
  s16 = __ushort_as_bfloat16(static_cast<unsigned short>(sb));
  const float sc = __uint_as_float(sb << 16);
  // rint((x - z) / s), between 0 and 15, the quotient rounded to fp32 as a division's: y = 1 / s correctly rounded by a Newton step (s has 8
  // bits, which keeps 1 / s away from halfway between two numbers), a quotient q within two units of the last place, and q + (d - q s) y,
  // Markstein's correction, where d - q s is exact and d / s is never halfway either.  (Below 2^-100 it might not be exact: those are
  // divided.)  Rounded by what is left of a mantissa; two at a time, numbers i and i + 4.
  if (sc > 0.f) {
    float y = ptx::rcp_approx(sc);
    y = fmaf(fmaf(-sc, y, 1.f), y, y);
    const uint64_t y2 = ptx::f32x2(y, y), s2 = ptx::f32x2(-sc, -sc), z2 = ptx::f32x2(-z, -z);
    const uint64_t sixteen = ptx::f32x2(16.f, 16.f), up = ptx::f32x2(12582912.f, 12582912.f), down = ptx::f32x2(-12582912.f, -12582912.f);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float x[8];
      unpack8<T>(u[k], x);
      uint64_t c[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t d = ptx::add_f32x2(ptx::f32x2(x[i], x[i + 4]), z2), q = ptx::mul_f32x2(d, y2);
        c[i] = ptx::fma_f32x2(ptx::fma_f32x2(q, s2, d), y2, q);
        c[i] = ptx::add_f32x2(ptx::add_f32x2(c[i], up), down);
      }
      if (sc < 7.9e-31f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = ptx::f32x2(rintf(__fdiv_rn(x[i] - z, sc)), rintf(__fdiv_rn(x[i + 4] - z, sc)));
      }
      // four codes are a number of 16 bits
      const float2 four = ptx::f32x2_get(ptx::add_f32x2(ptx::fma_f32x2(ptx::fma_f32x2(ptx::fma_f32x2(c[3], sixteen, c[2]), sixteen, c[1]), sixteen, c[0]), ptx::f32x2(8388608.f, 8388608.f)));
      word[k] = __byte_perm(__float_as_uint(four.x), __float_as_uint(four.y), 0x5410);
    }
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) word[k] = 0;
  }
}

// A lane's eight codes of token `tok` of a block (null: nowhere) and, by a group's first lane, its scale and offset.  Values of four tokens of a
// word go to `exchange` instead (quant_kv_write_quad follows); others write their bytes.  The whole warp calls.
template <int D, int GROUP>
__device__ __forceinline__ void quant_kv_write(uint8_t* block, int tok, int l, bool value, uint32_t* exchange, uint32_t word, __nv_bfloat16 s16, __nv_bfloat16 z16) {
  constexpr QuantKv F = quant_kv(D, GROUP);
  if (value) block = block ? block + F.part : nullptr;
  const uint32_t other = __shfl_xor_sync(0xffffffffu, word, 1);  // the eight dimensions beside these of a tile of 16
  if (exchange != nullptr) {
    exchange[l] = word;
  } else if (block != nullptr && !value) {
    reinterpret_cast<uint32_t*>(block + tok * (D / 2))[(l & 3) * (D / 32) + (l >> 2)] = word;
  } else if (block != nullptr) {
    // nibble i of this half of the tile beside nibble i of the other: even lanes write the first four such bytes, odd ones the rest
    const uint32_t low = l & 1 ? other : word, high = l & 1 ? word : other;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int g = (l & 1) * 4 + i;
      block[quant_kv_value_byte(tok, (l >> 1) * 16 + g)] = static_cast<uint8_t>(((low >> (4 * g)) & 15u) | (((high >> (4 * g)) & 15u) << 4));
    }
  }
  if (l % (GROUP / 8) == 0 && block != nullptr) {
    __nv_bfloat16* w = reinterpret_cast<__nv_bfloat16*>(block + F.codes) + tok * 2 * F.groups + l / (GROUP / 8);
    w[0] = s16;
    w[F.groups] = z16;
  }
}
// Nibbles of a tile of 16 dimensions: lane i looks after tile m and, of its dimensions, 2 a, 2 a + 1 and those 8 behind.
struct QuantTile {
  int m, a;
  __device__ __forceinline__ QuantTile() {
    const int i = threadIdx.x & 31;
    m = (i >> 4) * 4 + (i & 3);
    a = (i >> 2) & 3;
  }
  // of the first of its two words, of the four tokens from `tok` on, in the values' codes
  __device__ __forceinline__ int at(int tok) const { return (m >> 2) * 512 + a * 128 + (tok >> 2) * 16 + (m & 3) * 4; }
};
// The words of four tokens, from token `tok` of a block on, whose codes the warp has put into `codes` [4][PITCH].
template <int D, int GROUP, int PITCH = D / 8>
__device__ __forceinline__ void quant_kv_write_quad(uint8_t* block, int tok, const uint32_t* codes) {
  const QuantTile t;
  __syncwarp();
  if (t.m < D / 16) {
    // a word's bytes are tokens 0, 2, 1, 3, nibbles dimensions 16 m + g and 16 m + 8 + g; byte a of a row's word has g = 2 a and 2 a + 1
    uint2 w[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) w[b] = *reinterpret_cast<const uint2*>(codes + ((b & 1) * 2 + (b >> 1)) * PITCH + 2 * t.m);
    const uint32_t pick = t.a | (t.a + 4) << 4;
    const uint32_t low = __byte_perm(__byte_perm(w[0].x, w[1].x, pick), __byte_perm(w[2].x, w[3].x, pick), 0x5410);
    const uint32_t high = __byte_perm(__byte_perm(w[0].y, w[1].y, pick), __byte_perm(w[2].y, w[3].y, pick), 0x5410);
    uint8_t* const to = block + quant_kv(D, GROUP).part + t.at(tok);
    *reinterpret_cast<uint32_t*>(to) = (low & 0x0f0f0f0fu) | ((high << 4) & 0xf0f0f0f0u);
    *reinterpret_cast<uint32_t*>(to + 64) = ((low >> 4) & 0x0f0f0f0fu) | (high & 0xf0f0f0f0u);
  }
}

// ------------------------------------------------------------------ rows in
struct QuantStoreParams {
  const void *k, *v;  // [tokens][kv_heads * dim], pitches in elements
  int64_t k_row, v_row;
  const int32_t* slot;
  uint8_t* pool;
  int64_t units;  // (rows of a warp, head, keys or values) each
  int tokens, kv_heads, page_shift, max_pages;
  int* status;
};

// A warp takes keys or values of a head, of 8 rows (16 of 64 dimensions): a lane has 32 dimensions, so that what a group needs once, its ends
// and its scale, is worked out by the one lane, two or four that have it (with eight dimensions a lane that was half of 195 instructions for
// 256 numbers, and 8192 rows took 16.5 us).  The codes go through shared memory: keys leave in rows of 16 bytes a lane.  A word of the values
// holds four tokens of two dimensions: where four rows are the four tokens of a word (rows of a prompt) words are written, else (the tokens
// of a batch) every row's bytes.
//
// Measured, 8 heads of 128: 8192 rows 12.0 us (44 MB, 3.7 TB/s, bound by the issue of instructions), 256 rows in pages of their own 2.6 us, one
// row 2.0 us (latency: slot, row, code).  Blocks of 128 threads: of 256 they took 12.9, 3.1 and 2.15 us.
template <typename T, int D, int GROUP>
__global__ void __launch_bounds__(128) quant_kv_store_kernel(const QuantStoreParams p) {
  constexpr QuantKv F = quant_kv(D, GROUP);
  constexpr int LANES = D / 32, ROWS = 32 / LANES, PITCH = D / 8 + 4;  // (rows in different banks)
  __shared__ __align__(16) uint32_t s_codes[4][ROWS * PITCH];
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int lane = threadIdx.x & 31, l = lane % LANES, row = lane / LANES;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (unit >= p.units) return;
  const bool value = unit & 1;
  const int head = static_cast<int>((unit >> 1) % p.kv_heads);
  const int64_t t0 = (unit >> 1) / p.kv_heads * ROWS, t = t0 + row;
  uint32_t* const codes = s_codes[threadIdx.x >> 5];
  // lane i has the i-th slot
  int slots = lane < ROWS && t0 + lane < p.tokens ? p.slot[t0 + lane] : -1;
  uint4 raw[4];
  const T* from = reinterpret_cast<const T*>(value ? p.v : p.k) + t * (value ? p.v_row : p.k_row) + static_cast<int64_t>(head) * D + l * 32;
#pragma unroll
  for (int i = 0; i < 4; ++i) raw[i] = t < p.tokens ? *reinterpret_cast<const uint4*>(from + i * 8) : make_uint4(0, 0, 0, 0);
  if (slots >= 0 && slots >> p.page_shift >= p.max_pages) {
    if (p.status) atomicCAS(p.status, 0, kStatusBadIndex);
    slots = -1;
  }
  const int s0 = __shfl_sync(0xffffffffu, slots, lane & 28);  // of four rows, the first one's
  const uint32_t quads = __ballot_sync(0xffffffffu, s0 >= 0 && (s0 & 3) == 0 && slots == s0 + (lane & 3));
  const int s = __shfl_sync(0xffffffffu, slots, row);
  auto block_of = [&](int s) {
    const int page = s >> p.page_shift;
    return p.pool + (((static_cast<int64_t>(page) * p.kv_heads + head) << (p.page_shift - 4)) + ((s - (page << p.page_shift)) >> 4)) * F.block + (value ? F.part : 0);
  };
  uint32_t word[4];
  __nv_bfloat16 s16, z16;
  quant_kv_group<T, 4, GROUP / 32>(raw, word, s16, z16);
  const bool quad = ((quads >> (row & 28)) & 15u) == 15u;
  const int tok = s & 15;
  if (s >= 0) {
    uint8_t* const block = block_of(s);
    if (l % (GROUP / 32) == 0) {
      __nv_bfloat16* w = reinterpret_cast<__nv_bfloat16*>(block + F.codes) + tok * 2 * F.groups + l / (GROUP / 32);
      w[0] = s16;
      w[F.groups] = z16;
    }
  }
  if (!value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) codes[row * PITCH + i * LANES + l] = word[i];
    __syncwarp();
    if (s >= 0) *reinterpret_cast<uint4*>(block_of(s) + tok * (D / 2) + l * 16) = *reinterpret_cast<const uint4*>(codes + row * PITCH + l * 4);
    return;
  }
  *reinterpret_cast<uint4*>(codes + row * PITCH + l * 4) = make_uint4(word[0], word[1], word[2], word[3]);
  __syncwarp();
#pragma unroll
  for (int r = 0; r < ROWS; r += 4) {
    const int at = __shfl_sync(0xffffffffu, s0, r);
    if (((quads >> r) & 15u) == 15u) quant_kv_write_quad<D, GROUP, PITCH>(block_of(at) - F.part, at & 15, codes + r * PITCH);
  }
  if (__all_sync(0xffffffffu, quad || s < 0)) return;
  // a lane has a tile of 16 dimensions of a row, g = 0 .. 3 or 4 .. 7 of it: nibbles 16 m + g and 16 m + 8 + g are a byte
  constexpr int EACH = D / 8, TIMES = ROWS * EACH / 32;
  const int m = lane % EACH >> 1, half = lane & 1;
#pragma unroll 1
  for (int i = 0; i < TIMES; ++i) {
    const int r = i * (32 / EACH) + lane / EACH, to = __shfl_sync(0xffffffffu, slots, r);
    if (to < 0 || ((quads >> (r & 28)) & 15u) == 15u) continue;
    const uint2 w = *reinterpret_cast<const uint2*>(codes + r * PITCH + 2 * m);
    const uint32_t even = ((w.x & 0x0f0f0f0fu) | ((w.y << 4) & 0xf0f0f0f0u)) >> (16 * half), odd = (((w.x >> 4) & 0x0f0f0f0fu) | (w.y & 0xf0f0f0f0u)) >> (16 * half);
    uint8_t* const d = block_of(to) + quant_kv_value_byte(to & 15, m * 16) + half * 256;
    d[0] = static_cast<uint8_t>(even);
    d[64] = static_cast<uint8_t>(odd);
    d[128] = static_cast<uint8_t>(even >> 8);
    d[192] = static_cast<uint8_t>(odd >> 8);
  }
}

// ------------------------------------------------------------------ rotation and rows in
struct QuantRopeParams {
  void* qkv;  // [tokens][(q_heads + 2 kv_heads) * dim], queries and keys are rotated in place
  const int32_t *pos, *slot;
  uint8_t* pool;
  int tokens, q_heads, kv_heads, page_shift, max_pages;
  float log2_theta;
  int* status;
};

// Queries and keys of a fused projection rotated in place (half-split pairs, as rope_kv_store does), keys and values into the cache: what goes
// there is what the 16-bit rows hold.  A block takes R tokens, whose angles it computes once; a warp four (row, head) pairs at a time:
// four rows of a head (R = 4: values go out by words), or four heads of a row (R = 1: more blocks where there are few tokens).
// STATIC: positions and slots that no kernel in flight writes: angles are ready when the projection is.
// Measured, 32 query heads and 8 KV heads of 128: 8192 rows 46 us (195 MB, 4.2 TB/s; into a 16-bit cache 43 us), 256 rows 4.7 us, one row 2.9 us.  With
// 74 registers a thread, three blocks on an SM, 8192 rows took 51 us.
template <typename T, int D, int GROUP, int R, bool STATIC>
__global__ void __launch_bounds__(256, 4) quant_kv_rope_kernel(const QuantRopeParams p) {
  constexpr QuantKv F = quant_kv(D, GROUP);
  constexpr int LANES = D / 8, ROWS = 32 / LANES, HALF = D / 2;
  __shared__ float s_cos[R][HALF], s_sin[R][HALF];
  __shared__ __align__(8) uint32_t s_codes[8][R == 4 ? 4 * LANES : 1];
  ptx::griddep_launch_dependents();
  if (!STATIC) ptx::griddep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % LANES;
  const int t0 = blockIdx.x * R;
  int slots = lane < R && t0 + lane < p.tokens ? p.slot[t0 + lane] : -1;
  const bool bad = slots >= 0 && slots >> p.page_shift >= p.max_pages;
  if (bad) slots = -1;
  for (int i = threadIdx.x; i < R * HALF; i += 256) {
    const int r = i / HALF, k = i % HALF;
    const float x = static_cast<float>(t0 + r < p.tokens ? p.pos[t0 + r] : 0) * exp2f(-(2.0f * static_cast<float>(k) / static_cast<float>(D)) * p.log2_theta);
    sincosf(x, &s_sin[r][k], &s_cos[r][k]);
  }
  if (STATIC) ptx::griddep_wait();
  if (bad && warp == 0 && p.status) atomicCAS(p.status, 0, kStatusBadIndex);
  __syncthreads();
  const int s0 = __shfl_sync(0xffffffffu, slots, 0), turned = p.q_heads + p.kv_heads, heads = turned + p.kv_heads;
  const bool quad = R == 4 && s0 >= 0 && (s0 & 3) == 0 && __all_sync(0xffffffffu, lane >= 4 || slots == s0 + lane);
  const int64_t pitch = static_cast<int64_t>(heads) * D;
  auto block_of = [&](int s, int kv) {
    const int page = s >> p.page_shift;
    return p.pool + (((static_cast<int64_t>(page) * p.kv_heads + kv) << (p.page_shift - 4)) + ((s - (page << p.page_shift)) >> 4)) * F.block;
  };
  const int units = R == 4 ? heads : (heads + 3) / 4;
  uint4 raw[4 / ROWS], next[4 / ROWS];
  T *at[4 / ROWS], *next_at[4 / ROWS];
  auto fetch = [&](int unit) {
#pragma unroll
    for (int k = 0; k < 4 / ROWS; ++k) {
      const int i = k * ROWS + lane / LANES, row = R == 4 ? i : 0, h = R == 4 ? unit : unit * 4 + i;
      const bool real = t0 + row < p.tokens && h < heads;
      next_at[k] = real ? reinterpret_cast<T*>(p.qkv) + static_cast<int64_t>(t0 + row) * pitch + static_cast<int64_t>(h) * D + l * 8 : nullptr;
      next[k] = real ? *reinterpret_cast<const uint4*>(next_at[k]) : make_uint4(0, 0, 0, 0);
    }
  };
  if (warp < units) fetch(warp);
  for (int unit = warp; unit < units; unit += 8) {
#pragma unroll
    for (int k = 0; k < 4 / ROWS; ++k) {
      raw[k] = next[k];
      at[k] = next_at[k];
    }
    if (unit + 8 < units) fetch(unit + 8);  // (asked for a turn ahead)
#pragma unroll
    for (int k = 0; k < 4 / ROWS; ++k) {
      const int i = k * ROWS + lane / LANES, row = R == 4 ? i : 0, h = R == 4 ? unit : unit * 4 + i;
      if (R == 1 || h < turned) {
        // the other half of the pairs is LANES / 2 lanes away
        uint4 o;
        o.x = __shfl_xor_sync(0xffffffffu, raw[k].x, LANES / 2);
        o.y = __shfl_xor_sync(0xffffffffu, raw[k].y, LANES / 2);
        o.z = __shfl_xor_sync(0xffffffffu, raw[k].z, LANES / 2);
        o.w = __shfl_xor_sync(0xffffffffu, raw[k].w, LANES / 2);
        if (h < turned) {
          float x[8], y[8];
          unpack8<T>(raw[k], x);
          unpack8<T>(o, y);
          const float sign = l < LANES / 2 ? -1.f : 1.f;
          const int first = (l * 8) % HALF;
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = x[j] * s_cos[row][first + j] + sign * y[j] * s_sin[row][first + j];
          raw[k] = pack8<T>(x);
          if (at[k] != nullptr) *reinterpret_cast<uint4*>(at[k]) = raw[k];
        }
      }
      if (R == 4 ? h < p.q_heads : unit * 4 + 3 < p.q_heads) continue;  // (the whole warp: nothing but queries)
      uint32_t word[1];
      __nv_bfloat16 s16, z16;
      quant_kv_group<T, 1, GROUP / 8>({raw[k]}, word, s16, z16);
      const bool value = h >= turned;
      const int s = __shfl_sync(0xffffffffu, slots, row);
      uint8_t* const block = s >= 0 && h >= p.q_heads && h < heads ? block_of(s, value ? h - turned : h - p.q_heads) : nullptr;
      quant_kv_write<D, GROUP>(block, s & 15, l, value, R == 4 && value && quad ? s_codes[warp] + i * LANES : nullptr, word[0], s16, z16);
    }
    if (R == 4 && quad && unit >= turned) {
      quant_kv_write_quad<D, GROUP>(block_of(s0, unit - turned), s0 & 15, s_codes[warp]);
      __syncwarp();  // (the next head's codes)
    }
  }
}

// ------------------------------------------------------------------ rows back
struct QuantLoadParams {
  const uint8_t* pool;
  const int32_t* slot;
  void *k, *v;    // row r of both
  int64_t rows, units;  // (rows of a warp, head, keys or values) each
  int kv_heads, page_shift, max_pages, zeros;  // zeros: of rows without a slot, bit 0: in k, bit 1: in v (else they are left as they are)
  int* status;
};

// Rows of slots: a warp takes keys or values of a head, of 8 rows (16 of 64 dimensions), as the store does; a lane has four words of a row's codes,
// spread so that the lanes of a row write next to each other.  Values of four tokens of a word come 16 bytes a lane and are put into rows
// through shared memory; others byte by byte.  Measured, 8 heads of 128: 8192 rows 9.4 us (44 MB, 4.7 TB/s, most of them written), 256 rows
// in pages of their own 2.85 us, one row 2.0 us.
template <typename T, int D, int GROUP>
__global__ void __launch_bounds__(128) quant_kv_load_kernel(const QuantLoadParams p) {
  constexpr QuantKv F = quant_kv(D, GROUP);
  constexpr int LANES = D / 32, ROWS = 32 / LANES, PITCH = D / 8 + 4, G = F.groups, EACH = D / 8;
  __shared__ __align__(16) uint32_t s_codes[4][ROWS * PITCH], s_words[4][ROWS / 4 * (D / 2)];
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % LANES, row = lane / LANES;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + warp;
  if (unit >= p.units) return;
  const bool value = unit & 1;
  const int head = static_cast<int>((unit >> 1) % p.kv_heads);
  const int64_t t0 = (unit >> 1) / p.kv_heads * ROWS;
  uint32_t *const codes = s_codes[warp], *const words = s_words[warp];
  int slots = lane < ROWS && t0 + lane < p.rows ? p.slot[t0 + lane] : -1;
  if (slots >= 0 && slots >> p.page_shift >= p.max_pages) {
    if (p.status) atomicCAS(p.status, 0, kStatusBadIndex);
    slots = -1;
  }
  const int s0 = __shfl_sync(0xffffffffu, slots, lane & 28);  // of four rows, the first one's
  const uint32_t quads = __ballot_sync(0xffffffffu, s0 >= 0 && (s0 & 3) == 0 && slots == s0 + (lane & 3));
  auto is_quad = [&](int r) { return ((quads >> (r & 28)) & 15u) == 15u; };
  const int s = __shfl_sync(0xffffffffu, slots, row), tok = s & 15;
  auto block_of = [&](int s) {
    const int page = s >> p.page_shift;
    return p.pool + (((static_cast<int64_t>(page) * p.kv_heads + head) << (p.page_shift - 4)) + ((s - (page << p.page_shift)) >> 4)) * F.block + (value ? F.part : 0);
  };
  // a row's scales, then its offsets, two a word (one group: both in a word)
  uint32_t numbers[G];
  uint4 word = make_uint4(0, 0, 0, 0);
  if (s >= 0) {
    const uint8_t* block = block_of(s);
#pragma unroll
    for (int i = 0; i < G; ++i) numbers[i] = reinterpret_cast<const uint32_t*>(block + F.codes + tok * 4 * G)[i];
    if (!value) word = *reinterpret_cast<const uint4*>(block + tok * (D / 2) + l * 16);
  }
  uint32_t w[4] = {word.x, word.y, word.z, word.w};  // eight codes each, of dimensions dim(i) on
  auto dim = [&](int i) { return D == 128 ? 32 * i + 8 * l : 32 * (i & 1) + 16 * l + 8 * (i >> 1); };
  if (value) {
    // words (m / 4, g, of these four tokens, m % 4): 16 bytes are four tiles m of a g
    const int q = lane / EACH, mg = lane % EACH >> 3, g = lane & 7, from = __shfl_sync(0xffffffffu, s0, 4 * q);
    if (is_quad(4 * q)) {
      const uint4 v = *reinterpret_cast<const uint4*>(block_of(from) + mg * 512 + g * 64 + ((from & 15) >> 2) * 16);
      uint32_t* to = words + q * (D / 2) + mg * 32 + g;
      to[0] = v.x; to[8] = v.y; to[16] = v.z; to[24] = v.w;
    }
    __syncwarp();
    if (is_quad(row)) {
      // byte b of the words of a tile is this token's, nibbles dimensions 16 m + g and 16 m + 8 + g
      const int b = (row & 1) * 2 + ((row >> 1) & 1);
      const uint32_t pick = b | (b + 4) << 4;
      uint32_t row_words[4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t* at = words + (row >> 2) * (D / 2) + (2 * l + h) * 8;
        const uint4 x = *reinterpret_cast<const uint4*>(at), y = *reinterpret_cast<const uint4*>(at + 4);
        const uint32_t even = __byte_perm(__byte_perm(x.x, x.z, pick), __byte_perm(y.x, y.z, pick), 0x5410);
        const uint32_t odd = __byte_perm(__byte_perm(x.y, x.w, pick), __byte_perm(y.y, y.w, pick), 0x5410);
        row_words[2 * h] = (even & 0x0f0f0f0fu) | ((odd << 4) & 0xf0f0f0f0u);
        row_words[2 * h + 1] = ((even >> 4) & 0x0f0f0f0fu) | (odd & 0xf0f0f0f0u);
      }
      *reinterpret_cast<uint4*>(codes + row * PITCH + 4 * l) = make_uint4(row_words[0], row_words[1], row_words[2], row_words[3]);
    }
    if (!__all_sync(0xffffffffu, is_quad(row) || s < 0)) {
      const int m = lane % EACH >> 1, half = lane & 1;  // a tile, g = 0 .. 3 or 4 .. 7 of it
      constexpr int TIMES = ROWS * EACH / 32;
      uint32_t all[TIMES];
#pragma unroll
      for (int i = 0; i < TIMES; ++i) {  // (asked for together)
        const int r = i * (32 / EACH) + lane / EACH, at = __shfl_sync(0xffffffffu, slots, r);
        const uint8_t* d = block_of(max(at, 0)) + quant_kv_value_byte(max(at, 0) & 15, m * 16) + half * 256;
        all[i] = at < 0 || is_quad(r) ? 0u : d[0] | d[64] << 8 | d[128] << 16 | static_cast<uint32_t>(d[192]) << 24;
      }
#pragma unroll
      for (int i = 0; i < TIMES; ++i) {
        const int r = i * (32 / EACH) + lane / EACH;
        auto close = [](uint32_t x) { return static_cast<uint16_t>(((x | x >> 4) & 0xffu) | ((x >> 8 | x >> 12) & 0xff00u)); };  // four nibbles together
        uint16_t* to = reinterpret_cast<uint16_t*>(codes + r * PITCH + 2 * m) + half;
        if (!is_quad(r)) {
          to[0] = close(all[i] & 0x0f0f0f0fu);
          to[2] = close((all[i] >> 4) & 0x0f0f0f0fu);
        }
      }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = codes[row * PITCH + dim(i) / 8];
  }
  T* const to = reinterpret_cast<T*>(value ? p.v : p.k) + ((t0 + row) * p.kv_heads + head) * D;
  if (s < 0) {
    if (((p.zeros >> static_cast<int>(value)) & 1) && t0 + row < p.rows) {
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(to + dim(i)) = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  auto number = [&](int i) { return __uint_as_float(i & 1 ? numbers[i >> 1] & 0xffff0000u : numbers[i >> 1] << 16); };
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int group = (D == 128 ? 32 * i : 32 * (i & 1)) / GROUP;
    const float sc = number(group), z = number(G + group);
    uint64_t c[4];
    float x[8];
    quant_kv_codes(w[i], c);
    quant_kv_numbers(c, sc, z, x);
    constexpr float most = quant_kv_most<T>();
    if (quant_kv_past(sc, z, most)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = quant_kv_cut(x[j], most);
    }
    stf8<T>(to + dim(i), x);
  }
}

// ------------------------------------------------------------------ pages back
struct QuantPagesParams {
  const uint8_t* pool;
  const int32_t* pages;
  void *k, *v;       // page n's token `off` at row n * page_rows + off
  int64_t units;     // (page, 16 tokens of it, head) each
  int kv_heads, page_size, page_rows, max_pages;
  int* status;
  int pool_heads, head0;  // for attention of portions: heads of the pool, and the first of the kv_heads that are read
  // for attention of portions: records of the pass (see attn_prefill_paged.cu), whose page numbers count from `first` pages before the first one
  const int32_t* work;
  int entries, first, pages_read;
  float k_sign;       // what keys are multiplied by (a scale's sign, or zero)
  int32_t* table;     // numbers of the pages read back, for all of those that the records count
  uint4* spans;       // SCALED: [pages][kv_heads] what quant_kv_form takes, where a sequence's first page is; behind them whether some are held in bf16
  float2* forms;      // SCALED: [entries][kv_heads] powers of two taken out of keys and values (zeros: held in bf16)
};

// Tokens of page `n` (counted as the records do) that its sequence has, -1: no record has it; and the sequence's first page.  The whole warp asks.
struct QuantHeld {
  int tokens, start;
};
__device__ __forceinline__ QuantHeld quant_kv_held(const QuantPagesParams& p, int n) {
  QuantHeld held{-1, -1};
  for (int e = threadIdx.x & 31; e < p.entries; e += 32) {
    const int4 r = __ldg(reinterpret_cast<const int4*>(p.work + e * 8));
    if (r.z >= p.first && n >= r.z && n < r.z + r.w) {
      held.tokens = min(p.page_size, max(0, __ldg(p.work + e * 8 + 4) - (n - r.z) * p.page_size));
      held.start = r.z - p.first;
    }
  }
  return {__reduce_max_sync(0xffffffffu, held.tokens), __reduce_max_sync(0xffffffffu, held.start)};
}
// No magnitudes yet.
__global__ void __launch_bounds__(256) quant_kv_no_span_kernel(uint4* __restrict__ spans, int64_t n) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < n) spans[i] = make_uint4(0, 0, 0, 0);
}
// The largest and smallest magnitudes of the groups of a sequence's keys and values, by head (maxima: in whatever order).  A warp takes up to 64 tokens of
// a page and head, half of it looks at the scales of the keys of 16 tokens at a time, the other half at those of the values.
// Measured: 8192 tokens of 8 heads of 128 4.8 us, and 2 for the zeros before (latency: record, page, scales).
template <int D, int GROUP>
__global__ void __launch_bounds__(256) quant_kv_span_kernel(const QuantPagesParams p) {
  constexpr QuantKv F = quant_kv(D, GROUP);
  constexpr int G = F.groups, EACH = 4;
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int lane = threadIdx.x & 31, blocks = p.page_size >> 4, parts = (blocks + EACH - 1) / EACH;
  const int64_t units = p.units / blocks * parts;
  for (int64_t unit = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); unit < units; unit += static_cast<int64_t>(gridDim.x) * 8) {
    const int head = static_cast<int>(unit % p.kv_heads), b0 = static_cast<int>(unit / p.kv_heads % parts) * EACH;
    const int n = static_cast<int>(unit / p.kv_heads / parts), page = p.pages[n];
    const QuantHeld held = quant_kv_held(p, n + p.first);
    if (held.tokens <= b0 * 16 || page < 0 || page >= p.max_pages) continue;
    const uint8_t* block = p.pool + ((static_cast<int64_t>(page) * p.pool_heads + p.head0 + head) * blocks + b0) * F.block + (lane < 16 ? 0 : F.part) + F.codes + (lane & 15) * 4 * G;
    uint32_t w[EACH][G];
#pragma unroll
    for (int b = 0; b < EACH; ++b)
#pragma unroll
      for (int i = 0; i < G; ++i)  // (zeros: a group that does not count)
        w[b][i] = (b0 + b) * 16 + (lane & 15) < held.tokens ? reinterpret_cast<const uint32_t*>(block + b * F.block)[i] : 0u;
    auto number = [&](int b, int i) { return __uint_as_float(i & 1 ? w[b][i >> 1] & 0xffff0000u : w[b][i >> 1] << 16); };
    uint32_t most = 0, least = 0;
#pragma unroll
    for (int b = 0; b < EACH; ++b)
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const float s = number(b, i), z = number(b, G + i), m = fmaxf(fabsf(z), fabsf(fmaf(15.f, s, z)));
        if (m > 0.f) {  // (NaN: not counted)
          most = max(most, __float_as_uint(m));
          least = max(least, 0x7f800000u - __float_as_uint(m));
        }
      }
    const uint32_t both[4] = {__reduce_max_sync(0xffffffffu, lane < 16 ? most : 0u), __reduce_max_sync(0xffffffffu, lane < 16 ? least : 0u),
                              __reduce_max_sync(0xffffffffu, lane < 16 ? 0u : most), __reduce_max_sync(0xffffffffu, lane < 16 ? 0u : least)};
    const uint32_t mine = lane == 0 ? both[0] : lane == 1 ? both[1] : lane == 2 ? both[2] : both[3];
    if (lane < 4 && mine != 0) atomicMax(reinterpret_cast<uint32_t*>(p.spans + static_cast<int64_t>(held.start) * p.kv_heads + head) + lane, mine);
  }
}

// The codes of a warp's 16 tokens of a head, 8 x 8 blocks of (token, dimension) at a time as tensor-core fragments have them.
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// A warp takes 16 tokens of a head.  Keys: four lanes a token, 32 codes each.  Values: a lane has four tokens of eight dimensions 8 apart, which
// stmatrix turns into rows of a token.  Both go out from shared memory, whole rows at a time.
// Bound by the 16-bit rows that it writes (four times the codes): 1024 pages of 64 tokens of 8 heads of 128 62.6 us (352 MB, 5.6 TB/s), 37 pages of 4 heads
// of 64 2.9 us; for attention of portions 8192 tokens 13 us after their magnitudes are known.  Three blocks on an SM leave 80 registers a thread: heads of 128
// spill up to 96 bytes, beside 4 KB that a warp moves.
//
// For attention of portions (WORK) the tokens behind a sequence's end are zeros, whatever the cache has there, and a value that is no number is handed to
// those who see it by its token's key (products with values have a weight of zero for those who do not, which would not make it a number).  SCALED: keys and values of a bf16
// model go to fp16, divided by powers of two, or stay in bf16, as quant_kv_form says for their sequence and head.
template <typename T, int D, int GROUP, bool WORK, bool SCALED>
__global__ void __launch_bounds__(256, 3) quant_kv_pages_kernel(const QuantPagesParams p) {
  constexpr QuantKv F = quant_kv(D, GROUP);
  constexpr int W = D / 32, G = F.groups;
  // bytes from row to row in shared memory: pairs of rows in different halves of the banks (keys: 64 bytes of each a time), rows 4 banks on
  // (values: 16 bytes of eight a time)
  constexpr int KROW = D * 2 + 64, ROW = D * 2 + 16;
  __shared__ __align__(16) uint8_t s_rows[8][16 * KROW];
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  uint8_t* const rows = s_rows[warp];
  const int blocks = p.page_size >> 4;
  if (WORK && blockIdx.x == 0)
    for (int64_t i = threadIdx.x; i < static_cast<int64_t>(p.pages_read) + p.first; i += 256) p.table[i] = max(0, static_cast<int>(i) - p.first);
  if (SCALED)
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < static_cast<int64_t>(p.entries) * p.kv_heads; i += static_cast<int64_t>(gridDim.x) * 256) {
      const int e = static_cast<int>(i / p.kv_heads), start = min(max(__ldg(p.work + e * 8 + 2) - p.first, 0), p.pages_read - 1);
      const QuantForm form = quant_kv_form(__ldcg(p.spans + static_cast<int64_t>(start) * p.kv_heads + i % p.kv_heads));
      p.forms[i] = form.fp16 ? make_float2(1.f / form.k_down, 1.f / form.v_down) : make_float2(0.f, 0.f);
      if (!form.fp16) p.spans[static_cast<int64_t>(p.pages_read) * p.kv_heads].x = 1;
    }
  for (int64_t unit = static_cast<int64_t>(blockIdx.x) * 8 + warp; unit < p.units; unit += static_cast<int64_t>(gridDim.x) * 8) {
    const int head = static_cast<int>(unit % p.kv_heads), b = static_cast<int>(unit / p.kv_heads % blocks);
    const int64_t n = unit / p.kv_heads / blocks;
    const int page = p.pages[n];
    const bool bad = page < 0 || page >= p.max_pages;  // (the first page is read instead, and nothing written)
    const uint8_t* block = p.pool + ((static_cast<int64_t>(bad ? 0 : page) * (WORK ? p.pool_heads : p.kv_heads) + (WORK ? p.head0 : 0) + head) * blocks + b) * F.block;
    const int64_t row0 = n * p.page_rows + b * 16, pitch = static_cast<int64_t>(p.kv_heads) * D;
    // everything is asked for before anything is used
    uint32_t kw[2][W], vw[D / 16];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint8_t* at = block + (g + 8 * r) * (D / 2) + t4 * (D / 8);
      if (W == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(at);
        kw[r][0] = x.x; kw[r][1] = x.y; kw[r][2 % W] = x.z; kw[r][3 % W] = x.w;
      } else {
        const uint2 x = *reinterpret_cast<const uint2*>(at);
        kw[r][0] = x.x; kw[r][1] = x.y;
      }
    }
#pragma unroll
    for (int h = 0; h < D / 64; ++h) {
      const uint4 x = *reinterpret_cast<const uint4*>(block + F.part + h * 512 + lane * 16);
      vw[4 * h] = x.x; vw[4 * h + 1] = x.y; vw[4 * h + 2] = x.z; vw[4 * h + 3] = x.w;
    }
    // a token's scales and offsets, 2 G numbers of 16 bits
    uint32_t ks[2][G], vs[4][G];
    auto numbers = [&](const uint8_t* at, uint32_t (&to)[G]) {
      if (G == 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(at);
        to[0] = x.x; to[1 % G] = x.y; to[2 % G] = x.z; to[3 % G] = x.w;
      } else if (G == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(at);
        to[0] = x.x; to[1 % G] = x.y;
      } else {
        to[0] = *reinterpret_cast<const uint32_t*>(at);
      }
    };
    auto number = [](const uint32_t (&from)[G], int i) { return __uint_as_float(i & 1 ? from[i >> 1] & 0xffff0000u : from[i >> 1] << 16); };
#pragma unroll
    for (int r = 0; r < 2; ++r) numbers(block + F.codes + (g + 8 * r) * 4 * G, ks[r]);
#pragma unroll
    for (int j = 0; j < 4; ++j) numbers(block + F.part + F.codes + (4 * t4 + j) * 4 * G, vs[j]);
    int held = p.page_size;
    QuantForm form{true, 1.f, 1.f};
    if (WORK) {
      const QuantHeld h = quant_kv_held(p, static_cast<int>(n) + p.first);
      if (h.tokens < 0) continue;  // (no record has the page)
      held = h.tokens;
      if (SCALED) form = quant_kv_form(__ldcg(p.spans + static_cast<int64_t>(h.start) * p.kv_heads + head));
    }
    held -= b * 16;            // of these 16 tokens
    if (bad) {
      if (p.status && lane == 0) atomicCAS(p.status, 0, kStatusBadIndex);
      continue;
    }
    constexpr float most = SCALED ? quant_kv_most<__nv_bfloat16>() : quant_kv_most<T>();
    bool past = false;
    if (!SCALED || !form.fp16)
#pragma unroll
    for (int i = 0; i < G; ++i) {
#pragma unroll
      for (int r = 0; r < 2; ++r) past |= quant_kv_past(number(ks[r], i), number(ks[r], G + i), most);
#pragma unroll
      for (int j = 0; j < 4; ++j) past |= quant_kv_past(number(vs[j], i), number(vs[j], G + i), most);
    }
    // (WORK: tokens with a value that is no number)
    auto no_number = [&](const uint32_t (&w)[G], int i) { return !(fabsf(number(w, G + i)) < INFINITY); };
    uint32_t none = 0;
    if (WORK) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < G; ++i) none |= no_number(vs[j], i) ? 1u << (4 * t4 + j) : 0u;
      none = __reduce_or_sync(0xffffffffu, none);
    }
    auto two = [&](float a, float b) { return !SCALED || form.fp16 ? pk2<T>(a, b) : pk2<__nv_bfloat16>(a, b); };
    auto out = [&](void* to, int row_bytes) {
      T* const d = reinterpret_cast<T*>(to) + row0 * pitch + static_cast<int64_t>(head) * D;
      __syncwarp();
#pragma unroll
      for (int i = lane; i < 16 * D / 8; i += 32)
        *reinterpret_cast<uint4*>(d + (i / (D / 8)) * pitch + (i % (D / 8)) * 8) = *reinterpret_cast<const uint4*>(rows + (i / (D / 8)) * row_bytes + (i % (D / 8)) * 16);
      __syncwarp();
    };
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int w = 0; w < W; ++w) {
        float x[8];
        quant_kv_codes(kw[r][w], x);
        float sc = number(ks[r], w * 32 / GROUP), z = number(ks[r], G + w * 32 / GROUP);
        if (SCALED) sc *= form.k_down, z *= form.k_down;
        if (WORK) sc *= p.k_sign, z *= p.k_sign;
        if (WORK && ((none >> (g + 8 * r)) & 1u)) z = NAN;
        if (WORK && g + 8 * r >= held) sc = z = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = fmaf(sc, x[i], z);
        if (past) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = quant_kv_cut(x[i], most);
        }
        *reinterpret_cast<uint4*>(rows + (g + 8 * r) * KROW + (32 * w + 8 * t4) * 2) = make_uint4(two(x[0], x[1]), two(x[2], x[3]), two(x[4], x[5]), two(x[6], x[7]));
      }
    out(p.k, KROW);
#pragma unroll
    for (int m = 0; m < D / 16; ++m) {
      const int i = m * 16 / GROUP;
      // nibbles of a word: (token 0, dimension g), (0, g + 8), (2, g), (2, g + 8), and tokens 1 and 3 in the upper half
      float x[8];
      quant_kv_codes(vw[m], x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int tok = (j & 2) + (j >> 2);
        float sc = number(vs[tok], i), z = number(vs[tok], G + i);
        if (SCALED) sc *= form.v_down, z *= form.v_down;
        if (WORK && (4 * t4 + tok >= held || no_number(vs[tok], i))) sc = z = 0.f;
        x[j] = fmaf(sc, x[j], z);
      }
      if (past) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = quant_kv_cut(x[j], most);
      }
      // 8 x 8 blocks: dimensions 16 m + g by (tokens 4 t4, + 1), 16 m + 8 + g by the same, and both by (4 t4 + 2, + 3).  Lane i gives the address of
      // row i % 8 of block i / 8: its token (columns 2 t4, 2 t4 + 1 of a block are tokens 4 t4 (+ 2), + 1), eight dimensions.
      const int mat = lane >> 3, c = lane & 7, token = 4 * (c >> 1) + (c & 1) + (mat >> 1) * 2;
      stmatrix_x4_trans(ptx::smem_u32(rows + token * ROW + m * 32 + (mat & 1) * 16), two(x[0], x[4]), two(x[1], x[5]), two(x[2], x[6]), two(x[3], x[7]));
    }
    out(p.v, ROW);
  }
}

struct StoreLaunch {
  QuantStoreParams& p;
  cudaStream_t stream;
  template <typename T, int D, int GROUP>
  int operator()() const {
    constexpr int ROWS = 1024 / D;
    p.units = ((int64_t)p.tokens + ROWS - 1) / ROWS * p.kv_heads * 2;
    if (p.units > (int64_t)4 * 0x7fffffff) return -1;
    return (int)launch_pdl(quant_kv_store_kernel<T, D, GROUP>, dim3((unsigned)((p.units + 3) / 4)), dim3(128), 0, stream, p);
  }
};
struct LoadLaunch {
  QuantLoadParams& p;
  cudaStream_t stream;
  template <typename T, int D, int GROUP>
  int operator()() const {
    constexpr int ROWS = 1024 / D;
    p.units = (p.rows + ROWS - 1) / ROWS * p.kv_heads * 2;
    if (p.units > (int64_t)4 * 0x7fffffff) return -1;
    return (int)launch_pdl(quant_kv_load_kernel<T, D, GROUP>, dim3((unsigned)((p.units + 3) / 4)), dim3(128), 0, stream, p);
  }
};
struct RopeLaunch {
  const QuantRopeParams& p;
  int static_meta;
  cudaStream_t stream;
  template <typename T, int D, int GROUP>
  int operator()() const {
    // (four tokens a block where there are three such blocks for every SM, us with one token -> four: 1400 rows 11.6 -> 13.8, 2300 16.2 -> 14.1)
    if (p.tokens >= 12 * device_sm_count())
      return (int)launch_pdl(static_meta ? quant_kv_rope_kernel<T, D, GROUP, 4, true> : quant_kv_rope_kernel<T, D, GROUP, 4, false>,
                             dim3((unsigned)((p.tokens + 3) / 4)), dim3(256), 0, stream, p);
    return (int)launch_pdl(static_meta ? quant_kv_rope_kernel<T, D, GROUP, 1, true> : quant_kv_rope_kernel<T, D, GROUP, 1, false>,
                           dim3((unsigned)p.tokens), dim3(256), 0, stream, p);
  }
};
struct PagesLaunch {
  const QuantPagesParams& p;
  cudaStream_t stream;
  template <typename T, int D, int GROUP>
  int operator()() const {
    const int64_t blocks = (p.units + 7) / 8, most = (int64_t)device_sm_count() * 16;
    return (int)launch_pdl(quant_kv_pages_kernel<T, D, GROUP, false, false>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, stream, p);
  }
};
struct PortionLaunch {
  const QuantPagesParams& p;
  cudaStream_t stream;
  template <typename T, int D, int GROUP>
  int operator()() const {
    const int64_t blocks = (p.units + 7) / 8, most = (int64_t)device_sm_count() * 16;
    const unsigned page_blocks = (unsigned)(blocks < most ? blocks : most);
    if (std::is_same<T, __half>::value)
      return (int)launch_pdl(quant_kv_pages_kernel<__half, D, GROUP, true, false>, dim3(page_blocks), dim3(256), 0, stream, p);
    const int64_t spans = p.units / (p.page_size >> 4);  // (page, head) each
    int rc = (int)launch_pdl(quant_kv_no_span_kernel, dim3((unsigned)(spans / 256 + 1)), dim3(256), 0, stream, p.spans, spans + 1);
    if (rc) return rc;
    const int64_t span_blocks = (spans * ((p.page_size + 63) / 64) + 7) / 8;
    rc = (int)launch_pdl(quant_kv_span_kernel<D, GROUP>, dim3((unsigned)(span_blocks < most ? span_blocks : most)), dim3(256), 0, stream, p);
    if (rc) return rc;
    return (int)launch_pdl(quant_kv_pages_kernel<__half, D, GROUP, true, true>, dim3(page_blocks), dim3(256), 0, stream, p);
  }
};

}  // namespace blitz

extern "C" {
using namespace blitz;

// k, v: [num_tokens] rows of kv_heads * dim elements, pitches k_row and v_row (multiples of 8, 16-byte aligned).  slot[t] = page *
// page_size + offset, negative: the row is not written.  The same slot twice: some of both rows' bytes.
int blitz_quant_kv_store(const void* k, int64_t k_row, const void* v, int64_t v_row, const int32_t* slot, void* pool, int num_tokens,
                         int kv_heads, int dim, int group, int page_size, int max_pages, int* status, int dtype, cudaStream_t stream) {
  if (num_tokens <= 0) return 0;
  if (!quant_kv_supported(dim, group, page_size) || max_pages < 1 || kv_heads < 1 || ((k_row | v_row) & 7)) return -1;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(pool)) & 15) return -1;
  QuantStoreParams p{k, v, k_row, v_row, slot, (uint8_t*)pool, 0, num_tokens, kv_heads, quant_kv_shift(page_size), max_pages, status};
  return quant_kv_dispatch(dtype, dim, group, StoreLaunch{p, stream});
}

// qkv: [num_tokens][(q_heads + 2 kv_heads) * dim]: queries and keys are rotated in place to position pos[t] (half-split pairs, base rope_theta),
// keys and values written as blitz_quant_kv_store does.  static_meta != 0 promises that pos and slot are not written by kernels still running
// in this stream.
int blitz_quant_kv_rope(void* qkv, const int32_t* pos, const int32_t* slot, void* pool, int num_tokens, int q_heads, int kv_heads, int dim, int group,
                        int page_size, int max_pages, float rope_theta, int static_meta, int* status, int dtype, cudaStream_t stream) {
  if (num_tokens <= 0) return 0;
  if (!quant_kv_supported(dim, group, page_size) || max_pages < 1 || kv_heads < 1 || q_heads < 0) return -1;
  if ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(pool)) & 15) return -1;
  QuantRopeParams p{qkv, pos, slot, (uint8_t*)pool, num_tokens, q_heads, kv_heads, quant_kv_shift(page_size), max_pages, log2f(rope_theta), status};
  return quant_kv_dispatch(dtype, dim, group, RopeLaunch{p, static_meta, stream});
}

// Row slot[r] to row r of k and v, in 16 bits (a negative slot, or one that there is not: row r is left as it is, or zeros, in k where bit 0 of `zeros` is
// set, in v bit 1).
int blitz_quant_kv_load(const void* pool, const int32_t* slot, int64_t rows, void* k, void* v, int kv_heads, int dim, int group, int page_size,
                        int max_pages, int zeros, int* status, int dtype, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (!quant_kv_supported(dim, group, page_size) || max_pages < 1 || kv_heads < 1) return -1;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(pool)) & 15) return -1;
  QuantLoadParams p{(const uint8_t*)pool, slot, k, v, rows, 0, kv_heads, quant_kv_shift(page_size), max_pages, zeros, status};
  return quant_kv_dispatch(dtype, dim, group, LoadLaunch{p, stream});
}

// Page pages[n], in 16 bits, to rows n * page_rows .. of k and v (each row kv_heads * dim).
int blitz_quant_kv_pages(const void* pool, const int32_t* pages, int64_t count, void* k, void* v, int kv_heads, int dim, int group, int page_size,
                         int page_rows, int max_pages, int* status, int dtype, cudaStream_t stream) {
  if (count <= 0) return 0;
  if (!quant_kv_supported(dim, group, page_size) || max_pages < 1 || kv_heads < 1 || page_rows < page_size) return -1;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(pool)) & 15) return -1;
  QuantPagesParams p{(const uint8_t*)pool, pages, k, v, count * kv_heads * (page_size / 16), kv_heads, page_size, page_rows, max_pages, status};
  return quant_kv_dispatch(dtype, dim, group, PagesLaunch{p, stream});
}

// Scratch of blitz_quant_kv_portion for `pages` pages and `first` more that the records count, in the order of its layout: keys and values read
// back [pages][2][page_size][kv_heads][dim] in 16 bits, page numbers; of a bf16 model also the spans of keys and values, and what the `entries` records
// find of them.  offsets (may be null): where the 4 parts begin, and the end.
int64_t blitz_quant_kv_portion_bytes(int64_t pages, int64_t first, int entries, int kv_heads, int dim, int page_size, int dtype, int64_t* offsets) {
  const int64_t sizes[4] = {pages * 4 * page_size * kv_heads * dim, (pages + first) * 4, dtype == 1 ? (pages * kv_heads + 1) * 16 : 0,
                            dtype == 1 ? (int64_t)entries * kv_heads * 8 : 0};
  int64_t at = 0;
  for (int i = 0; i < 4; ++i) {
    if (offsets) offsets[i] = at;
    at += (sizes[i] + 255) / 256 * 256;
  }
  if (offsets) offsets[4] = at;
  return at;
}

// What attention of portions (blitz_attn_prefill_paged, or blitz_attn_prefill_scaled for a bf16 model) reads instead of a 4-bit cache: pages[n], the
// (first + n)-th page that the records of `work` count, of its pool_heads heads those from head0 on, in 16 bits (of a bf16 model: as quant_kv_form says), zeros behind the end of its sequence.
// Keys are multiplied by k_sign: hidden scores are infinities that the attention kernel multiplies by its scale, which has to be positive, so the sign
// of one that is not, or zero, goes into the keys.
int blitz_quant_kv_portion(const void* pool, const int32_t* pages, int64_t count, int64_t first, const int32_t* work, int entries, int pool_heads,
                           int head0, int kv_heads, int dim, int group, int page_size, int max_pages, float k_sign, void* scratch, int* status, int dtype, cudaStream_t stream) {
  if (count <= 0 || entries <= 0) return 0;
  if (!quant_kv_supported(dim, group, page_size) || max_pages < 1 || kv_heads < 1 || head0 < 0 || head0 + kv_heads > pool_heads || first < 0 ||
      count + first > 0x7fffffff)
    return -1;
  if ((reinterpret_cast<uintptr_t>(work) | reinterpret_cast<uintptr_t>(pool) | reinterpret_cast<uintptr_t>(scratch)) & 15) return -1;
  int64_t at[5];
  blitz_quant_kv_portion_bytes(count, first, entries, kv_heads, dim, page_size, dtype, at);
  char* s = (char*)scratch;
  QuantPagesParams p{(const uint8_t*)pool, pages, s, s + (int64_t)page_size * kv_heads * dim * 2, count * kv_heads * (page_size / 16), kv_heads, page_size, 2 * page_size, max_pages, status, pool_heads, head0};
  p.work = work; p.entries = entries; p.first = (int)first; p.table = (int32_t*)(s + at[1]); p.spans = (uint4*)(s + at[2]);
  p.pages_read = (int)count; p.k_sign = k_sign; p.forms = (float2*)(s + at[3]);
  return quant_kv_dispatch(dtype, dim, group, PortionLaunch{p, stream});
}

}  // extern "C"
