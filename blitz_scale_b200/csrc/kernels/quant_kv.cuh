// Paged key/value cache held in 4 bits: the format, shared by the kernels that write, read back and attend to it.
//
// A layer's cache is bytes [page][kv_head][page_size / 16][block].  A block is 16 tokens of one head: codes of the keys, their scales,
// codes of the values, their scales, so that a run of a head's tokens within a page is one contiguous copy whatever the page size.  A
// group of `group` dimensions has a scale s and an offset z in bf16, and a dimension is z + s c with a code c of 4 bits:
//
//   z = min x rounded down to bf16,  s = (max x - z) / 15 rounded up,  c = rint((x - z) / s), ties to even, in 0 .. 15 (s = 0: 0)
//
// in fp32 (z below and s above what they stand for: no number of the group leaves 0 .. 15 by more than fp32's rounding).  A group with an
// infinity or NaN, or wider than fp32, has z = NaN and s = c = 0: it reads back as NaN, and what does not see it stays clean.
//
// Keys: token after token, dim / 2 bytes.  32-bit word l W + w of them (W = dim / 32, l < 4) holds dimensions 32 w + 8 l .. + 7, low
// nibbles first: lane l of the four lanes that share a key in a tensor-core fragment loads its whole part of it at once, and the word
// w of every lane together is one group of 32 dimensions.
// Values: the fragment's pairs are neighbouring tokens of a dimension, so that a word holds 4 tokens (4 a .. 4 a + 3, in bytes 0, 2, 1,
// 3: masked nibbles are pairs of neighbours in the halves of a register) of dimensions 16 m + g (low nibbles) and 16 m + 8 + g.  The
// words are in the order [m / 4][g][a][m % 4], as the lanes of a warp load them, 16 bytes each (dim 64: one m / 4).
// Scales: per token the groups' s, then their z.
#pragma once
#include "common.cuh"
#include "ptx.cuh"

namespace blitz {

struct QuantKv {
  int codes, groups, part, block;  // bytes of 16 tokens' codes; groups of a head; bytes of keys or values in a block; of a block
};
__host__ __device__ constexpr QuantKv quant_kv(int dim, int group) {
  return {8 * dim, dim / group, 8 * dim + 64 * (dim / group), 2 * (8 * dim + 64 * (dim / group))};
}
inline bool quant_kv_supported(int dim, int group, int page_size) {
  return (dim == 64 || dim == 128) && (group == 32 || group == 64 || group == 128) && group <= dim && page_size >= 16 &&
         page_size <= (1 << 20) && (page_size & (page_size - 1)) == 0;
}
inline int quant_kv_shift(int page_size) {
  int n = 0;
  while ((1 << n) < page_size) ++n;
  return n;
}
// Byte of the values' codes that holds token t (of 16) of dimension d; the nibble is d / 8 % 2.
__host__ __device__ constexpr int quant_kv_value_byte(int t, int d) {
  return (d >> 6) * 512 + (d & 7) * 64 + (t >> 2) * 16 + ((d >> 4) & 3) * 4 + (t & 1) * 2 + ((t >> 1) & 1);
}

// (x & MASK) | BITS
template <uint32_t MASK, uint32_t BITS>
__device__ __forceinline__ uint32_t quant_kv_pick(uint32_t x) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(MASK), "r"(BITS));
  return y;
}
// The eight codes of a word, low nibbles first, as numbers: a nibble within the mantissa of a power of two that makes its lowest bit one.
__device__ __forceinline__ void quant_kv_codes(uint32_t w, float (&c)[8]) {
  const uint32_t v = w >> 12;  // nibbles 5 .. 7 where 2 .. 4 are
  c[0] = __uint_as_float(quant_kv_pick<0x0000fu, 0x4b000000u>(w)) - 8388608.f;
  c[1] = __uint_as_float(quant_kv_pick<0x000f0u, 0x49000000u>(w)) - 524288.f;
  c[2] = __uint_as_float(quant_kv_pick<0x00f00u, 0x47000000u>(w)) - 32768.f;
  c[3] = __uint_as_float(quant_kv_pick<0x0f000u, 0x45000000u>(w)) - 2048.f;
  c[4] = __uint_as_float(quant_kv_pick<0xf0000u, 0x43000000u>(w)) - 128.f;
  c[5] = __uint_as_float(quant_kv_pick<0x00f00u, 0x47000000u>(v)) - 32768.f;
  c[6] = __uint_as_float(quant_kv_pick<0x0f000u, 0x45000000u>(v)) - 2048.f;
  c[7] = __uint_as_float(quant_kv_pick<0xf0000u, 0x43000000u>(v)) - 128.f;
}
// The same, two an instruction (pairs of registers: where there is room for them).
__device__ __forceinline__ void quant_kv_codes(uint32_t w, uint64_t (&c)[4]) {
  const uint32_t v = w >> 12;
  auto two = [](uint32_t a, uint32_t b, float za, float zb) { return ptx::add_f32x2(ptx::f32x2(__uint_as_float(a), __uint_as_float(b)), ptx::f32x2(za, zb)); };
  c[0] = two(quant_kv_pick<0x0000fu, 0x4b000000u>(w), quant_kv_pick<0x000f0u, 0x49000000u>(w), -8388608.f, -524288.f);
  c[1] = two(quant_kv_pick<0x00f00u, 0x47000000u>(w), quant_kv_pick<0x0f000u, 0x45000000u>(w), -32768.f, -2048.f);
  c[2] = two(quant_kv_pick<0xf0000u, 0x43000000u>(w), quant_kv_pick<0x00f00u, 0x47000000u>(v), -128.f, -32768.f);
  c[3] = two(quant_kv_pick<0x0f000u, 0x45000000u>(v), quant_kv_pick<0xf0000u, 0x43000000u>(v), -2048.f, -128.f);
}
// s c + z
__device__ __forceinline__ void quant_kv_numbers(const uint64_t (&c)[4], float s, float z, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = ptx::f32x2_get(ptx::fma_f32x2(c[i], ptx::f32x2(s, s), ptx::f32x2(z, z)));
    x[2 * i] = v.x;
    x[2 * i + 1] = v.y;
  }
}
// The largest finite number of a type.  A scale that was rounded up can carry the largest number of a group past it: such groups are cut.
template <typename T>
__device__ __forceinline__ constexpr float quant_kv_most() { return std::is_same<T, __half>::value ? 65504.f : 3.3895313892515355e38f; }
__device__ __forceinline__ bool quant_kv_past(float s, float z, float most) { return fmaxf(fabsf(z), fabsf(fmaf(15.f, s, z))) > most; }
__device__ __forceinline__ float quant_kv_cut(float x, float most) { return fabsf(x) > most ? copysignf(most, x) : x; }
// Two weighted means of such numbers, rounded to T (a in the lower half): no number that was quantised is past the type's largest finite one, so no mean is.
template <typename T>
__device__ __forceinline__ uint32_t quant_kv_means(float a, float b) {
  uint32_t d;
  if (std::is_same<T, __half>::value) asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
  else asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
  return d;
}

// Calls f with the element type and the sizes as types and constants.
template <typename F>
static inline int quant_kv_dispatch(int dtype, int dim, int group, F&& f) {
  auto sizes = [&](auto type) {
    using T = decltype(type);
    if (dim == 128) return group == 32 ? f.template operator()<T, 128, 32>() : group == 64 ? f.template operator()<T, 128, 64>() : f.template operator()<T, 128, 128>();
    return group == 32 ? f.template operator()<T, 64, 32>() : f.template operator()<T, 64, 64>();
  };
  return dtype == 1 ? sizes(__nv_bfloat16{}) : sizes(__half{});
}

// 2^-e, 2^e <= x < 2^(e + 1): what brings numbers up to x to below 2
__device__ __forceinline__ float quant_kv_down(float x) {
  const int e = x > 0.f && x <= 3.4e38f ? max(-100, min(126, static_cast<int>(__float_as_uint(x) >> 23) - 127)) : 0;
  return __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
}

// How a pass reads back the keys and values of a sequence and KV head of a bf16 model: in fp16, which keeps three bits more of what z + s c is,
// divided by powers of two near the largest; or in bf16, as a 16-bit cache has them, where fp16 would not hold eleven bits of every group's
// largest number (one is below 2^-14 of the largest of all), or the powers leave 2^-100 .. 2^100.  So neither another sequence nor a token that a row
// does not see, or gives no weight, costs it more than those three bits.
struct QuantForm {
  bool fp16;
  float k_down, v_down;
};
// span: bits of the largest magnitude of the keys' groups, bits of infinity less those of the smallest one that is not zero, the same of the
// values' (zeros: there is nothing but zeros and what is no number).
__device__ __forceinline__ QuantForm quant_kv_form(uint4 span) {
  auto held = [](uint32_t most, uint32_t least) {
    const float m = __uint_as_float(most);
    return most == 0 || (m <= 0x1p100f && m >= 0x1p-100f && __uint_as_float(0x7f800000u - least) >= m * 0x1p-14f);
  };
  if (!held(span.x, span.y) || !held(span.z, span.w)) return {false, 1.f, 1.f};
  return {true, quant_kv_down(__uint_as_float(span.x)), quant_kv_down(__uint_as_float(span.z))};
}

// A row of bf16 numbers in a tile that TMA wrote with a 128-byte swizzle, to fp16 where it stands, divided by a power of two near the largest,
// which it returns.  row: of the first slab of 64 columns, `slab` bytes from one to the next; x: which exclusive-or its 16-byte pieces are at (lanes
// that have rows next to each other then read different banks).
template <int SLABS>
__device__ __forceinline__ float quant_kv_row_fp16(uint8_t* row, int slab, int x) {
  __nv_bfloat162 most = __float2bfloat162_rn(0.f);
#pragma unroll
  for (int i = 0; i < SLABS * 8; ++i) {
    const uint4 v = *reinterpret_cast<const uint4*>(row + (i >> 3) * slab + (((i & 7) ^ x) << 4));
    const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&v);
    most = __hmax2(most, __hmax2(__hmax2(__habs2(e[0]), __habs2(e[1])), __hmax2(__habs2(e[2]), __habs2(e[3]))));
  }
  const float down = quant_kv_down(fmaxf(__low2float(most), __high2float(most)));
#pragma unroll
  for (int i = 0; i < SLABS * 8; ++i) {
    uint4* const at = reinterpret_cast<uint4*>(row + (i >> 3) * slab + (((i & 7) ^ x) << 4));
    const uint4 v = *at;
    auto both = [&](uint32_t w) { return pk2<__half>(__uint_as_float(w << 16) * down, __uint_as_float(w & 0xffff0000u) * down); };
    *at = make_uint4(both(v.x), both(v.y), both(v.z), both(v.w));
  }
  return 1.f / down;
}

}  // namespace blitz
