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
// Byte of the values' codes that holds token t (of 16) of dimension d; the nibble is d / 8 % 2.
__host__ __device__ constexpr int quant_kv_value_byte(int t, int d) {
  return (d >> 6) * 512 + (d & 7) * 64 + (t >> 2) * 16 + ((d >> 4) & 3) * 4 + (t & 1) * 2 + ((t >> 1) & 1);
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

}  // namespace blitz
