// Writing rows of keys and values into a 4-bit cache, and reading them back in 16 bits (the format: quant_kv.cuh).
#include "launch.cuh"
#include "ptx.cuh"
#include "quant_kv.cuh"
#include "scalar.cuh"
#include "tmap.cuh"

namespace blitz {

// Eight numbers of a lane, whose group the lanes around it share: their codes, and the group's scale and offset.
template <typename T, int GROUP>
__device__ __forceinline__ void quant_kv_group(const uint4& u, uint32_t& word, __nv_bfloat16& s16, __nv_bfloat16& z16) {
  // the smallest number and the negative of the largest, as a pair (NaN where there is one)
  using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
  auto pair = [](uint32_t u) { return *reinterpret_cast<T2*>(&u); };
  auto bits = [](T2 v) { return *reinterpret_cast<uint32_t*>(&v); };
  uint32_t lo2 = bits(__hmin2_nan(__hmin2_nan(pair(u.x), pair(u.y)), __hmin2_nan(pair(u.z), pair(u.w))));
  uint32_t hi2 = bits(__hmax2_nan(__hmax2_nan(pair(u.x), pair(u.y)), __hmax2_nan(pair(u.z), pair(u.w)))) ^ 0x80008000u;
  uint32_t ends = bits(__hmin2_nan(pair(__byte_perm(lo2, hi2, 0x5410)), pair(__byte_perm(lo2, hi2, 0x7632))));
#pragma unroll
  for (int d = 1; d < GROUP / 8; d <<= 1) ends = bits(__hmin2_nan(pair(ends), pair(__shfl_xor_sync(0xffffffffu, ends, d))));
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
  word = 0;
  if (sc > 0.f) {
    float x[8];
    unpack8<T>(u, x);
    uint64_t c[4];
    if (sc >= 7.9e-31f) {
      float y = ptx::rcp_approx(sc);
      y = fmaf(fmaf(-sc, y, 1.f), y, y);
      const uint64_t y2 = ptx::f32x2(y, y), s2 = ptx::f32x2(-sc, -sc), z2 = ptx::f32x2(-z, -z);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint64_t d = ptx::add_f32x2(ptx::f32x2(x[i], x[i + 4]), z2), q = ptx::mul_f32x2(d, y2);
        c[i] = ptx::fma_f32x2(ptx::fma_f32x2(q, s2, d), y2, q);
        c[i] = ptx::add_f32x2(ptx::add_f32x2(c[i], ptx::f32x2(12582912.f, 12582912.f)), ptx::f32x2(-12582912.f, -12582912.f));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = ptx::f32x2(rintf(__fdiv_rn(x[i] - z, sc)), rintf(__fdiv_rn(x[i + 4] - z, sc)));
    }
    // four codes are a number of 16 bits
    const uint64_t sixteen = ptx::f32x2(16.f, 16.f);
    const float2 four = ptx::f32x2_get(ptx::add_f32x2(ptx::fma_f32x2(ptx::fma_f32x2(ptx::fma_f32x2(c[3], sixteen, c[2]), sixteen, c[1]), sixteen, c[0]), ptx::f32x2(8388608.f, 8388608.f)));
    word = __byte_perm(__float_as_uint(four.x), __float_as_uint(four.y), 0x5410);
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
// The words of four tokens, from token `tok` of a block on, whose codes the warp has put into `codes` [4][D / 8].
template <int D, int GROUP>
__device__ __forceinline__ void quant_kv_write_quad(uint8_t* block, int tok, const uint32_t* codes) {
  constexpr int LANES = D / 8;
  const QuantTile t;
  __syncwarp();
  if (t.m < D / 16) {
    // a word's bytes are tokens 0, 2, 1, 3, nibbles dimensions 16 m + g and 16 m + 8 + g; byte a of a row's word has g = 2 a and 2 a + 1
    uint2 w[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) w[b] = *reinterpret_cast<const uint2*>(codes + ((b & 1) * 2 + (b >> 1)) * LANES + 2 * t.m);
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
  int64_t units;  // (four rows, head) each
  int tokens, kv_heads, page_shift, max_pages;
  int* status;
};

// A warp takes four rows of one head, keys and values: D / 8 lanes a row, eight dimensions each; the lanes of a group find its smallest and
// largest number together.  (Bound by the chain of a warp, loads, shuffles, stores: slots, keys and values are asked for at once.)  Keys go out as they are, a word a lane.  A word of the values holds four tokens of two dimensions: where the four
// rows are the four tokens of a word (rows of a prompt) the lanes exchange their codes through shared memory and write words; else (the
// tokens of a batch) every row writes its bytes.
template <typename T, int D, int GROUP>
__global__ void __launch_bounds__(256) quant_kv_store_kernel(const QuantStoreParams p) {
  constexpr QuantKv F = quant_kv(D, GROUP);
  constexpr int LANES = D / 8, ROWS = 32 / LANES;  // rows a warp takes at a time
  __shared__ __align__(8) uint32_t s_codes[8][4 * LANES];
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int lane = threadIdx.x & 31, l = lane % LANES;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (unit >= p.units) return;
  const int head = static_cast<int>(unit % p.kv_heads);
  const int64_t t0 = unit / p.kv_heads * 4;
  uint32_t* const codes = s_codes[threadIdx.x >> 5];
  // the four slots: lane i has the i-th
  int slots = lane < 4 && t0 + lane < p.tokens ? p.slot[t0 + lane] : -1;
  uint4 raw[2][4 / ROWS];
#pragma unroll
  for (int r = 0; r < 4 / ROWS; ++r) {
    const int64_t t = t0 + r * ROWS + lane / LANES, at = static_cast<int64_t>(head) * D + l * 8;
    const bool real = t < p.tokens;
    raw[0][r] = real ? *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.k) + t * p.k_row + at) : make_uint4(0, 0, 0, 0);
    raw[1][r] = real ? *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.v) + t * p.v_row + at) : make_uint4(0, 0, 0, 0);
  }
  if (slots >= 0 && slots >> p.page_shift >= p.max_pages) {
    if (p.status) atomicCAS(p.status, 0, kStatusBadIndex);
    slots = -1;
  }
  const int s0 = __shfl_sync(0xffffffffu, slots, 0);
  const bool quad = s0 >= 0 && (s0 & 3) == 0 && __all_sync(0xffffffffu, lane >= 4 || slots == s0 + lane);
  auto block_of = [&](int s) {
    const int page = s >> p.page_shift;
    return p.pool + (((static_cast<int64_t>(page) * p.kv_heads + head) << (p.page_shift - 4)) + ((s - (page << p.page_shift)) >> 4)) * F.block;
  };
  auto rows = [&](auto plane) {
    constexpr bool value = decltype(plane)::value;
#pragma unroll
    for (int r = 0; r < 4 / ROWS; ++r) {
      const int s = __shfl_sync(0xffffffffu, slots, r * ROWS + lane / LANES);
      uint32_t word;
      __nv_bfloat16 s16, z16;
      quant_kv_group<T, GROUP>(raw[value][r], word, s16, z16);
      quant_kv_write<D, GROUP>(s >= 0 ? block_of(s) : nullptr, s & 15, l, value, value && quad ? codes + (r * ROWS + lane / LANES) * LANES : nullptr, word, s16, z16);
    }
    if (value && quad) quant_kv_write_quad<D, GROUP>(block_of(s0), s0 & 15, codes);
  };
  rows(std::false_type{});
  rows(std::true_type{});
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
template <typename T, int D, int GROUP, int R, bool STATIC>
__global__ void __launch_bounds__(256) quant_kv_rope_kernel(const QuantRopeParams p) {
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
  for (int unit = warp; unit < (R == 4 ? heads : (heads + 3) / 4); unit += 8) {
    uint4 raw[4 / ROWS];
    T* at[4 / ROWS];
#pragma unroll
    for (int k = 0; k < 4 / ROWS; ++k) {
      const int i = k * ROWS + lane / LANES, row = R == 4 ? i : 0, h = R == 4 ? unit : unit * 4 + i;
      const bool real = t0 + row < p.tokens && h < heads;
      at[k] = real ? reinterpret_cast<T*>(p.qkv) + static_cast<int64_t>(t0 + row) * pitch + static_cast<int64_t>(h) * D + l * 8 : nullptr;
      raw[k] = real ? *reinterpret_cast<const uint4*>(at[k]) : make_uint4(0, 0, 0, 0);
    }
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
      uint32_t word;
      __nv_bfloat16 s16, z16;
      quant_kv_group<T, GROUP>(raw[k], word, s16, z16);
      const bool value = h >= turned;
      const int s = __shfl_sync(0xffffffffu, slots, row);
      uint8_t* const block = s >= 0 && h >= p.q_heads && h < heads ? block_of(s, value ? h - turned : h - p.q_heads) : nullptr;
      quant_kv_write<D, GROUP>(block, s & 15, l, value, R == 4 && value && quad ? s_codes[warp] + i * LANES : nullptr, word, s16, z16);
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
  int64_t rows, units;  // (four rows, head) each
  int kv_heads, page_shift, max_pages;
  int* status;
};

// Rows of slots: a warp takes four of one head, as the store does.  Values of four tokens of a word come by words, through shared memory;
// others byte by byte.
template <typename T, int D, int GROUP>
__global__ void __launch_bounds__(256) quant_kv_load_kernel(const QuantLoadParams p) {
  constexpr QuantKv F = quant_kv(D, GROUP);
  constexpr int LANES = D / 8, ROWS = 32 / LANES;
  __shared__ uint32_t s_codes[8][4 * LANES];
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int lane = threadIdx.x & 31, l = lane % LANES;
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (unit >= p.units) return;
  const int head = static_cast<int>(unit % p.kv_heads);
  const int64_t t0 = unit / p.kv_heads * 4;
  uint32_t* const codes = s_codes[threadIdx.x >> 5];
  int slots = lane < 4 && t0 + lane < p.rows ? p.slot[t0 + lane] : -1;
  if (slots >= 0 && slots >> p.page_shift >= p.max_pages) {
    if (p.status) atomicCAS(p.status, 0, kStatusBadIndex);
    slots = -1;
  }
  const int s0 = __shfl_sync(0xffffffffu, slots, 0);
  const bool quad = s0 >= 0 && (s0 & 3) == 0 && __all_sync(0xffffffffu, lane >= 4 || slots == s0 + lane);
  auto block_of = [&](int s) {
    const int page = s >> p.page_shift;
    return p.pool + (((static_cast<int64_t>(page) * p.kv_heads + head) << (p.page_shift - 4)) + ((s - (page << p.page_shift)) >> 4)) * F.block;
  };
  auto scales = [&](const uint8_t* part, int tok) { return reinterpret_cast<const __nv_bfloat16*>(part + F.codes) + tok * 2 * F.groups; };
  uint32_t word[4 / ROWS];
  __nv_bfloat16 ks[4 / ROWS], kz[4 / ROWS], vs[4 / ROWS], vz[4 / ROWS];
  uint32_t vw[4 / ROWS];  // of the values, unless they come by quads
  const QuantTile own;
#pragma unroll
  for (int r = 0; r < 4 / ROWS; ++r) {
    const int s = max(0, __shfl_sync(0xffffffffu, slots, r * ROWS + lane / LANES)), tok = s & 15, g = l / (GROUP / 8);
    const uint8_t* block = block_of(s);
    word[r] = reinterpret_cast<const uint32_t*>(block + tok * (D / 2))[(l & 3) * (D / 32) + (l >> 2)];
    ks[r] = scales(block, tok)[g];
    kz[r] = scales(block, tok)[F.groups + g];
    vs[r] = scales(block + F.part, tok)[g];
    vz[r] = scales(block + F.part, tok)[F.groups + g];
    vw[r] = 0;
    if (!quad) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        vw[r] |= ((static_cast<uint32_t>(block[F.part + quant_kv_value_byte(tok, (l >> 1) * 16 + i)]) >> (4 * (l & 1))) & 15u) << (4 * i);
    }
  }
  if (quad && own.m < D / 16) {
    const uint8_t* from = block_of(s0) + F.part + own.at(s0 & 15);
    const uint32_t tile[2] = {*reinterpret_cast<const uint32_t*>(from), *reinterpret_cast<const uint32_t*>(from + 64)};
    // byte own.a of a row's words of the tile, tokens 0, 2, 1, 3
    const uint32_t low = (tile[0] & 0x0f0f0f0fu) | ((tile[1] << 4) & 0xf0f0f0f0u), high = ((tile[0] >> 4) & 0x0f0f0f0fu) | (tile[1] & 0xf0f0f0f0u);
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      uint8_t* to = reinterpret_cast<uint8_t*>(codes + ((b & 1) * 2 + (b >> 1)) * LANES + 2 * own.m) + own.a;
      to[0] = static_cast<uint8_t>(low >> (8 * b));
      to[4] = static_cast<uint8_t>(high >> (8 * b));
    }
  }
  if (quad) __syncwarp();
#pragma unroll
  for (int r = 0; r < 4 / ROWS; ++r) {
    const int row = r * ROWS + lane / LANES;
    if (__shfl_sync(0xffffffffu, slots, row) < 0) continue;
    const int64_t at = ((t0 + row) * p.kv_heads + head) * D + l * 8;
    const float k_s = __bfloat162float(ks[r]), k_z = __bfloat162float(kz[r]), v_s = __bfloat162float(vs[r]), v_z = __bfloat162float(vz[r]);
    float x[8], y[8];
    uint64_t c[4];
    quant_kv_codes(word[r], c);
    quant_kv_numbers(c, k_s, k_z, x);
    quant_kv_codes(quad ? codes[row * LANES + l] : vw[r], c);
    quant_kv_numbers(c, v_s, v_z, y);
    constexpr float most = quant_kv_most<T>();
    if (quant_kv_past(k_s, k_z, most) || quant_kv_past(v_s, v_z, most)) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] = quant_kv_cut(x[i], most);
        y[i] = quant_kv_cut(y[i], most);
      }
    }
    stf8<T>(reinterpret_cast<T*>(p.k) + at, x);
    stf8<T>(reinterpret_cast<T*>(p.v) + at, y);
  }
}

// ------------------------------------------------------------------ pages back
constexpr int kQuantSpanBlocks = 256;
struct QuantPagesParams {
  const uint8_t* pool;
  const int32_t* pages;
  void *k, *v;       // page n's token `off` at row n * page_rows + off
  int64_t units;     // (page, 16 tokens of it, head) each
  int kv_heads, page_size, page_rows, max_pages;
  int* status;
  // for attention of portions: records of the pass (see attn_prefill_paged.cu), whose page numbers count from `first` pages before the first one
  const int32_t* work;
  int entries, first;
  int32_t* table;     // numbers of the pages read back, for all of those that the records count
  const float* spans; // SCALED: [2][kv_heads][kQuantSpanBlocks] largest magnitudes, by block
  int span_blocks;
  float* up;          // SCALED: [2][kv_heads] powers of two that were taken out of keys and values
};

// Tokens of page `n` (counted as the records do) that its sequence has, -1: no record has it.  The whole warp asks.
__device__ __forceinline__ int quant_kv_held(const QuantPagesParams& p, int n) {
  int held = -1;
  for (int e = threadIdx.x & 31; e < p.entries; e += 32) {
    const int4 r = __ldg(reinterpret_cast<const int4*>(p.work + e * 8));
    if (n >= r.z && n < r.z + r.w) held = min(p.page_size, max(0, __ldg(p.work + e * 8 + 4) - (n - r.z) * p.page_size));
  }
  return __reduce_max_sync(0xffffffffu, held);
}
// The largest magnitudes of a pass's keys and values, by head: of every block, a part of them.  Half a warp looks at the scales of the
// keys of 16 tokens, the other half at those of the values.
template <int D, int GROUP>
__global__ void __launch_bounds__(256) quant_kv_span_kernel(const QuantPagesParams p, float* __restrict__ spans) {
  constexpr QuantKv F = quant_kv(D, GROUP);
  constexpr int G = F.groups;
  extern __shared__ int s_most[];  // [2][kv_heads] bits of numbers that are not negative
  for (int i = threadIdx.x; i < 2 * p.kv_heads; i += blockDim.x) s_most[i] = 0;
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  __syncthreads();
  const int lane = threadIdx.x & 31, blocks = p.page_size >> 4;
  for (int64_t unit = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5); unit < p.units; unit += static_cast<int64_t>(p.span_blocks) * 8) {
    const int head = static_cast<int>(unit % p.kv_heads), b = static_cast<int>(unit / p.kv_heads % blocks);
    const int n = static_cast<int>(unit / p.kv_heads / blocks), held = quant_kv_held(p, n + p.first), page = p.pages[n];
    if (held <= b * 16 || page < 0 || page >= p.max_pages) continue;
    const uint8_t* block = p.pool + ((static_cast<int64_t>(page) * p.kv_heads + head) * blocks + b) * F.block;
    const __nv_bfloat16* w = reinterpret_cast<const __nv_bfloat16*>(block + (lane < 16 ? 0 : F.part) + F.codes) + (lane & 15) * 2 * G;
    float most = 0.f;
    if (b * 16 + (lane & 15) < held) {
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const float s = __bfloat162float(w[i]), z = __bfloat162float(w[G + i]);
        most = fmaxf(most, fmaxf(fabsf(z), fabsf(fmaf(15.f, s, z))));  // (NaN: not counted)
      }
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
    if ((lane & 15) == 0) atomicMax(&s_most[(lane >> 4) * p.kv_heads + head], __float_as_int(most));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.kv_heads; i += blockDim.x) spans[i * kQuantSpanBlocks + blockIdx.x] = __int_as_float(s_most[i]);
}

// The codes of a warp's 16 tokens of a head, 8 x 8 blocks of (token, dimension) at a time as tensor-core fragments have them.
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// A warp takes 16 tokens of a head.  Keys: four lanes a token, 32 codes each.  Values: a lane has four tokens of eight dimensions 8 apart, which
// stmatrix turns into rows of a token.  Both go out from shared memory, whole rows at a time.
// Bound by the 16-bit rows that it writes (four times the codes).
//
// For attention of portions (WORK) the tokens behind a sequence's end are zeros, whatever the cache has there.  SCALED: keys and
// values of a bf16 model go to fp16, which keeps three bits more of what z + s c is, divided by a power of two near the largest of their head, so that
// the type's range does not matter.
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
    for (int64_t i = threadIdx.x; i < p.units / p.kv_heads / blocks + p.first; i += 256) p.table[i] = max(0, static_cast<int>(i) - p.first);
  __shared__ float s_down[SCALED ? 256 : 1];  // of keys, then of values, by head
  if (SCALED) {
    for (int i = warp; i < 2 * p.kv_heads; i += 8) {
      float most = 0.f;
#pragma unroll
      for (int c = 0; c < kQuantSpanBlocks; c += 32)
        if (c + lane < p.span_blocks) most = fmaxf(most, p.spans[i * kQuantSpanBlocks + c + lane]);
      const float down = quant_kv_down(warp_max(most));
      if (lane == 0) {
        s_down[i] = down;
        if (blockIdx.x == 0) p.up[i] = 1.f / down;
      }
    }
    __syncthreads();
  }
  for (int64_t unit = static_cast<int64_t>(blockIdx.x) * 8 + warp; unit < p.units; unit += static_cast<int64_t>(gridDim.x) * 8) {
    const int head = static_cast<int>(unit % p.kv_heads), b = static_cast<int>(unit / p.kv_heads % blocks);
    const int64_t n = unit / p.kv_heads / blocks;
    const int page = p.pages[n];
    const bool bad = page < 0 || page >= p.max_pages;  // (the first page is read instead, and nothing written)
    const float k_down = SCALED ? s_down[head] : 1.f, v_down = SCALED ? s_down[p.kv_heads + head] : 1.f;
    const uint8_t* block = p.pool + ((static_cast<int64_t>(bad ? 0 : page) * p.kv_heads + head) * blocks + b) * F.block;
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
    if (WORK) {
      held = quant_kv_held(p, static_cast<int>(n) + p.first);
      if (held < 0) continue;  // (no record has the page)
    }
    held -= b * 16;            // of these 16 tokens
    if (bad) {
      if (p.status && lane == 0) atomicCAS(p.status, 0, kStatusBadIndex);
      continue;
    }
    constexpr float most = quant_kv_most<T>();
    bool past = false;
    if (!SCALED)
#pragma unroll
    for (int i = 0; i < G; ++i) {
#pragma unroll
      for (int r = 0; r < 2; ++r) past |= quant_kv_past(number(ks[r], i), number(ks[r], G + i), most);
#pragma unroll
      for (int j = 0; j < 4; ++j) past |= quant_kv_past(number(vs[j], i), number(vs[j], G + i), most);
    }
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
        if (SCALED) sc *= k_down, z *= k_down;
        if (WORK && g + 8 * r >= held) sc = z = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = fmaf(sc, x[i], z);
        if (past) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = quant_kv_cut(x[i], most);
        }
        stf8<T>(reinterpret_cast<T*>(rows + (g + 8 * r) * KROW) + 32 * w + 8 * t4, x);
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
        if (SCALED) sc *= v_down, z *= v_down;
        if (WORK && 4 * t4 + tok >= held) sc = z = 0.f;
        x[j] = fmaf(sc, x[j], z);
      }
      if (past) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = quant_kv_cut(x[j], most);
      }
      // 8 x 8 blocks: dimensions 16 m + g by (tokens 4 t4, + 1), 16 m + 8 + g by the same, and both by (4 t4 + 2, + 3).  Lane i gives the address of
      // row i % 8 of block i / 8: its token (columns 2 t4, 2 t4 + 1 of a block are tokens 4 t4 (+ 2), + 1), eight dimensions.
      const int mat = lane >> 3, c = lane & 7, token = 4 * (c >> 1) + (c & 1) + (mat >> 1) * 2;
      stmatrix_x4_trans(ptx::smem_u32(rows + token * ROW + m * 32 + (mat & 1) * 16), pk2<T>(x[0], x[4]), pk2<T>(x[1], x[5]), pk2<T>(x[2], x[6]), pk2<T>(x[3], x[7]));
    }
    out(p.v, ROW);
  }
}

struct StoreLaunch {
  const QuantStoreParams& p;
  cudaStream_t stream;
  template <typename T, int D, int GROUP>
  int operator()() const {
    return (int)launch_pdl(quant_kv_store_kernel<T, D, GROUP>, dim3((unsigned)((p.units + 7) / 8)), dim3(256), 0, stream, p);
  }
};
struct LoadLaunch {
  const QuantLoadParams& p;
  cudaStream_t stream;
  template <typename T, int D, int GROUP>
  int operator()() const {
    return (int)launch_pdl(quant_kv_load_kernel<T, D, GROUP>, dim3((unsigned)((p.units + 7) / 8)), dim3(256), 0, stream, p);
  }
};
struct RopeLaunch {
  const QuantRopeParams& p;
  int static_meta;
  cudaStream_t stream;
  template <typename T, int D, int GROUP>
  int operator()() const {
    // (four tokens a block from four blocks on every SM on)
    if (p.tokens >= 16 * device_sm_count())
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
  QuantPagesParams& p;
  float* spans;
  cudaStream_t stream;
  template <typename T, int D, int GROUP>
  int operator()() const {
    const int64_t blocks = (p.units + 7) / 8, most = (int64_t)device_sm_count() * 16;
    const unsigned page_blocks = (unsigned)(blocks < most ? blocks : most);
    if (std::is_same<T, __half>::value)
      return (int)launch_pdl(quant_kv_pages_kernel<__half, D, GROUP, true, false>, dim3(page_blocks), dim3(256), 0, stream, p);
    p.spans = spans;
    p.span_blocks = (int)(blocks < kQuantSpanBlocks ? blocks : kQuantSpanBlocks);
    const int rc = (int)launch_pdl(quant_kv_span_kernel<D, GROUP>, dim3((unsigned)p.span_blocks), dim3(256), (size_t)2 * p.kv_heads * 4, stream, p, spans);
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
  if (!quant_kv_supported(dim, group, page_size) || kv_heads < 1 || ((k_row | v_row) & 7)) return -1;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(pool)) & 15) return -1;
  QuantStoreParams p{k, v, k_row, v_row, slot, (uint8_t*)pool, ((int64_t)num_tokens + 3) / 4 * kv_heads, num_tokens, kv_heads, quant_kv_shift(page_size), max_pages, status};
  if (p.units > (int64_t)8 * 0x7fffffff) return -1;
  return quant_kv_dispatch(dtype, dim, group, StoreLaunch{p, stream});
}

// qkv: [num_tokens][(q_heads + 2 kv_heads) * dim]: queries and keys are rotated in place to position pos[t] (half-split pairs, base rope_theta),
// keys and values written as blitz_quant_kv_store does.  static_meta != 0 promises that pos and slot are not written by kernels still running
// in this stream.
int blitz_quant_kv_rope(void* qkv, const int32_t* pos, const int32_t* slot, void* pool, int num_tokens, int q_heads, int kv_heads, int dim, int group,
                        int page_size, int max_pages, float rope_theta, int static_meta, int* status, int dtype, cudaStream_t stream) {
  if (num_tokens <= 0) return 0;
  if (!quant_kv_supported(dim, group, page_size) || kv_heads < 1 || q_heads < 0) return -1;
  if ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(pool)) & 15) return -1;
  QuantRopeParams p{qkv, pos, slot, (uint8_t*)pool, num_tokens, q_heads, kv_heads, quant_kv_shift(page_size), max_pages, log2f(rope_theta), status};
  return quant_kv_dispatch(dtype, dim, group, RopeLaunch{p, static_meta, stream});
}

// Row slot[r] to row r of k and v, in 16 bits (a negative slot: row r is left as it is).
int blitz_quant_kv_load(const void* pool, const int32_t* slot, int64_t rows, void* k, void* v, int kv_heads, int dim, int group, int page_size,
                        int max_pages, int* status, int dtype, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (!quant_kv_supported(dim, group, page_size) || kv_heads < 1) return -1;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(pool)) & 15) return -1;
  QuantLoadParams p{(const uint8_t*)pool, slot, k, v, rows, (rows + 3) / 4 * kv_heads, kv_heads, quant_kv_shift(page_size), max_pages, status};
  if (p.units > (int64_t)8 * 0x7fffffff) return -1;
  return quant_kv_dispatch(dtype, dim, group, LoadLaunch{p, stream});
}

// Page pages[n], in 16 bits, to rows n * page_rows .. of k and v (each row kv_heads * dim).
int blitz_quant_kv_pages(const void* pool, const int32_t* pages, int64_t count, void* k, void* v, int kv_heads, int dim, int group, int page_size,
                         int page_rows, int max_pages, int* status, int dtype, cudaStream_t stream) {
  if (count <= 0) return 0;
  if (!quant_kv_supported(dim, group, page_size) || kv_heads < 1 || page_rows < page_size) return -1;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(pool)) & 15) return -1;
  QuantPagesParams p{(const uint8_t*)pool, pages, k, v, count * kv_heads * (page_size / 16), kv_heads, page_size, page_rows, max_pages, status};
  return quant_kv_dispatch(dtype, dim, group, PagesLaunch{p, stream});
}

// Scratch of blitz_quant_kv_portion for `pages` pages and `first` more that the records count, in the order of its layout: keys and values read
// back [pages][2][page_size][kv_heads][dim] in 16 bits, page numbers; of a bf16 model also the powers of two of keys and values, and the parts of
// their largest magnitudes.  offsets (may be null): where the 4 parts begin, and the end.
int64_t blitz_quant_kv_portion_bytes(int64_t pages, int64_t first, int kv_heads, int dim, int page_size, int dtype, int64_t* offsets) {
  const int64_t h = dtype == 1 ? 2 * (int64_t)kv_heads : 0;
  const int64_t sizes[4] = {pages * 4 * page_size * kv_heads * dim, (pages + first) * 4, h * 4, h * 4 * kQuantSpanBlocks};
  int64_t at = 0;
  for (int i = 0; i < 4; ++i) {
    if (offsets) offsets[i] = at;
    at += (sizes[i] + 255) / 256 * 256;
  }
  if (offsets) offsets[4] = at;
  return at;
}

// What attention of portions (blitz_attn_prefill_paged, or blitz_attn_prefill_scaled for a bf16 model) reads instead of a 4-bit cache: pages[n], the
// (first + n)-th page that the records of `work` count, in 16 bits (of a bf16 model: fp16), zeros behind the end of its sequence.
int blitz_quant_kv_portion(const void* pool, const int32_t* pages, int64_t count, int64_t first, const int32_t* work, int entries, int kv_heads, int dim,
                           int group, int page_size, int max_pages, void* scratch, int* status, int dtype, cudaStream_t stream) {
  if (count <= 0 || entries <= 0) return 0;
  if (!quant_kv_supported(dim, group, page_size) || kv_heads < 1 || kv_heads > 128 || first < 0 || count + first > 0x7fffffff) return -1;
  if ((reinterpret_cast<uintptr_t>(work) | reinterpret_cast<uintptr_t>(pool) | reinterpret_cast<uintptr_t>(scratch)) & 15) return -1;
  int64_t at[5];
  blitz_quant_kv_portion_bytes(count, first, kv_heads, dim, page_size, dtype, at);
  char* s = (char*)scratch;
  QuantPagesParams p{(const uint8_t*)pool, pages, s, s + (int64_t)page_size * kv_heads * dim * 2, count * kv_heads * (page_size / 16), kv_heads, page_size, 2 * page_size, max_pages, status};
  p.work = work; p.entries = entries; p.first = (int)first; p.table = (int32_t*)(s + at[1]); p.up = (float*)(s + at[2]);
  return quant_kv_dispatch(dtype, dim, group, PortionLaunch{p, (float*)(s + at[3]), stream});
}

}  // extern "C"
