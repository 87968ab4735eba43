// Beam search over a paged cache: the best continuations of every request's beams, tables of the beams that go on, copies of
// what two of them cannot share, and the tables of a step from tables and lengths.
//
// The attention of such beams is in attn_beams.cu.
#include "launch.cuh"
#include "ptx.cuh"
#include "tmap.cuh"
#include "common.cuh"
#include "scalar.cuh"

namespace blitz {

constexpr int kBeamThreads = 256;
constexpr int kBeamMost = 64;  // beams of a request, and candidates of it

// ------------------------------------------------------------------ selection
// value(b, v) = score[b] + z[v] - log sum_u exp z[u], the n largest of a request's beams, ties to the lowest (b, v).
//
// The scan streams the logits once: a warp takes a stretch of a row, and leaves the sum of exponentials beside its largest logit, and the largest
// logit of every group of 512.  Nothing else is done beside the stream: a selection in it (bounds, lists and barriers for every 32 KB) took two to
// three times the stream's time.  The second kernel, a block per request, knows the sums, hence the values of the groups' largest; the n best elements are in
// the n best groups, which it reads again (1 KB each, out of L2 as a rule).  Values are pairs of fp32, 48 bits, so that a beam's candidates, and those of beams with equal
// logits, keep the order of their logits, which fp32 values would not tell apart.  The sums behind them are fp32: a score is off by 3e-8 as a rule and 5e-6 at
// most, and candidates of different rows that are nearer than that may come in either order.
//
// Measured, us in a graph (bytes once at the copy rate): 256 rows of 128256 logits in bf16, 8 beams, n = 24, 22.2 (10.0), of which the scan 15; 65 rows of 50257 in fp32
// 12.3 (2.0); one request of four beams 8.6 (0.2).  The scan is bound by its instructions, a fifth of them the exponentials, and the time until all warps have
// their first groups; the second kernel by a chain of some ten short rounds through shared memory.
constexpr int kSelGroup = 512;
constexpr int kSelWarps = 48;       // warps of an SM that the scan counts on
constexpr int kSelStretch = 32;     // groups of a stretch at most (sums of more lose digits)

// Numbers in the order of their bits (-0 as 0); minus infinity: 0.
__device__ __forceinline__ uint32_t sel_ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return x > -INFINITY ? (u ^ (u >> 31 ? 0xffffffffu : 0x80000000u)) : 0u;
}
__device__ __forceinline__ float sel_number(uint32_t o) { return o ? __uint_as_float(o ^ (o >> 31 ? 0x80000000u : 0xffffffffu)) : -INFINITY; }

template <typename T>
__device__ __forceinline__ void sel_unpack(const uint4& v, float (&f)[16 / sizeof(T)]) {
  if constexpr (sizeof(T) == 4) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  } else {
    unpack8<T>(v, f);
  }
}

// The largest of a piece.  (16-bit types: two at a time.)
template <typename T>
__device__ __forceinline__ float sel_max(const uint4& v) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  } else {
    using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
    auto two = [](uint32_t u) { return *reinterpret_cast<T2*>(&u); };
    const T2 a = __hmax2(__hmax2(two(v.x), two(v.y)), __hmax2(two(v.z), two(v.w)));
    const float2 f = cvt2<T>(*reinterpret_cast<const uint32_t*>(&a));
    return fmaxf(f.x, f.y);
  }
}

// A row in groups, which begin with its first element, wherever in memory that is: a row's sum does not depend on where it begins, so beams of equal logits and scores have equal
// values.  Copies go by pieces of 16 bytes on their boundaries; where the row begins behind one (by `lead` elements), a group has a piece more, and numbers are shifted as
// they are read (256 rows of 128257 logits in bf16 24.1 us where 128256 take 21.6; 65 rows of 50257 in fp32 12.3).
template <typename T>
struct SelRow {
  static constexpr int E = 16 / sizeof(T), NV = kSelGroup / (32 * E);      // elements of a piece, pieces of a group that a lane has
  static constexpr int kRing = sizeof(T) == 2 ? 4 : 3;                      // groups of a warp that wait in shared memory or are on their way
  static constexpr int kPieces = 32 * NV;                                   // pieces of a group, but for shifted ones' last
};
template <typename T>
__device__ __forceinline__ int sel_lead(const T* z) { return static_cast<int>((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T)); }
// Element `at` of a row and those behind it, a piece, into shared memory; outside the row: -inf.
template <typename T>
__device__ __forceinline__ void sel_piece(uint4* to, const T* z, int at, int vocab) {
  constexpr int E = 16 / sizeof(T);
  if (at >= 0 && at + E <= vocab) {
    ptx::cp_async_16(ptx::smem_u32(to), z + at, 16);
  } else {
#pragma unroll 1
    for (int e = 0; e < E; ++e) {
      if (at + e >= 0 && at + e < vocab) reinterpret_cast<T*>(to)[e] = z[at + e];
      else stf(reinterpret_cast<T*>(to) + e, -INFINITY);
    }
  }
}

// A piece's worth of numbers, from 32-bit word WORDS of piece a on (`half`: 16 bits behind it), the rest from b.
template <int WORDS>
__device__ __forceinline__ uint4 sel_shifted(const uint4& a, const uint4& b, int half) {
  const uint32_t w[9] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w, 0u};
  return make_uint4(__funnelshift_r(w[WORDS], w[WORDS + 1], half), __funnelshift_r(w[WORDS + 1], w[WORDS + 2], half), __funnelshift_r(w[WORDS + 2], w[WORDS + 3], half),
                    __funnelshift_r(w[WORDS + 3], w[WORDS + 4], half));
}

// The largest of a warp's numbers (those that are none apart).
__device__ __forceinline__ float sel_redux(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

struct SelPart {   // of a stretch: its largest logit m, the sum of exp(z - m)
  float m, s;
};

// A stretch is `length` groups of a row, `per_row` stretches and `groups` groups a row.  SHIFTED: some rows begin off the boundaries (a kernel apart, since
// the other one is 2 us of 23 faster without what these need).
template <typename T, bool SHIFTED>
__global__ void __launch_bounds__(kBeamThreads, sizeof(T) == 4 ? 4 : 6)
beam_scan_kernel(const T* __restrict__ logits, int64_t stride, int rows, int vocab, int groups, int per_row, int length, SelPart* __restrict__ parts,
                 float* __restrict__ largest) {
  constexpr int E = SelRow<T>::E, NV = SelRow<T>::NV, kRing = SelRow<T>::kRing;
  extern __shared__ __align__(16) uint4 sel_ring[];
  auto ring = reinterpret_cast<uint4 (*)[kRing][SelRow<T>::kPieces + SHIFTED]>(sel_ring);
  ptx::griddep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t self = static_cast<int64_t>(blockIdx.x) * (kBeamThreads / 32) + warp;
  if (self >= static_cast<int64_t>(rows) * per_row) return;
  const int row = static_cast<int>(self / per_row), g0 = static_cast<int>(self % per_row) * length, g1 = min(groups, g0 + length);
  const T* z = logits + row * stride;
  const int lead = SHIFTED ? sel_lead(z) : 0;
  int ahead = g0, put = 0;
  auto load = [&]() {
    if (ahead < g1) {
      const int first = ahead * kSelGroup - lead, at = first + lane * E;
      uint4* to = &ring[warp][put][lane];
      if (first >= 0 && first + kSelGroup + (SHIFTED ? E : 0) <= vocab) {
#pragma unroll
        for (int j = 0; j < NV; ++j) ptx::cp_async_16(ptx::smem_u32(to + j * 32), z + at + j * 32 * E, 16);
        if (SHIFTED && lane == 0) ptx::cp_async_16(ptx::smem_u32(to + NV * 32), z + at + kSelGroup, 16);
      } else {
#pragma unroll 1
        for (int j = 0; j < NV + SHIFTED; ++j)
          if (j < NV || lane == 0) sel_piece(to + j * 32, z, at + j * 32 * E, vocab);
      }
    }
    ptx::cp_async_commit();
    ++ahead;
    if (++put == kRing) put = 0;
  };
#pragma unroll 1
  for (int i = 0; i < kRing - 1; ++i) load();
  constexpr float kLog2e = 1.4426950408889634f;
  const uint64_t log2e = ptx::f32x2(kLog2e, kLog2e);
  float m = -INFINITY, sum = 0.f;       // (of the warp; of the lane)
  int get = 0;
#pragma unroll 1
  for (int g = g0; g < g1; ++g) {
    load();
    ptx::cp_async_wait<kRing - 1>();      // (a lane reads what it has copied itself, and where numbers are shifted what its neighbour has)
    uint4 cur[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) cur[j] = ring[warp][get][j * 32 + lane];
    if (SHIFTED && lead > 0) {
      __syncwarp();
      auto shift = [&](auto words) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
          cur[j] = sel_shifted<decltype(words)::value>(cur[j], ring[warp][get][j * 32 + lane + 1], sizeof(T) == 2 ? (lead & 1) * 16 : 0);
      };
      const int words = lead * static_cast<int>(sizeof(T)) / 4;
      if (words == 0) shift(std::integral_constant<int, 0>{});
      else if (words == 1) shift(std::integral_constant<int, 1>{});
      else if (words == 2) shift(std::integral_constant<int, 2>{});
      else shift(std::integral_constant<int, 3>{});
      __syncwarp();
    }
    if (++get == kRing) get = 0;
    float top = sel_max<T>(cur[0]);
#pragma unroll
    for (int j = 1; j < NV; ++j) top = fmaxf(top, sel_max<T>(cur[j]));
    top = sel_redux(top);
    if (lane == 0) largest[static_cast<int64_t>(row) * groups + g] = top;
    if (top > m) {
      sum *= ptx::ex2_approx((m - top) * kLog2e);
      m = top;
    }
    const float ref = m > -INFINITY ? -m : 0.f;      // (nothing but minus infinities: they add nothing, and a NaN stays one)
    const uint64_t back = ptx::f32x2(ref, ref);
    uint64_t part = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float f[E];
      sel_unpack<T>(cur[j], f);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 x = ptx::f32x2_get(ptx::mul_f32x2(ptx::add_f32x2(ptx::f32x2(f[e], f[e + 1]), back), log2e));
        part = ptx::add_f32x2(part, ptx::f32x2(ptx::ex2_approx(x.x), ptx::ex2_approx(x.y)));
      }
    }
    const float2 two = ptx::f32x2_get(part);
    sum += two.x + two.y;
  }
  // (not before: blocks of the next kernel that wait beside those of a scan took a quarter of its rate)
  ptx::griddep_launch_dependents();
  sum = warp_sum(sum);
  if (lane == 0) parts[self] = SelPart{m, sum};
}

struct SelOut {
  float* score;
  int32_t *parent, *token;
  int64_t pitch;      // from a request's to the next one's
};
// A value (two fp32 in the order of their bits, the larger first; 0: none), and behind it its place, the bits turned: of equal values the lowest place comes
// first.  Together one number of 128 bits, the larger the better.
struct SelCand {
  uint64_t v, early;
};
__device__ __forceinline__ SelCand sel_cand(uint64_t v, uint64_t place) { return SelCand{v, ~place}; }
// 1 if a comes before b.  (The borrow of b - a: a comparison with branches takes each lane by itself where values are equal, 250 cycles instead of 10.)
__device__ __forceinline__ uint32_t sel_before(const SelCand& a, const SelCand& b) {
  uint32_t less;
  asm("{\n\t.reg .u32 t;\n\t"
      "sub.cc.u32 t, %1, %5;\n\tsubc.cc.u32 t, %2, %6;\n\tsubc.cc.u32 t, %3, %7;\n\tsubc.cc.u32 t, %4, %8;\n\tsubc.u32 %0, 0, 0;\n\t}"
      : "=r"(less)
      : "r"(static_cast<uint32_t>(b.early)), "r"(static_cast<uint32_t>(b.early >> 32)), "r"(static_cast<uint32_t>(b.v)), "r"(static_cast<uint32_t>(b.v >> 32)),
        "r"(static_cast<uint32_t>(a.early)), "r"(static_cast<uint32_t>(a.early >> 32)), "r"(static_cast<uint32_t>(a.v)), "r"(static_cast<uint32_t>(a.v >> 32)));
  return -less;
}
__device__ __forceinline__ float sel_value(const SelCand& a) { return sel_number(static_cast<uint32_t>(a.v >> 32)); }
// a + b as the rounded sum and what the rounding left out
__device__ __forceinline__ float2 two_sum(float a, float b) {
  const float s = __fadd_rn(a, b), t = __fadd_rn(s, -a);
  return make_float2(s, __fadd_rn(__fadd_rn(a, -__fadd_rn(s, -t)), __fadd_rn(b, -t)));
}
// Of a row: its score, its largest logit, and the log of the sum of exp(z - largest) as hi + lo.  (Apart: a row that is masked by the type's lowest number everywhere
// has a largest logit in which the log of its sum disappears, in 64 bits too.)
struct SelNorm {
  float base, top, hi, lo;
};
// base + ((z - top) - log of the sum).  What is no number, or minus infinity, is no candidate.
__device__ __forceinline__ uint64_t sel_make(float z, const SelNorm& r) {
  const float2 d = two_sum(z, -r.top), e = two_sum(d.x, -r.hi), v = two_sum(e.x, r.base);
  const float rest = __fadd_rn(__fadd_rn(__fadd_rn(d.y, -r.lo), e.y), v.y), hi = __fadd_rn(v.x, rest), lo = __fadd_rn(rest, -__fadd_rn(hi, -v.x));
  const uint32_t o = sel_ordered(hi);
  return o ? static_cast<uint64_t>(o) << 32 | sel_ordered(lo) : 0ull;
}

constexpr int kSelRoom = 1024;       // candidates in shared memory
constexpr int kSelNear = 256;        // of them, those that are compared with one another
constexpr int kSelBounds = 128;      // numbers of which the n-th largest is a bound

struct SelShared {
  SelCand cand[kSelRoom], near[kSelNear], tops[kSelBounds], best[kBeamMost], bound;
  int found, close;
};

// A candidate that at least n are not behind: every thread has the best one of its own in `mine`, and of the best of pairs of threads it is the n-th.  (Threads
// without one have {0, thread}: each another one.)
__device__ __forceinline__ SelCand sel_bound(int n, SelCand mine, SelShared& sh) {
  const int tid = threadIdx.x;
  const SelCand other{__shfl_xor_sync(0xffffffffu, mine.v, 1), __shfl_xor_sync(0xffffffffu, mine.early, 1)};
  if (sel_before(other, mine)) mine = other;
  if ((tid & 1) == 0) sh.tops[tid >> 1] = mine;
  __syncthreads();
  int above = 0;
#pragma unroll 8
  for (int i = 0; i < kSelBounds / 2; ++i) above += sel_before(sh.tops[2 * i + (tid & 1)], mine);
  above += __shfl_xor_sync(0xffffffffu, above, 1);
  if (above == n - 1) sh.bound = mine;
  __syncthreads();
  return sh.bound;
}

// The n best of what `each` goes through, in order, into sh.best; `bound`: a candidate that at least n are not behind ({0, 0}: none known).  each(take) calls take(c) for
// all that may count, by all threads of the block.  Where there is no room for those that pass the bound, the n-th best of those that found room is the next bound.
template <typename Each>
__device__ __forceinline__ void sel_best(int n, SelCand bound, SelShared& sh, const Each& each) {
  const int tid = threadIdx.x;
  while (true) {
    if (tid == 0) sh.found = sh.close = 0;
    if (tid < n) sh.best[tid] = SelCand{0, 0};
    __syncthreads();
    each([&](const SelCand& c) {
      if (c.v && !sel_before(bound, c)) {
        const int at = atomicAdd(&sh.found, 1);
        if (at < kSelRoom) sh.cand[at] = c;
      }
    });
    __syncthreads();
    const int total = sh.found;
    const SelCand* list = sh.cand;
    int count = min(total, kSelRoom);
    if (count > kSelNear) {      // (few rows, small vocabularies: comparing a thousand with one another takes 20 us)
      SelCand mine{0, static_cast<uint64_t>(tid)};
      for (int i = tid; i < count; i += kBeamThreads)
        if (sel_before(sh.cand[i], mine)) mine = sh.cand[i];
      const SelCand least = sel_bound(n, mine, sh);
      for (int i = tid; i < count; i += kBeamThreads) {
        const SelCand c = sh.cand[i];
        if (!sel_before(least, c)) {
          const int at = atomicAdd(&sh.close, 1);
          if (at < kSelNear) sh.near[at] = c;
        }
      }
      __syncthreads();
      if (sh.close <= kSelNear) {
        list = sh.near;
        count = sh.close;
      }
    }
    for (int i = tid; i < count; i += kBeamThreads) {
      const SelCand c = list[i];
      int above = 0;
#pragma unroll 4
      for (int k = 0; k < count; ++k) above += sel_before(list[k], c);
      if (above < n) sh.best[above] = c;
    }
    __syncthreads();
    if (total <= kSelRoom) return;
    bound = sh.best[n - 1];
    __syncthreads();
  }
}

// (Three blocks of an SM: left to itself the compiler takes 64 registers, and spills; with two, which leaves it 108 instead of 77, 4096 requests of 8000 logits take 109 us
// instead of 89.)
template <typename T>
__global__ void __launch_bounds__(kBeamThreads, 3)
beam_pick_kernel(const T* __restrict__ logits, int64_t stride, int vocab, int groups, int per_row, const SelPart* __restrict__ parts,
                 const float* __restrict__ largest, const float* __restrict__ scores, int beams, int n, int keep, const int32_t* __restrict__ ended,
                 int num_ended, bool aligned, SelOut all, SelOut next) {
  constexpr int kWarps = kBeamThreads / 32, kAhead = 8;
  extern __shared__ __align__(16) uint4 held[];      // elements of the n best groups
  __shared__ SelShared sh;
  SelCand* best = sh.best;
  __shared__ __align__(16) SelNorm norm[kBeamMost];
  __shared__ float low[kBeamMost];
  __shared__ int from[kBeamMost], first[kBeamMost], start[kBeamMost], hits;
  __shared__ uint16_t hit[kSelRoom];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, num = beams * groups;
  const int64_t q = blockIdx.x;
  if (tid == 0) hits = 0;
  parts += q * beams * per_row;
  largest += q * num;
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  float ahead[kAhead];       // (on their way while the sums are added up)
#pragma unroll
  for (int k = 0; k < kAhead; ++k) ahead[k] = tid + k * kBeamThreads < num ? largest[tid + k * kBeamThreads] : -INFINITY;
  for (int b = warp; b < beams; b += kWarps) {
    const SelPart* row = parts + b * per_row;
    const float score = scores[q * beams + b];
    SelPart some[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) some[k] = lane + 32 * k < per_row ? row[lane + 32 * k] : SelPart{-INFINITY, 0.f};
    float m = some[0].m, s = 0.f;
#pragma unroll
    for (int k = 1; k < kAhead; ++k) m = fmaxf(m, some[k].m);
    for (int i = lane + 32 * kAhead; i < per_row; i += 32) m = fmaxf(m, row[i].m);
    m = warp_max(m);
    auto share = [&](const SelPart& x) { return x.s * (x.m > -INFINITY ? ptx::ex2_approx((x.m - m) * 1.4426950408889634f) : 1.f); };      // (1: 0 and NaN stay)
#pragma unroll
    for (int k = 0; k < kAhead; ++k) s += share(some[k]);
    for (int i = lane + 32 * kAhead; i < per_row; i += 32) s += share(row[i]);
    s = warp_sum(s);
    if (lane == 0) {
      // log s = log f + e log 2 with f from 1 to 2: in fp32 off by 2^-24, where log s would be by 2^-21
      int e = 1;
      const bool number = s > 0.f && s < INFINITY;
      const float f = number ? 2.f * frexpf(s, &e) : s;
      const double x = static_cast<double>(logf(f)) + (e - 1) * 0.69314718055994531;
      const float hi = static_cast<float>(x);
      norm[b] = SelNorm{score, m, hi, static_cast<float>(x - hi)};      // (an infinity: NaN)
    }
  }
  __syncthreads();
  auto group = [&](int i, float z) {
    const int b = min(i / groups, beams - 1);
    return sel_cand(sel_make(z, norm[b]), i);
  };
  SelCand mine{0, static_cast<uint64_t>(tid)};       // (each none another one)
  uint64_t mine_v[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    const SelCand c = group(tid + k * kBeamThreads, ahead[k]);
    mine_v[k] = c.v;
    if (c.v > mine.v) mine = c;       // (places rise)
  }
  for (int i = tid + kAhead * kBeamThreads; i < num; i += kBeamThreads) {
    const SelCand c = group(i, largest[i]);
    if (c.v > mine.v) mine = c;
  }
  const SelCand bound = sel_bound(n, mine, sh);
  sel_best(n, bound, sh, [&](auto&& take) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) take(sel_cand(mine_v[k], tid + k * kBeamThreads));
    for (int i = tid + kAhead * kBeamThreads; i < num; i += kBeamThreads) take(group(i, largest[i]));
  });
  // The n best elements are in these groups: one in any other group has their largest elements before it.  Those that reach the bound are in few pieces, which are
  // shared out by elements.
  constexpr int E = SelRow<T>::E, kPieces = SelRow<T>::kPieces;
  const int pieces = aligned ? kPieces : kPieces + 1;      // (of a group: the first and the last one may have elements of its neighbours, which do not count)
  auto group_of = [&](int i) { return aligned ? i / kPieces : i / (kPieces + 1); };
  if (tid < n) {
    const int f = best[tid].v ? static_cast<int>(~best[tid].early) : -1, b = f < 0 ? -1 : f / groups;
    from[tid] = b;
    if (f >= 0) {
      start[tid] = (f - b * groups) * kSelGroup;
      first[tid] = start[tid] - sel_lead(logits + (q * beams + b) * stride);
    }
  }
  SelCand least = best[n - 1].v ? SelCand{best[n - 1].v, 0} : SelCand{0, 0};
  auto lowest = [&] {      // a row's logits below this one are worth less than the bound
    if (tid < beams) {
      const SelNorm r = norm[tid];
      const float v = sel_value(least), x = v - r.base + r.hi + r.top, y = x - 1e-6f * (fabsf(v) + fabsf(r.base) + fabsf(r.hi) + fabsf(r.top));
      low[tid] = least.v && y > -INFINITY ? y : -INFINITY;
    }
  };
  lowest();
  __syncthreads();
#pragma unroll 2
  for (int i = tid; i < n * pieces; i += kBeamThreads) {
    const int at = group_of(i), b = from[at];
    if (b < 0) break;
    const T* z = logits + (q * beams + b) * stride;
    sel_piece(&held[i], z, first[at] + (i - at * pieces) * E, vocab);
  }
  ptx::cp_async_commit();
  ptx::cp_async_wait<0>();      // (a thread looks at what it has copied itself, until the next barrier)
  for (int turn = 0;; ++turn) {
#pragma unroll 2
    for (int i = tid; i < n * pieces; i += kBeamThreads) {
      const int b = from[group_of(i)];
      if (b < 0) break;
      if (sel_max<T>(held[i]) >= low[b]) {
        const int at = atomicAdd(&hits, 1);
        if (at < kSelRoom) hit[at] = static_cast<uint16_t>(i);
      }
    }
    __syncthreads();
    if (turn > 0 || hits <= kSelNear) break;
    // many pieces (small vocabularies, where few groups are not among the best): the n-th of their largest is a higher bound
    SelCand top{0, static_cast<uint64_t>(tid)};
#pragma unroll 1
    for (int t = tid; t < (hits <= kSelRoom ? hits : n * pieces); t += kBeamThreads) {
      const int i = hits <= kSelRoom ? hit[t] : t, at = group_of(i), b = from[at];
      if (b < 0) break;
      if (!aligned && (i == at * pieces || i == at * pieces + kPieces)) continue;
      const SelCand c = sel_cand(sel_make(sel_max<T>(held[i]), norm[b]), i);
      if (c.v && sel_before(c, top)) top = c;
    }
    const SelCand higher = sel_bound(n, top, sh);
    if (higher.v > least.v) least = SelCand{higher.v, 0};
    lowest();
    if (tid == 0) hits = 0;
    __syncthreads();
  }
  sel_best(n, least, sh, [&](auto&& take) {
    const bool few = hits <= kSelRoom;
#pragma unroll 1
    for (int t = tid; t < (few ? hits : n * pieces) * E; t += kBeamThreads) {
      const int i = few ? hit[t / E] : t / E, at = group_of(i), b = from[at];
      if (b < 0) break;
      const int token = first[at] + (i - at * pieces) * E + t % E;
      const float y = ldf(reinterpret_cast<const T*>(&held[i]) + t % E);
      if (y >= low[b] && static_cast<unsigned>(token - start[at]) < kSelGroup)
        take(sel_cand(sel_make(y, norm[b]), static_cast<uint64_t>(b) << 32 | static_cast<uint32_t>(token)));
    }
  });
  if (warp > 0) return;
  auto give = [](const SelOut& to, int64_t at, const SelCand& e) {
    to.score[at] = e.v ? sel_value(e) : -INFINITY;
    to.parent[at] = e.v ? static_cast<int32_t>(~e.early >> 32) : -1;
    to.token[at] = e.v ? static_cast<int32_t>(~e.early) : -1;
  };
  int before = 0;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int i = i0 + lane;
    if (i < n) give(all, q * all.pitch + i, best[i]);
    bool on = i < n && best[i].v != 0;
    for (int e = 0; on && e < num_ended; ++e) on = ended[e] != static_cast<int32_t>(~best[i].early);
    const unsigned who = __ballot_sync(0xffffffffu, on);
    const int at = before + __popc(who & ((1u << lane) - 1));
    if (on && at < keep) give(next, q * next.pitch + at, best[i]);
    before += __popc(who);
  }
  for (int i = before + lane; i < keep; i += 32) give(next, q * next.pitch + i, SelCand{0, 0});
}

// ------------------------------------------------------------------ tables of the beams that go on
struct ForkParams {
  const int32_t *table, *cached, *parents, *pool;
  int64_t table_stride, pool_stride, parents_stride;
  int width, from, to, pool_size, page, num_pages;   // from: beams of a request in `table`; to: children
  int32_t *out_table, *out_cached, *src, *dst, *tokens;
  int* status;
};

// A block per request.  A bit per page says which ones the children keep; the fresh ones are the first of the request's own without it.
// Latency bounds it: lengths, then tables, are two rounds of loads, all of a round at once (3.4 us for one request of 4 beams, 4.4 for 32 of 8; child after child 5.8 and 10.0).
__global__ void __launch_bounds__(kBeamThreads) beam_fork_kernel(const ForkParams p) {
  extern __shared__ uint32_t used[];
  __shared__ int par[kBeamMost], len[kBeamMost], again[kBeamMost], want[kBeamMost], fresh[kBeamMost], held[kBeamMost], sums[kBeamThreads / 32];
  __shared__ int wanted;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t q = blockIdx.x;
  const int words = (p.num_pages + 31) / 32;
  for (int i = tid; i < words; i += kBeamThreads) used[i] = 0;
  auto report = [&](int code) { if (p.status) atomicCAS(p.status, 0, code); };
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int first_pool = tid < p.pool_size ? p.pool[q * p.pool_stride + tid] : -1;
  if (tid < p.to) {
    par[tid] = p.parents[q * p.parents_stride + tid];
    fresh[tid] = -1;
  } else if (tid >= kBeamMost && tid < kBeamMost + p.from) {
    held[tid - kBeamMost] = p.cached[q * p.from + tid - kBeamMost];
  }
  __syncthreads();
  if (tid < p.to) {
    const int b = par[tid];
    int n = -1;
    if (b >= 0 && b < p.from) {
      n = max(held[b], -1);
      if (n / p.page >= p.width) {
        report(kStatusTooLarge);
        n = -1;
      }
    } else if (b >= p.from) {
      report(kStatusBadIndex);
    }
    int seen = 0;         // (children of one parent are all alive or all dead)
    for (int i = 0; i < tid; ++i) seen |= par[i] == b;
    len[tid] = n;
    again[tid] = seen;
  }
  __syncthreads();
  // children's tables without their fresh pages, and the pages that they keep (a parent's once)
#pragma unroll 4
  for (int it = tid; it < p.to * p.width; it += kBeamThreads) {
    const int j = it / p.width, i = it - j * p.width, n = len[j];
    const int keeps = n < 0 ? 0 : again[j] ? n / p.page : (n + p.page - 1) / p.page;
    int pg = -1;
    if (i < keeps) {
      pg = p.table[(q * p.from + par[j]) * p.table_stride + i];
      if (!again[j]) {
        if (pg >= 0 && pg < p.num_pages) atomicOr(&used[pg >> 5], 1u << (pg & 31));
        else report(kStatusBadIndex);
      }
    }
    p.out_table[q * p.to * p.width + it] = pg;
  }
  if (warp == 0) {       // which children want a fresh page: theirs is the one of their number among them
    int before = 0;
    for (int j0 = 0; j0 < p.to; j0 += 32) {
      const int j = j0 + lane;
      const bool wants = j < p.to && len[j] >= 0 && (len[j] % p.page == 0 || again[j]);
      const unsigned who = __ballot_sync(0xffffffffu, wants);
      if (j < p.to) want[j] = wants ? before + __popc(who & ((1u << lane) - 1)) : -1;
      before += __popc(who);
    }
    if (lane == 0) wanted = before;
  }
  __syncthreads();
  int got = 0;
  for (int i0 = 0; i0 < p.pool_size && got < wanted; i0 += kBeamThreads) {
    const int i = i0 + tid, pg = i0 == 0 ? first_pool : i < p.pool_size ? p.pool[q * p.pool_stride + i] : -1;
    const bool free = pg >= 0 && pg < p.num_pages && !(used[pg >> 5] >> (pg & 31) & 1);
    const unsigned who = __ballot_sync(0xffffffffu, free);
    if (lane == 0) sums[warp] = __popc(who);
    __syncthreads();
    int at = got + __popc(who & ((1u << lane) - 1)), total = 0;
    for (int k = 0; k < kBeamThreads / 32; ++k) {
      if (k < warp) at += sums[k];
      total += sums[k];
    }
    if (free && at < wanted) fresh[at] = pg;
    got += total;
    __syncthreads();
  }
  if (tid < p.to) {
    const int n = len[tid], page = want[tid] >= 0 ? fresh[want[tid]] : -1, full = n / p.page;
    const bool live = n >= 0 && (want[tid] < 0 || page >= 0), copies = live && want[tid] >= 0 && n % p.page > 0;
    const int64_t j = q * p.to + tid;
    if (live && want[tid] >= 0) p.out_table[j * p.width + full] = page;
    if (n >= 0 && !live) {
      report(kStatusNoPage);
      for (int i = 0; i < p.width; ++i) p.out_table[j * p.width + i] = -1;
    }
    p.out_cached[j] = live ? n : -1;
    p.src[j] = copies ? p.table[(q * p.from + par[tid]) * p.table_stride + full] : -1;
    p.dst[j] = copies ? page : -1;
    p.tokens[j] = copies ? n % p.page : 0;
  }
}

// ------------------------------------------------------------------ copies of pages and slots
struct CopyParams {
  uint8_t* base;
  int64_t layer_stride, page_stride, part_stride, part_bytes;   // bytes; a page is `parts` runs of part_bytes
  int64_t token_bytes;                                          // of a run, where `tokens` says how many there are
  int layers, parts, pages, pairs, pieces;
  const int32_t *src, *dst, *tokens;
  int* status;
};
constexpr int kCopyPiece = 32768;

// A block per piece of 32 KB, each thread with eight 16-byte loads under way; HBM bounds it (99 MB, 256 rows of 8 layers, 28.5 us, 6.9 TB/s read and written).  U: what all
// addresses are multiples of.
template <typename U>
__global__ void __launch_bounds__(kBeamThreads) copy_pages_kernel(const CopyParams p) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  const int pair = blockIdx.x / p.pieces, piece = blockIdx.x % p.pieces, tid = threadIdx.x;
  const int from = p.src[pair], to = p.dst[pair];
  if (from < 0 || to < 0) return;
  if (from >= p.pages || to >= p.pages) {
    if (p.status && tid == 0) atomicCAS(p.status, 0, kStatusBadIndex);
    return;
  }
  if (from == to) return;
  const int64_t bytes = p.tokens ? min(p.part_bytes, max(p.tokens[pair], 0) * p.token_bytes) : p.part_bytes;
  const int64_t lo = static_cast<int64_t>(piece) * kCopyPiece, hi = min(bytes, lo + kCopyPiece);
  if (lo >= hi) return;
  const int layer = blockIdx.y / p.parts, part = blockIdx.y % p.parts;
  uint8_t* at = p.base + layer * p.layer_stride + part * p.part_stride;
  const U* a = reinterpret_cast<const U*>(at + from * p.page_stride + lo);
  U* b = reinterpret_cast<U*>(at + to * p.page_stride + lo);
  const int count = static_cast<int>((hi - lo) / sizeof(U));
  constexpr int kTurn = 8;
  for (int i = tid; i < count; i += kTurn * kBeamThreads) {
    U x[kTurn];
#pragma unroll
    for (int k = 0; k < kTurn; ++k)
      if (i + k * kBeamThreads < count) x[k] = a[i + k * kBeamThreads];
#pragma unroll
    for (int k = 0; k < kTurn; ++k)
      if (i + k * kBeamThreads < count) b[i + k * kBeamThreads] = x[k];
  }
}

// ------------------------------------------------------------------ tables of a step
struct TableParams {
  const int32_t *table, *cached, *counts;
  int64_t table_stride;
  int rows, width, page, beams, entries, tokens;
  int32_t *indices, *indptr, *last, *pos, *slot, *tok_indptr, *shared;
  int* status;
};
constexpr int kTableMostRows = 8192;

// Every block adds up the rows' pages and tokens by itself (a few thousand numbers at most) and looks after its share of the entries: which row
// an entry belongs to is found by halves.  One launch and three rounds of loads: 3.5 us for 4 rows, 3.9 for 61 rows of 8192 new tokens.
__global__ void __launch_bounds__(kBeamThreads) step_tables_kernel(const TableParams p) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  extern __shared__ int ends[];
  int* pages = ends;                      // [rows + 1] where a row's pages begin
  int* toks = ends + p.rows + 1;
  __shared__ int wp[kBeamThreads / 32], wt[kBeamThreads / 32], taken, differ;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto report = [&](int code) { if (p.status) atomicCAS(p.status, 0, code); };
  const int per = (p.rows + kBeamThreads - 1) / kBeamThreads, r0 = min(p.rows, tid * per), r1 = min(p.rows, r0 + per);
  // tokens of a row after the step (0: it has no part in it)
  auto new_tokens = [&](int r) {
    const int c = p.cached[r], n = p.counts ? p.counts[r] : 1;
    if (c < 0 || n <= 0) return 0;
    if (c > static_cast<int64_t>(p.width) * p.page - n) {
      report(kStatusTooLarge);
      return 0;
    }
    return n;
  };
  int np = 0, nt = 0;
  for (int r = r0; r < r1; ++r) {
    const int n = new_tokens(r);
    toks[r + 1] = n;
    pages[r + 1] = n ? (p.cached[r] + n - 1) / p.page + 1 : 0;
    np += pages[r + 1];
    nt += n;
  }
  int sp = np, st = nt;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, sp, d), b = __shfl_up_sync(0xffffffffu, st, d);
    if (lane >= d) {
      sp += a;
      st += b;
    }
  }
  if (lane == 31) {
    wp[warp] = sp;
    wt[warp] = st;
  }
  if (tid == 0) {
    pages[0] = toks[0] = 0;
    taken = p.rows;
  }
  __syncthreads();
  sp -= np;
  st -= nt;
  for (int i = 0; i < warp; ++i) {
    sp += wp[i];
    st += wt[i];
  }
  for (int r = r0; r < r1; ++r) {
    pages[r + 1] = sp += pages[r + 1];
    toks[r + 1] = st += toks[r + 1];
    // rows are taken as long as there is room for their pages and tokens
    if (sp > p.entries || (p.counts && st > p.tokens)) atomicMin(&taken, r);
  }
  __syncthreads();
  const int rows = taken;
  if (rows < p.rows && tid == 0 && blockIdx.x == 0) report(kStatusTooLarge);
  const int total = pages[rows], total_t = toks[rows];
  const int self = blockIdx.x * kBeamThreads + tid, all = gridDim.x * kBeamThreads;
  auto slot_of = [&](int pg, int at) {       // (-1 where there is no page, or a number that can be none)
    const int64_t slot = static_cast<int64_t>(pg) * p.page + at % p.page;
    if (slot > 0x7fffffff) report(kStatusBadIndex);
    return pg >= 0 && slot <= 0x7fffffff ? static_cast<int>(slot) : -1;
  };
  auto row_of = [&](const int* begin, int x) {       // the last row that begins at or before x and is not empty
    int lo = 0, hi = rows;                           // begin[lo] <= x < begin[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (begin[mid] <= x) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  for (int e = self; e < p.entries; e += all) {
    int pg = 0;
    if (e < total) {
      const int r = row_of(pages, e);
      pg = p.table[r * p.table_stride + e - pages[r]];
    }
    p.indices[e] = pg;
  }
  for (int r = self; r <= p.rows; r += all) {
    p.indptr[r] = pages[min(r, rows)];
    if (p.tok_indptr) p.tok_indptr[r] = toks[min(r, rows)];
    if (r == p.rows) continue;
    const int n = r < rows ? toks[r + 1] - toks[r] : 0, c = p.cached[r];
    p.last[r] = n ? (c + n - 1) % p.page + 1 : 0;
    if (p.counts == nullptr) {
      p.pos[r] = n ? c : 0;
      p.slot[r] = n ? slot_of(p.table[r * p.table_stride + c / p.page], c) : -1;
    }
  }
  if (p.counts) {
    for (int t = self; t < p.tokens; t += all) {
      int at = 0, slot = -1;
      if (t < total_t) {
        const int r = row_of(toks, t);
        at = p.cached[r] + t - toks[r];
        slot = slot_of(p.table[r * p.table_stride + at / p.page], at);
      }
      p.pos[t] = at;
      p.slot[t] = slot;
    }
  }
  if (p.beams > 0) {
    // full pages that a request's rows have in common: up to the first one that differs, or the shortest row
    for (int q = blockIdx.x; q < p.rows / p.beams; q += gridDim.x) {
      __syncthreads();
      if (tid == 0) differ = 0x7fffffff;
      __syncthreads();
      int first = -1, most = 0x7fffffff;
      for (int r = q * p.beams; r < (q + 1) * p.beams; ++r) {
        const int n = r < rows ? toks[r + 1] - toks[r] : 0;
        if (!n) continue;
        if (first < 0) first = r;
        most = min(most, (p.cached[r] + n) / p.page);
      }
      if (first < 0) most = 0;
      for (int e = tid; e < most; e += kBeamThreads) {
        const int pg = p.table[first * p.table_stride + e];
        bool same = true;
        for (int r = first + 1; r < (q + 1) * p.beams; ++r)
          if (r < rows && toks[r + 1] > toks[r]) same &= p.table[r * p.table_stride + e] == pg;
        if (!same) {
          atomicMin(&differ, e);
          break;
        }
      }
      __syncthreads();
      if (tid == 0) p.shared[q] = min(most, differ);
    }
  }
}

// How a selection's rows are cut: groups and stretches of a row, groups of a stretch.
struct SelPlan {
  int groups, per_row, length;
  int64_t largest, bytes;       // where the groups' largest are in the scratch, its size
  SelPlan(int64_t rows, int vocab) {
    groups = static_cast<int>((static_cast<int64_t>(vocab) + kSelGroup - 1) / kSelGroup);
    const int64_t warps = static_cast<int64_t>(kSelWarps) * device_sm_count() / (rows < 1 ? 1 : rows);
    length = warps < 1 ? kSelStretch : static_cast<int>((groups + warps - 1) / warps);
    if (length > kSelStretch) length = kSelStretch;
    per_row = (groups + length - 1) / length;
    largest = (8 * rows * per_row + 255) / 256 * 256;
    bytes = largest + 4 * rows * groups;
  }
};

}  // namespace blitz

extern "C" {
using namespace blitz;

int64_t blitz_beam_select_workspace_bytes(int rows, int vocab, int n, int dtype) { return SelPlan(rows, vocab).bytes; }

// logits [rows][stride] in fp16 (0), bf16 (1) or fp32 (2); scores [rows]; a request's beams are consecutive rows.  score, parent and token:
// [rows / beams][n], pitch apart, next_*: [rows / beams][keep], next_pitch.  ended: tokens that end a sequence (num_ended of them).
int blitz_beam_select(const void* logits, int64_t stride, const float* scores, int rows, int vocab, int beams, int n, int keep, const int32_t* ended,
                      int num_ended, void* workspace, float* score, int32_t* parent, int32_t* token, float* next_score, int32_t* next_parent,
                      int32_t* next_token, int64_t pitch, int64_t next_pitch, int dtype, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (vocab < 1 || beams < 1 || beams > kBeamMost || rows % beams || n < 1 || n > kBeamMost || keep < 1 || keep > n || num_ended < 0) return -1;
  const SelPlan plan(rows, vocab);
  const int64_t blocks = (static_cast<int64_t>(rows) * plan.per_row + kBeamThreads / 32 - 1) / (kBeamThreads / 32);
  if (blocks > 0x7fffffff || static_cast<int64_t>(beams) * plan.groups > 0x7fffffff || vocab > 0x7fffffff - 2 * kSelGroup) return -1;
  SelPart* parts = reinterpret_cast<SelPart*>(workspace);
  float* largest = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + plan.largest);
  cudaError_t e = cudaSuccess;
  BLITZ_DISPATCH_DTYPE3(dtype, {
    constexpr int kRing = kBeamThreads / 32 * SelRow<T>::kRing * 16;       // bytes of the scan's rings for each piece of a group
    const bool aligned = ((reinterpret_cast<uintptr_t>(logits) | static_cast<uint64_t>(stride) * sizeof(T)) & 15) == 0;
    const int pieces = aligned ? SelRow<T>::kPieces : SelRow<T>::kPieces + 1;
    auto scan = aligned ? beam_scan_kernel<T, false> : beam_scan_kernel<T, true>;
    static PerDeviceOnce once;
    e = once.run([] {
      const cudaError_t first = cudaFuncSetAttribute(beam_scan_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing * (SelRow<T>::kPieces + 1));
      return first != cudaSuccess ? first
                                  : cudaFuncSetAttribute(beam_pick_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBeamMost * (SelRow<T>::kPieces + 1) * 16);
    });
    if (e == cudaSuccess)
      e = launch_pdl(scan, dim3((unsigned)blocks), dim3(kBeamThreads), kRing * pieces, stream, (const T*)logits, stride, rows, vocab, plan.groups, plan.per_row,
                     plan.length, parts, largest);
    if (e == cudaSuccess)
      e = launch_pdl(beam_pick_kernel<T>, dim3(rows / beams), dim3(kBeamThreads), n * pieces * 16, stream, (const T*)logits, stride, vocab, plan.groups, plan.per_row, (const SelPart*)parts, (const float*)largest, scores, beams, n, keep, ended, num_ended, aligned,
                     SelOut{score, parent, token, pitch}, SelOut{next_score, next_parent, next_token, next_pitch});
  });
  return (int)e;
}

// table [requests from][width], cached [requests from], parents [requests][to], pool [requests][pool_size]; the children's table
// [requests to][width], cached, and the copies to make (src, dst, tokens; -1: none).
int blitz_beam_fork(const int32_t* table, int64_t table_stride, const int32_t* cached, const int32_t* parents, int64_t parents_stride, const int32_t* pool, int64_t pool_stride,
                    int requests, int from, int to, int width, int pool_size, int page, int num_pages, int32_t* out_table, int32_t* out_cached, int32_t* src,
                    int32_t* dst, int32_t* tokens, int* status, cudaStream_t stream) {
  if (requests <= 0) return 0;
  if (from < 1 || to < 1 || from > kBeamMost || to > kBeamMost || width < 1 || page < 1 || num_pages < 1 || pool_size < 0) return -1;
  const size_t smem = static_cast<size_t>((num_pages + 31) / 32) * 4;
  if (smem > 200 * 1024) return -1;
  static PerDeviceOnce once;
  cudaError_t e = once.run([] { return cudaFuncSetAttribute(beam_fork_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024); });
  if (e != cudaSuccess) return (int)e;
  ForkParams p{table, cached, parents, pool, table_stride, pool_stride, parents_stride, width, from, to, pool_size, page, num_pages, out_table, out_cached, src, dst, tokens, status};
  return (int)launch_pdl(beam_fork_kernel, dim3(requests), dim3(kBeamThreads), smem, stream, p);
}

// Page (or slot) src[i] of every layer to dst[i], for pairs without a negative number.  A page is `parts` runs of part_bytes, part_stride
// apart; with tokens, the first tokens[i] token_bytes of each.
int blitz_copy_pages(void* base, int layers, int64_t layer_stride, int pages, int64_t page_stride, int parts, int64_t part_stride, int64_t part_bytes,
                     int64_t token_bytes, const int32_t* src, const int32_t* dst, const int32_t* tokens, int pairs, int* status, cudaStream_t stream) {
  if (pairs <= 0 || layers <= 0 || part_bytes <= 0) return 0;
  if (parts < 1 || pages < 1) return -1;
  const int64_t pieces = (part_bytes + kCopyPiece - 1) / kCopyPiece;
  if (pieces * pairs > 0x7fffffff || static_cast<int64_t>(layers) * parts > 65535) return -1;
  CopyParams p{static_cast<uint8_t*>(base), layer_stride, page_stride, part_stride, part_bytes, token_bytes, layers, parts, pages, pairs, (int)pieces, src, dst, tokens,
               status};
  const uint64_t align = reinterpret_cast<uintptr_t>(base) | layer_stride | page_stride | part_stride | part_bytes | (tokens ? token_bytes : 0);
  const dim3 grid((unsigned)(pieces * pairs), (unsigned)(layers * parts));
  if (align % 16 == 0) return (int)launch_pdl(copy_pages_kernel<uint4>, grid, dim3(kBeamThreads), 0, stream, p);
  if (align % 4 == 0) return (int)launch_pdl(copy_pages_kernel<uint32_t>, grid, dim3(kBeamThreads), 0, stream, p);
  return (int)launch_pdl(copy_pages_kernel<uint8_t>, grid, dim3(kBeamThreads), 0, stream, p);
}

// Page list, where each row's pages begin, tokens on its last page; of the new tokens positions and slots.  counts null: one new token for each
// row that has a length, in its row of pos and slot; else counts[r], one row's behind the other's (`tokens` places).  beams > 0: shared
// [rows / beams].
int blitz_step_tables(const int32_t* table, int64_t table_stride, const int32_t* cached, const int32_t* counts, int rows, int width, int page, int beams,
                      int entries, int tokens, int32_t* indices, int32_t* indptr, int32_t* last, int32_t* pos, int32_t* slot, int32_t* tok_indptr,
                      int32_t* shared, int* status, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (rows > kTableMostRows || width < 1 || page < 1 || entries < 0 || tokens < 0 || (beams > 0 && rows % beams)) return -1;
  TableParams p{table, cached, counts, table_stride, rows, width, page, beams, entries, tokens, indices, indptr, last, pos, slot, tok_indptr, shared, status};
  const size_t smem = static_cast<size_t>(rows + 1) * 8;
  static PerDeviceOnce once;
  cudaError_t e = once.run([] { return cudaFuncSetAttribute(step_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (kTableMostRows + 1) * 8); });
  if (e != cudaSuccess) return (int)e;
  const int64_t work = static_cast<int64_t>(entries) + (counts ? tokens : 0) + rows;
  int64_t blocks = (work + 4 * kBeamThreads - 1) / (4 * kBeamThreads);
  if (beams > 0 && blocks < rows / beams) blocks = rows / beams;
  const int most = 2 * device_sm_count();
  return (int)launch_pdl(step_tables_kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(kBeamThreads), smem, stream, p);
}

}  // extern "C"
