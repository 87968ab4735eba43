// Decode attention of beams: one query token per row, rows in groups (the beams of a request) whose first pages are the same.
//
// out = softmax(q K^T scale) V per head over the row's pages [page][K|V][token][kv_head][dim].  It is a stream over keys and values, so what counts is
// that those of the common pages come from HBM once: their query rows (beams times the query heads of a KV head, up to 32) are two tiles of
// 16 rows of one matrix product, mma.sync m16n8k16.  tcgen05 is not used on purpose: one SM streams 16 tokens of a head in the time of a thousand
// such instructions, and rows are few.
//
// Work.  A segment is the common part of a group, or what a row has behind it.  Per KV head (and block of beams, where they are more than 32 rows) the
// segments' steps of 16 tokens laid end to end are cut into equal ranges, and a warp takes one range of one head: neither long rows nor few of them leave
// warps idle.  Neighbouring warps have the heads of the same tokens, which are neighbours in memory.  A range is as many pieces as it meets segments; a piece leaves its
// sums in scratch (fp32), and a second kernel adds up a row's pieces, always in the same order.  Every block works out the ranges from the tables, so a
// captured launch follows them.
//
// A warp is by itself: it asks for its next step (TMA, boxes of 16 tokens x 64 columns) and computes the one that is there, and nothing in the
// loop waits for another warp.  (With cp.async instead a warp stood for 2000 to 4000 cycles of a step in its own requests, and computed, 750 to 1500, only then.)  Two
// steps of a warp, 128 KB an SM, are enough to keep memory busy; with three more requests wait in its queues, and SMs are served less evenly.
//
// Rounded to 16 bits: the weights, as operands of the second product, and the output.  Scores, maxima, sums and pieces are fp32.  Errors against 64 bits: bf16 0.0023 where the output's
// rounding alone is 0.0017, fp16 0.00027 (0.00021), as decode attention has them.  Weights as two 16-bit numbers take that away and cost 8 us of 67 (32 x 8 beams; 5 where only tiles
// of up to 16 rows have them).
//
// Measured, 32 query over 8 KV heads of 128, bf16, us in a graph (bytes of each token once, at the copy rate): 4 beams of 100144 tokens 74.5 to 75.5 (63.1), of 1014 tokens 9.7 (0.75);
// 32 x 8 beams of 1301 on average, 101 of them their own, 65.7 to 67.2 (44.5).  What bounds it: memory at 6.0 to 6.7 TB/s while all warps run, but
// equal ranges end between 41 and 57 us (32 x 8) or 57 and 66 (the long one); then 3 us for tables and first loads, 6.6 to 7.7 for the merge.
// Tried: three steps under way 72.9 (78.8 the long one), one 79.6 (84.3); queries and page ids of the next piece asked for a piece ahead 70.4; the heads of a range on one SM 72.8.
#include <cfloat>

#include "launch.cuh"
#include "ptx.cuh"
#include "tmap.cuh"
#include "common.cuh"
#include "mma.cuh"
#include "scalar.cuh"

namespace blitz {

constexpr int kBaWarps = 8, kBaThreads = 32 * kBaWarps;
constexpr int kBaStep = 16;            // tokens
constexpr int kBaRowsMost = 1024;      // rows of a launch
constexpr int kBaTile = 32;            // query rows of a segment

struct BeamAttnParams {
  const void* q;
  int64_t q_stride;
  const void* kv;
  const int32_t *indices, *indptr, *last_page_len, *shared;
  void* out;
  int64_t out_stride;
  int rows, beams, groups;      // groups of beams
  int q_heads, rep;             // query heads of a virtual head
  int kv_div, kv_heads;         // virtual heads of a KV head
  int per_block, blocks;        // beams of a block, blocks of a group
  int heads;                    // virtual heads x blocks
  int ranges_most;
  int page_shift, max_pages;
  float scale_log2, slack, cap_scale, cap_log2;      // the scale's size (1 under a cap, or where it is zero); keep and flip: zero or its sign, for the queries
  uint32_t keep, flip;
  const void* sink;
  int2* runs;                   // [blocks][groups + groups per_block] of each segment: its first piece's range, pieces
  float *o_common, *o_own;      // partial sums
  float2 *ml_common, *ml_own;   // reference (before the scale) and sum of each
  int static_table;
  int* status;
};

// Equal ranges of n steps of `segments` segments: as many as there are warps, but of two steps at least, or of one where there are more segments than that: a piece takes 3 us
// before its first product, one behind the other in a warp.  (Two steps against four: 1 x 4 beams of 1014 tokens 10.8 -> 9.9 us, 1 x 6 of 356 14.5 -> 11.4; with segments
// counted: 17 x 6 of 11 tokens 19.9 -> 11.2, 15 x 4 of 4 21.3 -> 14.3.)
struct BaRanges {
  int count, q, rem;
  __device__ __forceinline__ BaRanges(int n, int most, int segments) {
    count = max(1, min(most, max(n / 2, min(n, segments))));
    q = n / count;
    rem = n - q * count;
  }
  __device__ __forceinline__ int begin(int r) const { return r * q + min(r, rem); }
  __device__ __forceinline__ int of(int x) const { return x < rem * (q + 1) ? x / (q + 1) : rem + (x - rem * (q + 1)) / q; }
};

// Lengths, common pages and the line of segments, by all threads of a block; arrays in shared memory.
__device__ __forceinline__ void ba_line(const BeamAttnParams& p, int* line, int* len, int* common, int* sums) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int shared0 = tid < p.blocks * p.groups ? p.shared[tid % p.groups] : 0;      // (asked for together with the lengths)
  for (int r = tid; r < p.rows; r += kBaThreads) {
    const int pages = p.indptr[r + 1] - p.indptr[r];
    len[r] = pages > 0 ? ((pages - 1) << p.page_shift) + min(max(p.last_page_len[r], 0), 1 << p.page_shift) : 0;
  }
  __syncthreads();
  for (int i = tid; i < p.blocks * p.groups; i += kBaThreads) {
    const int b = i / p.groups, g = i % p.groups;
    int most = max(i == tid ? shared0 : p.shared[g], 0);
    bool any = false;
    for (int j = b * p.per_block; j < min((b + 1) * p.per_block, p.beams); ++j) {
      const int n = len[g * p.beams + j];
      if (n > 0) {
        any = true;
        most = min(most, n >> p.page_shift);
      }
    }
    common[i] = any ? most : 0;
  }
  __syncthreads();
  const int per = p.groups * (1 + p.per_block), total = p.blocks * per;
  const int each = (total + kBaThreads - 1) / kBaThreads, e0 = min(total, tid * each), e1 = min(total, e0 + each);
  auto steps = [&](int e) {
    const int b = e / per, i = e % per;
    if (i < p.groups) return common[b * p.groups + i] << (p.page_shift - 4);
    const int g = (i - p.groups) / p.per_block, j = b * p.per_block + (i - p.groups) % p.per_block;
    const int n = j < p.beams ? len[g * p.beams + j] : 0;
    return n > 0 ? (n - (common[b * p.groups + g] << p.page_shift) + kBaStep - 1) / kBaStep : 0;
  };
  int mine = 0;
  for (int e = e0; e < e1; ++e) mine += steps(e);
  int sum = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += up;
  }
  if (lane == 31) sums[warp] = sum;
  __syncthreads();
  sum -= mine;
  for (int w = 0; w < warp; ++w) sum += sums[w];
  for (int e = e0; e < e1; ++e) {
    line[e] = sum;
    sum += steps(e);
  }
  if (e1 == total && e0 < total) line[total] = sum;
  __syncthreads();
}

// A place on a warp's range: segment, and what of its row the steps are.
struct BaPlace {
  int seg, x;              // segment (of the block of beams), step on the line
  int seg_beg, seg_end;    // its steps
  int pages, tok0, len;    // first page in `indices`; token that its first step is; tokens of the row
};

// A wait that ran out: the status word, and as long again for each of the `count` copies that are under way from this stage on.
__device__ __noinline__ void ba_give_up(int* status, uint64_t* arrived, int stages, int stage, uint32_t phase, int count) {
  if (status) atomicCAS(status, 0, kStatusTimeoutProducer);
  for (; count > 0; --count) {
    int none = 0;
    ptx::bounded_mbar_wait(&arrived[stage], phase, &none);
    if (++stage == stages) {
      stage = 0;
      phase ^= 1;
    }
  }
}

// All weights are 2^-8 of what they are beside their reference, so that they are one at most and sums of bf16 values stay below tokens x values.  (fp16: its values are far
// from what fp32 holds, and small weights would lose digits.)
template <typename T>
__host__ __device__ constexpr float ba_small() { return std::is_same<T, __nv_bfloat16>::value ? 8.f : 0.f; }

template <typename T, int HD>
__global__ void __launch_bounds__(kBaThreads, 1) attn_beams_kernel(const __grid_constant__ CUtensorMap tmap, const BeamAttnParams p) {
  constexpr int kSlab = kBaStep * 128, kSlabs = HD / 64;       // 64 columns of a step's keys, 128 bytes a token, 16-byte columns turned by the token's number
  constexpr int kStage = 2 * kSlabs * kSlab;                  // keys, then values
  constexpr int kStages = HD == 128 ? 2 : 4;
  extern __shared__ uint8_t ba_raw[];
  uint8_t* ba_smem = ba_raw + (1024 - (ptx::smem_u32(ba_raw) & 1023)) % 1024;
  __shared__ int sums[kBaWarps];
  __shared__ uint64_t arrived[kBaWarps][kStages];
  __shared__ int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = p.groups * (1 + p.per_block);
  int* line = reinterpret_cast<int*>(ba_smem + kBaWarps * kStages * kStage);
  int* len = line + p.blocks * per + 1;
  int* common = len + p.rows;
  const int self = warp * gridDim.x + blockIdx.x;
  const int hv = self % p.heads, range = self / p.heads;
  const int block = hv % p.blocks, head = hv / p.blocks;       // head: virtual, of `rep` query heads
  if (threadIdx.x == 0) abort_flag = 0;
  if (lane < kStages) ptx::mbar_init(&arrived[warp][lane], 1);
  ptx::fence_mbar_init();
  if (threadIdx.x == 0) ptx::tma_prefetch_desc(&tmap);
  ptx::griddep_launch_dependents();
  if (!p.static_table) ptx::griddep_wait();
  ba_line(p, line, len, common, sums);
  ptx::griddep_wait();
  // where each segment's pieces are, for the merge
  for (int e = blockIdx.x + threadIdx.x * gridDim.x; e < p.blocks * per; e += gridDim.x * kBaThreads) {
    const int* of = line + e / per * per;
    const BaRanges ranges(of[per] - of[0], p.ranges_most, per);
    const int x0 = line[e] - of[0], x1 = line[e + 1] - of[0], r = x0 < x1 ? ranges.of(x0) : 0;
    p.runs[e] = make_int2(r, x0 < x1 ? ranges.of(x1 - 1) - r + 1 : 0);
  }

  line += block * per;
  common += block * p.groups;
  const int base = line[0];
  const BaRanges ranges(line[per] - base, p.ranges_most, per);
  if (range >= ranges.count) return;
  const int x_end = ranges.begin(range + 1);
  const int page = 1 << p.page_shift, kv_head = head / p.kv_div;

  auto enter = [&](BaPlace& a) {     // the segment that step a.x is in (a.seg: one at or before it)
    while (line[a.seg + 1] - base <= a.x) ++a.seg;
    a.seg_beg = line[a.seg] - base;
    a.seg_end = min(line[a.seg + 1] - base, x_end);
    int row, g;
    if (a.seg < p.groups) {
      g = a.seg;
      row = g * p.beams + block * p.per_block;
      while (len[row] == 0) ++row;                             // (a common part has a row with pages)
      a.tok0 = 0;
      a.len = common[g] << p.page_shift;
    } else {
      const int i = a.seg - p.groups;
      g = i / p.per_block;
      row = g * p.beams + block * p.per_block + i % p.per_block;
      a.tok0 = common[g] << p.page_shift;
      a.len = len[row];
    }
    a.pages = p.indptr[row];
  };
  BaPlace ld{}, at{};
  ld.x = at.x = ranges.begin(range);
  if (ld.x >= x_end) return;
  {
    int lo = 0, hi = per;      // line[lo] <= x < line[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (line[mid] - base <= ld.x) lo = mid;
      else hi = mid;
    }
    ld.seg = at.seg = lo;
  }
  enter(ld);
  enter(at);
  uint8_t* ring_at = ba_smem + warp * kStages * kStage;
  const uint32_t ring = ptx::smem_u32(ring_at);
  int win = 0, win_base = -64;       // page ids: lane l holds entry win_base + l of the row's list
  int ld_stage = 0;
  auto load = [&]() {                // requests the next step
    if (ld.x >= x_end) return;
    if (ld.x >= ld.seg_end) {
      enter(ld);
      win_base = -64;
    }
    const int t0 = ld.tok0 + (ld.x - ld.seg_beg) * kBaStep, pg = t0 >> p.page_shift;
    if (pg >= win_base + 32 || pg < win_base) {
      win_base = pg;
      const int last = (ld.len - 1) >> p.page_shift;
      win = pg + lane <= last ? p.indices[ld.pages + pg + lane] : 0;
      if (win < 0 || win >= p.max_pages) {
        if (p.status) atomicCAS(p.status, 0, kStatusBadIndex);
        win = 0;
      }
    }
    const int id = __shfl_sync(0xffffffffu, win, pg - win_base);
    if (ptx::elect_one()) {
      // (whole steps: pages are multiples of them)
      const int z = (id << (p.page_shift + 1)) + (t0 & (page - 1));
      uint8_t* to = ring_at + ld_stage * kStage;
      ptx::mbar_expect_tx(&arrived[warp][ld_stage], kStage);
#pragma unroll
      for (int i = 0; i < kSlabs; ++i) {
        ptx::tma_load_3d(to + i * kSlab, &tmap, &arrived[warp][ld_stage], i * 64, kv_head, z);
        ptx::tma_load_3d(to + (kSlabs + i) * kSlab, &tmap, &arrived[warp][ld_stage], i * 64, kv_head, z + page);
      }
    }
    ++ld.x;
    if (++ld_stage == kStages) ld_stage = 0;
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) load();
  const uint64_t scale2 = ptx::f32x2(p.scale_log2, p.scale_log2), small2 = ptx::f32x2(-ba_small<T>(), -ba_small<T>());
  const int g8 = lane >> 2, t4 = lane & 3, mi = lane >> 3, mr = lane & 7;
  // what the lane reads of a stage with ldmatrix: keys of its token from 16-byte column mi & 1 on, values of its token from column mi >> 1 on
  const int k_tok = (mi >> 1) * 8 + mr, v_tok = (mi & 1) * 8 + mr;
  const uint32_t k_at = ring + k_tok * 128 + (((mi & 1) ^ k_tok & 7) << 4);
  const uint32_t v_at = ring + kSlabs * kSlab + v_tok * 128 + (((mi >> 1) ^ v_tok & 7) << 4);
  int stage = 0;
  uint32_t phase = 0;
  bool ok = true;       // (a wait that ran out: the status word says so, and the warp ends when its copies have arrived)
  // A piece: TILES of 16 query rows.
  auto piece = [&](auto tiles) {
    constexpr int TILES = decltype(tiles)::value;
    const bool shared_part = at.seg < p.groups;
    const int i0 = at.seg - p.groups;
    const int row0 = shared_part ? at.seg * p.beams + block * p.per_block : i0 / p.per_block * p.beams + block * p.per_block + i0 % p.per_block;
    const int live = shared_part ? min(p.per_block, p.beams - block * p.per_block) * p.rep : p.rep;       // query rows
    uint32_t qa[TILES][HD / 16][4];
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int i = t * 16 + half * 8 + g8, r = i / p.rep;
        const T* q = reinterpret_cast<const T*>(p.q) + (row0 + r) * p.q_stride + (head * p.rep + i - r * p.rep) * HD;
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
          for (int hi = 0; hi < 2; ++hi)
            qa[t][ks][half + 2 * hi] = i < live ? *reinterpret_cast<const uint32_t*>(q + ks * 16 + hi * 8 + 2 * t4) & p.keep ^ p.flip : 0u;
      }
    float o[TILES][HD / 8][4], m[TILES][2], l[TILES][2], limit[TILES][2];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      m[t][0] = m[t][1] = -FLT_MAX;        // (finite: scores of minus infinity alone leave a piece of no weight)
      limit[t][0] = limit[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) o[t][i][0] = o[t][i][1] = o[t][i][2] = o[t][i][3] = 0.f;
    }
    for (; at.x < at.seg_end; ++at.x) {
      load();
      if (!__all_sync(0xffffffffu, ptx::bounded_mbar_wait(&arrived[warp][stage], phase, &abort_flag))) {
        if (lane == 0) ba_give_up(p.status, arrived[warp], kStages, stage, phase, ld.x - at.x);
        __syncwarp();
        ok = false;
        return;
      }
      const int valid = at.len - (at.tok0 + (at.x - at.seg_beg) * kBaStep);
      if (valid < kBaStep) {      // the row's last step: zeros for values behind its end, whatever the page holds there
        for (int i = lane; i < kBaStep * kSlabs * 8; i += 32)
          if (i / (kSlabs * 8) >= valid)
            *reinterpret_cast<uint4*>(ring_at + stage * kStage + (kSlabs + i / 8 % kSlabs) * kSlab + i / (kSlabs * 8) * 128 + i % 8 * 16) = make_uint4(0, 0, 0, 0);
        ptx::fence_proxy_async_smem();
      }
      __syncwarp();
      const uint32_t kbase = k_at + stage * kStage, vbase = v_at + stage * kStage;
      float s[TILES][2][4] = {};
      {
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) {
          uint32_t b0, b1, b2, b3;
          ldmatrix_x4((kbase ^ (ks * 2 & 7) << 4) + ks / 4 * kSlab, b0, b1, b2, b3);
#pragma unroll
          for (int t = 0; t < TILES; ++t) {
            mma16816<T>(s[t][0], qa[t][ks][0], qa[t][ks][1], qa[t][ks][2], qa[t][ks][3], b0, b1);
            mma16816<T>(s[t][1], qa[t][ks][0], qa[t][ks][1], qa[t][ks][2], qa[t][ks][3], b2, b3);
          }
        }
      }
      if (p.cap_log2 > 0.f) {
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int e = 0; e < 8; ++e) s[t][e >> 2][e & 3] = p.cap_log2 * ptx::tanh_ex2(s[t][e >> 2][e & 3] * p.cap_scale);
      }
      if (valid < kBaStep) {
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if ((e >> 2) * 8 + 2 * t4 + (e & 1) >= valid) s[t][e >> 2][e & 3] = -INFINITY;
      }
      // The weights' reference: the largest score at first, a later one only where a score is 2^8 above it (weights 256 times as large cost no precision; a maximum that is
      // followed costs four shuffles, and a vote, in every step).
      uint32_t pa[TILES][4];
      float top[TILES][2];
      bool over = false;
#pragma unroll
      for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          top[t][k] = fmaxf(fmaxf(s[t][0][2 * k], s[t][0][2 * k + 1]), fmaxf(s[t][1][2 * k], s[t][1][2 * k + 1]));
          over |= top[t][k] > limit[t][k];
        }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          float a[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float x = fmaxf(top[t][k], __shfl_xor_sync(0xffffffffu, top[t][k], 1));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
            x = fmaxf(x, m[t][k]);
            a[k] = ptx::ex2_approx((m[t][k] - x) * p.scale_log2);
            m[t][k] = x;
            limit[t][k] = x + p.slack;
            l[t][k] *= a[k];
          }
#pragma unroll
          for (int i = 0; i < HD / 8; ++i) {
            o[t][i][0] *= a[0];
            o[t][i][1] *= a[0];
            o[t][i][2] *= a[1];
            o[t][i][3] *= a[1];
          }
        }
      }
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        // (the reference is taken off before the scale: times it a large one is rounded by more than an exponential bears)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const float ref = -m[t][(e >> 1) & 1];
          float* x = &s[t][e >> 2][e & 3];
          const float2 y = ptx::f32x2_get(ptx::fma_f32x2(ptx::add_f32x2(ptx::f32x2(x[0], x[1]), ptx::f32x2(ref, ref)), scale2, small2));
          x[0] = ptx::ex2_approx(y.x);
          x[1] = ptx::ex2_approx(y.y);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) l[t][k] += (s[t][0][2 * k] + s[t][0][2 * k + 1]) + (s[t][1][2 * k] + s[t][1][2 * k + 1]);
        pa[t][0] = pk2<T>(s[t][0][0], s[t][0][1]);
        pa[t][1] = pk2<T>(s[t][0][2], s[t][0][3]);
        pa[t][2] = pk2<T>(s[t][1][0], s[t][1][1]);
        pa[t][3] = pk2<T>(s[t][1][2], s[t][1][3]);
      }
      {
#pragma unroll
        for (int np = 0; np < HD / 16; ++np) {
          uint32_t b0, b1, b2, b3;
          ldmatrix_x4_trans((vbase ^ (np * 2 & 7) << 4) + np / 4 * kSlab, b0, b1, b2, b3);
#pragma unroll
          for (int t = 0; t < TILES; ++t) {
            mma16816<T>(o[t][2 * np], pa[t][0], pa[t][1], pa[t][2], pa[t][3], b0, b1);
            mma16816<T>(o[t][2 * np + 1], pa[t][0], pa[t][1], pa[t][2], pa[t][3], b2, b3);
          }
        }
      }
      __syncwarp();       // the stage is free
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1;
      }
    }
    // the piece's sums: number `range` + segment of this head
    const int64_t slot = shared_part ? (static_cast<int64_t>(hv) * (p.ranges_most + p.groups) + range + at.seg) * kBaTile
                                     : (static_cast<int64_t>(hv) * (p.ranges_most + p.groups * p.per_block) + range + i0) * p.rep;
    float* po = shared_part ? p.o_common : p.o_own;
    float2* pml = shared_part ? p.ml_common : p.ml_own;
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float& sum = l[t][half];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const int i = t * 16 + half * 8 + g8;
        if (i < live) {
          if (t4 == 0) pml[slot + i] = make_float2(m[t][half], sum);
          float* to = po + (slot + i) * HD + 2 * t4;
#pragma unroll
          for (int k = 0; k < HD / 8; ++k) *reinterpret_cast<float2*>(to + k * 8) = make_float2(o[t][k][2 * half], o[t][k][2 * half + 1]);
        }
      }
  };
  while (ok && at.x < x_end) {
    if (at.x >= at.seg_end) enter(at);
    if (at.seg < p.groups && p.per_block * p.rep > 16) piece(std::integral_constant<int, 2>{});
    else piece(std::integral_constant<int, 1>{});
  }
}

// Adds up the pieces of a row and query head: those of its group's common part, then its own.  WARPS of them share one's pieces (few
// rows), or each warp has its own.
template <typename T, int HD, int WARPS>
__global__ void __launch_bounds__(kBaThreads, WARPS > 1 ? 2 : 4) attn_beams_merge_kernel(const BeamAttnParams p) {
  constexpr int kLanes = HD / 4, kTeams = WARPS * 32 / kLanes;      // lanes that hold a row of sums; teams that take every n-th piece
  ptx::griddep_launch_dependents();
  __shared__ float4 part[WARPS > 1 ? kTeams : 1][kLanes];
  const int item = WARPS > 1 ? blockIdx.x : blockIdx.x * kBaWarps + (threadIdx.x >> 5);
  const int tid = WARPS > 1 ? threadIdx.x : threadIdx.x & 31, lane = tid & 31, team = tid / kLanes, c = tid % kLanes;
  const int row = item / p.q_heads, qh = item - row * p.q_heads, head = qh / p.rep;
  const int g = row / p.beams, j = row - g * p.beams, block = j / p.per_block, jb = j - block * p.per_block;
  const int hv = head * p.blocks + block, own = g * p.per_block + jb;
  const int2* runs = p.runs + block * p.groups * (1 + p.per_block);
  ptx::griddep_wait();
  if (item >= p.rows * p.q_heads) return;
  const int2 c_run = runs[g], o_run = runs[p.groups + own];
  const float snk = p.sink ? ldf(reinterpret_cast<const T*>(p.sink) + qh) * 1.4426950408889634f : -INFINITY;
  // (a row without tokens has no own pieces and, where others of its group have tokens, must not have theirs)
  const int pages = p.indptr[row + 1] - p.indptr[row];
  const bool live = pages > 0 && ((pages - 1) << p.page_shift) + p.last_page_len[row] > 0;
  const int n0 = live ? c_run.y : 0, n = live ? n0 + o_run.y : 0;
  const int64_t common = (static_cast<int64_t>(hv) * (p.ranges_most + p.groups) + c_run.x + g) * kBaTile + jb * p.rep + qh - head * p.rep;
  const int64_t mine = (static_cast<int64_t>(hv) * (p.ranges_most + p.groups * p.per_block) + o_run.x + own - n0) * p.rep + qh - head * p.rep;
  auto at = [&](int i) { return i < n0 ? common + i * kBaTile : mine + static_cast<int64_t>(i) * p.rep; };
  auto ml = [&](int i) { return (i < n0 ? p.ml_common : p.ml_own)[at(i)]; };
  auto sums = [&](int i) { return *reinterpret_cast<const float4*>((i < n0 ? p.o_common : p.o_own) + at(i) * HD + 4 * c); };
  // Latency bounds this kernel: as many loads as registers hold are on their way at once, sums before their weights are known.  A lane holds the
  // maxima of every 32nd piece.
  constexpr int kHeld = WARPS > 1 ? 5 : 1, kEarly = 8;
  float2 held[kHeld];
  float4 early[kEarly];
#pragma unroll
  for (int k = 0; k < kHeld; ++k) held[k] = lane + 32 * k < n ? ml(lane + 32 * k) : make_float2(-INFINITY, 0.f);
#pragma unroll
  for (int k = 0; k < kEarly; ++k) early[k] = team + kTeams * k < n ? sums(team + kTeams * k) : make_float4(0.f, 0.f, 0.f, 0.f);
  float M = -INFINITY, L = 0.f;
#pragma unroll
  for (int k = 0; k < kHeld; ++k) M = fmaxf(M, held[k].x);
  for (int i = lane + 32 * kHeld; i < n; i += 32) M = fmaxf(M, ml(i).x);
  M = warp_max(M);
  const float ref = M > -INFINITY ? M : 0.f;
  // weights beside the largest reference, or beside the sink where that is larger
  const float sink_above = snk > -INFINITY ? snk - ref * p.scale_log2 : -INFINITY, less = fmaxf(sink_above, 0.f);
  auto weight = [&](float x) { return ptx::ex2_approx(fmaf(x - ref, p.scale_log2, -less)); };
#pragma unroll
  for (int k = 0; k < kHeld; ++k) {
    held[k].x = weight(held[k].x);
    L += held[k].y * held[k].x;
  }
  for (int i = lane + 32 * kHeld; i < n; i += 32) {
    const float2 x = ml(i);
    L += x.y * weight(x.x);
  }
  L = warp_sum(L) + (p.sink && live ? ptx::ex2_approx(fminf(sink_above, 0.f) - ba_small<T>()) : 0.f);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](const float4& x, float w) {
    acc.x += x.x * w;
    acc.y += x.y * w;
    acc.z += x.z * w;
    acc.w += x.w * w;
  };
#pragma unroll
  for (int k = 0; k < kEarly; ++k) {
    static_assert(kEarly * kTeams <= 32 * kHeld, "the early pieces' maxima are held");
    add(early[k], __shfl_sync(0xffffffffu, held[kTeams * k / 32].x, (team + kTeams * k) & 31));
  }
  for (int i0 = team + kTeams * kEarly; i0 < n; i0 += kTeams * kEarly) {
    float top[kEarly];
#pragma unroll
    for (int k = 0; k < kEarly; ++k) {
      const bool in = i0 + kTeams * k < n;
      top[k] = in ? ml(i0 + kTeams * k).x : -INFINITY;
      early[k] = in ? sums(i0 + kTeams * k) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int k = 0; k < kEarly; ++k) add(early[k], weight(top[k]));
  }
  if constexpr (WARPS > 1) {
    part[team][c] = acc;
    __syncthreads();
    if (team > 0) return;
    for (int i = 1; i < kTeams; ++i) {
      const float4 x = part[i][c];
      acc.x += x.x;
      acc.y += x.y;
      acc.z += x.z;
      acc.w += x.w;
    }
  } else if constexpr (kTeams > 1) {     // (two halves of a warp)
    acc.x += __shfl_xor_sync(0xffffffffu, acc.x, 16);
    acc.y += __shfl_xor_sync(0xffffffffu, acc.y, 16);
    acc.z += __shfl_xor_sync(0xffffffffu, acc.z, 16);
    acc.w += __shfl_xor_sync(0xffffffffu, acc.w, 16);
    if (team > 0) return;
  }
  const float f = live ? 1.f / L : 0.f;      // (live rows without weight: no number)
  stf4(reinterpret_cast<T*>(p.out) + row * p.out_stride + static_cast<int64_t>(qh) * HD + 4 * c, make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f));
}

// How a call is divided, and its scratch.
struct BaPlan {
  int rep, kv_div, per_block, blocks, heads, ranges, rows;       // rows: of a launch
  int64_t runs, ml_common, ml_own, o_common, o_own, bytes;       // offsets
};
static BaPlan ba_plan(int rows, int beams, int q_heads, int kv_heads, int hd) {
  BaPlan b;
  const int group = q_heads / kv_heads;
  b.kv_div = (group + 15) / 16;
  while (group % b.kv_div) ++b.kv_div;
  b.rep = group / b.kv_div;
  const int most = kBaTile / b.rep;
  b.blocks = (beams + most - 1) / most;
  b.per_block = (beams + b.blocks - 1) / b.blocks;
  b.blocks = (beams + b.per_block - 1) / b.per_block;
  b.heads = kv_heads * b.kv_div * b.blocks;
  b.ranges = device_sm_count() * kBaWarps / b.heads;
  if (b.ranges < 1) b.ranges = 1;
  b.rows = kBaRowsMost / beams * beams;
  if (b.rows > rows) b.rows = rows;
  const int64_t groups = b.rows / beams, n_common = b.heads * (b.ranges + groups) * kBaTile, n_own = b.heads * (b.ranges + groups * b.per_block) * b.rep;
  auto up = [](int64_t n) { return (n + 255) / 256 * 256; };
  b.runs = 0;
  b.ml_common = up(8 * b.blocks * groups * (1 + b.per_block));
  b.ml_own = b.ml_common + up(8 * n_common);
  b.o_common = b.ml_own + up(8 * n_own);
  b.o_own = b.o_common + up(4 * n_common * hd);
  b.bytes = b.o_own + up(4 * n_own * hd);
  return b;
}

template <typename T, int HD>
static int ba_launch(const CUtensorMap& tmap, const BeamAttnParams& p, cudaStream_t stream) {
  auto kern = attn_beams_kernel<T, HD>;
  constexpr int kRing = kBaWarps * (HD == 128 ? 2 : 4) * 2 * kBaStep * HD * 2;
  const int per = p.groups * (1 + p.per_block);
  static PerDeviceOnce once;
  cudaError_t e = once.run([&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - 1024); });
  if (e != cudaSuccess) return (int)e;
  const int workers = p.heads * p.ranges_most;
  const size_t smem = 1024 + kRing + 4 * static_cast<size_t>(p.blocks * per + 1 + p.rows + p.blocks * p.groups);
  e = launch_pdl(kern, dim3((workers + kBaWarps - 1) / kBaWarps), dim3(kBaThreads), smem, stream, tmap, p);
  if (e != cudaSuccess) return (int)e;
  const int items = p.rows * p.q_heads;
  // few rows: a block for each, so that the many pieces of a long one are added up by eight warps
  if (items <= 8 * device_sm_count()) return (int)launch_pdl(attn_beams_merge_kernel<T, HD, kBaWarps>, dim3(items), dim3(kBaThreads), 0, stream, p);
  return (int)launch_pdl(attn_beams_merge_kernel<T, HD, 1>, dim3((items + kBaWarps - 1) / kBaWarps), dim3(kBaThreads), 0, stream, p);
}

}  // namespace blitz

extern "C" {
using namespace blitz;

int64_t blitz_attn_beams_workspace_bytes(int rows, int beams, int q_heads, int kv_heads, int head_dim) {
  if (rows < 1 || beams < 1 || beams > 64 || kv_heads < 1 || q_heads < kv_heads) return 256;
  return ba_plan((rows + beams - 1) / beams * beams, beams, q_heads, kv_heads, head_dim).bytes;
}

// kv [max_pages][2][page][kv_heads][head_dim]; rows in groups of `beams`; shared [rows / beams].  page: 16 tokens times a power of two.  cap 0 and sink null: none.
// static_table != 0 promises that indices, indptr, last_page_len and shared are not written by kernels still running in this stream.
int blitz_attn_beams(const void* q, int64_t q_stride, const void* kv, const int32_t* indices, const int32_t* indptr, const int32_t* last_page_len,
                     const int32_t* shared, void* out, int64_t out_stride, void* workspace, int64_t workspace_bytes, int rows, int beams, int q_heads,
                     int kv_heads, int head_dim, int page, int max_pages, float scale, float cap, const void* sink, int static_table, int* status, int dtype,
                     cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (beams < 1 || beams > 64 || rows % beams || kv_heads < 1 || q_heads < 1 || q_heads % kv_heads || (head_dim != 64 && head_dim != 128) || page < 16 ||
      (page & (page - 1)) || max_pages < 1 || static_cast<int64_t>(max_pages) * 2 * page > 0x7fffffff || (q_stride & 7) || (out_stride & 7))
    return -1;
  const BaPlan b = ba_plan(rows, beams, q_heads, kv_heads, head_dim);
  if (workspace_bytes < b.bytes) return -1;
  // a pool as [token of a plane][head][64 columns]; a box is a step's
  CUtensorMap tmap;
  if (!get_tmap_3d(&tmap, kv, head_dim, kv_heads, (uint64_t)max_pages * 2 * page, (uint64_t)head_dim * 2, (uint64_t)head_dim * 2 * kv_heads, 64, 1, kBaStep)) return -2;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  BeamAttnParams p;
  p.q_stride = q_stride; p.kv = kv; p.indices = indices; p.out_stride = out_stride;
  p.beams = beams; p.q_heads = q_heads; p.rep = b.rep; p.kv_div = b.kv_div; p.kv_heads = kv_heads;
  p.per_block = b.per_block; p.blocks = b.blocks; p.heads = b.heads; p.ranges_most = b.ranges;
  p.page_shift = 31 - __builtin_clz(page); p.max_pages = max_pages;
  // scores enter the exponent with the scale's size (largest scores are looked for before it), its sign goes into the queries; under a cap they are log2 already
  const bool plain = !(cap > 0.f);
  p.keep = plain && scale == 0.f ? 0u : ~0u;
  p.flip = plain && scale < 0.f ? 0x80008000u : 0u;
  p.scale_log2 = plain && scale != 0.f ? fabsf(scale) * 1.4426950408889634f : 1.f;
  p.slack = 8.f / p.scale_log2;
  p.cap_scale = cap > 0.f ? scale / cap : 0.f;
  p.cap_log2 = cap * 1.4426950408889634f;
  p.sink = sink;
  p.runs = reinterpret_cast<int2*>(ws + b.runs);
  p.ml_common = reinterpret_cast<float2*>(ws + b.ml_common);
  p.ml_own = reinterpret_cast<float2*>(ws + b.ml_own);
  p.o_common = reinterpret_cast<float*>(ws + b.o_common);
  p.o_own = reinterpret_cast<float*>(ws + b.o_own);
  p.static_table = static_table; p.status = status;
  for (int r = 0; r < rows; r += b.rows) {
    p.rows = rows - r < b.rows ? rows - r : b.rows;
    p.groups = p.rows / beams;
    p.q = static_cast<const uint8_t*>(q) + 2 * r * q_stride;
    p.out = static_cast<uint8_t*>(out) + 2 * r * out_stride;
    p.indptr = indptr + r; p.last_page_len = last_page_len + r; p.shared = shared + r / beams;
    int rc;
    if (dtype == 1) rc = head_dim == 128 ? ba_launch<__nv_bfloat16, 128>(tmap, p, stream) : ba_launch<__nv_bfloat16, 64>(tmap, p, stream);
    else rc = head_dim == 128 ? ba_launch<__half, 128>(tmap, p, stream) : ba_launch<__half, 64>(tmap, p, stream);
    if (rc) return rc;
  }
  return 0;
}

}  // extern "C"
