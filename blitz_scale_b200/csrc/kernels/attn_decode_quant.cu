// Decode attention over a paged cache held in 4 bits (the format: quant_kv.cuh).
//
// One query token per sequence: o = sum_j p_j v_j, p = softmax_j(scale q.k_j), a stream over the sequence's codes and scales, which the
// tensor cores (mma.sync, m16n8k16) turn into products without ever forming a key or a value.  With k_d = z_g + s_g c_d for dimension d
// of group g:
//
//   q.k = sum_g s_g (sum_{d in g} q_d c_d) + z_g (sum_{d in g} q_d)
//   o_d = sum_j (p_j s_j) (c_jd - 8) + sum_j p_j (z_j + 8 s_j)
//
// A code becomes a 16-bit float by one mask and one "or" into the mantissa of a power of two, which adds a constant:
// keys: 1024 + c and 64 + c in fp16 (two nibbles a shift), the constants' part of the product is the accumulator's initial value;
// values: 128 + c in bf16, and a product of the weights with a constant matrix takes 136 off again (the codes around zero, so that
// the rounding of p_j s_j is not amplified by an offset that cancels).  Queries enter in fp16, a head divided by a power of two near its
// largest entry: bf16 and fp16 numbers are exact there (next to the largest, that is), and so are their products with codes.  p s is
// rounded to bf16 (its range is the scales'), as in attention over 16-bit caches; in fp16 models to two bf16 numbers, hi + lo.  The part
// of z_j stays in 32 bits; sum q_d z_g of the scores is one more product, of z as stored with sums of q in two bf16 numbers.
//
// S = Q K^T has queries as rows (at most 8 per KV head, 8 rows of padding), so that its accumulators hold a head's weights of neighbouring
// tokens as the second product, V^T P^T with dimensions as rows, wants them.  Scales of K multiply the accumulators of a group, scales of V
// the weights of a group.
//
// A warp takes chunks of 32 tokens by itself: a bulk copy (one contiguous piece of the cache) into its own ring of stages, no
// barrier but the copy's.  Four warps are a team, which takes a piece of a sequence (chunks dealt in turn) for one KV head and adds up what
// they have through shared memory at its end.  Three teams on an SM.
//
// Pieces.  num_splits = 1: whole (sequence, KV head) items, dealt to the teams.  Otherwise the chunks of all sequences, end to end, are cut
// into equal ranges, one per team and KV head; a range's first and last sequence may be incomplete, and whoever finishes a sequence's last
// piece adds them up (in the order of the ranges).
#include "launch.cuh"
#include "ptx.cuh"
#include "mma.cuh"
#include "quant_kv.cuh"
#include "scalar.cuh"
#include "tmap.cuh"

namespace blitz {

constexpr int kQdTeams = 3, kQdWarps = 4, kQdStages = 3, kQdThreads = kQdTeams * kQdWarps * 32;
constexpr int kQdChunk = 32;
constexpr int kQdMaxShared = 1024;  // sequences whose chunks can be dealt out
constexpr int kQdRow = 68;          // floats from head to head in the merge buffer: 64 and what keeps a warp's writes in different banks

struct DecodeQuantParams {
  const void* q;
  int64_t q_stride;
  const uint8_t* pool;
  const int32_t *indices, *indptr, *last_page_len;
  void* out;
  int64_t out_stride;
  unsigned* tickets;   // [batch][heads] pieces finished, zero between launches
  float* part;         // [2 teams][8 heads][D] sums, then [2 teams][8] of (maximum, sum of weights)
  int batch, kv_heads, heads, div, rep;  // heads: groups of at most 8 query heads, div of which share a KV head; rep: query heads of one
  int page_size, page_shift, max_pages, whole, static_table;
  float scale_log2, cap_scale, cap_log2;
  int window, keep_first;
  const void* sink;
  int* status;
};

template <int D, int GROUP>
struct QdCfg {
  static constexpr int kStage = 2 * quant_kv(D, GROUP).block;
  static constexpr int kRing = kQdStages * kStage;
  static constexpr int G = D / GROUP;
  static constexpr int kMergeFloats = kQdWarps * (8 * kQdRow + 16 + 8 * G);  // of a team: sums of 64 dimensions; m, l; offsets' sums
  static constexpr int kSmem = kQdTeams * (kQdWarps * kRing + kMergeFloats * 4) + (kQdMaxShared + 2 + kQdTeams) * 4 + kQdTeams * kQdWarps * kQdStages * 8;
};

struct QdPiece {
  int b, head, pg_beg, len, beg, end, all;  // chunks beg .. end of the visible chunks, of `all`
  int lo, first, n_first, c_window;         // visible keys: [0, first) and [lo, len); chunks of the former; first chunk of the latter
  int part;                                 // -1: the whole item
  __device__ __forceinline__ int token(int n) const { return (n < n_first ? n : c_window + n - n_first) * kQdChunk; }
};
__device__ __forceinline__ void qd_sequence(const DecodeQuantParams& p, int b, QdPiece& it) {
  it.b = b;
  it.pg_beg = p.indptr[b];
  const int pages = p.indptr[b + 1] - it.pg_beg;
  it.len = pages > 0 ? (pages - 1) * p.page_size + min(max(p.last_page_len[b], 0), p.page_size) : 0;
  it.lo = p.window > 0 ? max(0, it.len - p.window) : 0;
  it.first = min(p.keep_first, it.lo);
  it.n_first = (it.first + kQdChunk - 1) / kQdChunk;
  it.c_window = max(it.lo / kQdChunk, it.n_first);
  it.all = it.n_first + max(0, (it.len + kQdChunk - 1) / kQdChunk - it.c_window);
}
struct QdWalk {
  int x, end;   // items, or chunks of a range
  int b;        // (of a range) sequence of chunk x
  int first;    // nothing has been taken from the range yet
};
__device__ __forceinline__ unsigned qd_ranges(const DecodeQuantParams& p, unsigned chunks, unsigned teams) {
  return min((chunks + kQdWarps - 1) / kQdWarps, teams / static_cast<unsigned>(p.heads));
}
__device__ __forceinline__ int qd_begin(unsigned r, unsigned chunks, unsigned ranges) { return static_cast<int>(static_cast<uint64_t>(chunks) * r / ranges); }
__device__ __forceinline__ int qd_range_of(unsigned x, unsigned chunks, unsigned ranges) {
  return static_cast<int>(((static_cast<uint64_t>(x) + 1) * ranges + chunks - 1) / chunks) - 1;
}
__device__ __forceinline__ QdWalk qd_walk(const DecodeQuantParams& p, const int* before, int team, int teams) {
  QdWalk w{team, p.batch * p.heads, 0, 1};
  if (!p.whole) {
    const int chunks = before[p.batch], ranges = qd_ranges(p, chunks, teams), r = team / p.heads;
    w.x = w.end = 0;
    if (r < ranges) {
      w.x = qd_begin(r, chunks, ranges);
      w.end = qd_begin(r + 1, chunks, ranges);
      int lo = 0, hi = p.batch - 1;  // the last sequence that starts at or before x
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (before[mid] <= w.x) lo = mid;
        else hi = mid - 1;
      }
      w.b = lo;
    }
  }
  return w;
}
__device__ __forceinline__ bool qd_next(const DecodeQuantParams& p, const int* before, int team, int teams, QdWalk& w, QdPiece& it) {
  if (w.x >= w.end) return false;
  if (p.whole) {
    it.head = w.x % p.heads;
    qd_sequence(p, w.x / p.heads, it);
    it.beg = 0;
    it.end = it.all;
    it.part = -1;
    w.x += teams;
  } else {
    while (before[w.b + 1] <= w.x) ++w.b;
    qd_sequence(p, w.b, it);
    it.head = team % p.heads;
    it.beg = w.x - before[w.b];
    it.end = min(it.all, it.beg + w.end - w.x);
    it.part = it.end - it.beg == it.all ? -1 : team * 2 + (w.first ? 0 : 1);
    w.x += it.end - it.beg;
    w.first = 0;
  }
  return true;
}

// d = a b + (c0, c0, 0, 0): rows 8..15 of a are zero.
__device__ __forceinline__ void qd_mma_f16(float (&d)[4], uint32_t a0, uint32_t a2, uint32_t b0, uint32_t b1, float c0) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%5}, {%7,%8}, {%9,%9,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(0u), "r"(a2), "r"(b0), "r"(b1), "f"(c0), "f"(0.f));
}
__device__ __forceinline__ void qd_mma_f16_add(float (&d)[4], uint32_t a0, uint32_t a2, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%5}, {%7,%8}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(0u), "r"(a2), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void qd_mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// bf16 number `i` of consecutive ones.
template <int N>
__device__ __forceinline__ float qd_bf16(const uint32_t (&w)[N], int i) {
  return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
}

template <typename T, int D, int GROUP>
__global__ void __launch_bounds__(kQdThreads, 1) attn_decode_quant_kernel(const __grid_constant__ DecodeQuantParams p) {
  using Cfg = QdCfg<D, GROUP>;
  constexpr QuantKv F = quant_kv(D, GROUP);
  constexpr int G = D / GROUP, W = D / 32, WG = GROUP / 32, MT = D / 16;
  constexpr bool kTwo = std::is_same<T, __half>::value;  // weights as two bf16 numbers
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int local = warp / kQdWarps, w4 = warp % kQdWarps, tid = threadIdx.x % (kQdWarps * 32);
  uint8_t* ring = smem + warp * Cfg::kRing;
  float* mrg = reinterpret_cast<float*>(smem + kQdTeams * kQdWarps * Cfg::kRing) + local * Cfg::kMergeFloats;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kQdTeams * (kQdWarps * Cfg::kRing + Cfg::kMergeFloats * 4));
  uint64_t* full = bars + warp * kQdStages;
  int* before = reinterpret_cast<int*>(bars + kQdTeams * kQdWarps * kQdStages);  // [batch + 1] chunks of the sequences before each
  volatile int* abort_flag = before + kQdMaxShared + 1;
  volatile int* last_piece = abort_flag + 1;  // [team]
  const int teams = kQdTeams * static_cast<int>(gridDim.x), team = local * static_cast<int>(gridDim.x) + static_cast<int>(blockIdx.x);

  if (threadIdx.x < kQdTeams * kQdWarps * kQdStages) ptx::mbar_init(&bars[threadIdx.x], 1);
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  ptx::fence_proxy_async_smem();
  ptx::griddep_launch_dependents();
  if (!p.static_table) ptx::griddep_wait();
  if (!p.whole) {
    QdPiece seq;
    for (int b = threadIdx.x; b < p.batch; b += kQdThreads) {
      qd_sequence(p, b, seq);
      before[b + 1] = seq.all;
    }
    __syncthreads();
    if (warp == 0) {
      const int each = (p.batch + 31) / 32, b0 = min(p.batch, lane * each), b1 = min(p.batch, b0 + each);
      int sum = 0;
      for (int b = b0; b < b1; ++b) sum += before[b + 1];
      int total = sum;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, total, d);
        if (lane >= d) total += up;
      }
      int run = total - sum;
      if (lane == 0) before[0] = 0;
      for (int b = b0; b < b1; ++b) {
        run += before[b + 1];
        before[b + 1] = run;
      }
    }
  }
  __syncthreads();
  ptx::griddep_wait();

  T* const out = reinterpret_cast<T*>(p.out);
  if (!p.whole)  // sequences without a visible key are in nobody's range: their output is zero
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x)
      if (before[b] == before[b + 1])
        for (int e = threadIdx.x; e < p.heads * p.rep * D; e += kQdThreads) stf(out + b * p.out_stride + e, 0.f);

  auto meet = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(1 + local), "n"(kQdWarps * 32) : "memory"); };

  // ---------------------------------------------------------------- the copies, ahead of the products
  QdWalk ahead = qd_walk(p, before, team, teams);
  QdPiece ip{};
  int ic = 0, pieces_ahead = 0, issued = 0, taken = 0;
  bool more_ahead = qd_next(p, before, team, teams, ahead, ip);
  if (more_ahead) ic = ip.beg + w4;
  // (page ids of the chunk that is requested next: asked for one chunk earlier)
  int page0 = 0, page1 = 0;
  auto look = [&]() {
    while (more_ahead && ic >= ip.end) {
      more_ahead = qd_next(p, before, team, teams, ahead, ip);
      ++pieces_ahead;
      ic = ip.beg + ((w4 + pieces_ahead) & (kQdWarps - 1));
    }
    if (!more_ahead) return;
    const int tok = ip.token(ic);
    page0 = p.indices[ip.pg_beg + (tok >> p.page_shift)];
    if (p.page_shift == 4) page1 = tok + 16 < ip.len ? p.indices[ip.pg_beg + (tok >> 4) + 1] : page0;
  };
  auto request = [&]() {
    if (!more_ahead) return;
    if (lane == 0) {
      const int tok = ip.token(ic), stage = issued % kQdStages, blocks = min(kQdChunk, ip.len - tok + 15) >> 4;
      int pg[2] = {page0, page1};
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (pg[i] < 0 || pg[i] >= p.max_pages) {
          if (p.status && (i == 0 || p.page_shift == 4)) atomicCAS(p.status, 0, kStatusBadIndex);
          pg[i] = 0;
        }
      const int kv = ip.head / p.div;
      auto block = [&](int page, int off) { return p.pool + (((static_cast<int64_t>(page) * p.kv_heads + kv) << (p.page_shift - 4)) + (off >> 4)) * F.block; };
      uint8_t* to = ring + stage * Cfg::kStage;
      ptx::mbar_expect_tx(&full[stage], blocks * F.block);
      if (p.page_shift == 4) {
        ptx::bulk_load_1d(to, block(pg[0], 0), F.block, &full[stage]);
        if (blocks > 1) ptx::bulk_load_1d(to + F.block, block(pg[1], 0), F.block, &full[stage]);
      } else {
        ptx::bulk_load_1d(to, block(pg[0], tok & (p.page_size - 1)), blocks * F.block, &full[stage]);
      }
    }
    ++issued;
    ic += kQdWarps;
    look();
  };
  look();
#pragma unroll
  for (int i = 0; i < kQdStages; ++i) request();

  // ---------------------------------------------------------------- the products
  QdWalk walk = qd_walk(p, before, team, teams);
  QdPiece it{};
  bool ok = true;
  for (int piece = 0; qd_next(p, before, team, teams, walk, it); ++piece) {
    // queries: word w of a lane's key codes holds dimensions 32 w + 8 t4 .. + 7, pairs (i, i + 4) of which are a register's halves
    uint32_t qa[W][4], zq = 0;
    float qc[G], to_log2;
    {
      float x[W][8], most = 0.f;
      const T* row = reinterpret_cast<const T*>(p.q) + it.b * p.q_stride + static_cast<int64_t>(it.head * p.rep + g) * D + 8 * t4;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (g < p.rep) {
          ldf8<T>(row + 32 * w, x[w]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[w][i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(x[w][i]));
      }
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      // 2^-e with most in [2^e, 2^(e + 1)); an all-zero head, and one that is not finite, as it is
      const int e = most > 0.f && most <= 3.4e38f ? max(-126, min(126, static_cast<int>(__float_as_uint(most) >> 23) - 127)) : 0;
      const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      to_log2 = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      float sum[G];
#pragma unroll
      for (int gr = 0; gr < G; ++gr) sum[gr] = qc[gr] = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        float r[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          qa[w][i] = pk2<__half>(x[w][i] * down, x[w][i + 4] * down);
          const float2 f = cvt2<__half>(qa[w][i]);  // (as they enter the products)
          r[i] = f.x;
          r[i + 4] = f.y;
        }
        // the zero of a register's codes: 1024 in the first and third pair, 64 in the others
        sum[w / WG] += ((r[0] + r[4]) + (r[1] + r[5])) + ((r[2] + r[6]) + (r[3] + r[7]));
        qc[w / WG] -= 1024.f * ((r[0] + r[4]) + (r[2] + r[6])) + 64.f * ((r[1] + r[5]) + (r[3] + r[7]));
      }
      float hi[G], lo[G];
#pragma unroll
      for (int gr = 0; gr < G; ++gr) {
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
          sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], d);
          qc[gr] += __shfl_xor_sync(0xffffffffu, qc[gr], d);
        }
        hi[gr] = __bfloat162float(__float2bfloat16_rn(sum[gr]));
        lo[gr] = sum[gr] - hi[gr];
      }
      // row operand of the offsets' product: pairs of numbers as the scales' words of a token have them
      if (G == 4) zq = t4 == 0 ? pk2<__nv_bfloat16>(hi[0], hi[1 % G]) : t4 == 1 ? pk2<__nv_bfloat16>(hi[2 % G], hi[3 % G]) : t4 == 2 ? pk2<__nv_bfloat16>(lo[0], lo[1 % G]) : pk2<__nv_bfloat16>(lo[2 % G], lo[3 % G]);
      if (G == 2) zq = t4 == 0 ? pk2<__nv_bfloat16>(hi[0], hi[1 % G]) : t4 == 1 ? pk2<__nv_bfloat16>(lo[0], lo[1 % G]) : 0u;
      if (G == 1) zq = t4 == 0 ? pk2<__nv_bfloat16>(0.f, hi[0]) : t4 == 1 ? pk2<__nv_bfloat16>(0.f, lo[0]) : 0u;
    }
    const float scale = p.scale_log2 * to_log2, cap_in = p.cap_scale * to_log2;

    float o[MT][4], oc[G][4], zs[G], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int i = 0; i < MT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
    for (int i = 0; i < G; ++i) oc[i][0] = oc[i][1] = oc[i][2] = oc[i][3] = zs[i] = 0.f;

    for (int c = it.beg + ((w4 + piece) & (kQdWarps - 1)); c < it.end; c += kQdWarps) {
      const int stage = taken % kQdStages;
      if (ok && !ptx::bounded_mbar_wait(&full[stage], (taken / kQdStages) & 1, abort_flag)) {
        if (p.status && lane == 0) atomicCAS(p.status, 0, kStatusTimeoutProducer);
        ok = false;
      }
      if (ok) {
        const uint8_t* st = ring + stage * Cfg::kStage;
        const int tok0 = it.token(c), blocks = min(kQdChunk, it.len - tok0 + 15) >> 4;
        const bool edge = tok0 + kQdChunk > it.len || (tok0 < it.lo && tok0 + kQdChunk > it.first);  // some key is not visible
        float s[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          s[u][0] = s[u][1] = s[u][2] = s[u][3] = -INFINITY;
          if (u < blocks) {
            const uint8_t* kb = st + u * F.block;
            const uint8_t* sw = kb + F.codes;
            uint32_t sc[4 * G];  // scales and offsets of the lane's four tokens, 4 t4 ..
#pragma unroll
            for (int i = 0; i < G; ++i) {
              const uint4 v = *reinterpret_cast<const uint4*>(sw + t4 * 16 * G + 16 * i);
              sc[4 * i] = v.x; sc[4 * i + 1] = v.y; sc[4 * i + 2] = v.z; sc[4 * i + 3] = v.w;
            }
#pragma unroll
            for (int odd = 0; odd < 2; ++odd) {
              const int tau = 4 * (g >> 1) + (g & 1) + 2 * odd;  // the key that this lane brings to the product
              uint32_t kw[W];
              if (W == 4) {
                const uint4 v = *reinterpret_cast<const uint4*>(kb + tau * 64 + t4 * 16);
                kw[0] = v.x; kw[1] = v.y; kw[2 % W] = v.z; kw[3 % W] = v.w;
              } else {
                const uint2 v = *reinterpret_cast<const uint2*>(kb + tau * 32 + t4 * 8);
                kw[0] = v.x; kw[1] = v.y;
              }
              const uint32_t zw = *reinterpret_cast<const uint32_t*>(sw + tau * 4 * G + (G == 4 ? 8 + 4 * (t4 & 1) : G == 2 ? 4 : 0));
              float zp[4] = {0.f, 0.f, 0.f, 0.f};
              qd_mma_bf16(zp, zq, 0u, 0u, 0u, zw, 0u);
              float s0 = zp[0], s1 = zp[1];
#pragma unroll
              for (int gr = 0; gr < G; ++gr) {
                float acc[4];
#pragma unroll
                for (int w = gr * WG; w < (gr + 1) * WG; ++w) {
                  const uint32_t x = kw[w], y = x >> 8;
                  const uint32_t b0 = (x & 0x000f000fu) | 0x64006400u, b1 = (x & 0x00f000f0u) | 0x54005400u;
                  const uint32_t b2 = (y & 0x000f000fu) | 0x64006400u, b3 = (y & 0x00f000f0u) | 0x54005400u;
                  if (w == gr * WG) qd_mma_f16(acc, qa[w][0], qa[w][1], b0, b1, qc[gr]);
                  else qd_mma_f16_add(acc, qa[w][0], qa[w][1], b0, b1);
                  qd_mma_f16_add(acc, qa[w][2], qa[w][3], b2, b3);
                }
                s0 = fmaf(qd_bf16(sc, 2 * odd * 2 * G + gr), acc[0], s0);
                s1 = fmaf(qd_bf16(sc, (2 * odd + 1) * 2 * G + gr), acc[1], s1);
              }
              s[u][2 * odd] = s0;
              s[u][2 * odd + 1] = s1;
            }
          }
        }
        // scores in log2 units, and which of them count
        uint32_t seen = 0xff;
        if (edge) {
          seen = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int j = tok0 + (i >> 2) * 16 + 4 * t4 + (i & 3);
            if (j < it.len && (j >= it.lo || j < it.first)) seen |= 1u << i;
          }
        }
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float& x = s[i >> 2][i & 3];
          x = p.cap_log2 > 0.f ? p.cap_log2 * ptx::tanh_ex2(x * cap_in) : x * scale;
          if (edge && !((seen >> i) & 1u)) x = -INFINITY;
          top = fmaxf(top, x);
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (__any_sync(0xffffffffu, top > m)) {
          const float m_new = fmaxf(m, top), a = m_new > m ? ptx::ex2_approx(m - m_new) : 1.f;
          m = m_new;
          l *= a;
          const float a0 = __shfl_sync(0xffffffffu, a, 8 * t4), a1 = __shfl_sync(0xffffffffu, a, 8 * t4 + 4);  // of heads 2 t4, 2 t4 + 1
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            o[i][0] *= a0; o[i][1] *= a1; o[i][2] *= a0; o[i][3] *= a1;
          }
#pragma unroll
          for (int i = 0; i < G; ++i) {
            zs[i] *= a;
            oc[i][0] *= a0; oc[i][1] *= a1;
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float& x = s[i >> 2][i & 3];
          x = edge && !((seen >> i) & 1u) ? 0.f : ptx::ex2_approx(x - m);
          l += x;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (u < blocks) {
            const uint8_t* vb = st + u * F.block + F.part;
            uint32_t sc[4 * G];
#pragma unroll
            for (int i = 0; i < G; ++i) {
              const uint4 v = *reinterpret_cast<const uint4*>(vb + F.codes + t4 * 16 * G + 16 * i);
              sc[4 * i] = v.x; sc[4 * i + 1] = v.y; sc[4 * i + 2] = v.z; sc[4 * i + 3] = v.w;
            }
            if (edge) {  // (what is not visible may hold no numbers)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (!((seen >> (4 * u + i)) & 1u)) {
#pragma unroll
                  for (int k = 0; k < G; ++k) sc[i * G + k] = 0u;
                }
            }
            uint32_t vw[MT];
#pragma unroll
            for (int h = 0; h < D / 64; ++h) {
              const uint4 v = *reinterpret_cast<const uint4*>(vb + h * 512 + g * 64 + t4 * 16);
              vw[4 * h] = v.x; vw[4 * h + 1] = v.y; vw[4 * h + 2] = v.z; vw[4 * h + 3] = v.w;
            }
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
              float ps[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                ps[i] = s[u][i] * qd_bf16(sc, i * 2 * G + gr);
                zs[gr] = fmaf(s[u][i], qd_bf16(sc, i * 2 * G + G + gr), fmaf(8.f, ps[i], zs[gr]));
              }
              uint32_t b0 = pk2<__nv_bfloat16>(ps[0], ps[1]), b1 = pk2<__nv_bfloat16>(ps[2], ps[3]), c0 = 0, c1 = 0;
              if (kTwo) {
                const float2 x = cvt2<__nv_bfloat16>(b0), y = cvt2<__nv_bfloat16>(b1);
                c0 = pk2<__nv_bfloat16>(ps[0] - x.x, ps[1] - x.y);
                c1 = pk2<__nv_bfloat16>(ps[2] - y.x, ps[3] - y.y);
              }
              constexpr uint32_t kOff = 0xc308c308u;  // -136
              qd_mma_bf16(oc[gr], kOff, kOff, kOff, kOff, b0, b1);
              if (kTwo) qd_mma_bf16(oc[gr], kOff, kOff, kOff, kOff, c0, c1);
#pragma unroll
              for (int i = gr * (GROUP / 16); i < (gr + 1) * (GROUP / 16); ++i) {
                const uint32_t x = vw[i];
                const uint32_t a0 = (x & 0x000f000fu) | 0x43004300u, a1 = ((x >> 4) & 0x000f000fu) | 0x43004300u;
                const uint32_t a2 = ((x >> 8) & 0x000f000fu) | 0x43004300u, a3 = ((x >> 12) & 0x000f000fu) | 0x43004300u;
                qd_mma_bf16(o[i], a0, a1, a2, a3, b0, b1);
                if (kTwo) qd_mma_bf16(o[i], a0, a1, a2, a3, c0, c1);
              }
            }
          }
        }
        __syncwarp();  // every lane has read the stage
      }
      ++taken;
      if (ok) request();
    }

    // ---------------------------------------------------------------- the team adds up
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    float* ml = mrg + kQdWarps * 8 * kQdRow;  // [warp][8] maxima, [warp][8] sums, [warp][8][G]
    float* zo = ml + kQdWarps * 16;
    if (t4 == 0) {
      ml[w4 * 8 + g] = m;
      ml[kQdWarps * 8 + w4 * 8 + g] = l;
    }
#pragma unroll
    for (int i = 0; i < G; ++i) {
      zs[i] += __shfl_xor_sync(0xffffffffu, zs[i], 1);
      zs[i] += __shfl_xor_sync(0xffffffffu, zs[i], 2);
      if (t4 == 0) zo[(w4 * 8 + g) * G + i] = zs[i];
    }
    const int hh = tid >> 4, d4 = (tid & 15) * 4;  // head and four of 64 dimensions that this thread adds up
    const int head = it.head * p.rep + hh;
    float* const part = p.part + (static_cast<int64_t>(max(it.part, 0)) * 8 + hh) * D;
    float* const part_ml = p.part + static_cast<int64_t>(2 * teams) * 8 * D;
    const float snk = p.sink && hh < p.rep ? to_f<T>(reinterpret_cast<const T*>(p.sink)[head]) * 1.4426950408889634f : -INFINITY;
#pragma unroll
    for (int h = 0; h < D / 64; ++h) {
      float* row = mrg + (w4 * 8 + 2 * t4) * kQdRow + g;
#pragma unroll
      for (int i = 4 * h; i < 4 * h + 4; ++i) {
        const int gr = i * 16 / GROUP, at = (i - 4 * h) * 16;
        row[at] = o[i][0] + oc[gr][0];
        row[at + kQdRow] = o[i][1] + oc[gr][1];
        row[at + 8] = o[i][2] + oc[gr][0];
        row[at + 8 + kQdRow] = o[i][3] + oc[gr][1];
      }
      meet();
      float M = -INFINITY, L = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kQdWarps; ++w) M = fmaxf(M, ml[w * 8 + hh]);
#pragma unroll
      for (int w = 0; w < kQdWarps; ++w) {
        const float mw = ml[w * 8 + hh], f = mw == M ? 1.f : exp2f(mw - M);  // (no maximum at all: nothing to add)
        L = fmaf(f, ml[kQdWarps * 8 + w * 8 + hh], L);
        const float4 v = *reinterpret_cast<const float4*>(mrg + (w * 8 + hh) * kQdRow + d4);
        const float z = zo[(w * 8 + hh) * G + (64 * h + d4) / GROUP];
        acc[0] = fmaf(f, v.x + z, acc[0]);
        acc[1] = fmaf(f, v.y + z, acc[1]);
        acc[2] = fmaf(f, v.z + z, acc[2]);
        acc[3] = fmaf(f, v.w + z, acc[3]);
      }
      if (it.part < 0) {
        if (hh < p.rep) {
          const float top = fmaxf(M, snk), f = M == top ? 1.f : exp2f(M - top), sum = fmaf(f, L, snk > -INFINITY ? exp2f(snk - top) : 0.f);
          const float r = sum != 0.f ? f / sum : 0.f;
          stf4<T>(out + it.b * p.out_stride + static_cast<int64_t>(head) * D + 64 * h + d4, make_float4(acc[0] * r, acc[1] * r, acc[2] * r, acc[3] * r));
        }
      } else {
        __stcg(reinterpret_cast<float4*>(part + 64 * h + d4), make_float4(acc[0], acc[1], acc[2], acc[3]));
        if (h == 0 && (tid & 15) == 0) __stcg(reinterpret_cast<float2*>(part_ml) + static_cast<int64_t>(it.part) * 8 + hh, make_float2(M, L));
      }
      meet();
    }
    if (it.part < 0) continue;

    // ---------------------------------------------------------------- and whoever ends a sequence adds up its pieces
    const int chunks = before[p.batch], ranges = qd_ranges(p, chunks, teams), start = before[it.b];
    const int r0 = qd_range_of(start, chunks, ranges), r1 = qd_range_of(start + it.all - 1, chunks, ranges);
    __threadfence();
    meet();
    if (tid == 0) {
      unsigned* ticket = p.tickets + it.b * p.heads + it.head;
      const bool is_last = atomicAdd(ticket, 1u) == static_cast<unsigned>(r1 - r0);
      if (is_last) *ticket = 0u;
      last_piece[local] = is_last;
    }
    meet();
    if (!last_piece[local]) continue;
    __threadfence();
    if (hh < p.rep) {
      // (a range's first piece is in its team's first place)
      auto place = [&](int r) { return static_cast<int64_t>((r * p.heads + it.head) * 2 + (qd_begin(r, chunks, ranges) >= start ? 0 : 1)) * 8 + hh; };
      float M = snk;
      for (int r = r0; r <= r1; ++r) M = fmaxf(M, __ldcg(reinterpret_cast<const float2*>(part_ml) + place(r)).x);
      float sum = snk > -INFINITY ? exp2f(snk - M) : 0.f, acc[D / 16];
#pragma unroll
      for (int i = 0; i < D / 16; ++i) acc[i] = 0.f;
#pragma unroll 2
      for (int r = r0; r <= r1; ++r) {
        const int64_t at = place(r);
        const float2 v = __ldcg(reinterpret_cast<const float2*>(part_ml) + at);
        const float f = v.x == M ? 1.f : exp2f(v.x - M);
        sum = fmaf(f, v.y, sum);
#pragma unroll
        for (int h = 0; h < D / 64; ++h) {
          const float4 x = __ldcg(reinterpret_cast<const float4*>(p.part + at * D + 64 * h + d4));
          acc[4 * h] = fmaf(f, x.x, acc[4 * h]);
          acc[4 * h + 1] = fmaf(f, x.y, acc[4 * h + 1]);
          acc[4 * h + 2] = fmaf(f, x.z, acc[4 * h + 2]);
          acc[4 * h + 3] = fmaf(f, x.w, acc[4 * h + 3]);
        }
      }
      const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
      for (int h = 0; h < D / 64; ++h)
        stf4<T>(out + it.b * p.out_stride + static_cast<int64_t>(head) * D + 64 * h + d4,
                make_float4(acc[4 * h] * inv, acc[4 * h + 1] * inv, acc[4 * h + 2] * inv, acc[4 * h + 3] * inv));
    }
  }
  // (after a time-out: no copy may land in shared memory that another block has by then)
  for (; taken < issued; ++taken) ptx::bounded_mbar_wait(&full[taken % kQdStages], (taken / kQdStages) & 1, abort_flag);
}

struct DecodeQuantLaunch {
  const DecodeQuantParams& p;
  int sms;
  cudaStream_t stream;
  template <typename T, int D, int GROUP>
  int operator()() const {
    constexpr int smem = QdCfg<D, GROUP>::kSmem;
    static_assert(smem <= 232448, "more shared memory than a block may have");
    static PerDeviceOnce once;
    const cudaError_t e = once.run([&] { return cudaFuncSetAttribute(attn_decode_quant_kernel<T, D, GROUP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); });
    if (e != cudaSuccess) return (int)e;
    return (int)launch_pdl(attn_decode_quant_kernel<T, D, GROUP>, dim3(sms), dim3(kQdThreads), smem, stream, p);
  }
};

// Query heads in equal groups of at most 8 that share a KV head.
static inline int qd_groups(int rep) {
  int div = (rep + 7) / 8;
  while (rep % div) ++div;
  return div;
}

}  // namespace blitz

extern "C" {
using namespace blitz;

// Scratch of a call: tickets, which have to be zero before the first call and are again after each, then partial sums.
int64_t blitz_attn_decode_quant_workspace_bytes(int batch, int q_heads, int dim) {
  const int64_t teams = (int64_t)device_sm_count() * kQdTeams;
  return ((int64_t)batch * q_heads * 4 + 255) / 256 * 256 + 2 * teams * 8 * (dim + 2) * 4;
}

// q: [batch] rows with the query heads in their first q_heads * dim columns (pitch a multiple of 8, 16-byte aligned; so out).  A sequence
// without keys has an output of zeros.  num_splits = 1: sequences whole; otherwise equal shares of all chunks (up to 1024 sequences of as
// many heads as there are teams).  static_table != 0 promises that the tables are not written by kernels still running in this stream.
int blitz_attn_decode_quant(const void* q, int64_t q_stride, const void* pool, const int32_t* indices, const int32_t* indptr,
                            const int32_t* last_page_len, void* out, int64_t out_stride, void* workspace, int64_t workspace_bytes, int batch,
                            int q_heads, int kv_heads, int dim, int group, int page_size, int max_pages, int num_splits, float sm_scale, int window,
                            int keep_first, float softcap, const void* sink, int static_table, int* status, int dtype, cudaStream_t stream) {
  if (batch <= 0) return 0;
  if (!quant_kv_supported(dim, group, page_size) || kv_heads < 1 || q_heads % kv_heads || window < 0 || keep_first < 0 || softcap < 0.f) return -1;
  if (((q_stride | out_stride) & 7) || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(pool) | reinterpret_cast<uintptr_t>(workspace)) & 15)) return -1;
  const int sms = device_sm_count(), teams = sms * kQdTeams;
  DecodeQuantParams p;
  p.q = q; p.q_stride = q_stride; p.pool = (const uint8_t*)pool; p.indices = indices; p.indptr = indptr; p.last_page_len = last_page_len;
  p.out = out; p.out_stride = out_stride;
  p.div = qd_groups(q_heads / kv_heads); p.rep = q_heads / kv_heads / p.div; p.heads = kv_heads * p.div; p.kv_heads = kv_heads; p.batch = batch;
  p.whole = num_splits == 1 || batch > kQdMaxShared || p.heads > teams;
  if (!p.whole && (workspace == nullptr || workspace_bytes < blitz_attn_decode_quant_workspace_bytes(batch, q_heads, dim))) return -1;
  p.tickets = (unsigned*)workspace;
  p.part = workspace ? (float*)((char*)workspace + ((int64_t)batch * q_heads * 4 + 255) / 256 * 256) : nullptr;
  p.page_size = page_size; p.max_pages = max_pages; p.page_shift = 0;
  while ((1 << p.page_shift) < page_size) ++p.page_shift;
  p.scale_log2 = sm_scale * 1.4426950408889634f; p.cap_scale = softcap > 0.f ? sm_scale / softcap : 0.f; p.cap_log2 = softcap * 1.4426950408889634f;
  p.window = window; p.keep_first = keep_first; p.sink = sink; p.static_table = static_table; p.status = status;
  return quant_kv_dispatch(dtype, dim, group, DecodeQuantLaunch{p, sms, stream});
}

}  // extern "C"
