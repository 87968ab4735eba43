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
// A block takes a chunk of a row of logits: the sum of exponentials, and the chunk's n largest logits (those of a row order its values).
// The second kernel, a block per request, adds up the sums, turns logits into values and orders them in 64 bits: candidates of
// different beams may be nearer to one another than fp32 tells apart, and an exchange of two would be a wrong token.
//
// A chunk stays in registers between its two uses.  First the maxima of groups of threads: the n-th largest of them is a bound below the n-th
// largest logit, which few others pass (64 groups, n = 32: 1.4 n are expected).  Then exponentials, and what passes the bound goes to
// shared memory, where every candidate counts those above it.
constexpr int kSelVectors = 8;    // 16-byte pieces a thread holds
constexpr int kSelRoom = 1024;    // candidates of a chunk in shared memory

template <typename T>
struct SelRow {
  static constexpr int kElems = 16 / sizeof(T);
  static constexpr int kChunk = kBeamThreads * kSelVectors * kElems;
};

// Numbers in the order of their bits (-0 as 0); what has no number, or minus infinity, is no candidate: 0.
__device__ __forceinline__ uint32_t sel_ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return x > -INFINITY ? (u ^ (u >> 31 ? 0xffffffffu : 0x80000000u)) : 0u;
}
__device__ __forceinline__ float sel_number(uint32_t o) { return __uint_as_float(o ^ (o >> 31 ? 0x80000000u : 0xffffffffu)); }

template <typename T>
__device__ __forceinline__ void sel_unpack(const uint4& v, float (&f)[SelRow<T>::kElems]) {
  if constexpr (sizeof(T) == 4) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  } else {
    unpack8<T>(v, f);
  }
}

constexpr float kLog2e = 1.4426950408889634f;

struct SelPart {   // of a chunk: its largest logit m, the sum of exp(z - m)
  float m, s;
};

template <typename T>
__global__ void __launch_bounds__(kBeamThreads)
beam_scan_kernel(const T* __restrict__ logits, int64_t stride, int vocab, int chunks, int n, SelPart* __restrict__ parts, uint64_t* __restrict__ keys) {
  constexpr int E = SelRow<T>::kElems;
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  __shared__ float top[128];
  __shared__ float warp_top[kBeamThreads / 32], warp_sum_[kBeamThreads / 32];
  __shared__ float bound;
  __shared__ int found;
  __shared__ uint64_t cand[kSelRoom];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.x / chunks;
  const int chunk = blockIdx.x % chunks;
  const T* z = logits + row * stride;
  // pieces start on 16-byte boundaries, wherever the row does: the first one has `lead` elements before the row
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
  const int first = chunk * SelRow<T>::kChunk + tid * E - lead;   // element of the thread's first piece
  uint4 data[kSelVectors];
  auto again = [&] {       // (keeps the compiler from holding on to the unpacked numbers, twice as many registers)
#pragma unroll
    for (int j = 0; j < kSelVectors; ++j) asm volatile("" : "+r"(data[j].x), "+r"(data[j].y), "+r"(data[j].z), "+r"(data[j].w));
  };
#pragma unroll
  for (int j = 0; j < kSelVectors; ++j) {
    const int at = first + j * kBeamThreads * E;
    if (at >= 0 && at + E <= vocab) {
      data[j] = ld_nc16(z + at);
    } else {
      T piece[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (at + e >= 0 && at + e < vocab) piece[e] = z[at + e];
        else stf(&piece[e], -INFINITY);
      }
      memcpy(&data[j], piece, 16);
    }
  }
  float mine = -INFINITY;
#pragma unroll
  for (int j = 0; j < kSelVectors; ++j) {
    float f[E];
    sel_unpack<T>(data[j], f);
#pragma unroll
    for (int e = 0; e < E; ++e) mine = fmaxf(mine, f[e]);
  }
  // groups: 32, 64 or 128 of them, at least twice n
  const int groups = n <= 16 ? 32 : n <= 32 ? 64 : 128, width = kBeamThreads / groups;
  float g = mine;
  for (int d = 1; d < width; d <<= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, d));
  if ((tid & (width - 1)) == 0) top[tid / width] = g;
  const float w = warp_max(mine);
  if (lane == 0) warp_top[warp] = w;
  if (tid == 0) found = 0;
  __syncthreads();
  float m = warp_top[0];
#pragma unroll
  for (int i = 1; i < kBeamThreads / 32; ++i) m = fmaxf(m, warp_top[i]);
  if (tid < groups) {
    const float v = top[tid];
    int above = 0;
    for (int i = 0; i < groups; ++i) above += top[i] > v || (top[i] == v && i < tid);
    if (above == n - 1) bound = v;
  }
  __syncthreads();
  const float least = bound;
  const float ref = m > -INFINITY ? m : 0.f;    // (a chunk of minus infinities: its sum is 0)
  auto each = [&](auto&& take) {       // take(element, number) for all that pass the bound
#pragma unroll
    for (int j = 0; j < kSelVectors; ++j) {
      float f[E];
      sel_unpack<T>(data[j], f);
      bool any = false;
#pragma unroll
      for (int e = 0; e < E; ++e) any |= f[e] >= least;
      if (any) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (f[e] >= least && f[e] > -INFINITY) take(first + j * kBeamThreads * E + e, f[e]);
      }
    }
  };
  auto key = [](int at, float x) { return static_cast<uint64_t>(sel_ordered(x)) << 32 | (0xffffffffu - static_cast<uint32_t>(at)); };
  float sum = 0.f;
  again();
#pragma unroll
  for (int j = 0; j < kSelVectors; ++j) {
    float f[E];
    sel_unpack<T>(data[j], f);
    float part = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) part += ptx::ex2_approx((f[e] - ref) * kLog2e);
    sum += part;
  }
  again();
  each([&](int at, float x) {
    const int i = atomicAdd(&found, 1);
    if (i < kSelRoom) cand[i] = key(at, x);
  });
  sum = warp_sum(sum);
  if (lane == 0) warp_sum_[warp] = sum;
  __syncthreads();
  int count = found;
  if (count > kSelRoom) {
    // Many equal numbers, or large ones of few groups: the bound is moved up by halves until no more pass it than there is room for.  (Keys
    // differ from one another, so some bound lets n to kSelRoom through.)
    uint64_t lo = key(0x7fffffff, least), hi = ~0ull;
    for (int i = 0; i < 64; ++i) {
      const uint64_t mid = lo + (hi - lo) / 2;
      __syncthreads();
      if (tid == 0) found = 0;
      __syncthreads();
      int here = 0;
      each([&](int at, float x) { here += key(at, x) >= mid; });
      here = __reduce_add_sync(0xffffffffu, here);
      if (lane == 0 && here) atomicAdd(&found, here);
      __syncthreads();
      count = found;
      if (count > kSelRoom) lo = mid;
      else if (count < n) hi = mid;
      else {
        __syncthreads();
        if (tid == 0) found = 0;
        __syncthreads();
        each([&](int at, float x) {
          const uint64_t k = key(at, x);
          if (k >= mid) cand[atomicAdd(&found, 1)] = k;
        });
        __syncthreads();
        break;
      }
    }
  }
  uint64_t* out = keys + static_cast<int64_t>(blockIdx.x) * n;
  for (int i = tid; i < count; i += kBeamThreads) {
    const uint64_t mykey = cand[i];
    int above = 0;
    for (int k = 0; k < count; ++k) above += cand[k] > mykey;
    if (above < n) out[above] = mykey;
  }
  if (tid >= count && tid < n) out[tid] = 0;
  if (tid == 0) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kBeamThreads / 32; ++i) s += warp_sum_[i];
    parts[blockIdx.x] = SelPart{m, s};
  }
}

struct SelOut {
  float* score;
  int32_t *parent, *token;
};
struct SelCand {
  double v;
  int32_t row, token;
};
__device__ __forceinline__ bool sel_before(const SelCand& a, const SelCand& b) {
  return a.v > b.v || (a.v == b.v && (a.row < b.row || (a.row == b.row && a.token < b.token)));
}

// A block per request.  Of the chunks' lists those whose first entry is among the n best first entries are looked at: the n best are in them.
__global__ void __launch_bounds__(kBeamThreads)
beam_merge_kernel(const SelPart* __restrict__ parts, const uint64_t* __restrict__ keys, const float* __restrict__ scores, int beams, int chunks, int n,
                  int keep, const int32_t* __restrict__ ended, int num_ended, SelOut all, SelOut next) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  extern __shared__ __align__(16) uint8_t sel_smem[];
  SelCand* cand = reinterpret_cast<SelCand*>(sel_smem);               // [n n]
  SelCand* heads = cand + n * n;                                      // [beams chunks]
  SelCand* best = heads + beams * chunks;                             // [n]
  __shared__ double norm[kBeamMost], base[kBeamMost];
  __shared__ int lists[kBeamMost], found;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, num = beams * chunks;
  const int64_t q = blockIdx.x;
  parts += q * num;
  keys += q * num * n;
  if (tid == 0) found = 0;
  for (int b = warp; b < beams; b += kBeamThreads / 32) {
    const SelPart* row = parts + b * chunks;
    float m = -INFINITY;
    for (int i = lane; i < chunks; i += 32) m = fmaxf(m, row[i].m);
    m = warp_max(m);
    double s = 0.0;
    for (int i = lane; i < chunks; i += 32)
      s += static_cast<double>(row[i].s) * (row[i].m > -INFINITY ? exp(static_cast<double>(row[i].m) - m) : 1.0);   // (1: NaN stays, 0 does)
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    if (lane == 0) {
      norm[b] = m + log(s);
      base[b] = scores[q * beams + b];
    }
  }
  __syncthreads();
  auto entry = [&](int list, int i) {
    const uint64_t k = keys[static_cast<int64_t>(list) * n + i];
    const int b = list / chunks;
    const double x = k ? base[b] + (static_cast<double>(sel_number(static_cast<uint32_t>(k >> 32))) - norm[b]) : -INFINITY;
    const double v = x > -INFINITY ? x : -INFINITY;      // (what is no number is no candidate)
    return SelCand{v, b, static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(k))};
  };
  for (int i = tid; i < num; i += kBeamThreads) heads[i] = entry(i, 0);
  if (tid < n) {
    lists[tid] = -1;
    best[tid] = SelCand{-INFINITY, -1, -1};
  }
  __syncthreads();
  for (int i = tid; i < num; i += kBeamThreads) {
    const SelCand h = heads[i];
    if (!(h.v > -INFINITY)) continue;
    int above = 0;
    for (int k = 0; k < num; ++k) above += sel_before(heads[k], h);
    if (above < n) lists[above] = i;
  }
  __syncthreads();
  const bool cut = num >= n && lists[n - 1] >= 0;
  const SelCand least = cut ? heads[lists[n - 1]] : SelCand{-INFINITY, 0, 0};
  for (int i = tid; i < n * n; i += kBeamThreads) {
    const int list = lists[i / n];
    if (list < 0) continue;
    const SelCand e = entry(list, i % n);
    if (e.v > -INFINITY && !(cut && sel_before(least, e))) cand[atomicAdd(&found, 1)] = e;
  }
  __syncthreads();
  for (int i = tid; i < found; i += kBeamThreads) {
    const SelCand e = cand[i];
    int above = 0;
    for (int k = 0; k < found; ++k) above += sel_before(cand[k], e);
    if (above < n) best[above] = e;
  }
  __syncthreads();
  for (int i = tid; i < n; i += kBeamThreads) {
    all.score[q * n + i] = static_cast<float>(best[i].v);
    all.parent[q * n + i] = best[i].row;
    all.token[q * n + i] = best[i].token;
  }
  if (warp == 0) {
    int before = 0;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + lane;
      bool on = i < n && best[i].row >= 0;
      for (int e = 0; on && e < num_ended; ++e) on = ended[e] != best[i].token;
      const unsigned who = __ballot_sync(0xffffffffu, on);
      const int at = before + __popc(who & ((1u << lane) - 1));
      if (on && at < keep) {
        next.score[q * keep + at] = static_cast<float>(best[i].v);
        next.parent[q * keep + at] = best[i].row;
        next.token[q * keep + at] = best[i].token;
      }
      before += __popc(who);
    }
    for (int i = before + lane; i < keep; i += 32) {
      next.score[q * keep + i] = -INFINITY;
      next.parent[q * keep + i] = next.token[q * keep + i] = -1;
    }
  }
}

// ------------------------------------------------------------------ tables of the beams that go on
struct ForkParams {
  const int32_t *table, *cached, *parents, *pool;
  int64_t table_stride, pool_stride;
  int width, from, to, pool_size, page, num_pages;   // from: beams of a request in `table`; to: children
  int32_t *out_table, *out_cached, *src, *dst, *tokens;
  int* status;
};

// A block per request.  A bit per page says which ones the children keep; the fresh ones are the first of the request's own without it.
__global__ void __launch_bounds__(kBeamThreads) beam_fork_kernel(const ForkParams p) {
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  extern __shared__ uint32_t used[];
  __shared__ int par[kBeamMost], len[kBeamMost], again[kBeamMost], want[kBeamMost], fresh[kBeamMost], sums[kBeamThreads / 32];
  __shared__ int wanted;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t q = blockIdx.x;
  const int words = (p.num_pages + 31) / 32;
  for (int i = tid; i < words; i += kBeamThreads) used[i] = 0;
  auto report = [&](int code) { if (p.status) atomicCAS(p.status, 0, code); };
  if (tid < p.to) {
    const int b = p.parents[q * p.to + tid];
    int n = -1;
    if (b >= 0 && b < p.from) {
      n = p.cached[q * p.from + b];
      if (n >= 0 && n / p.page >= p.width) {
        report(kStatusTooLarge);
        n = -1;
      }
    } else if (b >= p.from) {
      report(kStatusBadIndex);
    }
    par[tid] = b;
    len[tid] = n < 0 ? -1 : n;
    fresh[tid] = -1;
  }
  __syncthreads();
  if (tid < p.to) {
    int seen = 0;
    for (int i = 0; i < tid; ++i) seen |= len[i] >= 0 && par[i] == par[tid];
    again[tid] = seen;
  }
  __syncthreads();
  // pages that children keep (a parent's once)
  for (int j = 0; j < p.to; ++j) {
    if (len[j] < 0 || again[j]) continue;
    const int32_t* row = p.table + (q * p.from + par[j]) * p.table_stride;
    const int keeps = (len[j] + p.page - 1) / p.page;
    for (int i = tid; i < keeps; i += kBeamThreads) {
      const int pg = row[i];
      if (pg >= 0 && pg < p.num_pages) atomicOr(&used[pg >> 5], 1u << (pg & 31));
      else report(kStatusBadIndex);
    }
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
    const int i = i0 + tid, pg = i < p.pool_size ? p.pool[q * p.pool_stride + i] : -1;
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
  for (int j = 0; j < p.to; ++j) {
    const int n = len[j], full = n / p.page, part = n % p.page;
    const bool wants = want[j] >= 0;
    const int page = wants ? fresh[want[j]] : -1;
    const bool live = n >= 0 && (!wants || page >= 0);
    const int keeps = !live ? 0 : wants ? full : (n + p.page - 1) / p.page;
    const int32_t* row = p.table + (q * p.from + par[j]) * p.table_stride;
    int32_t* to = p.out_table + (q * p.to + j) * p.width;
    for (int i = tid; i < p.width; i += kBeamThreads) to[i] = i < keeps ? row[i] : live && wants && i == full ? page : -1;
    if (tid == 0) {
      const bool copies = live && wants && part > 0;
      if (n >= 0 && !live) report(kStatusNoPage);
      p.out_cached[q * p.to + j] = live ? n : -1;
      p.src[q * p.to + j] = copies ? row[full] : -1;
      p.dst[q * p.to + j] = copies ? page : -1;
      p.tokens[q * p.to + j] = copies ? part : 0;
    }
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

// A block per piece of 32 KB.  U: what all addresses are multiples of.
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
// an entry belongs to is found by halves.
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
    pages[r + 1] = n ? (p.cached[r] + n + p.page - 1) / p.page : 0;
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
      const int pg = n ? p.table[r * p.table_stride + c / p.page] : -1;
      p.pos[r] = n ? c : 0;
      p.slot[r] = pg >= 0 ? pg * p.page + c % p.page : -1;
    }
  }
  if (p.counts) {
    for (int t = self; t < p.tokens; t += all) {
      int at = 0, slot = -1;
      if (t < total_t) {
        const int r = row_of(toks, t);
        at = p.cached[r] + t - toks[r];
        const int pg = p.table[r * p.table_stride + at / p.page];
        if (pg >= 0) slot = pg * p.page + at % p.page;
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

}  // namespace blitz

extern "C" {
using namespace blitz;

static int beam_chunks(int vocab, int dtype) {
  // (a row may begin behind a 16-byte boundary: up to 7 elements more)
  const int chunk = dtype == 2 ? SelRow<float>::kChunk : SelRow<__half>::kChunk, lead = dtype == 2 ? 3 : 7;
  return (vocab + lead + chunk - 1) / chunk;
}

int64_t blitz_beam_select_workspace_bytes(int rows, int vocab, int n, int dtype) {
  return static_cast<int64_t>(rows) * beam_chunks(vocab, dtype) * (static_cast<int64_t>(sizeof(SelPart)) + 8 * n);
}

// logits [rows][stride] in fp16 (0), bf16 (1) or fp32 (2); scores [rows]; a request's beams are consecutive rows.  score, parent and token:
// [rows / beams][n], next_*: [rows / beams][keep].  ended: tokens that end a sequence (num_ended of them).
int blitz_beam_select(const void* logits, int64_t stride, const float* scores, int rows, int vocab, int beams, int n, int keep, const int32_t* ended,
                      int num_ended, void* workspace, float* score, int32_t* parent, int32_t* token, float* next_score, int32_t* next_parent,
                      int32_t* next_token, int dtype, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (vocab < 1 || beams < 1 || beams > kBeamMost || rows % beams || n < 1 || n > kBeamMost || keep < 1 || keep > n || num_ended < 0) return -1;
  const int chunks = beam_chunks(vocab, dtype);
  if (static_cast<int64_t>(rows) * chunks > 0x7fffffff) return -1;
  SelPart* parts = reinterpret_cast<SelPart*>(workspace);
  uint64_t* keys = reinterpret_cast<uint64_t*>(parts + static_cast<int64_t>(rows) * chunks);
  cudaError_t e = cudaSuccess;
  BLITZ_DISPATCH_DTYPE3(dtype, (e = launch_pdl(beam_scan_kernel<T>, dim3(rows * chunks), dim3(kBeamThreads), 0, stream, (const T*)logits, stride, vocab, chunks, n,
                                               parts, keys)));
  if (e != cudaSuccess) return (int)e;
  const size_t smem = sizeof(SelCand) * (static_cast<size_t>(n) * n + static_cast<size_t>(beams) * chunks + n);
  if (smem > 200 * 1024) return -1;
  static PerDeviceOnce once;
  e = once.run([] { return cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024); });
  if (e != cudaSuccess) return (int)e;
  return (int)launch_pdl(beam_merge_kernel, dim3(rows / beams), dim3(kBeamThreads), smem, stream, parts, keys, scores, beams, chunks, n, keep, ended, num_ended,
                         SelOut{score, parent, token}, SelOut{next_score, next_parent, next_token});
}

// table [requests from][width], cached [requests from], parents [requests][to], pool [requests][pool_size]; the children's table
// [requests to][width], cached, and the copies to make (src, dst, tokens; -1: none).
int blitz_beam_fork(const int32_t* table, int64_t table_stride, const int32_t* cached, const int32_t* parents, const int32_t* pool, int64_t pool_stride,
                    int requests, int from, int to, int width, int pool_size, int page, int num_pages, int32_t* out_table, int32_t* out_cached, int32_t* src,
                    int32_t* dst, int32_t* tokens, int* status, cudaStream_t stream) {
  if (requests <= 0) return 0;
  if (from < 1 || to < 1 || from > kBeamMost || to > kBeamMost || width < 1 || page < 1 || num_pages < 1 || pool_size < 0) return -1;
  const size_t smem = static_cast<size_t>((num_pages + 31) / 32) * 4;
  if (smem > 200 * 1024) return -1;
  static PerDeviceOnce once;
  cudaError_t e = once.run([] { return cudaFuncSetAttribute(beam_fork_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024); });
  if (e != cudaSuccess) return (int)e;
  ForkParams p{table, cached, parents, pool, table_stride, pool_stride, width, from, to, pool_size, page, num_pages, out_table, out_cached, src, dst, tokens, status};
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
