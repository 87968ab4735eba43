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
// A chunk is looked at twice, so it waits in shared memory (cp.async; six blocks an SM, 192 KB under way; in registers it left room for one or two).
// First the maxima of groups of threads: the n-th largest of them is a bound below the n-th
// largest logit, which few others pass (64 groups, n = 32: 1.4 n are expected).  Then exponentials, and what passes the bound goes to
// a list, where every candidate counts those above it.
constexpr int kSelVectors = 8;    // 16-byte pieces a thread looks after
constexpr int kSelRoom = 512;     // candidates of a chunk

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

// Of a chunk: its largest logit m; c, and the sum of 2^(z L - c), L = log2 e in fp32 and c = m L rounded.  Off by the rounding of L for what lies
// between z and m alone, once the merge has taken out m's own part.  Where m is so large that the rounding of c would be of a term's size: `far`, and s the
// sum of exp(z - m).
struct SelPart {
  float m, c, s, far;
};
constexpr float kSelHuge = 65536.f;

template <typename T>
__global__ void __launch_bounds__(kBeamThreads, 6)
beam_scan_kernel(const T* __restrict__ logits, int64_t stride, int vocab, int chunks, int n, SelPart* __restrict__ parts, uint64_t* __restrict__ keys) {
  constexpr int E = SelRow<T>::kElems;
  __shared__ uint4 data[kSelVectors * kBeamThreads];
  __shared__ __align__(16) float top[128];
  __shared__ float warp_top[kBeamThreads / 32], warp_sum_[kBeamThreads / 32];
  __shared__ float bound;
  __shared__ int found, passed;
  __shared__ uint64_t cand[kSelRoom];
  __shared__ uint16_t pieces[kSelVectors * kBeamThreads];     // that have a number which passes the bound
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = blockIdx.x / chunks;
  const int chunk = blockIdx.x % chunks;
  const T* z = logits + row * stride;
  // pieces start on 16-byte boundaries, wherever the row does: the first one has `lead` elements before the row
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
  const int first = chunk * SelRow<T>::kChunk + tid * E - lead;   // element of the thread's first piece
  if (tid == 0) found = passed = 0;
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
#pragma unroll
  for (int j = 0; j < kSelVectors; ++j) {
    const int at = first + j * kBeamThreads * E;
    if (at >= 0 && at + E <= vocab) {
      ptx::cp_async_16(ptx::smem_u32(&data[j * kBeamThreads + tid]), z + at, 16);
    } else {
      T* piece = reinterpret_cast<T*>(&data[j * kBeamThreads + tid]);
      for (int e = 0; e < E; ++e) {
        if (at + e >= 0 && at + e < vocab) piece[e] = z[at + e];
        else stf(&piece[e], -INFINITY);
      }
    }
  }
  ptx::cp_async_commit();
  ptx::cp_async_wait<0>();        // (a thread reads what it has copied itself)
  float largest[kSelVectors], mine = -INFINITY;      // of each piece
#pragma unroll
  for (int j = 0; j < kSelVectors; ++j) {
    largest[j] = sel_max<T>(data[j * kBeamThreads + tid]);
    mine = fmaxf(mine, largest[j]);
  }
  // groups: 32, 64 or 128 of them, at least twice n
  const int groups = n <= 16 ? 32 : n <= 32 ? 64 : 128, width = kBeamThreads / groups;
  float g = mine;
  for (int d = 1; d < width; d <<= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, d));
  if ((tid & (width - 1)) == 0) top[tid / width] = g;
  const float w = warp_max(mine);
  if (lane == 0) warp_top[warp] = w;
  __syncthreads();
  float m = warp_top[0];
#pragma unroll
  for (int i = 1; i < kBeamThreads / 32; ++i) m = fmaxf(m, warp_top[i]);
  if (tid < groups) {
    const float v = top[tid];
    int above = 0;
    for (int i = 0; i < groups; i += 4) {
      const float4 o = *reinterpret_cast<const float4*>(&top[i]);
      above += (o.x > v || (o.x == v && i < tid)) + (o.y > v || (o.y == v && i + 1 < tid)) + (o.z > v || (o.z == v && i + 2 < tid)) +
               (o.w > v || (o.w == v && i + 3 < tid));
    }
    if (above == n - 1) bound = v;
  }
  __syncthreads();
  const float least = bound;
  const bool huge = fabsf(m) > kSelHuge && m > -INFINITY;
  const float c = m > -INFINITY ? m * kLog2e : 0.f;    // (a chunk of minus infinities: its sum is 0)
  auto key = [](int at, float x) { return static_cast<uint64_t>(sel_ordered(x)) << 32 | (0xffffffffu - static_cast<uint32_t>(at)); };
#pragma unroll
  for (int j = 0; j < kSelVectors; ++j)
    if (largest[j] >= least && largest[j] > -INFINITY) pieces[atomicAdd(&passed, 1)] = static_cast<uint16_t>(j * kBeamThreads + tid);
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < kSelVectors; ++j) {
    float f[E];
    sel_unpack<T>(data[j * kBeamThreads + tid], f);
    float part = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) part += ptx::ex2_approx(fmaf(f[e], kLog2e, -c));
    sum += part;
  }
  if (huge) {
    sum = 0.f;
#pragma unroll 1
    for (int i = 0; i < kSelVectors * E; ++i)
      sum += ptx::ex2_approx((ldf(reinterpret_cast<const T*>(&data[i / E * kBeamThreads + tid]) + i % E) - m) * kLog2e);
  }
  sum = warp_sum(sum);
  if (lane == 0) warp_sum_[warp] = sum;
  __syncthreads();
  // candidates: numbers of those pieces from the bound on.  Where there are too many (equal numbers, or large ones of few groups) the bound is
  // moved up by halves until there is room for them.  (Keys differ from one another, so some bound lets n to kSelRoom through.)
  uint64_t lo = 0, hi = ~0ull, mid = key(0x7fffffff, least);
  int count;
  for (int turn = 0;; ++turn) {
#pragma unroll 1
    for (int i = tid; i < passed * E; i += kBeamThreads) {
      const int piece = pieces[i / E], e = i % E;
      const uint64_t k = key(chunk * SelRow<T>::kChunk + piece * E - lead + e, ldf(reinterpret_cast<const T*>(&data[piece]) + e));
      if (k >= mid && k >> 32) {
        const int at = atomicAdd(&found, 1);
        if (at < kSelRoom) cand[at] = k;
      }
    }
    __syncthreads();
    count = found;
    if (count <= kSelRoom && (count >= n || turn == 0)) break;
    if (turn > 64) break;      // (not reached)
    (count > kSelRoom ? lo : hi) = mid;
    mid = lo + (hi - lo) / 2;
    __syncthreads();
    if (tid == 0) found = 0;
    __syncthreads();
  }
  count = min(count, kSelRoom);
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
    parts[blockIdx.x] = SelPart{m, c, s, huge ? 1.f : 0.f};
  }
}

struct SelOut {
  float* score;
  int32_t *parent, *token;
};
// A candidate: its value as 64 bits in the order of the numbers (0: none), its beam and token.  (Comparisons of doubles took half the kernel's time.)
struct SelCand {
  uint64_t v, place;
};
__device__ __forceinline__ bool sel_before(const SelCand& a, const SelCand& b) { return a.v > b.v || (a.v == b.v && a.place < b.place); }
__device__ __forceinline__ float sel_value(const SelCand& a) {
  return static_cast<float>(__longlong_as_double(static_cast<long long>(a.v ^ (a.v >> 63 ? 1ull << 63 : ~0ull))));
}

// A block per request: of the chunks' candidates the n best, by a bound as in the scan.  Neighbouring candidates of a list are in different groups, so that lists
// that have most of the best ones do not let more through.  (An earlier form took heads of the lists one after the other: 20 us for n = 24.)
constexpr int kSelListRoom = 8192;      // keys that wait in shared memory, where they are no more
constexpr int kSelBestRoom = 1024;
__global__ void __launch_bounds__(kBeamThreads)
beam_merge_kernel(const SelPart* __restrict__ parts, const uint64_t* __restrict__ keys, const float* __restrict__ scores, int beams, int chunks, int n,
                  int keep, const int32_t* __restrict__ ended, int num_ended, SelOut all, SelOut next) {
  constexpr int kWarps = kBeamThreads / 32;
  extern __shared__ __align__(16) uint64_t held[];
  __shared__ __align__(16) uint64_t top[kBeamThreads];
  __shared__ SelCand cand[kSelBestRoom], best[kBeamMost];
  __shared__ double norm[kBeamMost], base[kBeamMost];
  __shared__ uint64_t bound;
  __shared__ int found;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, num = beams * chunks * n;
  const int64_t q = blockIdx.x;
  parts += q * beams * chunks;
  keys += q * num;
  const bool in_shared = num <= kSelListRoom;
  if (tid == 0) found = 0;
  if (tid < n) best[tid] = SelCand{0, ~0ull};
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();
  if (in_shared) {
#pragma unroll 8
    for (int i = tid; i < num; i += kBeamThreads) held[i] = keys[i];
  }
  for (int b = warp; b < beams; b += kWarps) {
    const SelPart* row = parts + b * chunks;
    const float score = scores[q * beams + b];
    const SelPart one = lane < chunks ? row[lane] : SelPart{-INFINITY, 0.f, 0.f, 0.f};
    float m = one.m;
    for (int i = lane + 32; i < chunks; i += 32) m = fmaxf(m, row[i].m);
    m = warp_max(m);
    // sum of exp(z - m): of a chunk, s exp(c ln 2 - m) exp(-d m'), L ln 2 = 1 + d, m' its largest
    constexpr double kLn2 = 0.69314718055994531, kD = static_cast<double>(kLog2e) * kLn2 - 1.0;
    auto share = [&](const SelPart& x) {
      if (!(x.m > -INFINITY)) return x.s;      // (0, or NaN)
      return x.s * (x.far != 0.f ? expf(x.m - m) : expf(static_cast<float>(x.c * kLn2 - m - kD * x.m)));
    };
    float s = share(one);
    for (int i = lane + 32; i < chunks; i += 32) s += share(row[i]);
    s = warp_sum(s);
    if (lane == 0) {
      // log s = log f + e log 2 with f from 1 to 2: in fp32 off by 2^-24, where log s would be by 2^-21
      int e = 1;
      const bool number = s > 0.f && s < INFINITY;
      const float f = number ? 2.f * frexpf(s, &e) : s;
      norm[b] = static_cast<double>(m) + (static_cast<double>(logf(f)) + (e - 1) * kLn2);
      base[b] = score;
    }
  }
  __syncthreads();
  auto made = [&](int i) {
    const uint64_t k = in_shared ? held[i] : keys[i];
    if (k == 0) return SelCand{0, ~0ull};
    const int b = i / (chunks * n);
    const double v = base[b] + (static_cast<double>(sel_number(static_cast<uint32_t>(k >> 32))) - norm[b]) + 0.0;      // (-0 as 0)
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v));
    // (what is no number is no candidate)
    return v > -INFINITY ? SelCand{u ^ (u >> 63 ? ~0ull : 1ull << 63), static_cast<uint64_t>(b) << 32 | (0xffffffffu - static_cast<uint32_t>(k))} : SelCand{0, ~0ull};
  };
  uint64_t mine = 0;
#pragma unroll 4
  for (int i = tid; i < num; i += kBeamThreads) mine = max(mine, made(i).v);
  top[tid] = mine;
  __syncthreads();
  const int groups = n <= 32 ? 64 : 128;
  if (tid < groups) {
    for (int i = tid + groups; i < kBeamThreads; i += groups) mine = max(mine, top[i]);
    top[tid] = mine;
  }
  __syncthreads();
  if (tid < groups) {
    int above = 0;
#pragma unroll 8
    for (int i = 0; i < groups; ++i) above += top[i] > mine || (top[i] == mine && i < tid);
    if (above == n - 1) bound = mine;
  }
  __syncthreads();
  const uint64_t least = bound > 0 ? bound : 1;
#pragma unroll 4
  for (int i = tid; i < num; i += kBeamThreads) {
    const SelCand e = made(i);
    if (e.v >= least) {
      const int at = atomicAdd(&found, 1);
      if (at < kSelBestRoom) cand[at] = e;
    }
  }
  __syncthreads();
  const int count = found;
  if (count <= kSelBestRoom) {
    for (int i = tid; i < count; i += kBeamThreads) {
      const SelCand e = cand[i];
      int above = 0;
#pragma unroll 4
      for (int k = 0; k < count; ++k) above += sel_before(cand[k], e);
      if (above < n) best[above] = e;
    }
  } else {
    // many equal values: one after the other, the best of those behind the last one
    SelCand last{~0ull, 0};
    for (int j = 0; j < n; ++j) {
      SelCand first{0, ~0ull};
      for (int i = tid; i < num; i += kBeamThreads) {
        const SelCand e = made(i);
        if (e.v && sel_before(last, e) && sel_before(e, first)) first = e;
      }
      __syncthreads();
      cand[tid] = first;
      __syncthreads();
      for (int i = 0; i < kBeamThreads; ++i)
        if (sel_before(cand[i], first)) first = cand[i];
      if (tid == 0) best[j] = first;
      last = first;
      if (first.v == 0) break;
    }
  }
  __syncthreads();
  if (warp > 0) return;
  auto give = [](const SelOut& to, int64_t at, const SelCand& e) {
    to.score[at] = e.v ? sel_value(e) : -INFINITY;
    to.parent[at] = e.v ? static_cast<int32_t>(e.place >> 32) : -1;
    to.token[at] = e.v ? static_cast<int32_t>(e.place) : -1;
  };
  int before = 0;
  for (int i0 = 0; i0 < n; i0 += 32) {
    const int i = i0 + lane;
    if (i < n) give(all, q * n + i, best[i]);
    bool on = i < n && best[i].v != 0;
    for (int e = 0; on && e < num_ended; ++e) on = ended[e] != static_cast<int32_t>(best[i].place);
    const unsigned who = __ballot_sync(0xffffffffu, on);
    const int at = before + __popc(who & ((1u << lane) - 1));
    if (on && at < keep) give(next, q * keep + at, best[i]);
    before += __popc(who);
  }
  for (int i = before + lane; i < keep; i += 32) give(next, q * keep + i, SelCand{0, ~0ull});
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
// Latency bounds it: lengths, then tables, are two rounds of loads, all of a round at once.
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
    par[tid] = p.parents[q * p.to + tid];
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
  const int64_t num = static_cast<int64_t>(beams) * chunks * n;
  if (num > 0x7fffffff) return -1;
  static PerDeviceOnce once;
  e = once.run([] { return cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * kSelListRoom); });
  if (e != cudaSuccess) return (int)e;
  return (int)launch_pdl(beam_merge_kernel, dim3(rows / beams), dim3(kBeamThreads), num <= kSelListRoom ? 8 * (size_t)num : 0, stream, parts, keys, scores, beams, chunks, n, keep, ended, num_ended,
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
