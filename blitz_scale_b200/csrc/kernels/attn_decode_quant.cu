// Decode attention over a paged cache held in 4 bits (the format: quant_kv.cuh).
//
// One query token per sequence: o = sum_j p_j v_j, p = softmax_j(scale q.k_j), a stream over the sequence's codes and scales, which the
// tensor cores (mma.sync, m16n8k16) turn into products without ever forming a key or a value.  With k_d = z_g + s_g c_d for dimension d
// of group g:
//
//   q.k = sum_g s_g (sum_{d in g} q_d c_d) + z_g (sum_{d in g} q_d)
//   o_d = sum_j (p_j s_j) (c_jd - 8) + sum_j p_j (z_j + 8 s_j)
//
// A code, or 16 times one, is an fp16 number as its bits stand in a half's low byte: a denormal, c 2^-24, which the tensor cores multiply like any
// other.  A word of 8 codes takes five instructions and no constant has to come off again.  Queries enter in fp16, a head divided by a power of
// two that brings its largest entry to 2^14 .. 2^15 (2^10 .. 2^11 for what meets 16 times a code): bf16 and fp16 numbers are exact there down to
// 2^-24 of the largest, and so are their products with codes.  Weights times scales are rounded to fp16, times a power of two of the
// head's that brings the largest scale so far that has a weight to 2^6 .. 2^7 (less, where tokens without one have larger scales): 2^-11 of each down to scales 2^-20 of
// the largest, less below.  Their product with -8, one more matrix
// product a group, makes the codes lie around zero, so that this rounding is not amplified by what cancels.  The part of z_j + 8 s_j stays in 32
// bits; the sums of q_d z_g in the scores are one more product, in bf16, of z as stored with sums of q in two numbers.
//
// The maximum that weights refer to follows the scores only when they pass it by 2^8 (fp16 has room for that): nearly every chunk finds
// that out with a vote, without a maximum over its lanes or a rescaling.
//
// S^T = K Q^T has 16 tokens as rows and at most 8 query heads as columns, O^T = V^T P^T dimensions as rows and the same columns: a lane
// has the same heads in both.  Between them the weights' 8 x 8 blocks are transposed by movmatrix.  Scales of K multiply the accumulators
// of a group, scales of V the weights of a group.  Where at most 4 query heads share a KV head, the columns are 4 heads x 2
// halves of the groups (HALVES): lanes of columns 0..3 handle the scales of the first half of the groups, the others those of the second.
//
// A warp takes chunks of 32 tokens by itself, through a ring of stages of its own; one more warp issues the copies (bulk copies: a
// head's tokens in a page are one contiguous piece), a lane for each of the others.  Eleven warps have 168 registers each, which is enough but for
// five to eight query heads over a KV head of 128 in groups of 32 (12 bytes spilled); fifteen with 128 took 43.4 us where these took 40.3 (256 sequences of 512
// tokens, 32 query heads over 8 of 128, groups of 32).
//
// The chunks of all sequences of all heads, end to end, are cut into equal ranges, one per warp of the GPU, so that neither lengths nor the
// number of sequences leave warps idle.  A sequence that is cut leaves its pieces' sums in shared memory, where the warps that end with it
// wait for them and add them up, a head each (the warp it begins in comes to it last, the next one began with it: nobody waits long);
// pieces in several blocks go through scratch and a ticket per head, and the last block adds up.  The order is that of the ranges,
// whoever is last.  Where there are no more sequences of heads than blocks, and the longest costs less beside an equal share than
// that hand-over (2.5 us), a block takes one of them whole.
//
// Measured, bf16, 32 query heads over 8 of 128: 256 sequences of 512 tokens in groups of 32 41.3 us (172 MB, 4.2 TB/s; the 16-bit kernel
// 98 us); one of 100003 in groups of 128 29.8 us (3.65 TB/s); 61 of 1100 on average in groups of 64 24.7 us (fp16); one of 977 9.7 us.  Bound by the stream where
// it is long (5.6 TB/s beside the ends; the warps issue in half of the cycles); 9 to 11 us of every call are its ends: tables, first
// pages, and pieces added up.
#include "launch.cuh"
#include "ptx.cuh"
#include "mma.cuh"
#include "quant_kv.cuh"
#include "scalar.cuh"
#include "tmap.cuh"

namespace blitz {

constexpr int kQdWarps = 11, kQdThreads = (kQdWarps + 1) * 32;
constexpr int kQdChunk = 32;
constexpr int kQdMaxBatch = 1024;   // sequences of a launch
constexpr int kQdMaxStages = 4;
constexpr int kQdSmem = 232448;     // bytes of shared memory a block may have

struct DecodeQuantParams {
  const void* q;
  int64_t q_stride;
  const uint8_t* pool;
  const int32_t *indices, *indptr, *last_page_len;
  void* out;
  int64_t out_stride;
  unsigned* tickets;   // [batch][query heads] chunks finished, zero between launches
  float* part;         // [2 blocks][rep][D] sums, then [2 blocks][rep] of (maximum, sum of weights)
  int batch, kv_heads, heads, div, rep;  // heads: groups of at most 8 query heads, div of which share a KV head; rep: query heads of one
  int page_size, page_shift, max_pages, stages, static_table;
  unsigned slack, alone;  // chunks in the time that adding up pieces of several blocks takes: of all blocks together, of a block by itself
  float sign, scale_log2, cap_scale, cap_log2;  // the scale's sign (0, NaN: itself) goes into the queries, its magnitude into the factors
  int window, keep_first;
  const void* sink;
  int* status;
  int give_up;  // test aid: every other block begins as if a wait had run out
};

// Shared memory: rings, a slot per warp for the sums of its first piece (the last one's go into the ring), tables of the sequences, barriers.
__host__ __device__ constexpr int qd_slot_floats(int D, int rep) { return rep * (D + 4) + 16; }  // rows in different banks, then maxima and sums
__host__ __device__ constexpr int qd_table_bytes() { return (3 * kQdMaxBatch + 4 + 8 + kQdWarps * 16) * 4; }
inline int qd_smem(int D, int stage, int rep, int stages) { return kQdWarps * (stages * stage + qd_slot_floats(D, rep) * 4) + qd_table_bytes() + kQdWarps * kQdMaxStages * 16; }

struct QdTables {
  int *before, *len, *page;  // chunks of the sequences before each ([batch + 1]), lengths, places of the first page ids
};
// Visible keys of a sequence: [0, first) and [lo, len), in chunks.
struct QdSeen {
  int len, lo, first, n_first, c_window;
  __device__ __forceinline__ int token(int n) const { return (n < n_first ? n : c_window + n - n_first) * kQdChunk; }
  __device__ __forceinline__ int chunks() const { return n_first + max(0, (len + kQdChunk - 1) / kQdChunk - c_window); }
};
__device__ __forceinline__ QdSeen qd_seen(const DecodeQuantParams& p, int len) {
  QdSeen v;
  v.len = len;
  v.lo = p.window > 0 ? max(0, len - p.window) : 0;
  v.first = min(p.keep_first, v.lo);
  v.n_first = (v.first + kQdChunk - 1) / kQdChunk;
  v.c_window = max(v.lo / kQdChunk, v.n_first);
  return v;
}
// How `all` chunks are cut into equal ranges: `each` warps of a block take one (all of them where there are chunks enough; few chunks go to
// more blocks, whose warps then have an SM's pipes to themselves).
struct QdCut {
  unsigned each, base, rem;
  __device__ __forceinline__ QdCut(unsigned all, unsigned blocks) {
    each = min(static_cast<unsigned>(kQdWarps), max(4u, (all + blocks - 1) / blocks));
    base = all / (blocks * each);
    rem = all % (blocks * each);
  }
  __device__ __forceinline__ unsigned begin(unsigned v) const { return v * base + min(v, rem); }
  __device__ __forceinline__ unsigned range(unsigned x) const { return x < rem * (base + 1) ? x / (base + 1) : rem + (x - rem * (base + 1)) / base; }
};
// The ranges of a block's warps.  Where there is work enough, those that share their quarter of the SM with one more and the warp that copies,
// not with two others, get 8 chunks where the others get 7: with equal ranges they were done 14 % earlier (one sequence of 100003 tokens
// 30.0 -> 29.0 us, 256 of 512 40.1 -> 39.7).
struct QdRanges {
  unsigned x0, n, base, rem;
  bool weighted;
  __device__ __forceinline__ unsigned begin(unsigned w) const {
    static_assert(kQdWarps == 11, "warps 3 and 7");
    return x0 + (weighted ? n * (7 * w + (w > 3 ? 1 : 0) + (w > 7 ? 1 : 0)) / 79 : w * base + min(w, rem));
  }
  // (kept in shared memory: the products need the registers)
  __device__ __forceinline__ void keep(volatile int* to) const {
    to[0] = x0; to[1] = n; to[2] = base; to[3] = rem; to[4] = weighted;
  }
};
__device__ __forceinline__ QdRanges qd_ranges(const volatile int* kept) {
  return {static_cast<unsigned>(kept[0]), static_cast<unsigned>(kept[1]), static_cast<unsigned>(kept[2]), static_cast<unsigned>(kept[3]), kept[4] != 0};
}
__device__ __forceinline__ QdRanges qd_ranges(const QdCut& cut, unsigned block) {
  const unsigned first = block * cut.each, x0 = cut.begin(first);
  return {x0, cut.begin(first + cut.each) - x0, cut.base, cut.rem > first ? min(cut.rem - first, cut.each) : 0u, cut.each == kQdWarps && cut.base >= 8};
}
__device__ __forceinline__ QdRanges qd_ranges(unsigned begin, unsigned end) {
  const unsigned n = end - begin;
  return {begin, n, n / kQdWarps, n % kQdWarps, n >= 8 * kQdWarps};
}
// A walk over the pieces of a range of chunks.
struct QdWalk {
  unsigned x, end;
  int head, b;
};
struct QdPiece {
  int head, b, beg, end;   // chunks beg .. end of the sequence's
  unsigned start, stop;    // where the whole sequence of this head lies among all chunks
};
__device__ __forceinline__ QdWalk qd_walk(const QdTables& t, int batch, unsigned x, unsigned end) {
  QdWalk w{x, end, 0, 0};
  if (x < end) {
    const unsigned each = t.before[batch];
    w.head = x / each;
    const int y = x - w.head * each;
    int lo = 0, hi = batch - 1;  // the last sequence that starts at or before y
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (t.before[mid] <= y) lo = mid;
      else hi = mid - 1;
    }
    w.b = lo;
  }
  return w;
}
__device__ __forceinline__ bool qd_next(const QdTables& t, int batch, QdWalk& w, QdPiece& it) {
  if (w.x >= w.end) return false;
  const unsigned each = t.before[batch], base = w.head * each;
  while (static_cast<unsigned>(t.before[w.b + 1]) <= w.x - base) ++w.b;
  it.head = w.head;
  it.b = w.b;
  it.start = base + t.before[w.b];
  it.stop = base + t.before[w.b + 1];
  it.beg = w.x - it.start;
  it.end = min(it.stop, w.end) - it.start;
  w.x += it.end - it.beg;
  if (w.x == base + each) {
    ++w.head;
    w.b = 0;
  }
  return true;
}

__device__ __forceinline__ void qd_keep(volatile int* to, const QdPiece& it) {
  to[0] = it.head; to[1] = it.b; to[2] = it.start; to[3] = it.stop;
}
__device__ __forceinline__ QdPiece qd_kept(const volatile int* from) {
  return {from[0], from[1], 0, 0, static_cast<unsigned>(from[2]), static_cast<unsigned>(from[3])};
}

// Waits (in a converged warp) until words of shared memory that other warps of the block write are not zero: a lane for each that counts.
// Once a wait of the block has run out, none is waited for.
__device__ __forceinline__ bool qd_wait(const volatile int* word, bool counts, volatile int* abort_flag) {
  const uint64_t since = ptx::globaltimer_ns();
  for (uint32_t it = 1;; ++it) {
    if (__any_sync(0xffffffffu, *abort_flag != 0 || ((it & 63u) == 0 && ptx::globaltimer_ns() - since > ptx::kDefaultWaitNs))) {
      *abort_flag = 1;
      return false;
    }
    if (__all_sync(0xffffffffu, !counts || *word != 0)) break;
    __nanosleep(32);
  }
  __threadfence_block();
  return true;
}

__device__ __forceinline__ void qd_mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void qd_mma_f16_add(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void qd_mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t qd_transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float qd_low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float qd_high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Exponent of a positive number; 2^e, -126 <= e <= 127.
__device__ __forceinline__ int qd_exponent(float x) { return static_cast<int>(__float_as_uint(x) >> 23) - 127; }
__device__ __forceinline__ float qd_power(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }

// Scales and offsets of a token, of the groups that a lane's columns stand for (all, or half x of them).
template <int G, bool HALVES>
struct QdScales {
  static constexpr int N = HALVES ? G / 2 : G;
  float s[N];
  __device__ __forceinline__ void keys(const uint8_t* token, int x) {  // the scales alone
    if (G == 4 && HALVES) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(token + 4 * x);
      s[0] = qd_low(w); s[1 % N] = qd_high(w);
    } else if (G == 4) {
      const uint2 w = *reinterpret_cast<const uint2*>(token);
      s[0] = qd_low(w.x); s[1 % N] = qd_high(w.x); s[2 % N] = qd_low(w.y); s[3 % N] = qd_high(w.y);
    } else if (G == 2 && HALVES) {
      s[0] = qd_low(*reinterpret_cast<const uint16_t*>(token + 2 * x));
    } else {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(token);
      s[0] = qd_low(w);
      if (G == 2) s[1 % N] = qd_high(w);
    }
  }
  float mid[N];  // z + 8 s
  __device__ __forceinline__ void values(const uint8_t* token, int x) {
    uint32_t a, b = 0, c, d = 0;
    if (G == 4 && HALVES) {
      a = *reinterpret_cast<const uint32_t*>(token + 4 * x);
      c = *reinterpret_cast<const uint32_t*>(token + 8 + 4 * x);
    } else if (G == 4) {
      const uint4 w = *reinterpret_cast<const uint4*>(token);
      a = w.x; b = w.y; c = w.z; d = w.w;
    } else if (G == 2 && HALVES) {
      a = *reinterpret_cast<const uint16_t*>(token + 2 * x);
      c = *reinterpret_cast<const uint16_t*>(token + 4 + 2 * x);
    } else if (G == 2) {
      const uint2 w = *reinterpret_cast<const uint2*>(token);
      a = w.x; c = w.y;
    } else {
      a = *reinterpret_cast<const uint32_t*>(token);
      c = a >> 16;
    }
    s[0] = qd_low(a);
    mid[0] = fmaf(8.f, s[0], qd_low(c));
    if (N >= 2) {
      s[1 % N] = qd_high(a);
      mid[1 % N] = fmaf(8.f, s[1 % N], qd_high(c));
    }
    if (N == 4) {
      s[2 % N] = qd_low(b); s[3 % N] = qd_high(b);
      mid[2 % N] = fmaf(8.f, s[2 % N], qd_low(d)); mid[3 % N] = fmaf(8.f, s[3 % N], qd_high(d));
    }
  }
  __device__ __forceinline__ void none() {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = mid[i] = 0.f;
  }
  __device__ __forceinline__ float largest() const {
    float v = s[0];
#pragma unroll
    for (int i = 1; i < N; ++i) v = fmaxf(v, s[i]);
    return v;
  }
};

template <typename T, int D, int GROUP, bool HALVES>
__global__ void __launch_bounds__(kQdThreads, 1) attn_decode_quant_kernel(const __grid_constant__ DecodeQuantParams p) {
  constexpr QuantKv F = quant_kv(D, GROUP);
  constexpr int G = D / GROUP, W = D / 32, WG = GROUP / 32, MT = D / 16, N = QdScales<G, HALVES>::N;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ring_bytes = p.stages * 2 * F.block, slot = qd_slot_floats(D, p.rep);
  float* const slots = reinterpret_cast<float*>(smem + kQdWarps * ring_bytes);
  QdTables tab;
  tab.before = reinterpret_cast<int*>(slots + kQdWarps * slot);
  tab.len = tab.before + kQdMaxBatch + 4;
  tab.page = tab.len + kQdMaxBatch;
  volatile int* const abort_flag = tab.page + kQdMaxBatch;
  // [warp][16]: where its walk is, the piece it is at (kept here: the products need the registers), whether its sums are in its slot, its ring, the
  // block's ranges
  volatile int* const records = abort_flag + 8;
  uint64_t* const full = reinterpret_cast<uint64_t*>(tab.page + kQdMaxBatch + 8 + kQdWarps * 16);  // [warp][stage]
  uint64_t* const empty = full + kQdWarps * kQdMaxStages;

  if (threadIdx.x < kQdWarps * kQdMaxStages) {
    ptx::mbar_init(&full[threadIdx.x], 1);
    ptx::mbar_init(&empty[threadIdx.x], 1);
  }
  if (threadIdx.x == 0) {
    *abort_flag = p.give_up && (blockIdx.x & 1);
  }
  if (threadIdx.x < kQdWarps) records[threadIdx.x * 16 + 8] = records[threadIdx.x * 16 + 9] = 0;
  ptx::fence_mbar_init();
  ptx::fence_proxy_async_smem();
  ptx::griddep_launch_dependents();
  if (!p.static_table) ptx::griddep_wait();
  for (int b = threadIdx.x; b < p.batch; b += kQdThreads) {
    const int beg = p.indptr[b], pages = p.indptr[b + 1] - beg;
    const int len = pages > 0 ? (pages - 1) * p.page_size + min(max(p.last_page_len[b], 0), p.page_size) : 0;
    tab.len[b] = len;
    tab.page[b] = beg;
    tab.before[b + 1] = qd_seen(p, len).chunks();
  }
  __syncthreads();
  if (warp == 0) {
    const int each = (p.batch + 31) / 32, b0 = min(p.batch, lane * each), b1 = min(p.batch, b0 + each);
    int sum = 0, most = 0;
    for (int b = b0; b < b1; ++b) {
      sum += tab.before[b + 1];
      most = max(most, tab.before[b + 1]);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) abort_flag[1] = most;
    int total = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, total, d);
      if (lane >= d) total += up;
    }
    int run = total - sum;
    if (lane == 0) tab.before[0] = 0;
    for (int b = b0; b < b1; ++b) {
      run += tab.before[b + 1];
      tab.before[b + 1] = run;
    }
  }
  __syncthreads();
  const unsigned each = tab.before[p.batch], all = each * p.heads, items = p.batch * p.heads;
  // Measured, equal shares -> whole sequences, us, 32 heads over 8 of 128: 1 of 977 tokens 10.3 -> 9.2, 8 of 1000 11.6 -> 9.8, 16 of 2000 17.7 -> 13.7, 18 of 3000
  // 21.0 -> 17.4; but 1 of 1500 11.0 -> 11.4.
  const bool whole = items <= gridDim.x && static_cast<unsigned>(abort_flag[1]) <= all / gridDim.x + min(p.alone, p.slack / items);
  ptx::griddep_wait();

  T* const out = reinterpret_cast<T*>(p.out);
  const unsigned own_head = blockIdx.x / p.batch, own_b = blockIdx.x % p.batch;  // (blocks behind the last one: nothing)
  const QdRanges mine = !whole ? qd_ranges(QdCut(all, gridDim.x), blockIdx.x) : blockIdx.x >= items ? qd_ranges(all, all) : qd_ranges(own_head * each + tab.before[own_b], own_head * each + tab.before[own_b + 1]);
  const int warps = whole ? kQdWarps : QdCut(all, gridDim.x).each;
  // (sequences without a visible key are in nobody's range: their output is zero)
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x)
    if (tab.before[b] == tab.before[b + 1])
      for (int e = threadIdx.x; e < p.heads * p.rep * D; e += kQdThreads) stf(out + b * p.out_stride + e, 0.f);

  if (warp == kQdWarps) {
    // ---------------------------------------------------------------- copies: a lane for each warp
    const unsigned v = min(lane, warps - 1);
    QdWalk walk = qd_walk(tab, p.batch, mine.begin(v), lane < warps ? mine.begin(v + 1) : 0u);
    QdPiece it{};
    QdSeen see{};
    bool more = qd_next(tab, p.batch, walk, it);
    int c = it.beg, stage = 0, kv = 0, pages = 0;
    uint32_t phase = 1;
    if (more) {
      see = qd_seen(p, tab.len[it.b]);
      kv = it.head / p.div;
      pages = tab.page[it.b];
    }
    // page ids of the next chunk, asked for ahead of its turn
    int id0 = 0, id1 = 0;
    auto look = [&]() {
      const int tok = see.token(c);
      id0 = p.indices[pages + (tok >> p.page_shift)];
      if (p.page_shift == 4) id1 = tok + 16 < see.len ? p.indices[pages + (tok >> 4) + 1] : id0;
    };
    if (more) look();
    uint64_t since = ptx::globaltimer_ns();
    uint32_t idle = 0;
    while (__any_sync(0xffffffffu, more)) {
      const bool go = more && ptx::mbar_test_wait(&empty[lane * kQdMaxStages + stage], phase);
      if (go) {
        const int tok = see.token(c), blocks = min(kQdChunk, see.len - tok + 15) >> 4;
        if (id0 < 0 || id0 >= p.max_pages || (p.page_shift == 4 && (id1 < 0 || id1 >= p.max_pages))) {
          if (p.status) atomicCAS(p.status, 0, kStatusBadIndex);
          id0 = id1 = 0;
        }
        uint64_t* bar = &full[lane * kQdMaxStages + stage];
        uint8_t* to = smem + lane * ring_bytes + stage * 2 * F.block;
        auto block = [&](int page, int off) { return p.pool + (((static_cast<int64_t>(page) * p.kv_heads + kv) << (p.page_shift - 4)) + (off >> 4)) * F.block; };
        ptx::mbar_expect_tx(bar, blocks * F.block);
        if (p.page_shift == 4) {
          ptx::bulk_load_1d(to, block(id0, 0), F.block, bar);
          if (blocks > 1) ptx::bulk_load_1d(to + F.block, block(id1, 0), F.block, bar);
        } else {
          ptx::bulk_load_1d(to, block(id0, tok & (p.page_size - 1)), blocks * F.block, bar);
        }
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
        if (++c == it.end) {
          more = qd_next(tab, p.batch, walk, it);
          if (more) {
            c = it.beg;
            see = qd_seen(p, tab.len[it.b]);
            kv = it.head / p.div;
            pages = tab.page[it.b];
          }
        }
        if (more) look();
      }
      if (__any_sync(0xffffffffu, go)) {
        idle = 0;
      } else {
        __nanosleep(200);
        if ((++idle & 63u) == 0) {
          const uint64_t now = ptx::globaltimer_ns();
          if (idle == 64) since = now;
          if (__any_sync(0xffffffffu, *abort_flag != 0 || now - since > ptx::kDefaultWaitNs)) {
            if (lane == 0) {
              if (p.status) atomicCAS(p.status, 0, kStatusTimeoutProducer);
              *abort_flag = 1;
            }
            break;
          }
        }
      }
    }
    // (no copy may land in shared memory that another block has by then: a warp that gave up has not waited for its own)
    if (lane < warps) {
      since = ptx::globaltimer_ns();
      for (int s = 0; s < p.stages; ++s) {
        if (stage == 0) phase ^= 1u;
        stage = stage == 0 ? p.stages - 1 : stage - 1;
        while (!ptx::mbar_try_wait(&full[lane * kQdMaxStages + stage], phase ^ 1u) && ptx::globaltimer_ns() - since < 10000000ull) {
        }
      }
    }
  } else if (warp < warps) {
    // ---------------------------------------------------------------- products
    const int g = lane >> 2, t4 = lane & 3;
    const int x = HALVES ? t4 >> 1 : 0;                     // half of the groups that this lane's columns 2 t4, 2 t4 + 1 stand for
    const int col = HALVES ? (2 * t4) & 3 : 2 * t4;         // first of the lane's two heads
    const int tau = 4 * (g >> 1) + (g & 1);                 // rows g and g + 8 of a block of 16 are its tokens tau and tau + 2
    const uint8_t* const ring = smem + warp * ring_bytes;
    uint64_t* const my_full = full + warp * kQdMaxStages;
    uint64_t* const my_empty = empty + warp * kQdMaxStages;
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    volatile int* const rec = records + warp * 16;
    {
      const QdWalk walk = qd_walk(tab, p.batch, mine.begin(warp), mine.begin(warp + 1));
      rec[0] = walk.x; rec[1] = walk.end; rec[2] = walk.head; rec[3] = walk.b;
      mine.keep(rec + 10);
    }
    for (;;) {
      QdPiece it;
      {
        QdWalk walk{static_cast<unsigned>(rec[0]), static_cast<unsigned>(rec[1]), rec[2], rec[3]};
        __syncwarp();
        if (!qd_next(tab, p.batch, walk, it)) break;
        rec[0] = walk.x; rec[2] = walk.head; rec[3] = walk.b;
        qd_keep(rec + 4, it);
        __syncwarp();
      }
      const QdSeen see = qd_seen(p, tab.len[it.b]);
      // queries: word w of a lane's key codes holds dimensions 32 w + 8 t4 .. + 7, pairs (i, i + 4) of which are a register's halves
      uint32_t qb[W][4], zb0, zb1 = 0;
      float scale[2];
      {
        const int hq = HALVES ? g & 3 : g, xq = HALVES ? g >> 2 : 0;  // head and half of column g
        float v[W][8], most = 0.f;
        const T* row = reinterpret_cast<const T*>(p.q) + it.b * p.q_stride + static_cast<int64_t>(it.head * p.rep + hq) * D + 8 * t4;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          if (hq < p.rep) {
            ldf8<T>(row + 32 * w, v[w]);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[w][i] = 0.f;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(v[w][i]));
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        // 2^-e with most in [2^e, 2^(e + 1)); an all-zero head, and one that is not finite, as it is
        const int e = most > 0.f && most <= 3.4e38f ? max(-126, min(126, static_cast<int>(__float_as_uint(most) >> 23) - 127)) : 0;
        const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23), up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
        const float turn = down * p.sign;
        float sum[G];
#pragma unroll
        for (int i = 0; i < G; ++i) sum[i] = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const bool mine = !HALVES || (w / WG) / N == xq;
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // (odd pairs meet codes times 16)
            const float by = i & 1 ? 1024.f : 16384.f, back = i & 1 ? 0x1p-20f : 0x1p-24f;
            qb[w][i] = mine ? pk2<__half>(v[w][i] * turn * by, v[w][i + 4] * turn * by) : 0u;
            const float2 f = cvt2<__half>(qb[w][i]);  // (as they enter the products)
            sum[w / WG] += (f.x + f.y) * back;
          }
        }
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
#pragma unroll
          for (int i = 0; i < G; ++i) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], d);
        }
        float hi[G], lo[G];
#pragma unroll
        for (int i = 0; i < G; ++i) {
          hi[i] = __bfloat162float(__float2bfloat16_rn(sum[i]));
          lo[i] = sum[i] - hi[i];
        }
        // column operand of the offsets' product: pairs of numbers as a token's words have them
        using B = __nv_bfloat16;
        if (G == 1) zb0 = pk2<B>(0.f, hi[0]), zb1 = pk2<B>(0.f, lo[0]);
        else zb0 = pk2<B>(hi[0], hi[1 % G]), zb1 = pk2<B>(lo[0], lo[1 % G]);
        if (G == 4 && t4 == 1) zb0 = pk2<B>(hi[2 % G], hi[3 % G]), zb1 = pk2<B>(lo[2 % G], lo[3 % G]);
        if (t4 >= (G == 4 ? 2 : 1)) zb0 = zb1 = 0u;
        // what the lane's own columns need
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          scale[k] = fmaxf(0x1p-126f, __shfl_sync(0xffffffffu, up, (2 * t4 + k) * 4) * (1024.f * (p.cap_log2 > 0.f ? p.cap_scale : p.scale_log2)));
        }
      }

      // `down` takes weights times scales to 16 bits, of a column each; scales up to `lim` are within it, weights up to 2^8 taken into account.  `weighed`:
      // exponent of the largest scale with a weight to speak of, and (times 32) how many times that weight may still be halved
      float o[MT][4], eight[N][4], zs[N][2], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, down[2] = {0x1p100f, 0x1p100f}, lim = 0.f;
      int weighed[2] = {-200 * 32, -200 * 32};
#pragma unroll
      for (int i = 0; i < MT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) zs[i][0] = zs[i][1] = eight[i][0] = eight[i][1] = eight[i][2] = eight[i][3] = 0.f;

      for (int c = it.beg; c < it.end; ++c) {
        if (ok && !__all_sync(0xffffffffu, ptx::bounded_mbar_wait(&my_full[stage], phase, abort_flag))) {
          if (p.status && lane == 0) atomicCAS(p.status, 0, kStatusTimeoutEpilogue);
          ok = false;
        }
        if (!ok) continue;
        const uint8_t* st = ring + stage * 2 * F.block;
        const int tok0 = see.token(c);
        const bool edge = tok0 + kQdChunk > see.len || (tok0 < see.lo && tok0 + kQdChunk > see.first);  // some key is not visible
        // (16 tokens that a short last chunk does not have: whatever the stage holds, and not visible)
        float s[2][4];  // (tau, first head), (tau, second), (tau + 2, first), (tau + 2, second)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint8_t* ka = st + u * F.block + tau * (D / 2) + t4 * (D / 8);
          const uint8_t* sa = st + u * F.block + F.codes + tau * 4 * G;
          uint32_t ku[W], kv[W];
          if (W == 4) {
            const uint4 a = *reinterpret_cast<const uint4*>(ka), b = *reinterpret_cast<const uint4*>(ka + D);
            ku[0] = a.x; ku[1] = a.y; ku[2 % W] = a.z; ku[3 % W] = a.w;
            kv[0] = b.x; kv[1] = b.y; kv[2 % W] = b.z; kv[3 % W] = b.w;
          } else {
            const uint2 a = *reinterpret_cast<const uint2*>(ka), b = *reinterpret_cast<const uint2*>(ka + D);
            ku[0] = a.x; ku[1] = a.y;
            kv[0] = b.x; kv[1] = b.y;
          }
          const int z_at = G == 4 ? 8 + 4 * (t4 & 1) : G == 2 ? 4 : 0;
          const uint32_t za = *reinterpret_cast<const uint32_t*>(sa + z_at), zb = *reinterpret_cast<const uint32_t*>(sa + 8 * G + z_at);
          QdScales<G, HALVES> fa, fb;
          fa.keys(sa, x);
          fb.keys(sa + 8 * G, x);
          qd_mma_bf16(s[u], za, zb, za, zb, zb0, zb1);
          float acc[N][4];
#pragma unroll
          for (int w = 0; w < W; ++w) {
            const int i = (w / WG) % N;
            const uint32_t a = ku[w], b = kv[w], ah = a >> 8, bh = b >> 8;
            const uint32_t even = 0x000f000fu, odd = 0x00f000f0u;
            if (w % WG == 0 && w / WG < N) qd_mma_f16(acc[i], a & even, b & even, a & odd, b & odd, qb[w][0], qb[w][1]);
            else qd_mma_f16_add(acc[i], a & even, b & even, a & odd, b & odd, qb[w][0], qb[w][1]);
            qd_mma_f16_add(acc[i], ah & even, bh & even, ah & odd, bh & odd, qb[w][2], qb[w][3]);
          }
#pragma unroll
          for (int i = 0; i < N; ++i) {
            s[u][0] = fmaf(fa.s[i], acc[i][0], s[u][0]);
            s[u][1] = fmaf(fa.s[i], acc[i][1], s[u][1]);
            s[u][2] = fmaf(fb.s[i], acc[i][2], s[u][2]);
            s[u][3] = fmaf(fb.s[i], acc[i][3], s[u][3]);
          }
          if (HALVES) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[u][i] += __shfl_xor_sync(0xffffffffu, s[u][i], 2);
          }
        }
        // scores in log2 units are these times a factor, which the maximum and the exponent's argument take in
        float by[2] = {scale[0], scale[1]};
        if (p.cap_log2 > 0.f) {
#pragma unroll
          for (int i = 0; i < 8; ++i) s[i >> 2][i & 3] = p.cap_log2 * ptx::tanh_ex2(s[i >> 2][i & 3] * scale[i & 1]);
          by[0] = by[1] = 1.f;
        }
        QdScales<G, HALVES> f[4];  // of the values of tokens tau, tau + 2, 16 + tau, 18 + tau
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i].values(st + (i >> 1) * F.block + F.part + F.codes + (tau + 2 * (i & 1)) * 4 * G, x);
        if (edge) {  // (what is not visible has no weight, and may hold no numbers)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = tok0 + (i >> 1) * 16 + tau + 2 * (i & 1);
            if (j >= see.len || (j < see.lo && j >= see.first)) {
              s[i >> 1][2 * (i & 1)] = s[i >> 1][2 * (i & 1) + 1] = -INFINITY;
              f[i].none();
            }
          }
        }
        const float large[4] = {f[0].largest(), f[1].largest(), f[2].largest(), f[3].largest()};
        float top[2] = {s[0][0], s[0][1]}, wide = fmaxf(fmaxf(large[0], large[1]), fmaxf(large[2], large[3]));
#pragma unroll
        for (int i = 2; i < 8; ++i) top[i & 1] = fmaxf(top[i & 1], s[i >> 2][i & 3]);
        if (__builtin_expect(__any_sync(0xffffffffu, top[0] * by[0] > m[0] + 8.f || top[1] * by[1] > m[1] + 8.f || wide > lim), 0)) {
          float narrow = INFINITY;  // the smallest scale that is not zero
#pragma unroll
          for (int i = 0; i < 4; ++i) narrow = large[i] > 0.f ? fminf(narrow, large[i]) : narrow;
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) {
            top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], d));
            top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], d));
            wide = fmaxf(wide, __shfl_xor_sync(0xffffffffu, wide, d));
            narrow = fminf(narrow, __shfl_xor_sync(0xffffffffu, narrow, d));
          }
          float grown[2], a[2], mine[2] = {wide, wide};
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            top[k] *= by[k];
            grown[k] = top[k] > m[k] ? top[k] - m[k] : 0.f;
            m[k] = fmaxf(m[k], top[k]);
            a[k] = ptx::ex2_approx(-grown[k]);
            l[k] *= a[k];
#pragma unroll
            for (int i = 0; i < N; ++i) zs[i][k] *= a[k];
          }
          // scales of very different sizes, or none with a weight to speak of: the largest one that has one (below 2^-16 counted as if with it)
          if (__builtin_expect(__any_sync(0xffffffffu, wide > 16.f * narrow || top[0] < m[0] - 16.f || top[1] < m[1] - 16.f), 0)) {
            mine[0] = mine[1] = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              mine[i & 1] = fmaxf(mine[i & 1], large[i >> 1] * fminf(1.f, 65536.f * ptx::ex2_approx(fmaf(s[i >> 2][i & 3], by[i & 1], -m[i & 1]))));
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) {
              mine[0] = fmaxf(mine[0], __shfl_xor_sync(0xffffffffu, mine[0], d));
              mine[1] = fmaxf(mine[1], __shfl_xor_sync(0xffffffffu, mine[1], d));
            }
          }
          int low = 126;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            // (what was counted before has 2^-grown of its weight now; the first 24 of that, from 2^8 to 2^-16, leave it one to speak of)
            const int credit = (weighed[k] & 31) - static_cast<int>(ceilf(fminf(grown[k], 500.f))), old = (weighed[k] >> 5) + min(0, credit), now = max(old, qd_exponent(mine[k]));
            weighed[k] = now * 32 + (qd_exponent(mine[k]) >= old ? 24 : max(0, credit));
            // scales below 2^e are at 2^7 then: all that count, and others up to 2^12 times as large (no other chunk comes here for those)
            const int was = 7 - qd_exponent(down[k]);
            const int e = min(126, max(-93, max(now + 1, min(max(qd_exponent(wide) + 1, was), now + 13))));
            a[k] = ptx::ex2_approx(static_cast<float>(was - e) - grown[k]);
            down[k] = qd_power(7 - e);
            low = min(low, e);
          }
          lim = qd_power(low);
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            o[i][0] *= a[0]; o[i][1] *= a[1]; o[i][2] *= a[0]; o[i][3] *= a[1];
          }
#pragma unroll
          for (int i = 0; i < N; ++i) {
            eight[i][0] *= a[0]; eight[i][1] *= a[1]; eight[i][2] *= a[0]; eight[i][3] *= a[1];
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float& v = s[i >> 2][i & 3];
          v = ptx::ex2_approx(fmaf(v, by[i & 1], -m[i & 1]));  // (a chunk has a visible key, whose score m has seen: zero for what is not visible)
          l[i & 1] += v;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint8_t* vb = st + u * F.block + F.part;
          const QdScales<G, HALVES>&fa = f[2 * u], &fb = f[2 * u + 1];
          uint32_t vw[MT];
#pragma unroll
          for (int h = 0; h < D / 64; ++h) {
            const uint4 v = *reinterpret_cast<const uint4*>(vb + h * 512 + g * 64 + t4 * 16);
            vw[4 * h] = v.x; vw[4 * h + 1] = v.y; vw[4 * h + 2] = v.z; vw[4 * h + 3] = v.w;
          }
          uint32_t b0[N], b1[N];
          if constexpr (N == 1) {
            zs[0][0] = fmaf(s[u][0], fa.mid[0], fmaf(s[u][2], fb.mid[0], zs[0][0]));
            zs[0][1] = fmaf(s[u][1], fa.mid[0], fmaf(s[u][3], fb.mid[0], zs[0][1]));
            b0[0] = qd_transposed(pk2<__half>(s[u][0] * (fa.s[0] * down[0]), s[u][1] * (fa.s[0] * down[1])));
            b1[0] = qd_transposed(pk2<__half>(s[u][2] * (fb.s[0] * down[0]), s[u][3] * (fb.s[0] * down[1])));
          } else {  // two groups an instruction
            const uint64_t down0 = ptx::f32x2(down[0], down[0]), down1 = ptx::f32x2(down[1], down[1]);
            const uint64_t w0 = ptx::f32x2(s[u][0], s[u][0]), w1 = ptx::f32x2(s[u][1], s[u][1]), w2 = ptx::f32x2(s[u][2], s[u][2]), w3 = ptx::f32x2(s[u][3], s[u][3]);
#pragma unroll
            for (int i = 0; i < N; i += 2) {
              const uint64_t sa = ptx::f32x2(fa.s[i], fa.s[(i + 1) % N]), sb = ptx::f32x2(fb.s[i], fb.s[(i + 1) % N]);
              const uint64_t ma = ptx::f32x2(fa.mid[i], fa.mid[(i + 1) % N]), mb = ptx::f32x2(fb.mid[i], fb.mid[(i + 1) % N]);
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const float2 z = ptx::f32x2_get(ptx::fma_f32x2(k ? w1 : w0, ma, ptx::fma_f32x2(k ? w3 : w2, mb, ptx::f32x2(zs[i][k], zs[(i + 1) % N][k]))));
                zs[i][k] = z.x;
                zs[(i + 1) % N][k] = z.y;
              }
              const float2 p0 = ptx::f32x2_get(ptx::mul_f32x2(w0, ptx::mul_f32x2(sa, down0))), p1 = ptx::f32x2_get(ptx::mul_f32x2(w1, ptx::mul_f32x2(sa, down1)));
              const float2 p2 = ptx::f32x2_get(ptx::mul_f32x2(w2, ptx::mul_f32x2(sb, down0))), p3 = ptx::f32x2_get(ptx::mul_f32x2(w3, ptx::mul_f32x2(sb, down1)));
              b0[i] = qd_transposed(pk2<__half>(p0.x, p1.x));
              b1[i] = qd_transposed(pk2<__half>(p2.x, p3.x));
              b0[(i + 1) % N] = qd_transposed(pk2<__half>(p0.y, p1.y));
              b1[(i + 1) % N] = qd_transposed(pk2<__half>(p2.y, p3.y));
            }
          }
#pragma unroll
          for (int i = 0; i < N; ++i) qd_mma_f16_add(eight[i], 0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u, b0[i], b1[i]);  // -8, -8 times 16
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const int j = (i * 16 / GROUP) % N;
            const uint32_t v = vw[i], vh = v >> 8, even = 0x000f000fu, odd = 0x00f000f0u;
            qd_mma_f16_add(o[i], v & even, v & odd, vh & even, vh & odd, b0[j], b1[j]);
          }
        }
        __syncwarp();  // every lane has read the stage
        if (lane == 0) ptx::mbar_arrive(&my_empty[stage]);
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }

      // ------------------------------------------------------------ the end of a piece
      it = qd_kept(rec + 4);
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          l[k] += __shfl_xor_sync(0xffffffffu, l[k], d);
#pragma unroll
          for (int i = 0; i < N; ++i) zs[i][k] += __shfl_xor_sync(0xffffffffu, zs[i][k], d);
        }
      }
      const float up[2] = {1.f / down[0], 1.f / down[1]};
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int j = (i * 16 / GROUP) % N;
        o[i][0] = fmaf((o[i][0] + eight[j][0]) * 0x1p24f, up[0], zs[j][0]); o[i][1] = fmaf((o[i][1] + eight[j][1]) * 0x1p24f, up[1], zs[j][1]);
        o[i][2] = fmaf((o[i][2] + eight[j][2]) * 0x1p20f, up[0], zs[j][0]); o[i][3] = fmaf((o[i][3] + eight[j][3]) * 0x1p20f, up[1], zs[j][1]);
      }
      const QdRanges mine = qd_ranges(rec + 10);
      const unsigned X0 = mine.x0, X1 = mine.x0 + mine.n, x0 = mine.begin(warp), x1 = mine.begin(warp + 1);
      if (it.start >= x0 && it.stop <= x1) {
        float r[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float f = 1.f, sum = l[k];
          if (p.sink != nullptr && col + k < p.rep) {
            const float snk = ldf<T>(reinterpret_cast<const T*>(p.sink) + it.head * p.rep + col + k) * 1.4426950408889634f, top = fmaxf(snk, m[k]);
            f = ptx::ex2_approx(m[k] - top);
            sum = fmaf(f, l[k], ptx::ex2_approx(snk - top));
          }
          r[k] = sum != 0.f ? f * ptx::rcp_approx(sum) : 0.f;
        }
        // rounded, and 8 x 8 blocks transposed, so that a lane has two neighbouring dimensions of head g
        const int hq = HALVES ? g & 3 : g, xq = HALVES ? g >> 2 : 0;
        T* to = out + it.b * p.out_stride + static_cast<int64_t>(it.head * p.rep + hq) * D + 2 * t4;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const uint32_t a = qd_transposed(quant_kv_means<T>(o[i][0] * r[0], o[i][1] * r[1])), b = qd_transposed(quant_kv_means<T>(o[i][2] * r[0], o[i][3] * r[1]));
          if (hq < p.rep && (!HALVES || (i * 16 / GROUP) / N == xq)) {
            *reinterpret_cast<uint32_t*>(to + 16 * i) = a;
            *reinterpret_cast<uint32_t*>(to + 16 * i + 8) = b;
          }
        }
        continue;
      }

      // ------------------------------------------------------------ a piece: its sums into the slot, or the ring, which takes no more
      const bool in_slot = x0 >= it.start;
      {
        float* to = in_slot ? slots + warp * slot : reinterpret_cast<float*>(smem + warp * ring_bytes);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          if (!HALVES || (i * 16 / GROUP) / N == x) {
            if (col < p.rep) {
              to[col * (D + 4) + 16 * i + g] = o[i][0];
              to[col * (D + 4) + 16 * i + 8 + g] = o[i][2];
            }
            if (col + 1 < p.rep) {
              to[(col + 1) * (D + 4) + 16 * i + g] = o[i][1];
              to[(col + 1) * (D + 4) + 16 * i + 8 + g] = o[i][3];
            }
          }
        }
        if (g == 0 && x == 0) {
          float* ml = to + p.rep * (D + 4);
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (col + k < p.rep) {
              ml[2 * (col + k)] = m[k];
              ml[2 * (col + k) + 1] = l[k];
            }
        }
        __threadfence_block();
        __syncwarp();
        if (lane == 0) rec[in_slot ? 8 : 9] = 1;
      }
      // The warps of this block that end with the sequence share its heads (one that goes on with the next sequence has them to itself, where
      // nobody else has a piece); the i-th lane looks after the i-th of all warps that have one.
      const unsigned at = mine.begin(min(lane, warps)), behind = mine.begin(min(lane + 1, warps));
      const bool has = lane < warps && at < it.stop && behind > it.start;
      const uint32_t having = __ballot_sync(0xffffffffu, has), ending = __ballot_sync(0xffffffffu, has && behind <= it.stop);
      const int w0 = __ffs(having) - 1, n = __popc(having), each = max(1, __popc(ending)), h0 = warp - w0;
      if (h0 >= p.rep || (n > 1 && x1 > it.stop)) continue;
      const unsigned begin = mine.begin(min(w0 + lane, warps));
      const int from = (lane < n && begin < it.start ? (w0 + lane) * (ring_bytes / 4) : kQdWarps * ring_bytes / 4 + min(w0 + lane, kQdWarps - 1) * slot);
      // (a wait that ran out is an error that the host reads; the chunks are counted all the same, so that the tickets are zero after this call too)
      const bool there = qd_wait(records + min(w0 + lane, kQdWarps - 1) * 16 + (begin < it.start ? 9 : 8), lane < n, abort_flag);
      if (!there && p.status && lane == 0) atomicCAS(p.status, 0, kStatusTimeoutEpilogue);
      constexpr int C = D / 32;  // dimensions of a lane
      const bool inside = it.start >= X0 && it.stop <= X1;
      float* const part_ml = p.part + static_cast<int64_t>(2) * gridDim.x * p.rep * D;
      const int64_t place = (blockIdx.x * 2 + (it.start < X0 ? 0 : 1)) * p.rep;
      auto store = [&](int hh, const float (&acc)[C], float M, float L) {  // the sum of all pieces, divided
        float f = 1.f, sum = L;
        if (p.sink != nullptr) {
          const float snk = ldf<T>(reinterpret_cast<const T*>(p.sink) + it.head * p.rep + hh) * 1.4426950408889634f, most = fmaxf(snk, M);
          f = ptx::ex2_approx(M - most);
          sum = fmaf(f, L, ptx::ex2_approx(snk - most));
        }
        const float r = sum != 0.f ? f * ptx::rcp_approx(sum) : 0.f;
        T* to = out + it.b * p.out_stride + static_cast<int64_t>(it.head * p.rep + hh) * D + lane * C;
#pragma unroll
        for (int i = 0; i < C; i += 2) *reinterpret_cast<uint32_t*>(to + i) = quant_kv_means<T>(acc[i] * r, acc[i + 1] * r);
      };
      auto four = [&](const float* v, float f, float (&acc)[C], bool global) {
        if (C == 4) {
          const float4 t = global ? __ldcg(reinterpret_cast<const float4*>(v)) : *reinterpret_cast<const float4*>(v);
          acc[0] = fmaf(f, t.x, acc[0]); acc[1] = fmaf(f, t.y, acc[1]); acc[2 % C] = fmaf(f, t.z, acc[2 % C]); acc[3 % C] = fmaf(f, t.w, acc[3 % C]);
        } else {
          const float2 t = global ? __ldcg(reinterpret_cast<const float2*>(v)) : *reinterpret_cast<const float2*>(v);
          acc[0] = fmaf(f, t.x, acc[0]); acc[1] = fmaf(f, t.y, acc[1]);
        }
      };
      auto add_up = [&](auto heads) {  // H heads at a time: their loads follow one another without a wait
        constexpr int H = decltype(heads)::value;
        const float* const all = reinterpret_cast<const float*>(smem);
#pragma unroll 1
        for (int hb = h0; hb < p.rep; hb += H * each) {
          float2 ml[H];
          float M[H], L[H], f[H], acc[H][C];
          int hh[H];
#pragma unroll
          for (int h = 0; h < H; ++h) {  // (fewer heads than H: the first one again)
            hh[h] = hb + h * each < p.rep ? hb + h * each : hb;
            ml[h] = lane < n ? *reinterpret_cast<const float2*>(all + from + p.rep * (D + 4) + 2 * hh[h]) : make_float2(-INFINITY, 0.f);
          }
#pragma unroll
          for (int h = 0; h < H; ++h) {
            M[h] = warp_max(ml[h].x);
            f[h] = ml[h].x == M[h] ? 1.f : ptx::ex2_approx(ml[h].x - M[h]);
            L[h] = warp_sum(lane < n ? f[h] * ml[h].y : 0.f);
#pragma unroll
            for (int i = 0; i < C; ++i) acc[h][i] = 0.f;
          }
          for (int v = 0; v < n; ++v) {
            const float* o = all + __shfl_sync(0xffffffffu, from, v) + lane * C;
#pragma unroll
            for (int h = 0; h < H; ++h) four(o + hh[h] * (D + 4), __shfl_sync(0xffffffffu, f[h], v), acc[h], false);
          }
#pragma unroll
          for (int h = 0; h < H; ++h) {
            if (inside) {
              store(hh[h], acc[h], M[h], L[h]);
            } else {
              float* to = p.part + (place + hh[h]) * D + lane * C;
              if (C == 4) __stcg(reinterpret_cast<float4*>(to), make_float4(acc[h][0], acc[h][1], acc[h][2 % C], acc[h][3 % C]));
              else __stcg(reinterpret_cast<float2*>(to), make_float2(acc[h][0], acc[h][1]));
              if (lane == 0) __stcg(reinterpret_cast<float2*>(part_ml) + place + hh[h], make_float2(M[h], L[h]));
            }
          }
        }
      };
      if (!there) {
      } else if (h0 + each < p.rep) {
        add_up(std::integral_constant<int, 4>{});
      } else {
        add_up(std::integral_constant<int, 1>{});
      }
      if (inside) continue;

      // ------------------------------------------------------------ pieces of several blocks: for each head, whoever is last adds them up
      // (a ticket counts chunks; which blocks have them is worked out while it is on its way)
      __syncwarp();
      const unsigned have = min(it.stop, X1) - max(it.start, X0);
      const bool asks = h0 + lane * each < p.rep;
      unsigned* const ticket = p.tickets + (it.b * p.heads + it.head) * p.rep + h0 + lane * each;
      unsigned before = 0;
      if (asks) {
        __threadfence();
        before = atomicAdd(ticket, have);
      }
      const QdCut cut(static_cast<unsigned>(tab.before[p.batch]) * p.heads, gridDim.x);
      const int c0 = cut.range(it.start) / warps, blocks = static_cast<int>(cut.range(it.stop - 1) / warps) - c0 + 1;
      const bool is_last = asks && before + have == it.stop - it.start;
      if (is_last) {
        *ticket = 0u;
        __threadfence();
      }
      __syncwarp();
      uint32_t todo = __ballot_sync(0xffffffffu, is_last && there);
      // H heads at a time, UNROLL of their pieces: eight loads are on their way
      auto merge = [&](auto heads, auto unroll) {
        constexpr int H = decltype(heads)::value, UNROLL = decltype(unroll)::value;
        const float* from[H];
        const float2* ml_from[H];
        int hh[H];
        float M[H], L[H], acc[H][C];
#pragma unroll
        for (int h = 0; h < H; ++h) {  // (fewer heads than H: the last one again)
          hh[h] = h0 + (__ffs(todo) - 1) * each;
          if (todo & (todo - 1) || h == H - 1) todo &= todo - 1;
          // the first block has its piece in its second place, the others in their first: piece c is 2 c - 1 places behind that
          from[h] = p.part + (static_cast<int64_t>(2 * c0 + 1) * p.rep + hh[h]) * D + lane * C;
          ml_from[h] = reinterpret_cast<const float2*>(part_ml) + static_cast<int64_t>(2 * c0 + 1) * p.rep + hh[h];
          M[h] = -INFINITY;
          L[h] = 0.f;
#pragma unroll
          for (int i = 0; i < C; ++i) acc[h][i] = 0.f;
        }
        for (int c = 0; c < blocks; c += 32) {
          const int n = min(32, blocks - c);
          float f[H], ahead[UNROLL][H][C];  // (the first pieces are asked for beside what they are worth)
          float2 ml[H];
#pragma unroll
          for (int v = 0; v < UNROLL; ++v)
#pragma unroll
            for (int h = 0; h < H; ++h) {
              const float* o = from[h] + static_cast<int64_t>(max(0, 2 * (c + v) - 1)) * p.rep * D;
              if (v >= n) {
#pragma unroll
                for (int i = 0; i < C; ++i) ahead[v][h][i] = 0.f;
              } else if (C == 4) {
                const float4 t = __ldcg(reinterpret_cast<const float4*>(o));
                ahead[v][h][0] = t.x; ahead[v][h][1] = t.y; ahead[v][h][2 % C] = t.z; ahead[v][h][3 % C] = t.w;
              } else {
                const float2 t = __ldcg(reinterpret_cast<const float2*>(o));
                ahead[v][h][0] = t.x; ahead[v][h][1] = t.y;
              }
            }
#pragma unroll
          for (int h = 0; h < H; ++h) ml[h] = lane < n ? __ldcg(ml_from[h] + max(0, 2 * (c + lane) - 1) * p.rep) : make_float2(-INFINITY, 0.f);
#pragma unroll
          for (int h = 0; h < H; ++h) {
            const float top = fmaxf(M[h], warp_max(ml[h].x)), a = M[h] == top ? 1.f : ptx::ex2_approx(M[h] - top);
            M[h] = top;
            f[h] = ml[h].x == top ? 1.f : ptx::ex2_approx(ml[h].x - top);
            L[h] = fmaf(a, L[h], warp_sum(lane < n ? f[h] * ml[h].y : 0.f));
#pragma unroll
            for (int i = 0; i < C; ++i) acc[h][i] *= a;
          }
#pragma unroll
          for (int v = 0; v < UNROLL; ++v)
#pragma unroll
            for (int h = 0; h < H; ++h) {
              const float fv = __shfl_sync(0xffffffffu, f[h], v);
#pragma unroll
              for (int i = 0; i < C; ++i)
                if (v < n) acc[h][i] = fmaf(fv, ahead[v][h][i], acc[h][i]);
            }
#pragma unroll UNROLL
          for (int v = UNROLL; v < n; ++v) {
            const int64_t at = static_cast<int64_t>(max(0, 2 * (c + v) - 1)) * p.rep * D;
#pragma unroll
            for (int h = 0; h < H; ++h) four(from[h] + at, __shfl_sync(0xffffffffu, f[h], v), acc[h], true);
          }
        }
#pragma unroll
        for (int h = 0; h < H; ++h) store(hh[h], acc[h], M[h], L[h]);
      };
      while (todo) {
        if (todo & (todo - 1)) merge(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{});
        else merge(std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
      }
    }
  }
}

struct DecodeQuantLaunch {
  DecodeQuantParams& p;
  int sms;
  cudaStream_t stream;
  template <typename T, int D, int GROUP>
  int operator()() const {
    if (D / GROUP > 1 && p.rep <= 4) return run<T, D, GROUP, (D / GROUP > 1)>();
    return run<T, D, GROUP, false>();
  }
  template <typename T, int D, int GROUP, bool HALVES>
  int run() const {
    constexpr int stage = 2 * quant_kv(D, GROUP).block;
    static PerDeviceOnce once;
    const cudaError_t e = once.run([&] { return cudaFuncSetAttribute(attn_decode_quant_kernel<T, D, GROUP, HALVES>, cudaFuncAttributeMaxDynamicSharedMemorySize, kQdSmem); });
    if (e != cudaSuccess) return (int)e;
    p.stages = kQdMaxStages;
    while (p.stages > 2 && qd_smem(D, stage, p.rep, p.stages) > kQdSmem) --p.stages;
    const int smem = qd_smem(D, stage, p.rep, p.stages);
    if (smem > kQdSmem) return -1;
    return (int)launch_pdl(attn_decode_quant_kernel<T, D, GROUP, HALVES>, dim3(sms), dim3(kQdThreads), smem, stream, p);
  }
};

// Query heads in equal groups of at most 8 that share a KV head.
static inline int qd_groups(int rep) {
  int div = (rep + 7) / 8;
  while (rep % div) ++div;
  return div;
}
static std::atomic<int> g_qd_give_up{0};

// Bytes of the partial sums in a workspace, whatever a call's batch and heads: calls of any size share one, and nobody's sums may be where
// another has its tickets.
static inline int64_t qd_part_bytes() { return ((int64_t)2 * device_sm_count() * 8 * (128 + 2) * 4 + 255) / 256 * 256; }

}  // namespace blitz

extern "C" {
using namespace blitz;

// Scratch of a call: partial sums, then tickets, which have to be zero before the first call and are again after each.
int64_t blitz_attn_decode_quant_workspace_bytes(int batch, int q_heads, int dim) {
  return qd_part_bytes() + (int64_t)batch * q_heads * 4;
}

// Test aid: while `on` is not zero, every other block of the following launches begins as if a wait had run out.
void blitz_attn_decode_quant_give_up(int on) { blitz::g_qd_give_up = on != 0; }

// q: [batch] rows with the query heads in their first q_heads * dim columns (pitch a multiple of 8, 16-byte aligned; so out).  A sequence
// without keys has an output of zeros.  static_table != 0 promises that the tables are not written by kernels still running in this
// stream.  More than 1024 sequences go in several launches.
int blitz_attn_decode_quant(const void* q, int64_t q_stride, const void* pool, const int32_t* indices, const int32_t* indptr,
                            const int32_t* last_page_len, void* out, int64_t out_stride, void* workspace, int64_t workspace_bytes, int batch,
                            int q_heads, int kv_heads, int dim, int group, int page_size, int max_pages, float sm_scale, int window,
                            int keep_first, float softcap, const void* sink, int static_table, int* status, int dtype, cudaStream_t stream) {
  if (batch <= 0) return 0;
  if (!quant_kv_supported(dim, group, page_size) || max_pages < 1 || kv_heads < 1 || q_heads % kv_heads || window < 0 || keep_first < 0 || softcap < 0.f) return -1;
  if (((q_stride | out_stride) & 7) || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(pool) | reinterpret_cast<uintptr_t>(workspace)) & 15)) return -1;
  if (workspace == nullptr || workspace_bytes < blitz_attn_decode_quant_workspace_bytes(batch, q_heads, dim)) return -1;
  DecodeQuantParams p;
  p.div = qd_groups(q_heads / kv_heads); p.rep = q_heads / kv_heads / p.div; p.heads = kv_heads * p.div; p.kv_heads = kv_heads;
  p.q_stride = q_stride; p.pool = (const uint8_t*)pool; p.indices = indices; p.out_stride = out_stride;
  p.part = (float*)workspace;
  p.page_size = page_size; p.max_pages = max_pages; p.page_shift = 0; p.stages = 2;
  while ((1 << p.page_shift) < page_size) ++p.page_shift;
  p.slack = 15000000u / (2 * quant_kv(dim, group).block);  // 2.5 us at 6 TB/s
  p.alone = 184320u / (2 * quant_kv(dim, group).block);    // (what eleven warps compute in that time)
  const float size = sm_scale < 0.f ? -sm_scale : sm_scale > 0.f ? sm_scale : 1.f;
  p.sign = sm_scale < 0.f ? -1.f : sm_scale > 0.f ? 1.f : sm_scale;
  p.scale_log2 = size * 1.4426950408889634f; p.cap_scale = softcap > 0.f ? size / softcap : 0.f; p.cap_log2 = softcap * 1.4426950408889634f;
  p.window = window; p.keep_first = keep_first; p.sink = sink; p.static_table = static_table; p.status = status; p.give_up = g_qd_give_up;
  for (int b = 0; b < batch; b += kQdMaxBatch) {
    p.batch = batch - b < kQdMaxBatch ? batch - b : kQdMaxBatch;
    p.q = (const char*)q + (int64_t)b * q_stride * 2;
    p.out = (char*)out + (int64_t)b * out_stride * 2;
    p.indptr = indptr + b; p.last_page_len = last_page_len + b;
    p.tickets = (unsigned*)((char*)workspace + qd_part_bytes()) + (int64_t)b * q_heads;
    const int rc = quant_kv_dispatch(dtype, dim, group, DecodeQuantLaunch{p, device_sm_count(), stream});
    if (rc) return rc;
  }
  return 0;
}

}  // extern "C"
