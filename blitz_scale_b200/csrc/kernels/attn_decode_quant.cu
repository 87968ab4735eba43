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
// values: 128 + c in bf16, and a product of a constant matrix with the weights takes 136 off again (the codes around zero, so that
// the rounding of p_j s_j is not amplified by an offset that cancels).  Queries enter in fp16, a head divided by a power of two near its
// largest entry: bf16 and fp16 numbers are exact there (next to the largest, that is), and so are their products with codes.  p s is
// rounded to bf16 (its range is the scales'), as in attention over 16-bit caches; in fp16 models to two bf16 numbers, hi + lo.  The part
// of z_j stays in 32 bits; the sums of q_d z_g in the scores are one more product, of z as stored with sums of q in two bf16 numbers.
//
// S^T = K Q^T has 16 tokens as rows and at most 8 query heads as columns, O^T = V^T P^T dimensions as rows and the same columns: a lane
// has the same heads in both.  Between them the weights' 8 x 8 blocks are transposed by movmatrix.  Scales of K multiply the accumulators
// of a group, scales of V the weights of a group.  Where at most 4 query heads share a KV head, the columns are 4 heads x 2
// halves of the groups (HALVES): lanes of columns 0..3 handle the scales of the first half of the groups, the others those of the second.
//
// A warp takes chunks of 32 tokens by itself, through a ring of stages of its own; one more warp issues the copies (bulk copies: a
// head's tokens in a page are one contiguous piece), a lane for each of the others.
//
// The chunks of all sequences of all heads, end to end, are cut into equal ranges, one per warp of the GPU, so that neither lengths nor the
// number of sequences leave warps idle.  A sequence of a head that is whole within a range is stored at once; pieces are added up, in the order
// of the ranges, at the end of the launch: through shared memory within a block, through scratch and a ticket between blocks.
#include "launch.cuh"
#include "ptx.cuh"
#include "mma.cuh"
#include "quant_kv.cuh"
#include "scalar.cuh"
#include "tmap.cuh"

namespace blitz {

constexpr int kQdWarps = 15, kQdThreads = (kQdWarps + 1) * 32;
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
  unsigned* tickets;   // [batch][heads] pieces finished, zero between launches
  float* part;         // [2 blocks][rep][D] sums, then [2 blocks][rep] of (maximum, sum of weights)
  int batch, kv_heads, heads, div, rep;  // heads: groups of at most 8 query heads, div of which share a KV head; rep: query heads of one
  int page_size, page_shift, max_pages, stages, static_table;
  float scale_log2, cap_scale, cap_log2;
  int window, keep_first;
  const void* sink;
  int* status;
};

// Shared memory: rings, a slot per warp for the first piece's sums, tables of the sequences, barriers.
__host__ __device__ constexpr int qd_slot_floats(int D, int rep) { return rep * (D + 4) + 16; }  // rows in different banks, then maxima and sums
__host__ __device__ constexpr int qd_table_bytes() { return (3 * kQdMaxBatch + 4 + 16) * 4; }
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
// How `all` chunks are cut into `n` ranges.
struct QdCut {
  unsigned base, rem;
  __device__ __forceinline__ QdCut(unsigned all, unsigned n) : base(all / n), rem(all % n) {}
  __device__ __forceinline__ unsigned begin(unsigned v) const { return v * base + min(v, rem); }
  __device__ __forceinline__ unsigned range(unsigned x) const { return x < rem * (base + 1) ? x / (base + 1) : rem + (x - rem * (base + 1)) / base; }
};
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

// d = a b + (c0, c1, c0, c1)
__device__ __forceinline__ void qd_mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, float c0, float c1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
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
__device__ __forceinline__ void qd_mma_bf16_add(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t qd_transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float qd_low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float qd_high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

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
  __device__ __forceinline__ void values(const uint8_t* token, int x, bool on) {
    uint32_t a = 0, b = 0, c = 0, d = 0;
    if (on) {  // (what is not visible may hold no numbers)
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
};

template <typename T, int D, int GROUP, bool HALVES>
__global__ void __launch_bounds__(kQdThreads, 1) attn_decode_quant_kernel(const __grid_constant__ DecodeQuantParams p) {
  constexpr QuantKv F = quant_kv(D, GROUP);
  constexpr int G = D / GROUP, W = D / 32, WG = GROUP / 32, MT = D / 16, N = QdScales<G, HALVES>::N;
  constexpr bool kTwo = std::is_same<T, __half>::value;  // weights as two bf16 numbers
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ring_bytes = p.stages * 2 * F.block, slot = qd_slot_floats(D, p.rep);
  float* const slots = reinterpret_cast<float*>(smem + kQdWarps * ring_bytes);
  QdTables tab;
  tab.before = reinterpret_cast<int*>(slots + kQdWarps * slot);
  tab.len = tab.before + kQdMaxBatch + 4;
  tab.page = tab.len + kQdMaxBatch;
  int* const across = tab.page + kQdMaxBatch;  // [2]: sequence and head that goes on before, after this block (-1: none); [2] flag of the last piece
  volatile int* const abort_flag = across + 8;
  uint64_t* const full = reinterpret_cast<uint64_t*>(across + 16);  // [warp][stage]
  uint64_t* const empty = full + kQdWarps * kQdMaxStages;

  if (threadIdx.x < kQdWarps * kQdMaxStages) {
    ptx::mbar_init(&full[threadIdx.x], 1);
    ptx::mbar_init(&empty[threadIdx.x], 1);
  }
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    across[0] = across[1] = -1;
  }
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
    int sum = 0;
    for (int b = b0; b < b1; ++b) sum += tab.before[b + 1];
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
  ptx::griddep_wait();

  T* const out = reinterpret_cast<T*>(p.out);
  const QdCut cut(static_cast<unsigned>(tab.before[p.batch]) * p.heads, kQdWarps * gridDim.x);
  const unsigned first_warp = blockIdx.x * kQdWarps;
  // (sequences without a visible key are in nobody's range: their output is zero)
  for (int b = blockIdx.x; b < p.batch; b += gridDim.x)
    if (tab.before[b] == tab.before[b + 1])
      for (int e = threadIdx.x; e < p.heads * p.rep * D; e += kQdThreads) stf(out + b * p.out_stride + e, 0.f);

  QdPiece first_piece{}, last_piece{};  // of this warp's range
  if (warp == kQdWarps) {
    // ---------------------------------------------------------------- copies: a lane for each warp
    const unsigned v = first_warp + min(lane, kQdWarps - 1);
    QdWalk walk = qd_walk(tab, p.batch, cut.begin(v), lane < kQdWarps ? cut.begin(v + 1) : 0u);
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
        __nanosleep(100);
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
    // (after a time-out: no copy may land in shared memory that another block has by then)
    if (lane < kQdWarps && *abort_flag) {
      since = ptx::globaltimer_ns();
      for (int s = 0; s < p.stages; ++s) {
        if (stage == 0) phase ^= 1u;
        stage = stage == 0 ? p.stages - 1 : stage - 1;
        while (!ptx::mbar_try_wait(&full[lane * kQdMaxStages + stage], phase ^ 1u) && ptx::globaltimer_ns() - since < 10000000ull) {
        }
      }
    }
  } else {
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
    const unsigned x0 = cut.begin(first_warp + warp), x1 = cut.begin(first_warp + warp + 1);
    QdWalk walk = qd_walk(tab, p.batch, x0, x1);
    QdPiece it{};
    for (bool first = true; qd_next(tab, p.batch, walk, it); first = false) {
      if (first) first_piece = it;
      last_piece = it;
      const QdSeen see = qd_seen(p, tab.len[it.b]);
      // queries: word w of a lane's key codes holds dimensions 32 w + 8 t4 .. + 7, pairs (i, i + 4) of which are a register's halves
      uint32_t qb[W][4], zb0, zb1 = 0;
      float qc[N][2], scale[2];
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
        float sum[G], zero[N];
#pragma unroll
        for (int i = 0; i < G; ++i) sum[i] = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) zero[i] = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const bool mine = !HALVES || (w / WG) / N == xq;
          float r[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            qb[w][i] = mine ? pk2<__half>(v[w][i] * down, v[w][i + 4] * down) : 0u;
            const float2 f = cvt2<__half>(qb[w][i]);  // (as they enter the products)
            r[i] = f.x;
            r[i + 4] = f.y;
          }
          // the zero of a register's codes: 1024 in the first and third pair, 64 in the others
          sum[w / WG] += ((r[0] + r[4]) + (r[1] + r[5])) + ((r[2] + r[6]) + (r[3] + r[7]));
          zero[(w / WG) % N] -= 1024.f * ((r[0] + r[4]) + (r[2] + r[6])) + 64.f * ((r[1] + r[5]) + (r[3] + r[7]));
        }
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) {
#pragma unroll
          for (int i = 0; i < G; ++i) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], d);
#pragma unroll
          for (int i = 0; i < N; ++i) zero[i] += __shfl_xor_sync(0xffffffffu, zero[i], d);
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
          scale[k] = __shfl_sync(0xffffffffu, up, (2 * t4 + k) * 4);
#pragma unroll
          for (int i = 0; i < N; ++i) qc[i][k] = __shfl_sync(0xffffffffu, zero[i], (2 * t4 + k) * 4);
        }
      }

      float o[MT][4], oc[N][4], zs[N][2], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < MT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) oc[i][0] = oc[i][1] = oc[i][2] = oc[i][3] = zs[i][0] = zs[i][1] = 0.f;

      for (int c = it.beg; c < it.end; ++c) {
        if (ok && !__all_sync(0xffffffffu, ptx::bounded_mbar_wait(&my_full[stage], phase, abort_flag))) {
          if (p.status && lane == 0) atomicCAS(p.status, 0, kStatusTimeoutEpilogue);
          ok = false;
        }
        if (!ok) continue;
        const uint8_t* st = ring + stage * 2 * F.block;
        const int tok0 = see.token(c), blocks = min(kQdChunk, see.len - tok0 + 15) >> 4;
        const bool edge = tok0 + kQdChunk > see.len || (tok0 < see.lo && tok0 + kQdChunk > see.first);  // some key is not visible
        float s[2][4];  // (tau, first head), (tau, second), (tau + 2, first), (tau + 2, second)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          s[u][0] = s[u][1] = s[u][2] = s[u][3] = 0.f;
          if (u < blocks) {
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
              const uint32_t a0 = (a & 0x000f000fu) | 0x64006400u, a1 = (b & 0x000f000fu) | 0x64006400u;
              const uint32_t a2 = (a & 0x00f000f0u) | 0x54005400u, a3 = (b & 0x00f000f0u) | 0x54005400u;
              const uint32_t c0 = (ah & 0x000f000fu) | 0x64006400u, c1 = (bh & 0x000f000fu) | 0x64006400u;
              const uint32_t c2 = (ah & 0x00f000f0u) | 0x54005400u, c3 = (bh & 0x00f000f0u) | 0x54005400u;
              if (w % WG == 0 && w / WG < N) qd_mma_f16(acc[i], a0, a1, a2, a3, qb[w][0], qb[w][1], qc[i][0], qc[i][1]);
              else qd_mma_f16_add(acc[i], a0, a1, a2, a3, qb[w][0], qb[w][1]);
              qd_mma_f16_add(acc[i], c0, c1, c2, c3, qb[w][2], qb[w][3]);
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
        }
        // scores in log2 units, and which of them count: bit 2 u + (0: token tau, 1: tau + 2)
        uint32_t seen = 15u;
        if (edge) {
          seen = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = tok0 + (i >> 1) * 16 + tau + 2 * (i & 1);
            if (j < see.len && (j >= see.lo || j < see.first)) seen |= 1u << i;
          }
        }
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float& v = s[i >> 2][i & 3];
          v = p.cap_log2 > 0.f ? p.cap_log2 * ptx::tanh_ex2(v * scale[i & 1] * p.cap_scale) : v * scale[i & 1] * p.scale_log2;
          if (edge && !((seen >> (i >> 1)) & 1u)) v = -INFINITY;
          top[i & 1] = fmaxf(top[i & 1], v);
        }
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], d));
          top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], d));
        }
        if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
          float a[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            a[k] = top[k] > m[k] ? ptx::ex2_approx(m[k] - top[k]) : 1.f;
            m[k] = fmaxf(m[k], top[k]);
            l[k] *= a[k];
          }
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            o[i][0] *= a[0]; o[i][1] *= a[1]; o[i][2] *= a[0]; o[i][3] *= a[1];
          }
#pragma unroll
          for (int i = 0; i < N; ++i) {
            oc[i][0] *= a[0]; oc[i][1] *= a[1];
            zs[i][0] *= a[0]; zs[i][1] *= a[1];
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float& v = s[i >> 2][i & 3];
          v = edge && !((seen >> (i >> 1)) & 1u) ? 0.f : ptx::ex2_approx(v - m[i & 1]);
          l[i & 1] += v;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (u < blocks) {
            const uint8_t* vb = st + u * F.block + F.part;
            QdScales<G, HALVES> fa, fb;
            fa.values(vb + F.codes + tau * 4 * G, x, !edge || ((seen >> (2 * u)) & 1u));
            fb.values(vb + F.codes + (tau + 2) * 4 * G, x, !edge || ((seen >> (2 * u + 1)) & 1u));
            uint32_t vw[MT];
#pragma unroll
            for (int h = 0; h < D / 64; ++h) {
              const uint4 v = *reinterpret_cast<const uint4*>(vb + h * 512 + g * 64 + t4 * 16);
              vw[4 * h] = v.x; vw[4 * h + 1] = v.y; vw[4 * h + 2] = v.z; vw[4 * h + 3] = v.w;
            }
            uint32_t b0[N], b1[N], c0[N], c1[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const float p0 = s[u][0] * fa.s[i], p1 = s[u][1] * fa.s[i], p2 = s[u][2] * fb.s[i], p3 = s[u][3] * fb.s[i];
              zs[i][0] = fmaf(s[u][0], fa.mid[i], fmaf(s[u][2], fb.mid[i], zs[i][0]));
              zs[i][1] = fmaf(s[u][1], fa.mid[i], fmaf(s[u][3], fb.mid[i], zs[i][1]));
              const uint32_t r0 = pk2<__nv_bfloat16>(p0, p1), r1 = pk2<__nv_bfloat16>(p2, p3);
              b0[i] = qd_transposed(r0);
              b1[i] = qd_transposed(r1);
              if (kTwo) {
                c0[i] = qd_transposed(pk2<__nv_bfloat16>(p0 - qd_low(r0), p1 - qd_high(r0)));
                c1[i] = qd_transposed(pk2<__nv_bfloat16>(p2 - qd_low(r1), p3 - qd_high(r1)));
              }
              constexpr uint32_t kOff = 0xc308c308u;  // -136
              qd_mma_bf16_add(oc[i], kOff, kOff, kOff, kOff, b0[i], b1[i]);
              if (kTwo) qd_mma_bf16_add(oc[i], kOff, kOff, kOff, kOff, c0[i], c1[i]);
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              const int j = (i * 16 / GROUP) % N;
              const uint32_t v = vw[i];
              const uint32_t a0 = (v & 0x000f000fu) | 0x43004300u, a1 = ((v >> 4) & 0x000f000fu) | 0x43004300u;
              const uint32_t a2 = ((v >> 8) & 0x000f000fu) | 0x43004300u, a3 = ((v >> 12) & 0x000f000fu) | 0x43004300u;
              qd_mma_bf16_add(o[i], a0, a1, a2, a3, b0[j], b1[j]);
              if (kTwo) qd_mma_bf16_add(o[i], a0, a1, a2, a3, c0[j], c1[j]);
            }
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
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          l[k] += __shfl_xor_sync(0xffffffffu, l[k], d);
#pragma unroll
          for (int i = 0; i < N; ++i) zs[i][k] += __shfl_xor_sync(0xffffffffu, zs[i][k], d);
        }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int j = (i * 16 / GROUP) % N;
        o[i][0] += oc[j][0] + zs[j][0]; o[i][1] += oc[j][1] + zs[j][1];
        o[i][2] += oc[j][0] + zs[j][0]; o[i][3] += oc[j][1] + zs[j][1];
      }
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
          r[k] = sum != 0.f ? f / sum : 0.f;
        }
        // rounded, and 8 x 8 blocks transposed, so that a lane has two neighbouring dimensions of head g
        const int hq = HALVES ? g & 3 : g, xq = HALVES ? g >> 2 : 0;
        T* to = out + it.b * p.out_stride + static_cast<int64_t>(it.head * p.rep + hq) * D + 2 * t4;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const uint32_t a = qd_transposed(pk2<T>(o[i][0] * r[0], o[i][1] * r[1])), b = qd_transposed(pk2<T>(o[i][2] * r[0], o[i][3] * r[1]));
          if (hq < p.rep && (!HALVES || (i * 16 / GROUP) / N == xq)) {
            *reinterpret_cast<uint32_t*>(to + 16 * i) = a;
            *reinterpret_cast<uint32_t*>(to + 16 * i + 8) = b;
          }
        }
      } else {
        // a piece: the range's first one has a slot, the last one the ring, which has nothing to take any more
        float* to = first ? slots + warp * slot : reinterpret_cast<float*>(smem + warp * ring_bytes);
        if (!first) __syncwarp();
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
      }
    }
  }
  __syncthreads();

  // -------------------------------------------------------------------- pieces within the block
  const unsigned X0 = cut.begin(first_warp), X1 = cut.begin(first_warp + kQdWarps);
  float* const part_ml = p.part + static_cast<int64_t>(2) * gridDim.x * p.rep * D;
  // the sum of a sequence's pieces is written as its output or, where other blocks have some, to scratch
  auto store = [&](int b, int hd, int d, const float (&acc)[4], float M, float L) {
    float f = 1.f, sum = L;
    if (p.sink != nullptr) {
      const float snk = ldf<T>(reinterpret_cast<const T*>(p.sink) + hd) * 1.4426950408889634f, top = fmaxf(snk, M);
      f = exp2f(M - top);
      sum = fmaf(f, L, exp2f(snk - top));
    }
    const float r = sum != 0.f ? f / sum : 0.f;
    stf4<T>(out + b * p.out_stride + static_cast<int64_t>(hd) * D + d, make_float4(acc[0] * r, acc[1] * r, acc[2] * r, acc[3] * r));
  };
  if (warp < kQdWarps) {
    const unsigned x0 = cut.begin(first_warp + warp), x1 = cut.begin(first_warp + warp + 1);
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
      const QdPiece& it = k ? last_piece : first_piece;
      if (x0 == x1 || (k && first_piece.start == last_piece.start)) continue;  // (one piece only)
      const bool whole = it.start >= x0 && it.stop <= x1;
      if (whole || (it.start < x0 && warp != 0)) continue;   // stored already, or an earlier warp's to add up
      const bool inside = it.start >= X0 && it.stop <= X1;
      const int place = blockIdx.x * 2 + (it.start < X0 ? 0 : 1);
      auto source = [&](int v) -> const float* {  // where warp v has its piece
        return max(it.start, cut.begin(first_warp + v)) == cut.begin(first_warp + v) ? slots + v * slot : reinterpret_cast<const float*>(smem + v * ring_bytes);
      };
      for (int e = lane; e < p.rep * (D / 4); e += 32) {
        const int hh = e / (D / 4), d = (e % (D / 4)) * 4;
        float M = -INFINITY, L = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
        for (int v = warp; v < kQdWarps && cut.begin(first_warp + v) < it.stop; ++v) M = fmaxf(M, source(v)[p.rep * (D + 4) + 2 * hh]);
        for (int v = warp; v < kQdWarps && cut.begin(first_warp + v) < it.stop; ++v) {
          const float* from = source(v);
          const float mv = from[p.rep * (D + 4) + 2 * hh], f = mv == M ? 1.f : exp2f(mv - M);
          L = fmaf(f, from[p.rep * (D + 4) + 2 * hh + 1], L);
          const float4 o = *reinterpret_cast<const float4*>(from + hh * (D + 4) + d);
          acc[0] = fmaf(f, o.x, acc[0]);
          acc[1] = fmaf(f, o.y, acc[1]);
          acc[2] = fmaf(f, o.z, acc[2]);
          acc[3] = fmaf(f, o.w, acc[3]);
        }
        if (inside) {
          store(it.b, it.head * p.rep + hh, d, acc, M, L);
        } else {
          __stcg(reinterpret_cast<float4*>(p.part + (static_cast<int64_t>(place) * p.rep + hh) * D + d), make_float4(acc[0], acc[1], acc[2], acc[3]));
          if (d == 0) __stcg(reinterpret_cast<float2*>(part_ml) + static_cast<int64_t>(place) * p.rep + hh, make_float2(M, L));
        }
      }
      if (!inside) {
        __threadfence();
        if (lane == 0) {
          across[it.start < X0 ? 0 : 1] = it.b * p.heads + it.head;
        }
      }
    }
  }
  __syncthreads();

  // -------------------------------------------------------------------- pieces of several blocks: whoever is last adds them up
#pragma unroll 1
  for (int k = 0; k < 2; ++k) {
    const int item = across[k];
    if (item < 0) continue;
    const int b = item / p.heads, head = item % p.heads;
    const unsigned start = static_cast<unsigned>(head) * tab.before[p.batch] + tab.before[b], stop = start + tab.before[b + 1] - tab.before[b];
    const unsigned c0 = cut.range(start) / kQdWarps, c1 = cut.range(stop - 1) / kQdWarps;
    if (threadIdx.x == 0) {
      __threadfence();
      const bool is_last = atomicAdd(p.tickets + item, 1u) == c1 - c0;
      if (is_last) p.tickets[item] = 0u;
      __threadfence();
      across[2 + k] = is_last;
    }
    __syncthreads();
    if (!across[2 + k]) continue;
    for (int e = threadIdx.x; e < p.rep * (D / 4); e += kQdThreads) {
      const int hh = e / (D / 4), d = (e % (D / 4)) * 4;
      auto place = [&](unsigned c) { return static_cast<int64_t>(c * 2 + (start < cut.begin(c * kQdWarps) ? 0 : 1)) * p.rep + hh; };
      float M = -INFINITY, L = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (unsigned c = c0; c <= c1; ++c) M = fmaxf(M, __ldcg(reinterpret_cast<const float2*>(part_ml) + place(c)).x);
#pragma unroll 4
      for (unsigned c = c0; c <= c1; ++c) {
        const int64_t at = place(c);
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(part_ml) + at);
        const float f = ml.x == M ? 1.f : exp2f(ml.x - M);
        const float4 o = __ldcg(reinterpret_cast<const float4*>(p.part + at * D + d));
        L = fmaf(f, ml.y, L);
        acc[0] = fmaf(f, o.x, acc[0]);
        acc[1] = fmaf(f, o.y, acc[1]);
        acc[2] = fmaf(f, o.z, acc[2]);
        acc[3] = fmaf(f, o.w, acc[3]);
      }
      store(b, head * p.rep + hh, d, acc, M, L);
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

}  // namespace blitz

extern "C" {
using namespace blitz;

// Scratch of a call: tickets, which have to be zero before the first call and are again after each, then partial sums.
int64_t blitz_attn_decode_quant_workspace_bytes(int batch, int q_heads, int dim) {
  return ((int64_t)batch * q_heads * 4 + 255) / 256 * 256 + (int64_t)2 * device_sm_count() * 8 * (dim + 2) * 4;
}

// q: [batch] rows with the query heads in their first q_heads * dim columns (pitch a multiple of 8, 16-byte aligned; so out).  A sequence
// without keys has an output of zeros.  static_table != 0 promises that the tables are not written by kernels still running in this
// stream.  More than 1024 sequences go in several launches.
int blitz_attn_decode_quant(const void* q, int64_t q_stride, const void* pool, const int32_t* indices, const int32_t* indptr,
                            const int32_t* last_page_len, void* out, int64_t out_stride, void* workspace, int64_t workspace_bytes, int batch,
                            int q_heads, int kv_heads, int dim, int group, int page_size, int max_pages, float sm_scale, int window,
                            int keep_first, float softcap, const void* sink, int static_table, int* status, int dtype, cudaStream_t stream) {
  if (batch <= 0) return 0;
  if (!quant_kv_supported(dim, group, page_size) || kv_heads < 1 || q_heads % kv_heads || window < 0 || keep_first < 0 || softcap < 0.f) return -1;
  if (((q_stride | out_stride) & 7) || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(pool) | reinterpret_cast<uintptr_t>(workspace)) & 15)) return -1;
  if (workspace == nullptr || workspace_bytes < blitz_attn_decode_quant_workspace_bytes(batch, q_heads, dim)) return -1;
  DecodeQuantParams p;
  p.div = qd_groups(q_heads / kv_heads); p.rep = q_heads / kv_heads / p.div; p.heads = kv_heads * p.div; p.kv_heads = kv_heads;
  p.q_stride = q_stride; p.pool = (const uint8_t*)pool; p.indices = indices; p.out_stride = out_stride;
  p.part = (float*)((char*)workspace + ((int64_t)batch * q_heads * 4 + 255) / 256 * 256);
  p.page_size = page_size; p.max_pages = max_pages; p.page_shift = 0; p.stages = 2;
  while ((1 << p.page_shift) < page_size) ++p.page_shift;
  p.scale_log2 = sm_scale * 1.4426950408889634f; p.cap_scale = softcap > 0.f ? sm_scale / softcap : 0.f; p.cap_log2 = softcap * 1.4426950408889634f;
  p.window = window; p.keep_first = keep_first; p.sink = sink; p.static_table = static_table; p.status = status;
  for (int b = 0; b < batch; b += kQdMaxBatch) {
    p.batch = batch - b < kQdMaxBatch ? batch - b : kQdMaxBatch;
    p.q = (const char*)q + (int64_t)b * q_stride * 2;
    p.out = (char*)out + (int64_t)b * out_stride * 2;
    p.indptr = indptr + b; p.last_page_len = last_page_len + b;
    p.tickets = (unsigned*)workspace + (int64_t)b * p.heads;
    const int rc = quant_kv_dispatch(dtype, dim, group, DecodeQuantLaunch{p, device_sm_count(), stream});
    if (rc) return rc;
  }
  return 0;
}

}  // extern "C"
