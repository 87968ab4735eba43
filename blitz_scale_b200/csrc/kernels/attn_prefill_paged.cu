// Causal prefill attention over the paged KV cache on tcgen05 for sm_100a: GQA, heads of up to 128, queries of
// the current chunk against everything the cache holds for the sequence (earlier chunks and the chunk itself).
//
// Q comes from the fused QKV activation of the chunk (2-D TMA boxes); K and V come from the paged pool, where
// rope_kv_store has already put the chunk's own keys and values, as 3-D TMA boxes of one page (or 64 tokens of
// one) each, looked up through the page table.  A prompt that does not fit one batch is therefore prefetched in
// chunks with no other kernel: the first chunk has an empty prefix, later ones a prefix of whole earlier chunks.
//
// A work item is 256 query rows of one sequence and one q head, as two tiles of 128 rows that walk the KV blocks
// of 128 tokens up to the diagonal once for both:
//
//   S_t = Q_t K^T      tcgen05.mma, A = Q_t (smem), B = K block (smem), S_t in TMEM                      t = 0, 1
//   P_t = softmax      warpgroup t (4 warps, thread = row): one tcgen05.ld pass over S_t, running max and sum in
//                      fp32, P_t written back over S_t's first 64 columns (two 16-bit values per column)
//   O_t += P_t V       tcgen05.mma with A = P_t from tensor memory, accumulating in TMEM over all blocks
//
// A ninth warp issues the MMAs (one thread), a tenth the TMA loads.  While warpgroup 0 turns S_0 into P_0 the
// tensor core works on S_1 and on O_1, and the other way round: the two tiles ping-pong, and every K and V block
// feeds two tiles from one load.  O stays in TMEM for the whole walk: the maximum a row's probabilities refer to
// only moves when the true maximum has grown by more than 2^8 (the probabilities then stay below 256, harmless in
// 16 bits and fp32), and only then the warp rescales its O rows in place (tcgen05.ld, multiply, tcgen05.st); with
// ordinary inputs that happens in the first block or two of a row and never again.
//
// The grid is persistent: one CTA per SM takes work items in a fixed order (heaviest first, dealt back and forth
// over the CTAs so that every CTA gets a similar sum).  The three roles walk the same list on their own, all
// barrier phases come from running counts, and nothing is drained between items: the next item's Q, K and V are
// loaded and its first S products issued while the warpgroups still write the previous item's output, so the
// latency of starting an item (its page ids, its first loads, the first MMA) is paid once per CTA, not per item.
//
// Models that ask for it (template parameter EXT) get a sliding window with kept first tokens, soft-capped scores and a
// per-head sink.  The two tiles of an item then walk the key blocks of the kept tokens and those from the first row's
// window edge on; blocks in between are never loaded.  A block that is wholly visible to a tile needs no mask.  The cap,
// cap * tanh(s / cap), is applied to the scores as they turn into probabilities.  Where all of a warp's scores of the
// block stay below half the cap (one vote per block, the usual case), that is an odd polynomial on the FMA pipe, two
// scores per instruction, and the largest magnitude serves as the row's reference instead of its maximum, so that one
// pass over the scores decides both; else the special-function unit does it (tanh being monotonic, the row maximum is
// capped alone).  The sink is one more term of the row sum at the end.
//
// Keys and values may differ in size, and either may be smaller than the tile it is computed in (64 or 128 columns, a
// multiple of 8): TMA fills the columns behind a head's end with zeros.  A gate (one number per head and row, through a
// sigmoid) multiplies a head's output rows as they leave tensor memory.
//
// A bias by distance per head (template parameter BIAS): bias[h][min(i - j, bias_len - 1)] is added to the scaled scores.  A
// block of 128 keys against a tile of 128 rows has 255 distances; the tile's warpgroup fetches their biases (two a thread,
// requested before it waits for the scores) into shared memory, where the lanes of a warp, rows that follow one another, read
// neighbouring words.  Blocks whose every distance is beyond the table share its last entry, which moves the reference.
//
// The window may be a chunk counted from position 0 (`chunked`): a row sees the keys of its own chunk.  Weights may be sigmoids of
// the scores (template parameter SIG; EXT with it): no maximum, no row sum, no rescaling.  sigmoid(x) = 1 / (1 + e^-x); four
// neighbours share a reciprocal, 1 / a = b (c d) / (a b c d), unless a product of some four leaves the range of fp32 (one vote per
// half a block).
//
// Operands in fp16 for a bf16 model (IO: the type of queries, sink and output): keys and values were divided by powers of two (of a sequence and KV
// head) so that fp16 holds them, and each thread turns its row of queries into fp16 in shared memory, divided by a power of two near the row's
// largest entry, as an item begins.  The row's scale and the output's factor make up for both.  A 4-bit cache read back for a pass
// comes so (quant_kv.cu).  8192 rows of nine prompts, 32 heads of 128: 192 us where a bf16 cache takes 174 (what an item waits for at its start, and
// registers); with queries converted by a pass before it 184 us behind 20 us of that.
// Sequences and heads that fp16 does not hold come in bf16: a block takes its items with operands in fp16 first, then, where the pass has any, those in
// bf16, with code, barriers and descriptors of their own (the type chosen item by item took 8 us more; a second launch 5 us in every pass).
//
// Replaces FlashInfer's BatchPrefillWithRaggedKVCacheWrapper / paged wrapper calls and their host Plan()
// (src/kernel/attention_prefill.cu:11-45, src/kernel/flashinfer_types.cu:24-49).
#include "launch.cuh"
#include "ptx.cuh"
#include "tmap.cuh"
#include "common.cuh"
#include "quant_kv.cuh"
#include <cmath>

namespace blitz {

constexpr int kPpThreads = 320;  // warpgroup 0, warpgroup 1, MMA warp, load warp
constexpr int kPpTile = 128;     // q rows per tile and kv tokens per block
constexpr float kPpRescaleAt = 8.f;  // log2 units
constexpr int kPpWorkInts = 8;   // per (sequence, pair of tiles): first row, rows, first page entry, pages, cached tokens, pair

struct PagedPrefillParams {
  void* out;  // [tokens, q_heads * vdim]
  const void* gate;  // [tokens][gate_stride], a column per query head, or null
  int64_t out_stride, gate_stride;
  const int32_t* page_indices;  // page ids of every sequence, back to back
  const int32_t* work;          // [entries][kPpWorkInts], heaviest first
  int entries, q_heads, kv_heads, vdim, page_size, page_rows, box_tokens, oob_row;  // page n's token `off`: pool row n * page_rows + off
  float scale_log2;
  int chunked;                // EXT: the window is a chunk
  int window, keep_first;     // EXT: a row sees the last `window` positions (0: all) and the first `keep_first`
  float cap_scale, cap_log2;  // EXT: soft cap (cap_log2 > 0): score in log2 units = cap_log2 * tanh(q.k * cap_scale)
  float small_max;            // EXT: largest |q.k| the polynomial takes (0: never)
  float poly[4];              // EXT: score in log2 units = x (poly[0] + poly[1] x^2 + poly[2] x^4 + poly[3] x^6), x = q.k
  const void* sink;           // EXT: [q_heads] in the activation type, or null
  const void* bias;           // BIAS: [q_heads][bias_len] in the activation type (SIG: [q_heads], or null)
  int bias_len;
  const float2* forms;        // IO: [entries][kv_heads] powers of two taken out of keys and values, zeros where those are in bf16
  const int* some_bf16;       // IO: whether any are
  float least_up;             // IO: what makes the factor of scores 2^-126
  int* status;
  long long* trace;  // profiling aid (null in production): clock stamps of CTA 0's first item, see the set_trace call
};

constexpr int kPpTraceIters = 32, kPpTraceSlots = 8;
// role 0 / 1: first lane of warpgroup 0 / 1; role 2: the MMA thread
__device__ __forceinline__ void pp_trace(const PagedPrefillParams& p, bool on, int role, int j, int slot) {
  if (on && p.trace != nullptr && j < kPpTraceIters) p.trace[(role * kPpTraceIters + j) * kPpTraceSlots + slot] = clock64();
}

template <int HD, int VD>
struct PpCfg {
  static constexpr int kSlabBytes = kPpTile * 128;     // 64 columns of a tile: 128 rows x 128 bytes
  static constexpr int kSlabs = HD / 64, kValueSlabs = VD / 64;
  static constexpr int kTileBytes = kSlabs * kSlabBytes, kValueBytes = kValueSlabs * kSlabBytes;  // a Q or K tile, a V tile
  static constexpr int kBarBytes = 256;
  static constexpr int kBiasFloats = 2 * 2 * 256;  // per tile: two blocks' distances
  static constexpr int kSmemBytes = 4 * kTileBytes + 2 * kValueBytes + 1024 + kBarBytes;  // Q x 2 tiles, K x 2 stages, V x 2 stages
};

struct PpItem {
  int seq_start, q_len, pg0, npages, kv_len, prefix, q0, nt, nblk, head, kv_head;
  int nblk_t[2];
  float k_up;             // IO: the power of two taken out of the keys
  int n_first, b_window;  // key blocks walked: [0, n_first), then from b_window on
  __device__ __forceinline__ int block(int j) const { return j < n_first ? j : b_window + j - n_first; }
};
// Work item `idx` of the flattened list (entry x q head; the heads of one entry are neighbours, so CTAs that run
// at the same time share its K and V in L2).
// MIXED: an item of the other type has no blocks.
template <bool EXT, bool MIXED, bool SCALED>
__device__ __forceinline__ PpItem pp_item(const PagedPrefillParams& p, int idx) {
  PpItem it;
  const int entry = idx / p.q_heads;
  it.head = idx - entry * p.q_heads;
  it.kv_head = it.head / (p.q_heads / p.kv_heads);
  const int4 a = __ldg(reinterpret_cast<const int4*>(p.work + entry * kPpWorkInts));
  const int4 b = __ldg(reinterpret_cast<const int4*>(p.work + entry * kPpWorkInts + 4));
  it.seq_start = a.x; it.q_len = a.y; it.pg0 = a.z; it.npages = a.w; it.kv_len = b.x;
  it.prefix = it.kv_len - it.q_len;  // tokens of earlier chunks
  it.q0 = b.y * 2 * kPpTile;
  it.nt = (it.q0 + kPpTile < it.q_len) ? 2 : 1;
#pragma unroll
  for (int t = 0; t < 2; ++t) {  // blocks tile t needs: keys up to its last row's position
    const int last = min(it.kv_len, it.prefix + min(it.q_len, it.q0 + kPpTile * (t + 1)));
    it.nblk_t[t] = t < it.nt ? (last + kPpTile - 1) / kPpTile : 0;
  }
  it.n_first = it.b_window = 0;
  if (EXT && p.window > 0) {
    const int p0 = it.prefix + it.q0, lo = p.chunked ? p0 - p0 % p.window : max(0, p0 - p.window + 1);  // first key in the window of the item's first row
    it.n_first = (min(p.keep_first, lo) + kPpTile - 1) / kPpTile;
    it.b_window = max(lo / kPpTile, it.n_first);
#pragma unroll
    for (int t = 0; t < 2; ++t)
      if (it.nblk_t[t] > 0) it.nblk_t[t] = it.n_first + max(0, it.nblk_t[t] - it.b_window);
  }
  if (MIXED) {
    it.k_up = __ldg(&p.forms[static_cast<int64_t>(entry) * p.kv_heads + it.kv_head].x);
    if ((it.k_up != 0.f) != SCALED) it.nblk_t[0] = it.nblk_t[1] = 0;
  }
  it.nblk = max(it.nblk_t[0], it.nblk_t[1]);
  return it;
}
// The r-th item of this CTA: rounds alternate direction over the CTAs.  -1: this CTA has none in round r.
__device__ __forceinline__ int pp_index(int r, int total) {
  const int G = gridDim.x;
  const int idx = r * G + ((r & 1) ? G - 1 - static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x));
  return idx < total ? idx : -1;
}

template <typename OP, int HD, int VD, bool POLY, bool EXT, bool BIAS, bool SIG, typename IO = OP>
__global__ void __launch_bounds__(kPpThreads, 1)
attn_prefill_paged_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                          const __grid_constant__ CUtensorMap tmap_v, const PagedPrefillParams p) {
  using C = PpCfg<HD, VD>;
  constexpr bool MIXED = !std::is_same<OP, IO>::value;
  constexpr int TB = C::kTileBytes, VB = C::kValueBytes, SB = C::kSlabBytes;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = ptx::smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023u) & ~1023u) - raw_addr);
  uint8_t* sQ = smem;            // [2 tiles]
  uint8_t* sK = sQ + 2 * TB;     // [2 stages]
  uint8_t* sV = sK + 2 * TB;     // [2 stages]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + 2 * VB);
  uint64_t* q_full = bars;        // [2] per tile and item
  uint64_t* q_empty = bars + 2;   // once per item: its last S products are done
  uint64_t* k_full = bars + 3;    // [2] per block
  uint64_t* k_empty = bars + 5;   // [2]
  uint64_t* v_full = bars + 7;    // [2]
  uint64_t* v_empty = bars + 9;   // [2]
  uint64_t* s_full = bars + 11;   // [2] per tile and block
  uint64_t* p_ready = bars + 13;  // [2]
  uint64_t* o_full = bars + 15;   // [2]
  uint64_t* o_free = bars + 17;   // [2] per tile and item: the warpgroup has read its output rows
  uint64_t* q_fp16 = bars + 19;   // [2] per tile and item, IO: the warpgroup has turned its queries into fp16
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 21);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* s_bias = reinterpret_cast<float*>(sV + 2 * VB + C::kBarBytes);  // BIAS only

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int total = p.entries * p.q_heads;

  if (threadIdx.x == 0) {
    for (int set = 0; set < (MIXED ? 2 : 1); ++set) {
      uint64_t* const more = bars + set * (C::kBarBytes / 8);  // MIXED: a second set behind the first
      ptx::mbar_init(&q_empty[more - bars], 1);
      for (int i = 0; i < 2; ++i) {
        ptx::mbar_init(&q_full[more - bars + i], 1);
        ptx::mbar_init(&q_fp16[more - bars + i], 128);
        ptx::mbar_init(&k_full[more - bars + i], 1);
        ptx::mbar_init(&k_empty[more - bars + i], 1);
        ptx::mbar_init(&v_full[more - bars + i], 1);
        ptx::mbar_init(&v_empty[more - bars + i], 1);
        ptx::mbar_init(&s_full[more - bars + i], 1);
        ptx::mbar_init(&p_ready[more - bars + i], 128);
        ptx::mbar_init(&o_full[more - bars + i], 1);
        ptx::mbar_init(&o_free[more - bars + i], 128);
      }
    }
    *abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::tma_prefetch_desc(&tmap_q);
    ptx::tma_prefetch_desc(&tmap_k);
    ptx::tma_prefetch_desc(&tmap_v);
  }
  if (warp == 8) {
    ptx::tmem_alloc(tmem_slot, 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  ptx::griddep_launch_dependents();
  ptx::griddep_wait();  // queries, keys, values and the work list come from earlier kernels
  const uint32_t tmem_S = tmem_base;        // S_t (and P_t over its first 64 columns) at + 128 t
  const uint32_t tmem_O = tmem_base + 256;  // O_t at + VD t

  if constexpr (!MIXED) {
    using T = OP;
    constexpr bool SCALED = false;
#include "attn_prefill_roles.cuh"
  } else {
    auto items_of = [&](auto operand, int set) {
      using T = decltype(operand);
      constexpr bool SCALED = std::is_same<T, __half>::value;
      const int more = set * (C::kBarBytes / 8);
      uint64_t *const all[] = {q_full, q_empty, k_full, k_empty, v_full, v_empty, s_full, p_ready, o_full, o_free, q_fp16};
      uint64_t* const q_full = all[0] + more;
      uint64_t* const q_empty = all[1] + more;
      uint64_t* const k_full = all[2] + more;
      uint64_t* const k_empty = all[3] + more;
      uint64_t* const v_full = all[4] + more;
      uint64_t* const v_empty = all[5] + more;
      uint64_t* const s_full = all[6] + more;
      uint64_t* const p_ready = all[7] + more;
      uint64_t* const o_full = all[8] + more;
      uint64_t* const o_free = all[9] + more;
      uint64_t* const q_fp16 = all[10] + more;
#include "attn_prefill_roles.cuh"
    };
    items_of(OP{}, 0);
    if (__ldg(p.some_bf16) != 0) {
      ptx::tc_fence_before_sync();
      __syncthreads();  // every product is done, and its output read
      ptx::tc_fence_after_sync();
      items_of(IO{}, 1);
    }
  }

  ptx::tc_fence_before_sync();
  __syncthreads();
  if (warp == 8) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem_base, 512);
  }
}

template <typename T, int HD, int VD, bool POLY, bool EXT, bool BIAS, bool SIG, typename IO = T>
static int launch_paged_prefill(const CUtensorMap (&tm)[3], const PagedPrefillParams& p, int grid, cudaStream_t stream) {
  using C = PpCfg<HD, VD>;
  constexpr int kSmem = C::kSmemBytes + (BIAS ? C::kBiasFloats * 4 : 0) + (std::is_same<T, IO>::value ? 0 : C::kBarBytes);
  static PerDeviceOnce once;
  cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(attn_prefill_paged_kernel<T, HD, VD, POLY, EXT, BIAS, SIG, IO>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
  });
  if (e != cudaSuccess) return (int)e;
  return (int)launch_pdl(attn_prefill_paged_kernel<T, HD, VD, POLY, EXT, BIAS, SIG, IO>, dim3(grid), dim3(kPpThreads), (size_t)kSmem, stream, tm[0], tm[1], tm[2], p);
}

static long long* g_pp_trace = nullptr;

}  // namespace blitz

extern "C" {
using namespace blitz;

// Profiling aid: while `buf` (3 roles x 32 iterations x 8 int64 clock stamps, device memory) is set, CTA 0 of every
// following launch records when its warpgroups and its MMA thread pass each phase of its first work item.
void blitz_attn_prefill_paged_set_trace(long long* buf) { blitz::g_pp_trace = buf; }

// q: [num_tokens, q_stride >= q_heads * dim] of the current chunk, rotated; k_pool, v_pool: the layer's pools
// [max_pages][page_rows][kv_heads][dim or vdim], a page's tokens in its first page_size rows (one tensor for keys and values:
// page_rows = 2 page_size, v_pool at the first value plane), which already hold the chunk's keys and values;
// out: [num_tokens, q_heads * vdim].  page_indices: device array of the sequences' page ids, back to back (the
// lists cover prefix + chunk).  work: device array (16-byte aligned) of `entries` records of 8 int32, one per
// (sequence, 256 rows of it), heaviest first: first row of the sequence in qkv, rows of the sequence in this chunk,
// index of its first page id, number of its pages, tokens cached for it (chunk included), which 256-row pair, 0, 0.
// page_size: a power of two >= 8.  dim and vdim: multiples of 8 up to 128.  flags bit 0: compute a quarter of the
// exponentials on the FMA pipe (not with a window, cap or sink).  window (0 = none) / keep_first, softcap (0 = none), sink
// and gate (null = none), chunked and sigmoid: see the top of the file.  bias: [q_heads][bias_len] in the activation type, or null
// (not with a window, cap or sink; with sigmoid weights only bias_len 1).
static int prefill_paged(const void* q, int64_t q_stride, const void* k_pool, const void* v_pool, void* out, int64_t out_stride,
                             const int32_t* page_indices, const int32_t* work, int entries, int num_tokens,
                             int q_heads, int kv_heads, int dim, int vdim, int page_size, int page_rows, int max_pages,
                             float sm_scale, int flags, int window, int keep_first, int chunked, int sigmoid, float softcap, const void* sink,
                             const void* bias, int bias_len, const void* gate, int64_t gate_stride, const float2* forms, const int* some_bf16, int* status,
                             int dtype, cudaStream_t stream) {
  if (num_tokens <= 0 || entries <= 0) return 0;
  if (dim < 8 || dim > 128 || (dim & 7) || vdim < 8 || vdim > 128 || (vdim & 7)) return -1;
  if (kv_heads < 1 || (q_heads % kv_heads) != 0 || (out_stride & 7) || (q_stride & 7)) return -1;
  if (window < 0 || keep_first < 0 || softcap < 0.f) return -1;
  if ((chunked && (window < 1 || keep_first)) || (sigmoid && (sink || softcap > 0.f || keep_first || (bias && bias_len != 1)))) return -1;
  if (page_size < 8 || (page_size & (page_size - 1)) != 0 || page_rows < page_size || work == nullptr) return -1;
  if ((reinterpret_cast<uintptr_t>(work) & 15) != 0 || (reinterpret_cast<uintptr_t>(out) & 15) != 0) return -1;
  const int bt = page_size < 64 ? page_size : 64;
  // rows of a pool: those of the last page end with its tokens
  const uint64_t rows = (uint64_t)(max_pages - 1) * page_rows + page_size;
  CUtensorMap tm[3];
  if (!get_tmap_3d(&tm[0], q, (uint64_t)dim, (uint64_t)q_heads, (uint64_t)num_tokens, (uint64_t)dim * 2, (uint64_t)q_stride * 2, 64, 1, kPpTile))
    return -2;
  for (int i = 1; i < 3; ++i) {
    const uint64_t d = i == 1 ? dim : vdim;
    if (!get_tmap_3d(&tm[i], i == 1 ? k_pool : v_pool, d, (uint64_t)kv_heads, rows, d * 2, d * 2 * kv_heads, 64, 1, (uint32_t)bt)) return -2;
  }
  PagedPrefillParams p;
  p.out = out; p.out_stride = out_stride; p.page_indices = page_indices; p.work = work; p.entries = entries;
  p.gate = gate; p.gate_stride = gate_stride; p.vdim = vdim; p.page_rows = page_rows;
  p.q_heads = q_heads; p.kv_heads = kv_heads; p.page_size = page_size; p.box_tokens = bt;
  p.oob_row = (int)rows;
  p.scale_log2 = sm_scale * 1.4426950408889634f; p.status = status; p.trace = g_pp_trace;
  p.chunked = chunked; p.forms = forms; p.some_bf16 = some_bf16; p.least_up = 0x1p-126f / p.scale_log2;
  p.window = window; p.keep_first = keep_first; p.sink = sink; p.bias = bias; p.bias_len = bias_len;
  p.cap_scale = softcap > 0.f ? sm_scale / softcap : 0.f; p.cap_log2 = softcap * 1.4426950408889634f;
  // tanh(z) = z (k0 + k1 z^2 + k2 z^4 + k3 z^6) for |z| <= 0.5 (Chebyshev interpolation of tanh(z) / z in z^2, absolute
  // error 2.5e-7), with z = q.k * cap_scale folded in.  Scores below 40 log2 units keep every probability that refers to
  // the largest magnitude above 2^-80.  A tiny scale / cap would underflow in the coefficients: no polynomial then.
  const double z = p.cap_scale, k[4] = {0.99999945, -0.33326284, 0.13189939, -0.04439274};
  double zn = z * p.cap_log2;
  for (int i = 0; i < 4; ++i, zn *= z * z) p.poly[i] = (float)(k[i] * zn);
  p.small_max = z > 1e-5 ? (float)fmin(0.5 / z, 40.0 / p.scale_log2) : 0.f;
  const long long total = (long long)entries * q_heads;
  const int sms = device_sm_count();
  const int grid = (int)(total < sms ? total : sms);
  const bool poly = (flags & 1) != 0, ext = window > 0 || softcap > 0.f || sink != nullptr;
  if (bias != nullptr && !sigmoid && (ext || bias_len < 1)) return -1;
  auto sized = [&](auto type, auto poly_, auto ext_, auto bias_, auto sig_) {
    using T = decltype(type);
    constexpr bool P = decltype(poly_)::value, X = decltype(ext_)::value, B = decltype(bias_)::value, G = decltype(sig_)::value;
    if (dim > 64)
      return vdim > 64 ? launch_paged_prefill<T, 128, 128, P, X, B, G>(tm, p, grid, stream)
                       : launch_paged_prefill<T, 128, 64, P, X, B, G>(tm, p, grid, stream);
    return vdim > 64 ? launch_paged_prefill<T, 64, 128, P, X, B, G>(tm, p, grid, stream)
                     : launch_paged_prefill<T, 64, 64, P, X, B, G>(tm, p, grid, stream);
  };
  auto launch = [&](auto type) {
    const std::false_type no{};
    const std::true_type yes{};
    if (sigmoid) return sized(type, no, yes, no, yes);
    if (bias != nullptr) return sized(type, no, no, yes, no);
    if (ext) return sized(type, no, yes, no, no);
    if (poly) return sized(type, yes, no, no, no);
    return sized(type, no, no, no, no);
  };
  if (forms != nullptr) {
    if (dim != vdim || (dim != 64 && dim != 128)) return -1;
    auto mixed = [&](auto ext_) {
      constexpr bool X = decltype(ext_)::value;
      return dim > 64 ? launch_paged_prefill<__half, 128, 128, false, X, false, false, __nv_bfloat16>(tm, p, grid, stream)
                      : launch_paged_prefill<__half, 64, 64, false, X, false, false, __nv_bfloat16>(tm, p, grid, stream);
    };
    return ext ? mixed(std::true_type{}) : mixed(std::false_type{});
  }
  return dtype == 1 ? launch(__nv_bfloat16{}) : launch(__half{});
}

int blitz_attn_prefill_paged(const void* q, int64_t q_stride, const void* k_pool, const void* v_pool, void* out, int64_t out_stride,
                             const int32_t* page_indices, const int32_t* work, int entries, int num_tokens,
                             int q_heads, int kv_heads, int dim, int vdim, int page_size, int page_rows, int max_pages,
                             float sm_scale, int flags, int window, int keep_first, int chunked, int sigmoid, float softcap, const void* sink,
                             const void* bias, int bias_len, const void* gate, int64_t gate_stride, int* status, int dtype, cudaStream_t stream) {
  return prefill_paged(q, q_stride, k_pool, v_pool, out, out_stride, page_indices, work, entries, num_tokens, q_heads, kv_heads, dim, vdim, page_size,
                       page_rows, max_pages, sm_scale, flags, window, keep_first, chunked, sigmoid, softcap, sink, bias, bias_len, gate, gate_stride,
                       nullptr, nullptr, status, dtype, stream);
}

// The same for a bf16 model (q, sink and out) whose keys and values blitz_quant_kv_portion has read back: forms is the fourth part of its scratch,
// some_bf16 what is behind the spans.  dim 64 or 128.
int blitz_attn_prefill_scaled(const void* q, int64_t q_stride, const void* k_pool, const void* v_pool, void* out, int64_t out_stride,
                              const int32_t* page_indices, const int32_t* work, int entries, int num_tokens, int q_heads, int kv_heads, int dim,
                              int page_size, int page_rows, int max_pages, float sm_scale, int window, int keep_first, float softcap, const void* sink,
                              const void* forms, const int* some_bf16, int* status, cudaStream_t stream) {
  if (forms == nullptr || some_bf16 == nullptr) return -1;
  return prefill_paged(q, q_stride, k_pool, v_pool, out, out_stride, page_indices, work, entries, num_tokens, q_heads, kv_heads, dim, dim, page_size,
                       page_rows, max_pages, sm_scale, 0, window, keep_first, 0, 0, softcap, sink, nullptr, 0, nullptr, 0, (const float2*)forms, some_bf16,
                       status, 0, stream);
}

}  // extern "C"
