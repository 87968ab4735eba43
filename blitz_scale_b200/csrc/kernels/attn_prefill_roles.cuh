// What the warps of the paged prefill kernel do: included in its body, once for every type of operands (T; SCALED: queries are turned into fp16), where
// tiles, barriers and the table of items have their names (attn_prefill_paged.cu).
  constexpr uint32_t kFmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  constexpr uint32_t kIdescS = ptx::make_idesc_f16(kFmt, 0u, 0u, 128, 128);
  constexpr uint32_t kIdescPV = ptx::make_idesc_f16(kFmt, 0u, 1u, 128, VD);
  if (warp == 9) {
    // ------------------------------------------------------------ load warp: Q, then K and V block by block
    // K or V block j -> one tile of 128 token rows: every lane fetches one box (a page, or 64 tokens of one)
    const int bt = p.box_tokens;
    const bool mine = lane < kPpTile / bt;
    auto box_row = [&](const PpItem& it, int j) {  // this lane's first row of block j in the pools
      const int tok = it.block(j) * kPpTile + lane * bt;
      const int slot = tok / p.page_size;
      if (!mine || slot >= it.npages) return p.oob_row;  // past the pool: the box arrives as zeros
      return p.page_indices[it.pg0 + slot] * p.page_rows + (tok & (p.page_size - 1));
    };
    auto load_kv = [&](uint8_t* dst, const CUtensorMap* map, int slabs, uint64_t* bar, int kv_head, int row) {
      if (lane == 0) ptx::mbar_expect_tx(bar, slabs * SB);
      __syncwarp();
      if (mine) {
#pragma unroll
        for (int s = 0; s < slabs; ++s) ptx::tma_load_3d(dst + s * SB + lane * bt * 128, map, bar, s * 64, kv_head, row);
      }
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      int ok = 1;
      if (lane == 0) ok = ptx::bounded_mbar_wait(bar, parity, abort_flag) ? 1 : 0;
      return __shfl_sync(0xffffffffu, ok, 0) != 0;
    };
    bool ok = true;
    uint32_t g = 0, n_items = 0;  // blocks and items loaded so far
    for (int r = 0; r * static_cast<int>(gridDim.x) < total && ok; ++r) {
      const int idx = pp_index(r, total);
      if (idx < 0) continue;
      const PpItem it = pp_item<EXT, MIXED, SCALED>(p, idx);
      if (MIXED && it.nblk == 0) continue;
      if (n_items > 0) ok = wait(q_empty, (n_items - 1) & 1);  // the previous item's S products have read Q
      if (!ok) break;
      if (lane == 0) {
        for (int t = 0; t < 2; ++t) {
          if (it.nblk_t[t] == 0) continue;
          ptx::mbar_expect_tx(&q_full[t], TB);
#pragma unroll
          for (int s = 0; s < C::kSlabs; ++s)
            ptx::tma_load_3d(sQ + t * TB + s * SB, &tmap_q, &q_full[t], s * 64, it.head, it.seq_start + it.q0 + t * kPpTile);
        }
      }
      if constexpr (SCALED) {  // the next item's queries into L2: what brings them to fp16 waits for them
        const int next = (r + 1) * static_cast<int>(gridDim.x) < total ? pp_index(r + 1, total) : -1;
        if (next >= 0 && lane < 2 * C::kSlabs) {
          const PpItem n = pp_item<EXT, MIXED, SCALED>(p, next);
          const int t = lane / C::kSlabs;
          if (n.nblk_t[t] > 0) ptx::tma_prefetch_3d(&tmap_q, lane % C::kSlabs * 64, n.head, n.seq_start + n.q0 + t * kPpTile);
        }
      }
      int row = box_row(it, 0);
      for (int j = 0; j < it.nblk && ok; ++j, ++g) {
        const int row_next = j + 1 < it.nblk ? box_row(it, j + 1) : p.oob_row;  // looked up a block ahead of its use
        // a block's K goes where the K of two blocks ago was, once the S products of that block are done; V likewise
        if (g >= 2) ok = wait(&k_empty[g & 1], ((g - 2) >> 1) & 1);
        if (!ok) break;
        load_kv(sK + (g & 1) * TB, &tmap_k, C::kSlabs, &k_full[g & 1], it.kv_head, row);
        if (g >= 2) ok = wait(&v_empty[g & 1], ((g - 2) >> 1) & 1);
        if (!ok) break;
        load_kv(sV + (g & 1) * VB, &tmap_v, C::kValueSlabs, &v_full[g & 1], it.kv_head, row);
        row = row_next;
      }
      ++n_items;
    }
    if (!ok && lane == 0 && p.status) atomicCAS(p.status, 0, kStatusTimeoutProducer);
  } else if (warp == 8) {
    // ------------------------------------------------------------ MMA warp: one thread issues
    if (ptx::elect_one()) {
      auto issue_S = [&](int t, int stage) {
        const uint32_t a = ptx::smem_u32(sQ + t * TB), bb = ptx::smem_u32(sK + stage * TB);
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint32_t off = (k >> 2) * SB + (k & 3) * 32;
          ptx::umma_f16_ss(tmem_S + t * 128, ptx::make_smem_desc(a + off, 16, 1024, ptx::kLayoutSw128),
                           ptx::make_smem_desc(bb + off, 16, 1024, ptx::kLayoutSw128), kIdescS, k != 0 ? 1u : 0u);
        }
        ptx::umma_commit(&s_full[t]);
      };
      auto issue_PV = [&](int t, int stage, bool accumulate) {
        const uint32_t bb = ptx::smem_u32(sV + stage * VB);
#pragma unroll
        for (int k = 0; k < kPpTile / 16; ++k) {
          // A = P in tensor memory: row = lane, 16 tokens = 8 columns.  B = V: N-major, slabs of 64 head-dim
          // columns; 16 tokens (K) advance 2 KB.
          ptx::umma_f16_ts(tmem_O + t * VD, tmem_S + t * 128 + k * 8,
                           ptx::make_smem_desc(bb + k * 2048, SB, 1024, ptx::kLayoutSw128), kIdescPV,
                           (accumulate || k != 0) ? 1u : 0u);
        }
        ptx::umma_commit(&o_full[t]);
      };
      auto wait = [&](uint64_t* bar, uint32_t parity) { return ptx::bounded_mbar_wait(bar, parity, abort_flag); };
      // Everything this thread touches between two MMAs stays in registers (no arrays indexed by the tile number):
      // it is the one thread the tensor pipe waits for.
      bool ok = true;
      uint32_t g = 0, n_items = 0;   // blocks and items started so far
      uint32_t cnt0 = 0, cnt1 = 0;   // blocks tile t has been through
      uint32_t outs0 = 0, outs1 = 0; // items tile t has produced output for
      for (int r = 0; r * static_cast<int>(gridDim.x) < total && ok; ++r) {
        const int idx = pp_index(r, total);
        if (idx < 0) continue;
        const PpItem it = pp_item<EXT, MIXED, SCALED>(p, idx);
        if (MIXED && it.nblk == 0) continue;
        const int nb0 = it.nblk_t[0], nb1 = it.nblk_t[1], nblk = it.nblk;
        const bool tr = n_items == 0 && blockIdx.x == 0;
        uint64_t* const q_there = SCALED ? q_fp16 : q_full;
        ok = (nb0 == 0 || wait(&q_there[0], outs0 & 1)) && wait(&k_full[g & 1], (g >> 1) & 1);
        if (!ok) break;
        ptx::tc_fence_after_sync();
        // S of the first block: the tiles' score columns are free (their last P of the previous item was waited for)
        if (nb0 > 0) issue_S(0, g & 1);
        if (nb1 > 0) {
          ok = wait(&q_there[1], outs1 & 1);
          if (!ok) break;
          ptx::tc_fence_after_sync();
          issue_S(1, g & 1);
        }
        ptx::umma_commit(&k_empty[g & 1]);
        if (nblk == 1) ptx::umma_commit(q_empty);
        for (int j = 0; j < nblk && ok; ++j) {
          const uint32_t gj = g + j;
          pp_trace(p, tr, 2, j, 0);
          bool v_here = false, k_next = false;
          // one tile's turn: wait for its P, then its P V and its next S
          auto turn = [&](const int t, const int nbt, const uint32_t cnt_t, const uint32_t outs_t) {
            if (j >= nbt || !ok) return;
            ok = wait(&p_ready[t], (cnt_t + j) & 1);  // P_t of block j is written; S_t and (after a rescale) O_t are settled
            pp_trace(p, tr, 2, j, 2 + 2 * t);
            if (ok && !v_here) {
              ok = wait(&v_full[gj & 1], (gj >> 1) & 1);
              v_here = true;
            }
            if (ok && j + 1 < nbt && !k_next) {
              ok = wait(&k_full[(gj + 1) & 1], ((gj + 1) >> 1) & 1);
              k_next = true;
            }
            // the first product of an item overwrites O_t: the warpgroup must have read the previous item's rows
            if (ok && j == 0 && outs_t > 0) ok = wait(&o_free[t], (outs_t - 1) & 1);
            if (!ok) return;
            ptx::tc_fence_after_sync();
            issue_PV(t, gj & 1, j > 0);
            if (j + 1 < nbt) issue_S(t, (gj + 1) & 1);
            pp_trace(p, tr, 2, j, 3 + 2 * t);
          };
          turn(0, nb0, cnt0, outs0);
          turn(1, nb1, cnt1, outs1);
          if (!ok) break;
          if (k_next) ptx::umma_commit(&k_empty[(gj + 1) & 1]);
          ptx::umma_commit(&v_empty[gj & 1]);
          if (j + 2 == nblk) ptx::umma_commit(q_empty);  // the S products of the last block have just been issued
        }
        cnt0 += nb0;
        cnt1 += nb1;
        outs0 += nb0 > 0 ? 1 : 0;
        outs1 += nb1 > 0 ? 1 : 0;
        g += nblk;
        ++n_items;
      }
      if (!ok && p.status) atomicCAS(p.status, 0, kStatusTimeoutMma);
    }
  } else {
    // ------------------------------------------------------------ softmax warpgroups (thread = query row)
    const int t = warp >> 2;
    const int r_ = (warp & 3) * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem_S + t * 128 + lane_addr;
    const uint32_t tO = tmem_O + t * VD + lane_addr;
    bool ok = true;
    uint32_t cnt = 0;  // blocks this tile has been through
    bool first = true;
    uint32_t items = 0;  // that have the tile
    for (int r = 0; r * static_cast<int>(gridDim.x) < total && ok; ++r) {
      const int idx = pp_index(r, total);
      if (idx < 0) continue;
      const PpItem it = pp_item<EXT, MIXED, SCALED>(p, idx);
      const int my_blocks = it.nblk_t[t];
      if (my_blocks == 0) continue;  // a short last pair has no second tile
      const bool tracer = first && blockIdx.x == 0 && (warp & 3) == 0 && lane == 0;
      first = false;
      const int q_idx = it.q0 + t * kPpTile + r_;  // row within the chunk
      const int limit = it.prefix + q_idx;         // last key position this row may see
      const int chunk_from = EXT && p.chunked ? limit - limit % p.window : -1;  // first key of the row's chunk
      float m_ref = 0.f, l = 0.f;
      float row_up = 1.f;
      if constexpr (SCALED) {
        if (!ptx::bounded_mbar_wait(&q_full[t], items++ & 1, abort_flag)) {
          ok = false;
          break;
        }
        row_up = quant_kv_row_fp16<C::kSlabs>(sQ + t * TB + r_ * 128, SB, r_ & 7) * it.k_up;
        row_up = fmaxf(row_up, p.least_up);  // (a factor of zero would make numbers that are none of what is hidden)
        ptx::fence_proxy_async_smem();
        ptx::mbar_arrive(&q_fp16[t]);
      }
      auto scale_log2 = [&]() { return SCALED ? p.scale_log2 * row_up : p.scale_log2; };
      auto cap_scale = [&]() { return SCALED ? p.cap_scale * row_up : p.cap_scale; };
      const float sig_bias = SIG && p.bias ? -1.4426950408889634f * to_f<T>(reinterpret_cast<const T*>(p.bias)[it.head]) : 0.f;
      const T* bias_row = BIAS ? reinterpret_cast<const T*>(p.bias) + static_cast<int64_t>(it.head) * p.bias_len : nullptr;
      const float far_bias = BIAS ? to_f<T>(bias_row[p.bias_len - 1]) * 1.4426950408889634f : 0.f;
      for (int j = 0; j < my_blocks; ++j) {
        pp_trace(p, tracer, t, j, 0);
        // the block's smallest distance; is any of them inside the table?
        const int nearest = it.prefix + it.q0 + t * kPpTile - (it.block(j) * kPpTile + kPpTile - 1);
        const bool near = BIAS && nearest < p.bias_len - 1;
        float bias_pair[2];
        if (near) {
#pragma unroll
          for (int k = 0; k < 2; ++k)
            bias_pair[k] = to_f<T>(bias_row[min(max(nearest + r_ + k * kPpTile, 0), p.bias_len - 1)]) * 1.4426950408889634f;
        }
        if (!ptx::bounded_mbar_wait(&s_full[t], (cnt + j) & 1, abort_flag)) {
          ok = false;
          break;
        }
        pp_trace(p, tracer, t, j, 1);
        ptx::tc_fence_after_sync();
        if constexpr (SIG) {
          const int kv0 = it.block(j) * kPpTile, row0 = it.prefix + it.q0 + t * kPpTile;
          // the block's visible keys, of this row and of all rows of the tile
          const int from = p.window > 0 ? chunk_from >= 0 ? chunk_from : limit - p.window + 1 : 0;
          const int lo = from - kv0, hi = limit - kv0, last = row0 + kPpTile - 1;
          const bool early = p.window > 0 && kv0 < (p.chunked ? last / p.window * p.window : last - p.window + 1);  // keys before some row's first
          const bool masked = kv0 + kPpTile - 1 > row0 || early;
          const uint64_t scale2 = ptx::f32x2(-p.scale_log2, -p.scale_log2), bias2 = ptx::f32x2(sig_bias, sig_bias),
                         one2 = ptx::f32x2(1.f, 1.f);
          auto weights = [&](auto&& hidden) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // 64 scores -> 32 columns of pairs
              uint32_t v[2][32], pk[32];
              ptx::tmem_ld_32x32(tS + h * 64, v[0]);
              ptx::tmem_ld_32x32(tS + h * 64 + 32, v[1]);
              ptx::tmem_ld_wait();
              // 1 + e^-x of scores c and c + 1
              auto denominators = [&](int c) {
                const int k = c - h * 64;
                const float2 x = ptx::f32x2_get(
                    ptx::fma_f32x2(ptx::f32x2(__uint_as_float(v[k >> 5][k & 31]), __uint_as_float(v[k >> 5][(k & 31) + 1])), scale2, bias2));
                return ptx::fma_f32x2(ptx::f32x2(ptx::ex2_approx(x.x), ptx::ex2_approx(x.y)), one2, one2);
              };
              float smallest = 1.f;
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                const int c = h * 64 + 2 * i;
                const uint64_t ab = denominators(c), cd = denominators(c + 2);
                const float2 f = ptx::f32x2_get(ab), g = ptx::f32x2_get(cd);
                const float fp = f.x * f.y, gp = g.x * g.y, r = ptx::rcp_approx(fp * gp);
                smallest = fminf(smallest, r);
                const float rf = r * gp, rg = r * fp;
                const float2 w = ptx::f32x2_get(ptx::mul_f32x2(ptx::f32x2(f.y, f.x), ptx::f32x2(rf, rf)));
                const float2 z = ptx::f32x2_get(ptx::mul_f32x2(ptx::f32x2(g.y, g.x), ptx::f32x2(rg, rg)));
                pk[i] = pk2<T>(hidden(c) ? 0.f : w.x, hidden(c + 1) ? 0.f : w.y);
                pk[i + 1] = pk2<T>(hidden(c + 2) ? 0.f : z.x, hidden(c + 3) ? 0.f : z.y);
              }
              if (__any_sync(0xffffffffu, !(smallest > 1e-36f))) {  // a product left the range: one reciprocal each
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                  const int c = h * 64 + 2 * i;
                  const float2 d = ptx::f32x2_get(denominators(c));
                  pk[i] = pk2<T>(hidden(c) ? 0.f : ptx::rcp_approx(d.x), hidden(c + 1) ? 0.f : ptx::rcp_approx(d.y));
                }
              }
              ptx::tmem_st_32x32(tS + h * 32, pk);
            }
          };
          if (!masked) weights([](int) { return false; });
          else if (!early) weights([&](int i) { return i > hi; });
          else weights([&](int i) { return i > hi || i < lo; });
          ptx::tmem_st_wait();
          ptx::tc_fence_before_sync();
          ptx::mbar_arrive(&p_ready[t]);
          l = 1.f;
          continue;
        }
        uint32_t v0[32], v1[32], v2[32], v3[32];  // the row's 128 scores (fp32 bits)
        ptx::tmem_ld_32x32(tS, v0);
        ptx::tmem_ld_32x32(tS + 32, v1);
        ptx::tmem_ld_32x32(tS + 64, v2);
        ptx::tmem_ld_32x32(tS + 96, v3);
        ptx::tmem_ld_wait();
        pp_trace(p, tracer, t, j, 2);
        auto score = [&](int i) -> uint32_t& { return i < 32 ? v0[i] : i < 64 ? v1[i - 32] : i < 96 ? v2[i - 64] : v3[i - 96]; };
        const int kv0 = it.block(j) * kPpTile;
        const int row0 = it.prefix + it.q0 + t * kPpTile;  // position of the tile's first row
        // does the block hold a key that some row of the tile may not see?
        bool masked = kv0 + kPpTile - 1 > row0;
        if (EXT && p.window > 0)
          masked = masked || (p.chunked ? kv0 < (row0 + kPpTile - 1) / p.window * p.window
                                        : kv0 <= row0 + kPpTile - 1 - p.window && kv0 + kPpTile > p.keep_first);
        const int from = (EXT && p.window > 0) ? chunk_from >= 0 ? chunk_from : limit - p.window + 1 : 0;
        auto visible = [&](int i) {  // key i of the block to this row
          return kv0 + i <= limit && (!EXT || kv0 + i >= from || kv0 + i < p.keep_first);
        };
        const bool capped = EXT && p.cap_log2 > 0.f;
        float bias = 0.f;  // of every score of the block, in log2 units
        if (near) {
          float* sb = s_bias + (t * 2 + (j & 1)) * 256;  // (the buffer of two blocks ago: every warp has passed the last barrier)
          sb[r_] = bias_pair[0];
          sb[r_ + kPpTile] = bias_pair[1];
          if (t == 0) asm volatile("bar.sync 1, 128;" ::: "memory");
          else asm volatile("bar.sync 2, 128;" ::: "memory");
          // distance of key i to this row: nearest + r_ + 127 - i
#pragma unroll
          for (int i = 0; i < kPpTile; ++i)
            score(i) = __float_as_uint(fmaf(__uint_as_float(score(i)), scale_log2(), sb[r_ + kPpTile - 1 - i]));
        } else if (BIAS) {
          bias = far_bias;
        }
        const float score_scale = near ? 1.f : scale_log2();
        // largest of the row's 128 scores, or of their magnitudes: eight independent chains of three-input maxima (with two
        // softmax warps per scheduler nothing else hides a serial one)
        auto largest = [&](auto&& max3) {
          float mxs[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) mxs[i] = __uint_as_float(score(i));
#pragma unroll
          for (int i = 8; i < kPpTile - 8; i += 16)
#pragma unroll
            for (int k = 0; k < 8; ++k)
              mxs[k] = max3(mxs[k], __uint_as_float(score(i + 2 * k)), __uint_as_float(score(i + 2 * k + 1)));
#pragma unroll
          for (int i = kPpTile - 8; i < kPpTile; ++i) mxs[i & 7] = max3(mxs[i & 7], __uint_as_float(score(i)), __uint_as_float(score(i)));
          const float mx = fmaxf(max3(mxs[0], mxs[1], mxs[2]), max3(mxs[3], mxs[4], mxs[5]));
          return max3(mx, mxs[6], mxs[7]);
        };
        float mx = 0.f;
        bool small = false;
        if (capped && std::is_same<T, __nv_bfloat16>::value) {  // (fp16 probabilities need the maximum itself)
          mx = largest([](float a, float b, float c) { return ptx::fmax3_abs(a, b, c); });
          small = __all_sync(0xffffffffu, mx <= p.small_max);
        }
        if (small) {
          mx *= scale_log2();  // |cap tanh(x / cap)| <= |x|
        } else {
          if (masked) {
#pragma unroll
            for (int i = 0; i < kPpTile; ++i)
              if (!visible(i)) score(i) = 0xff800000u;  // -inf
          }
          mx = largest([](float a, float b, float c) { return ptx::fmax3(a, b, c); });
          if (capped) mx = mx == -INFINITY ? mx : p.cap_log2 * ptx::tanh_ex2(mx * cap_scale());
          else mx = BIAS ? fmaf(mx, score_scale, bias) : mx * scale_log2();
        }
        // (S of this block was issued after P V of the previous one, so that product is complete: O_t is stable and
        // the columns P is about to overwrite have been read)
        if (j == 0) {
          m_ref = (!EXT && mx == -INFINITY) ? 0.f : mx;  // EXT: a row may see nothing of its first blocks
        } else {
          const bool grow = mx > m_ref + kPpRescaleAt;
          if (__any_sync(0xffffffffu, grow)) {
            const float alpha = grow ? ptx::ex2_approx(m_ref - mx) : 1.f;
#pragma unroll 1
            for (int c = 0; c < VD; c += 32) {
              uint32_t o[32];
              ptx::tmem_ld_32x32(tO + c, o);
              ptx::tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              ptx::tmem_st_32x32(tO + c, o);
            }
            ptx::tmem_st_wait();
            l *= alpha;
            if (grow) m_ref = mx;
          }
        }
        pp_trace(p, tracer, t, j, 3);
        // probabilities (16 bit) -> tensor memory over the scores; row sum
        float rs[4] = {0.f, 0.f, 0.f, 0.f};
        const float neg_m = ((EXT && m_ref == -INFINITY) ? 0.f : -m_ref) + (BIAS ? bias : 0.f);
        auto probabilities = [&](auto&& exponents) {  // exponents(c): those of scores c and c + 1
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // 64 scores -> 32 columns of pairs
            uint32_t pk[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float2 x = exponents(h * 64 + 2 * i);
              const float e0 = ptx::ex2_approx(x.x);
              const float e1 = (POLY && (i & 1)) ? ptx::ex2_poly(x.y) : ptx::ex2_approx(x.y);
              rs[i & 3] += e0 + e1;
              pk[i] = pk2<T>(e0, e1);
            }
            ptx::tmem_st_32x32(tS + h * 32, pk);
          }
        };
        if (EXT && small) {
          const uint64_t c0 = ptx::f32x2(p.poly[0], p.poly[0]), c1 = ptx::f32x2(p.poly[1], p.poly[1]),
                         c2 = ptx::f32x2(p.poly[2], p.poly[2]), c3 = ptx::f32x2(p.poly[3], p.poly[3]), nm = ptx::f32x2(neg_m, neg_m);
          auto poly = [&](int c) {
            const uint64_t x = ptx::f32x2(__uint_as_float(score(c)), __uint_as_float(score(c + 1)));
            const uint64_t y = ptx::mul_f32x2(x, x);
            uint64_t r = ptx::fma_f32x2(c3, y, c2);
            r = ptx::fma_f32x2(r, y, c1);
            r = ptx::fma_f32x2(r, y, c0);
            return ptx::f32x2_get(ptx::fma_f32x2(x, r, nm));
          };
          if (masked) {
            probabilities([&](int c) {
              float2 e = poly(c);
              if (!visible(c)) e.x = -INFINITY;
              if (!visible(c + 1)) e.y = -INFINITY;
              return e;
            });
          } else {
            probabilities(poly);
          }
        } else if (capped) {
          auto cap = [&](float x) { return x == -INFINITY ? x : fmaf(ptx::tanh_ex2(x * cap_scale()), p.cap_log2, neg_m); };
          probabilities([&](int c) { return make_float2(cap(__uint_as_float(score(c))), cap(__uint_as_float(score(c + 1)))); });
        } else {
          probabilities([&](int c) {
            return make_float2(fmaf(__uint_as_float(score(c)), BIAS ? score_scale : scale_log2(), neg_m),
                               fmaf(__uint_as_float(score(c + 1)), BIAS ? score_scale : scale_log2(), neg_m));
          });
        }
        pp_trace(p, tracer, t, j, 4);
        ptx::tmem_st_wait();
        l += (rs[0] + rs[1]) + (rs[2] + rs[3]);
        ptx::tc_fence_before_sync();
        ptx::mbar_arrive(&p_ready[t]);
        pp_trace(p, tracer, t, j, 5);
      }
      if (ok) ok = ptx::bounded_mbar_wait(&o_full[t], (cnt + my_blocks - 1) & 1, abort_flag);
      if (!ok) break;
      cnt += my_blocks;
      ptx::tc_fence_after_sync();
      if (EXT && p.sink != nullptr && l > 0.f)
        l += ptx::ex2_approx(to_f<IO>(reinterpret_cast<const IO*>(p.sink)[it.head]) * 1.4426950408889634f - m_ref);
      float inv = l > 0.f ? 1.f / l : 0.f;
      if constexpr (SCALED) inv *= __ldg(&p.forms[static_cast<int64_t>(idx / p.q_heads) * p.kv_heads + it.kv_head].y);
      if (p.gate != nullptr && q_idx < it.q_len) {
        const T z = reinterpret_cast<const T*>(p.gate)[static_cast<int64_t>(it.seq_start + q_idx) * p.gate_stride + it.head];
        inv /= 1.f + expf(-to_f<T>(z));
      }
      IO* dst = reinterpret_cast<IO*>(p.out) + static_cast<int64_t>(it.seq_start + q_idx) * p.out_stride + it.head * p.vdim;
#pragma unroll 1
      for (int c = 0; c < VD; c += 32) {
        uint32_t o[32];
        ptx::tmem_ld_32x32(tO + c, o);
        ptx::tmem_ld_wait();
        if (c + 32 >= VD) {  // all of this item's output rows are in registers: the next item may overwrite them
          ptx::tc_fence_before_sync();
          ptx::mbar_arrive(&o_free[t]);
        }
        if (q_idx < it.q_len) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            if (c + i < p.vdim) *reinterpret_cast<uint4*>(dst + c + i) = make_uint4(
                pk2<IO>(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv),
                pk2<IO>(__uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv),
                pk2<IO>(__uint_as_float(o[i + 4]) * inv, __uint_as_float(o[i + 5]) * inv),
                pk2<IO>(__uint_as_float(o[i + 6]) * inv, __uint_as_float(o[i + 7]) * inv));
          }
        }
      }
    }
    if (!ok && p.status && lane == 0) atomicCAS(p.status, 0, kStatusTimeoutEpilogue);
  }
