// Attention over pages with many rows per key head (trees of drafted tokens, runs, prompts behind a cached prefix): tcgen05
// products of 128 rows x 128 keys.  A row is a (token, query head of the key head) pair.
//
// Built like the dense two-stream forward (fb_fwd_s_sm100.cuh): two softmax warpgroups share a row tile and take its key tiles in
// turn, with logits and probabilities of their own in tensor memory, one output accumulator and one running reference maximum
// per row that they hand to one another behind each tile's row maximum.
//   warps 0-3, 4-7  softmax of the even / odd key tiles, thread = row; queries into shared memory; epilogue
//   warp 8          TMA producer: a copy per page (and 64 columns), a lane looks up a page
//   warp 9          S = Q.K^T          warp 10   O += P.V
//   warp 11         V behind its copy: places that hold no key become zero, and so do values that are not finite where not every
//                   row sees the key (0 x inf would reach the rows that do not): the epilogue adds them to the rows that do
// The schedule is that of fb_paged.cuh: equal parts of all key tiles per CTA, parts of an item joined by a second launch.
// Key tiles are taken from the newest down: a bias that falls with the distance then shows its maximum first.
#pragma once

#include <mutex>

#include "fb_paged.cuh"

namespace fb {

constexpr int kTileThreads = 384;

template <int TD>
struct TileCfg {
  static constexpr int Q_BYTES = tile_bytes(TD), ST = 2;
  static constexpr int OFF_K = Q_BYTES, OFF_V = OFF_K + ST * Q_BYTES, OFF_BAR = OFF_V + ST * Q_BYTES, OFF_ML = OFF_BAR + 256,
                       OFF_M = OFF_ML + 2 * 2 * 128 * 8, SMEM = OFF_M + 2 * 128 * 4 + 1024;
  static constexpr int T_S = 0, T_P = 256, T_O = 384;  // stream x: S + 128 x, P + 64 x
};

// The 32 keys from drafted token td0 on (negative: cached ones) that a row of token t (global token n) sees, as bits.
__device__ __forceinline__ uint32_t seen_bits(const fb_paged_params& p, int n, int t, int td0) {
  if (!p.tree_mask) return td0 > t ? 0u : t - td0 >= 31 ? 0xffffffffu : (2u << (t - td0)) - 1u;
  const int64_t* words = p.tree_mask + n * p.mask_stride;
  auto word = [&](int w) { return w < 0 ? ~0ull : w < p.mask_words ? (uint64_t)words[w] : 0ull; };
  const int w = td0 >> 6, s = td0 & 63;
  return (uint32_t)(s ? (word(w) >> s) | (word(w + 1) << (64 - s)) : word(w));
}

template <typename T, int TD, bool SLOPES>
__global__ void __launch_bounds__(kTileThreads, 1)
paged_tile_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PagedArgs a) {
  using Cfg = TileCfg<TD>;
  constexpr int ST = Cfg::ST, NB = TD / 64, CH = TD / 8;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem), sQ = sbase, sK = sbase + Cfg::OFF_K, sV = sbase + Cfg::OFF_V, bar0 = sbase + Cfg::OFF_BAR;
  // (two slots: one per stream, or per stage)
  const uint32_t q_ready = bar0, q_free = bar0 + 8, o_free = bar0 + 16, s_full = bar0 + 24, p_ready = bar0 + 40, pv_done = bar0 + 56,
                 k_full = bar0 + 72, k_free = bar0 + 88, v_full = bar0 + 104, v_free = bar0 + 120, s_read = bar0 + 136, v_ok = bar0 + 152;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Cfg::OFF_BAR + 168);
  const uint32_t abort_flag = bar0 + 172;
  // per tile, eight deep (the producer is four tiles ahead of a softmax at most): which of the tile's pages exist
  volatile uint32_t* s_pages = reinterpret_cast<volatile uint32_t*>(smem + Cfg::OFF_BAR + 176);
  // per segment, eight deep: its number + 1 if it has values that were taken out
  volatile int* s_taken = reinterpret_cast<volatile int*>(smem + Cfg::OFF_BAR + 208);

  const fb_paged_params& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 8) {
    if (lane == 0) {
      st_shared_flag(abort_flag, 0u);
      mbar_init(q_ready, 8);
      mbar_init(q_free, 1);
      mbar_init(o_free, 8);
      for (int i = 0; i < 2; ++i) {
        mbar_init(s_full + 8 * i, 1);
        mbar_init(p_ready + 8 * i, 4);
        mbar_init(pv_done + 8 * i, 1);
        mbar_init(s_read + 8 * i, 4);
        mbar_init(k_full + 8 * i, 1);
        mbar_init(k_free + 8 * i, 1);
        mbar_init(v_full + 8 * i, 1);
        mbar_init(v_free + 8 * i, 1);
        mbar_init(v_ok + 8 * i, 1);
      }
      for (int i = 0; i < 8; ++i) s_taken[i] = 0;
      mbar_fence_init();
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
  } else if (warp == 9) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  grid_dep_wait();
  if (threadIdx.x == 0) a.desc[blockIdx.x].x = -1;
  PagedWalk<128, 128, kTileThreads> walk;
  walk.start(a, p.Hk);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  Segment seg;
  auto key0 = [](const Segment& s, int j) { return (s.t1 - 1 - j) * 128; };  // first key of the j-th tile visited

  if (warp >= 8) {
    setmaxnreg_dec<88>();
    if (warp == 8) {
      // ------------------------------------------------------------------ TMA producer
      const int rows = min(p.page_size, 128), pieces = 128 / rows;  // copies of a tile
      auto wait_all = [&](uint32_t bar, int parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)); };  // (the warp leaves together)
      auto produce = [&] {
        int t = 0;
        while (walk.next(a, seg)) {
          const int32_t* table = p.block_table + (int64_t)min(seg.b, p.B - 1) * p.table_stride;
          for (int j = 0; j < seg.t1 - seg.t0; ++j, ++t) {
            const int st = t % ST, key = key0(seg, j) + lane * rows;
            int page = (int)p.num_pages, place = 0;  // behind the cache: the copy fills in zeros
            bool bad = false;
            if (lane < pieces && key < seg.r.keys) {
              const int col = a.page_div.quot32(key), pg = table[col];
              bad = pg < 0 || pg >= p.num_pages;
              if (!bad) {
                page = pg;
                place = key - col * p.page_size;
              } else {
                paged_bad_index(p);
              }
            }
            const uint32_t there = ~__ballot_sync(0xffffffffu, bad);
            if (t >= ST && !wait_all(k_free + 8 * st, (t / ST - 1) & 1)) return;
            if (lane == 0) {
              s_pages[t & 7] = there;
              mbar_expect_tx(k_full + 8 * st, Cfg::Q_BYTES);
            }
            __syncwarp();
            if (lane < pieces) {
#pragma unroll
              for (int c = 0; c < NB; ++c)
                tma_load_4d(sK + st * Cfg::Q_BYTES + c * 128 * 128 + lane * rows * 128, &tmK, k_full + 8 * st, c * 64, place, seg.hg, page);
            }
            if (t >= ST && !wait_all(v_free + 8 * st, (t / ST - 1) & 1)) return;
            if (lane == 0) mbar_expect_tx(v_full + 8 * st, Cfg::Q_BYTES);
            __syncwarp();
            if (lane < pieces) {
#pragma unroll
              for (int c = 0; c < NB; ++c)
                tma_load_4d(sV + st * Cfg::Q_BYTES + c * 128 * 128 + lane * rows * 128, &tmV, v_full + 8 * st, c * 64, place, seg.hg, page);
            }
          }
        }
      };
      produce();
    } else if (warp == 9) {
      // ------------------------------------------------------------------ S = Q.K^T
      if (elect_one()) {
        constexpr uint32_t idS = instr_desc(kBf16, false, false, 128, 128);
        const DescBase dQ = kmajor_base<TD>(sQ), dK = kmajor_base<TD>(sK);
        int t = 0, n = 0, c0 = 0, c1 = 0;  // key tiles, segments; key tiles of either stream
        for (; walk.next(a, seg); ++n) {
          mbar_wait(q_ready, n & 1, abort_flag);
          tc_fence_after_sync();
          for (int j = 0; j < seg.t1 - seg.t0; ++j, ++t) {
            const int x = j & 1, c = x ? c1++ : c0++, st = t % ST;
            if (c > 0) mbar_wait(s_read + 8 * x, (c - 1) & 1, abort_flag);
            mbar_wait(k_full + 8 * st, (t / ST) & 1, abort_flag);
            tc_fence_after_sync();
#pragma unroll
            for (int s = 0; s < TD / 16; ++s)
              umma_ss(tmem + Cfg::T_S + 128 * x, desc_at(dQ, kmajor_step<TD>(s)), desc_at(dK, st * Cfg::Q_BYTES + kmajor_step<TD>(s)), idS, s > 0);
            umma_commit(s_full + 8 * x);
            umma_commit(k_free + 8 * st);
          }
          umma_commit(q_free);  // Q of this segment is no longer read
        }
      }
    } else if (warp == 10) {
      // ------------------------------------------------------------------ O += P.V
      if (elect_one()) {
        constexpr uint32_t idO = instr_desc(kBf16, false, true, 128, TD);
        const DescBase dV = mnmajor_base<TD>(sV);
        int t = 0, n = 0, c0 = 0, c1 = 0;
        for (; walk.next(a, seg); ++n) {
          for (int j = 0; j < seg.t1 - seg.t0; ++j, ++t) {
            const int x = j & 1, c = x ? c1++ : c0++, st = t % ST;
            mbar_wait(v_ok + 8 * st, (t / ST) & 1, abort_flag);
            mbar_wait(p_ready + 8 * x, c & 1, abort_flag);
            if (j == 0 && n > 0) mbar_wait(o_free, (n - 1) & 1, abort_flag);  // the accumulator of the last segment has been read
            tc_fence_after_sync();
#pragma unroll
            for (int s = 0; s < 8; ++s)
              umma_ts(tmem + Cfg::T_O, tmem + Cfg::T_P + 64 * x + s * 8, desc_at(dV, st * Cfg::Q_BYTES + mnmajor_step<TD>(s)), idO, (j > 0 || s > 0) ? 1u : 0u);
            umma_commit(pv_done + 8 * x);
            umma_commit(v_free + 8 * st);
          }
        }
      }
    } else {
      // ------------------------------------------------------------------ V behind its copy
      int t = 0, n = 0;
      for (; walk.next(a, seg); ++n) {
        for (int j = 0; j < seg.t1 - seg.t0; ++j, ++t) {
          const int st = t % ST, k0 = key0(seg, j);
          mbar_wait(v_full + 8 * st, (t / ST) & 1, abort_flag);
          const int r0 = max(seg.r.len - k0, 0), live = seg.r.keys - k0;  // first row that not all see; rows that hold keys
          if (r0 < 128) {
            bool taken = false;
            for (int i = r0 * CH + lane; i < 128 * CH; i += 32) {
              const int row = i / CH;
              const uint32_t at = sV + st * Cfg::Q_BYTES + tile_chunk_offset<TD>(row, (i - row * CH) * 8);
              if (row >= live) {
                st_shared_v4(at, 0u, 0u, 0u, 0u);
                continue;
              }
              uint32_t w[4];
              ld_shared_v4(at, w[0], w[1], w[2], w[3]);
              bool odd = false;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                constexpr uint32_t E = kBf16 ? 0x7f80u : 0x7c00u;
                if ((w[e] & E) == E) w[e] &= 0xffff0000u, odd = true;
                if (((w[e] >> 16) & E) == E) w[e] &= 0xffffu, odd = true;
              }
              if (odd) st_shared_v4(at, w[0], w[1], w[2], w[3]);
              taken |= odd;
            }
            if (taken) s_taken[n & 7] = n + 1;
            fence_proxy_async_smem();
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(v_ok + 8 * st);
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax + epilogue
    setmaxnreg_inc<208>();
    const int x = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + Cfg::T_S + 128 * x + lane_off, tP = tmem + Cfg::T_P + 64 * x + lane_off, tO = tmem + Cfg::T_O + lane_off;
    const uint32_t m_own = sbase + Cfg::OFF_M + (x * 128 + row) * 4, m_other = sbase + Cfg::OFF_M + ((x ^ 1) * 128 + row) * 4;
    const float sl2 = a.scale_log2;
    const uint64_t sl2p = f2(sl2, sl2);
    int c = 0, co = 0, n = 0, t0 = 0;  // key tiles of this stream and of the other, segments and key tiles so far
    uint32_t s[4][32];                 // the thread's row of the logit tile
    int tok, head;                     // the row's token (of the request) and query head; -1: padding
    // Half a row of queries per thread; ahead of the last segment's epilogue.
    auto load_q = [&](const Segment& sg, int nth) {
      const int gr = sg.rt * 128 + row;
      tok = -1;
      head = 0;
      if (gr < sg.r.tokens * a.G) {
        tok = a.group_div.quot32(gr);
        head = sg.hg * a.G + gr - tok * a.G;
      }
      const T* src = reinterpret_cast<const T*>(p.q) + (int64_t)(sg.r.first + max(tok, 0)) * p.q_stride[0] + head * p.q_stride[1];
      if (nth > 0) mbar_wait(q_free, (nth - 1) & 1, abort_flag);
#pragma unroll
      for (int ch = 0; ch < CH / 2; ++ch) {
        const int col = (x * CH / 2 + ch) * 8;
        const uint4 w = tok >= 0 && col < p.D ? *reinterpret_cast<const uint4*>(src + col) : make_uint4(0u, 0u, 0u, 0u);
        st_shared_v4(sQ + tile_chunk_offset<TD>(row, col), w.x, w.y, w.z, w.w);
      }
      fence_proxy_async_smem();
      mbar_arrive_warp(q_ready);
    };
    Segment nxt;
    bool more = walk.next(a, nxt);
    if (more) load_q(nxt, 0);
    for (; more; ++n) {
      seg = nxt;
      const int n_kv = seg.t1 - seg.t0, tk = tok, hd = head, gn = seg.r.first + max(tk, 0);
      float m_used = -INFINITY, l = 0.f;  // reference maximum (log2 units: logit * log2 e); row sum of this stream's tiles, relative to it
      const int c0 = c, co0 = co;
      const float slope2 = SLOPES && tk >= 0 ? p.slopes[hd] * kLog2eP : 0.f;
      const int my_pos = SLOPES && tk >= 0 ? (p.positions ? p.positions[gn] : seg.r.len + tk) : 0;
      for (int j = x; j < n_kv; j += 2, ++c) {
        const int k0 = key0(seg, j);
        mbar_wait(s_full + 8 * x, c & 1, abort_flag);
        tc_fence_after_sync();
        const uint32_t there = s_pages[(t0 + j) & 7];
        const bool dead = there != 0xffffffffu || k0 + 128 > seg.r.len;
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        const float abase = SLOPES ? slope2 * (float)(k0 - my_pos) : 0.f;
        auto complete = [&](int ch) {
          if (dead) {
            const int j0 = k0 + ch * 32, left = seg.r.keys - j0;
            uint32_t bits = left >= 32 ? 0xffffffffu : left > 0 ? (1u << left) - 1u : 0u;
            if (tk >= 0 && bits && j0 + 32 > seg.r.len) bits &= seen_bits(p, gn, tk, j0 - seg.r.len);
            if (there != 0xffffffffu) {  // (rare)
              const int rows = min(p.page_size, 128);
              for (int i = 0; i < 32; ++i)
                if (!(there >> ((ch * 32 + i) / rows) & 1)) bits &= ~(1u << i);
            }
            if (SLOPES && p.positions) {
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const int key = j0 + i, pos = key >= seg.r.len && key < seg.r.keys ? p.positions[seg.r.first + key - seg.r.len] : key;
                s[ch][i] = __float_as_uint(fmaf(slope2, (float)(pos - my_pos), __uint_as_float(s[ch][i]) * sl2));
              }
            } else if (SLOPES) {
#pragma unroll
              for (int i = 0; i < 32; ++i) s[ch][i] = __float_as_uint(fmaf(slope2, (float)(j0 + i - my_pos), __uint_as_float(s[ch][i]) * sl2));
            }
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(bits >> i & 1)) s[ch][i] = __float_as_uint(-INFINITY);
#pragma unroll
            for (int i = 0; i < 32; i += 2) mx4[(i >> 1) & 3] = fmax3(mx4[(i >> 1) & 3], __uint_as_float(s[ch][i]), __uint_as_float(s[ch][i + 1]));
            __syncwarp();  // (the loads from tensor memory want the warp together)
            return;
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float v0 = __uint_as_float(s[ch][i]), v1 = __uint_as_float(s[ch][i + 1]);
            if (SLOPES) {
              f2_unpack(f2_fma(f2(v0, v1), sl2p, f2(fmaf((float)(ch * 32 + i), slope2, abase), fmaf((float)(ch * 32 + i + 1), slope2, abase))), v0, v1);
              s[ch][i] = __float_as_uint(v0);
              s[ch][i + 1] = __float_as_uint(v1);
            }
            mx4[(i >> 1) & 3] = fmax3(mx4[(i >> 1) & 3], v0, v1);
          }
        };
        tmem_ld32(tS, s[0]);
        tmem_wait_ld(s[0]);
        tmem_ld32(tS + 32, s[1]);
        complete(0);
        tmem_wait_ld(s[1]);
        tmem_ld32(tS + 64, s[2]);
        complete(1);
        tmem_wait_ld(s[2]);
        tmem_ld32(tS + 96, s[3]);
        complete(2);
        tmem_wait_ld(s[3]);
        tc_fence_before_sync();
        mbar_arrive_warp(s_read + 8 * x);  // the tensor core may start on the stream's next tile
        complete(3);
        float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        if (!SLOPES) mx *= sl2;  // sl2 > 0
        // ---- the reference maximum, from tile to tile: it moves only when the maximum has grown by more than 2^8 (exact: the row
        // sums carry the same reference)
        const float m_last = m_used;
        if (j > 0) {
          asm volatile("bar.sync %0, 256;" ::"r"(2 + (x ^ 1)) : "memory");
          m_used = __uint_as_float(ld_shared_flag(m_other));
          const float m_new = fmaxf(m_used, mx);
          if (__any_sync(0xffffffffu, m_new - m_used > 8.f)) {  // (from -inf: the difference is +inf, or NaN where both are)
            // O is stable behind the product of tile j - 1.  The wait tests a parity, so the other stream's product before it, tile
            // j - 3, must be known to have completed: tile j's logits are here, K(j) was loaded behind V(j - 1), and V(j - 1), in a
            // ring of two, where V(j - 3) had been, behind that product.
            static_assert(ST == 2, "a deeper ring does not order the products of tiles j - 3 and j");
            mbar_wait(pv_done + 8 * (x ^ 1), (co0 + ((j - 1) >> 1)) & 1, abort_flag);
            tc_fence_after_sync();
            const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_used - m_new);
            m_used = m_new;
#pragma unroll 1
            for (int ch = 0; ch < TD / 32; ++ch) {
              uint32_t r[32];
              tmem_ld32(tO + ch * 32, r);
              tmem_wait_ld(r);
#pragma unroll
              for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
              tmem_st32(tO + ch * 32, r);
            }
            tmem_wait_st();
          }
        } else {
          m_used = mx;
        }
        if (j + 1 < n_kv) {
          st_shared_f32(m_own, m_used);
          asm volatile("bar.arrive %0, 256;" ::"r"(2 + x) : "memory");
        }
        if (c > 0) mbar_wait(pv_done + 8 * x, (c - 1) & 1, abort_flag);  // P has been read
        // ---- p = exp2(logit2 - m), row sum, P -> tensor memory (the A operand of O += P.V), rounded to the 16 bits of V
        const float msub = m_used == -INFINITY ? 0.f : m_used;
        l *= fast_exp2(m_last - msub);  // (0 at the stream's first tile, where l is 0)
        uint64_t l2a = f2(0.f, 0.f), l2b = f2(0.f, 0.f);
        const uint64_t nm = f2(-msub, -msub);
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {
          uint32_t pw[16];  // 32 keys = 16 packed words
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const uint64_t v = f2(__uint_as_float(s[ch][i]), __uint_as_float(s[ch][i + 1]));
            float a0, a1;
            f2_unpack(!SLOPES ? f2_fma(v, sl2p, nm) : f2_add(v, nm), a0, a1);
            const float p0 = fast_exp2(a0), p1 = fast_exp2(a1);
            if (i & 2) l2b = f2_add(l2b, f2(p0, p1)); else l2a = f2_add(l2a, f2(p0, p1));
            pw[i / 2] = Pack2<T>::pack(p0, p1);
          }
          tmem_st16(tP + ch * 16, pw);
        }
        {
          float x0, x1, x2, x3;
          f2_unpack(l2a, x0, x1);
          f2_unpack(l2b, x2, x3);
          l += (x0 + x1) + (x2 + x3);
        }
        tmem_wait_st();
        tc_fence_before_sync();
        mbar_arrive_warp(p_ready + 8 * x);
      }
      t0 += n_kv;
      more = walk.next(a, nxt);
      if (more) load_q(nxt, n + 1);
      // ---- epilogue, this warpgroup's half of the columns.  The stream of the last tile knows its product to have completed (its
      // commit covers the ones before it, which the same thread issued); the other learns it from the warpgroups' barrier.
      c = c0 + ((n_kv + 1 - x) >> 1);
      co = co0 + ((n_kv + x) >> 1);
      const int xl = (n_kv - 1) & 1;  // stream of the last tile
      if (xl == x) mbar_wait(pv_done + 8 * x, (c - 1) & 1, abort_flag);
      float2* ml = reinterpret_cast<float2*>(smem + Cfg::OFF_ML) + (n & 1) * 256;
      ml[x * 128 + row] = make_float2(m_used, l);
      asm volatile("bar.sync 1, 256;" ::: "memory");  // both warpgroups
      tc_fence_after_sync();
      const float2 other = ml[(x ^ 1) * 128 + row];
      const float m = fmaxf(m_used, other.x), ms = m == -INFINITY ? 0.f : m;  // the last reference is the largest
      const float ls = l * fast_exp2(m_used - ms) + other.y * fast_exp2(other.x - ms);
      const bool whole = seg.t0 == 0 && seg.t1 == seg.tiles, taken = s_taken[n & 7] == n + 1;
      const float inv = !whole ? 1.f : ls > 0.f ? 1.f / ls : ls == 0.f ? 0.f : ls;
      const int64_t prow = ((int64_t)blockIdx.x * 2 + (seg.t0 == 0 ? 1 : 0)) * 128 + row;  // slot 1: the CTA in which the item begins
#pragma unroll 1
      for (int ch = 0; ch < TD / 64; ++ch) {
        const int col0 = x * (TD / 2) + ch * 32;
        uint32_t r[32];
        tmem_ld32(tO + col0, r);
        tmem_wait_ld(r);
        if (tk >= 0) {
          if (taken) {  // (rare) values that are not finite, for the rows that see their keys
            const int32_t* table = p.block_table + (int64_t)seg.b * p.table_stride;
            for (int key = max(seg.r.len, seg.t0 * 128); key < min(seg.r.keys, seg.t1 * 128); ++key) {
              const int col = a.page_div.quot32(key), pg = table[col];
              if (pg < 0 || pg >= p.num_pages || !tree_sees(p, gn, tk, key - seg.r.len)) continue;
              const T* v = reinterpret_cast<const T*>(p.value_cache) + pg * p.value_cache_stride[0] + (key - col * p.page_size) * p.value_cache_stride[1] +
                           seg.hg * p.value_cache_stride[2] + col0;
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                const float e = col0 + i < p.D ? to_f32(v[i]) : 0.f;
                if (!(fabsf(e) <= 3.4e38f)) r[i] = __float_as_uint(__uint_as_float(r[i]) + e);
              }
            }
          }
          if (whole) {
            T* orow = reinterpret_cast<T*>(p.o) + (int64_t)gn * p.o_stride[0] + hd * p.o_stride[1];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              if (col0 + g * 8 >= p.D) break;  // D is a multiple of 8
              auto p2 = [&](int i) {
                return ls == 0.f ? 0u : Pack2<T>::pack(__uint_as_float(r[g * 8 + i]) * inv, __uint_as_float(r[g * 8 + i + 1]) * inv);
              };
              *reinterpret_cast<uint4*>(orow + col0 + g * 8) = make_uint4(p2(0), p2(2), p2(4), p2(6));
            }
          } else {
            float4* dst = reinterpret_cast<float4*>(a.part + prow * TD + col0);
#pragma unroll
            for (int g = 0; g < 8; ++g)
              dst[g] = make_float4(__uint_as_float(r[4 * g]), __uint_as_float(r[4 * g + 1]), __uint_as_float(r[4 * g + 2]), __uint_as_float(r[4 * g + 3]));
          }
        }
        __syncwarp();
      }
      if (x == 0 && tk >= 0) {
        if (!whole) a.ml[prow] = make_float2(m, ls);
        else if (p.lse) p.lse[(int64_t)gn * p.Hq + hd] = ls > 0.f ? (m + fast_log2(ls)) * kLn2P : ls == 0.f ? -INFINITY : ls;
      }
      if (!whole && seg.t0 == 0 && threadIdx.x == 0) a.desc[blockIdx.x] = make_int4(seg.b, seg.rt, seg.hg, seg.last_cta);
      tc_fence_before_sync();
      mbar_arrive_warp(o_free);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  report_expired_wait(abort_flag, p.status);
  if (warp == 9) {
    settle_expired_wait(abort_flag);
    __syncwarp();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int TD, bool SLOPES>
int launch_paged_tile_t(const PagedArgs& a, const PagedPlan& plan, const CUtensorMap& tk, const CUtensorMap& tv, cudaStream_t st) {
  auto kern = paged_tile_kernel<T, TD, SLOPES>;
  static std::mutex mu;
  static bool attr_done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lk(mu);
    if (!attr_done[dev & 63]) {
      const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, TileCfg<TD>::SMEM);
      if (e != cudaSuccess) return (int)e;
      attr_done[dev & 63] = true;
    }
  }
  return launch_pdl(kern, plan.ctas, kTileThreads, TileCfg<TD>::SMEM, st, tk, tv, a);
}

template <int TD>
int launch_paged_tile(const PagedArgs& a, const PagedPlan& plan, cudaStream_t st) {
  const fb_paged_params& p = a.p;
  CUtensorMap tk, tv;
  const int rows = p.page_size < 128 ? p.page_size : 128;
  int rc;
  if ((rc = make_tmap_4d(&tk, p.key_cache, p.D, p.page_size, p.Hk, p.num_pages, p.key_cache_stride[1], p.key_cache_stride[2], p.key_cache_stride[0], 64, rows)))
    return rc;
  if ((rc = make_tmap_4d(&tv, p.value_cache, p.D, p.page_size, p.Hk, p.num_pages, p.value_cache_stride[1], p.value_cache_stride[2], p.value_cache_stride[0], 64, rows)))
    return rc;
  auto go = [&](auto t) {
    using T = decltype(t);
    return p.slopes ? launch_paged_tile_t<T, TD, true>(a, plan, tk, tv, st) : launch_paged_tile_t<T, TD, false>(a, plan, tk, tv, st);
  };
  if ((rc = p.dtype == FB_DTYPE_F16 ? go(__half()) : go(__nv_bfloat16()))) return rc;
  return launch_paged_join<TD>(a, plan, st);
}

}  // namespace fb
