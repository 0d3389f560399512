// Attention over pages with many rows per key head (trees of drafted tokens, runs, prompts behind a cached prefix): tcgen05
// products of 128 rows x 128 keys.  A row is a (token, query head of the key head) pair.
//
// Built like the dense two-stream forward (fb_fwd_s_sm100.cuh): two softmax warpgroups share a row tile and take its key tiles in
// turn, with logits and probabilities of their own in tensor memory, one output accumulator and one running reference maximum
// per row that they hand to one another behind each tile's row maximum.
//   warps 0-3, 4-7  softmax of the even / odd key tiles, thread = row; epilogue
//   warp 8          walks the schedule, one segment ahead of all others; copies of K: TMA, one per page (and 64 columns), a lane
//                   looks up a page.  K does not wait for V's ring: the logits run ahead of the products P.V
//   warp 9          S = Q.K^T          warp 10   O += P.V
//   warp 11         copies of V, and V behind its copy: places that hold no key become zero, and so do values that are not finite
//                   where not every row sees the key (0 x inf would reach the rows that do not): the epilogue adds them to the
//                   rows that do; the next segment's queries
// The schedule's state is registers that a softmax thread, with a row of logits in its own, does not have: the others read the
// segments from shared memory.
// The schedule is that of fb_paged.cuh: equal parts of all key tiles per CTA, parts of an item joined by a second launch.
// Key tiles are taken from the newest down: a bias that falls with the distance then shows its maximum first.
// 8 trees of up to 60 tokens over up to 6000, H32-8 D128, slopes: 64 us (139 MB, 24 GFLOP; the general kernel 24059).  Bound by a
// tile's chain of steps (tensor pipe 33 %) and, 25 us of it, by the segments' beginnings and ends and the join.
#pragma once

#include <mutex>

#include "fb_paged.cuh"

namespace fb {

constexpr int kTileThreads = 384;

template <int TD>
struct TileCfg {
  static constexpr int Q_BYTES = tile_bytes(TD);
  // Stages of K and V.  A copy from HBM takes about as long as two tiles' work, and V's stage is held until its product is done:
  // with two the products wait for V (2200 clk a tile).
  static constexpr int KST = TD == 128 ? 2 : 3, VST = TD == 128 ? 3 : 4;
  static constexpr int OFF_K = Q_BYTES, OFF_V = OFF_K + KST * Q_BYTES, OFF_BAR = OFF_V + VST * Q_BYTES, OFF_SEG = OFF_BAR + 512,
                       OFF_ML = OFF_SEG + 8 * 64, OFF_M = OFF_ML + 2 * 2 * 128 * 8, OFF_POS = OFF_M + 2 * 128 * 4, SMEM = OFF_POS + 8 * 128 * 4 + 1024;
  static constexpr int T_S = 0, T_P = 256, T_O = 384;  // stream x: S + 128 x, P + 64 x
};

// A segment as the other warps read it; n_kv = 0: there are no more.
struct TileSeg {
  int n_kv, t0, t1, tiles, b, rt, hg, last_cta, first, tokens, len, keys;
};
static_assert(sizeof(TileSeg) <= 64, "room in shared memory");

template <typename T, int TD, bool SLOPES>
__global__ void __launch_bounds__(kTileThreads, 1)
paged_tile_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ PagedArgs a) {
  using Cfg = TileCfg<TD>;
  constexpr int KST = Cfg::KST, VST = Cfg::VST, NB = TD / 64, CH = TD / 8;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  static_assert(KST + 3 < 8, "rings of pages and positions");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem), sQ = sbase, sK = sbase + Cfg::OFF_K, sV = sbase + Cfg::OFF_V, bar0 = sbase + Cfg::OFF_BAR;
  // one slot per stream, stage (up to four), product in turn and stream, segment (eight)
  const uint32_t q_ready = bar0, q_free = bar0 + 8, o_free = bar0 + 16, s_full = bar0 + 24, p_ready = bar0 + 40, s_read = bar0 + 56,
                 k_full = bar0 + 72, k_free = bar0 + 104, v_full = bar0 + 136, v_free = bar0 + 168, v_ok = bar0 + 320, pv_done = bar0 + 352,
                 seg_full = bar0 + 384;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Cfg::OFF_BAR + 200);
  const uint32_t abort_flag = bar0 + 204;
  // per tile, eight deep: K's place is filled again when S of KST tiles before is done, for which a stream has taken the logits of
  // the tile before that, or two before, and may still read positions (it signals ahead of its last 32 keys): the producer is up to
  // KST + 3 tiles ahead of a softmax.  Which of the tile's pages exist, and the
  // positions of its keys behind its first place, where they are not their places (behind the first new token's where positions are
  // given: they may lie anywhere, and what counts between new tokens is small beside that)
  volatile uint32_t* s_pages = reinterpret_cast<volatile uint32_t*>(smem + Cfg::OFF_BAR + 208);
  float* s_pos = reinterpret_cast<float*>(smem + Cfg::OFF_POS);
  // per segment, eight deep: its number + 1 if it has values that were taken out; the segment
  volatile int* s_taken = reinterpret_cast<volatile int*>(smem + Cfg::OFF_BAR + 240);
  volatile TileSeg* s_seg = reinterpret_cast<volatile TileSeg*>(smem + Cfg::OFF_SEG);

  const fb_paged_params& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 8) {
    if (lane == 0) {
      st_shared_flag(abort_flag, 0u);
      mbar_init(q_ready, 1);
      mbar_init(q_free, 1);
      mbar_init(o_free, 8);  // every softmax warp has read the accumulator of the segment
      for (int i = 0; i < 2; ++i) {
        mbar_init(s_full + 8 * i, 1);
        mbar_init(p_ready + 8 * i, 4);  // the stream's warps
        mbar_init(s_read + 8 * i, 4);   // the logits of the tile are in registers
      }
      for (int i = 0; i < 4; ++i) {
        mbar_init(k_full + 8 * i, 1);
        mbar_init(k_free + 8 * i, 1);
        mbar_init(v_full + 8 * i, 1);
        mbar_init(v_free + 8 * i, 1);
        mbar_init(v_ok + 8 * i, 1);
        mbar_init(pv_done + 8 * i, 1);
      }
      for (int i = 0; i < 8; ++i) {
        mbar_init(seg_full + 8 * i, 1);
        s_taken[i] = 0;
      }
      mbar_fence_init();
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
  } else if (warp == 9) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  grid_dep_wait();
  if (threadIdx.x == 0) a.desc[2 * blockIdx.x].x = -1;
  PagedWalk<128, 128, kTileThreads> walk;
  walk.start(a, p.Hk, blockIdx.x, gridDim.x);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  // Product number c of stream x: two barriers in turn, so that a wait cannot take the product before it for its own.
  auto pv_bar = [&](int x, int c) { return pv_done + 16 * x + 8 * (c & 1); };
  // Segment n, once it is known; none if there is none.
  auto segment = [&](int n) -> const volatile TileSeg* {
    const volatile TileSeg* sg = s_seg + (n & 7);
    return mbar_wait(seg_full + 8 * (n & 7), (n >> 3) & 1, abort_flag) && sg->n_kv > 0 ? sg : nullptr;
  };

  if (warp >= 8) {
    setmaxnreg_dec<88>();
    if (warp == 8) {
      // ------------------------------------------------------------------ schedule, copies of K
      const int rows = min(p.page_size, 128), pieces = 128 / rows;  // copies of a tile
      auto wait_all = [&](uint32_t bar, int parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)); };  // (the warp leaves together)
      auto publish = [&](const Segment& sg, bool there, int n) {
        if (lane == 0) {
          volatile TileSeg* d = s_seg + (n & 7);
          d->n_kv = there ? sg.t1 - sg.t0 : 0;
          d->t0 = sg.t0;
          d->t1 = sg.t1;
          d->tiles = sg.tiles;
          d->b = sg.b;
          d->rt = sg.rt;
          d->hg = sg.hg;
          d->last_cta = sg.last_cta;
          d->first = sg.r.first;
          d->tokens = sg.r.tokens;
          d->len = sg.r.len;
          d->keys = sg.r.keys;
          mbar_arrive(seg_full + 8 * (n & 7));
        }
      };
      auto load_q = [&](const Segment& sg, int n) {
        if (n > 0 && !wait_all(q_free, (n - 1) & 1)) return false;
        const int live_rows = min(sg.r.tokens * a.G - sg.rt * 128, 128), col = (lane % CH) * 8;
#pragma unroll 4
        for (int r = lane / CH; r < 128; r += 32 / CH) {
          const bool live = r < live_rows && col < p.D;
          const int gr = sg.rt * 128 + r, tok = live ? a.group_div.quot32(gr) : 0, head = sg.hg * a.G + (live ? gr - tok * a.G : 0);
          const T* src = reinterpret_cast<const T*>(p.q) + (int64_t)(sg.r.first + tok) * p.q_stride[0] + head * p.q_stride[1] + col;
          cp_async16_zfill(sQ + tile_chunk_offset<TD>(r, col), live ? src : reinterpret_cast<const T*>(p.q), live);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_ready);
        return true;
      };
      auto produce = [&] {
        Segment seg, nxt = {};
        bool more = walk.next(a, nxt);
        publish(nxt, more, 0);
        for (int t = 0, n = 0; more; ++n) {
          seg = nxt;
          more = walk.next(a, nxt);
          publish(nxt, more, n + 1);
          const int32_t* table = p.block_table + (int64_t)min(seg.b, p.B - 1) * p.table_stride;
          for (int j = 0; j < seg.t1 - seg.t0; ++j, ++t) {
            const int st = t % KST, k0 = (seg.t1 - 1 - j) * 128, key = k0 + lane * rows;
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
            if (t >= KST && !wait_all(k_free + 8 * st, (t / KST - 1) & 1)) return;
            if (SLOPES && k0 + 128 > seg.r.len) {
              const int at0 = p.positions ? p.positions[seg.r.first] : k0;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int k = k0 + e * 32 + lane;
                s_pos[(t & 7) * 128 + e * 32 + lane] =
                    (float)((p.positions && k >= seg.r.len && k < seg.r.keys ? p.positions[seg.r.first + k - seg.r.len] : k) - at0);
              }
            }
            if (lane == 0) s_pages[t & 7] = there;
            __syncwarp();
            if (lane == 0) mbar_expect_tx(k_full + 8 * st, Cfg::Q_BYTES);
            __syncwarp();
            if (lane < pieces) {
#pragma unroll
              for (int c = 0; c < NB; ++c)
                tma_load_4d(sK + st * Cfg::Q_BYTES + c * 128 * 128 + lane * rows * 128, &tmK, k_full + 8 * st, c * 64, place, seg.hg, page);
            }
            if (j == 0 && !load_q(seg, n)) return;  // (behind the first copy of K, which need not wait for the last segment's end)
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
        for (const volatile TileSeg* sg; (sg = segment(n)); ++n) {
          const int n_kv = sg->n_kv;
          mbar_wait(q_ready, n & 1, abort_flag);
          tc_fence_after_sync();
          for (int j = 0; j < n_kv; ++j, ++t) {
            const int x = j & 1, c = x ? c1++ : c0++, st = t % KST;
            if (c > 0) mbar_wait(s_read + 8 * x, (c - 1) & 1, abort_flag);
            mbar_wait(k_full + 8 * st, (t / KST) & 1, abort_flag);
            tc_fence_after_sync();
#pragma unroll
            for (int s = 0; s < TD / 16; ++s)
              umma_ss(tmem + Cfg::T_S + 128 * x, desc_at(dQ, kmajor_step<TD>(s)), desc_at(dK, st * Cfg::Q_BYTES + kmajor_step<TD>(s)), idS, s > 0);
            umma_commit(s_full + 8 * x);
            umma_commit(k_free + 8 * st);
          }
          umma_commit(q_free);  // the segment's queries are no longer read
        }
      }
    } else if (warp == 10) {
      // ------------------------------------------------------------------ O += P.V
      if (elect_one()) {
        constexpr uint32_t idO = instr_desc(kBf16, false, true, 128, TD);
        const DescBase dV = mnmajor_base<TD>(sV);
        int t = 0, n = 0, c0 = 0, c1 = 0;
        for (const volatile TileSeg* sg; (sg = segment(n)); ++n) {
          const int n_kv = sg->n_kv;
          for (int j = 0; j < n_kv; ++j, ++t) {
            const int x = j & 1, c = x ? c1++ : c0++, st = t % VST;
            mbar_wait(v_ok + 8 * st, (t / VST) & 1, abort_flag);
            mbar_wait(p_ready + 8 * x, c & 1, abort_flag);
            if (j == 0 && n > 0) mbar_wait(o_free, (n - 1) & 1, abort_flag);  // the accumulator of the last segment has been read
            tc_fence_after_sync();
#pragma unroll
            for (int s = 0; s < 8; ++s)
              umma_ts(tmem + Cfg::T_O, tmem + Cfg::T_P + 64 * x + s * 8, desc_at(dV, st * Cfg::Q_BYTES + mnmajor_step<TD>(s)), idO, (j > 0 || s > 0) ? 1u : 0u);
            umma_commit(pv_bar(x, c));
            umma_commit(v_free + 8 * st);
          }
        }
      }
    } else {
      // ------------------------------------------------------------------ copies of V, and V behind them
      auto segment_warp = [&](int n) {  // (the warp leaves together)
        const volatile TileSeg* sg = segment(n);
        return __all_sync(0xffffffffu, sg != nullptr) ? sg : nullptr;
      };
      // V of tile number t (of the CTA), the j-th of a segment
      const int rows = min(p.page_size, 128), pieces = 128 / rows;
      auto load_v = [&](const volatile TileSeg* sg, int j, int t) {
        const int st = t % VST, key = (sg->t1 - 1 - j) * 128 + lane * rows;
        int page = (int)p.num_pages, place = 0;  // behind the cache: the copy fills in zeros
        if (lane < pieces && key < sg->keys) {
          const int col = a.page_div.quot32(key), pg = p.block_table[(int64_t)min(sg->b, p.B - 1) * p.table_stride + col];
          if (pg >= 0 && pg < p.num_pages) {
            page = pg;
            place = key - col * p.page_size;
          }
        }
        if (t >= VST && !__all_sync(0xffffffffu, mbar_wait(v_free + 8 * st, (t / VST - 1) & 1, abort_flag))) return;
        if (lane == 0) mbar_expect_tx(v_full + 8 * st, Cfg::Q_BYTES);
        __syncwarp();
        if (lane < pieces) {
#pragma unroll
          for (int c = 0; c < NB; ++c)
            tma_load_4d(sV + st * Cfg::Q_BYTES + c * 128 * 128 + lane * rows * 128, &tmV, v_full + 8 * st, c * 64, place, sg->hg, page);
        }
      };
      int t = 0, n = 0;
      const volatile TileSeg *sg = segment_warp(0), *nx = nullptr;
      // The copies run VST - 1 tiles ahead, across segments: tile lj of segment ls is copied next.
      const volatile TileSeg* ls = sg;
      int lj = 0, lt = 0, ln = 0;
      auto load_next = [&] {
        if (!ls) return;
        load_v(ls, lj, lt++);
        if (++lj == ls->n_kv) {
          ls = segment_warp(++ln);  // (known before the first copy of K of the one before)
          lj = 0;
        }
      };
      for (int i = 0; i < VST - 1; ++i) load_next();
      for (; sg; sg = nx, ++n) {
        const int n_kv = sg->n_kv, t1 = sg->t1, len = sg->len, keys = sg->keys;
        for (int j = 0; j < n_kv; ++j, ++t) {
          const int st = t % VST, k0 = (t1 - 1 - j) * 128;
          mbar_wait(v_full + 8 * st, (t / VST) & 1, abort_flag);
          const int r0 = max(len - k0, 0), live = keys - k0;  // first row that not all see; rows that hold keys
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
          load_next();  // (behind the product of tile t - 1; ahead of the arrival it would hold up the next product)
        }
        nx = segment_warp(n + 1);
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax + epilogue
    setmaxnreg_inc<208>();
    const int x = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + Cfg::T_S + 128 * x + lane_off, tP = tmem + Cfg::T_P + 64 * x + lane_off, tO = tmem + Cfg::T_O + lane_off;
    const uint32_t m_own = sbase + Cfg::OFF_M + (x * 128 + row) * 4, m_other = sbase + Cfg::OFF_M + ((x ^ 1) * 128 + row) * 4;
    // Maxima are kept in quarters of a log2 unit, in which no finite logit overflows.
    const float sl2 = a.scale_log2, sl2q = 0.25f * sl2;
    const uint64_t sl2p = f2(sl2, sl2);
    int c = 0, co = 0, n = 0, t0 = 0;  // key tiles of this stream and of the other, segments and key tiles so far
    uint32_t s[4][32];                 // the thread's row of the logit tile
    auto segment_both = [&](int n) {  // (the warpgroups leave together: behind an expired wait, too)
      const volatile TileSeg* sg = segment(n);
      uint32_t all;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\t"
          "setp.ne.b32 p, %1, 0;\n\t"
          "barrier.cta.red.and.pred q, 1, 256, p;\n\t"
          "selp.b32 %0, 1, 0, q;\n\t}"
          : "=r"(all)
          : "r"(sg ? 1u : 0u)
          : "memory");
      return all ? sg : nullptr;
    };
    for (const volatile TileSeg* sg; (sg = segment_both(n)); ++n) {
      const int n_kv = sg->n_kv, t1 = sg->t1, len = sg->len, keys = sg->keys;
      // the row's token (of the request, -1: padding) and query head
      const int gr = sg->rt * 128 + row, tk = gr < sg->tokens * a.G ? a.group_div.quot32(gr) : -1, gn = sg->first + max(tk, 0);
      const int hd = sg->hg * a.G + (tk >= 0 ? gr - tk * a.G : 0);
      float m_used = -INFINITY, l = 0.f;  // reference maximum (logit * log2 e / 4); row sum of this stream's tiles, relative to it
      const int c0 = c, co0 = co;
      // the bias in units of q.k, so that a logit costs one product more: s + slope_r (pos - k0), times sl2, plus 4 baseq; in a tile of new
      // tokens s + slope_r (pos - mine)
      const float slope2 = SLOPES && tk >= 0 ? p.slopes[hd] * kLog2eP : 0.f, slope_r = slope2 / sl2;
      const int my_pos = SLOPES && tk >= 0 ? (p.positions ? p.positions[gn] : len + tk) : 0;
      const int own_pos = SLOPES && p.positions && tk >= 0 ? my_pos - p.positions[sg->first] : 0;
      for (int j = x; j < n_kv; j += 2, ++c) {
        const int k0 = (t1 - 1 - j) * 128;
        const bool own = k0 + 128 > len;  // the tile holds new tokens' keys, or places behind them
        uint32_t bits[4] = {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu};
        if (own) {  // the row's view of them, ahead of the wait
#pragma unroll
          for (int ch = 0; ch < 4; ++ch) {
            const int j0 = k0 + ch * 32, left = keys - j0;
            bits[ch] = left >= 32 ? 0xffffffffu : left > 0 ? (1u << left) - 1u : 0u;
            if (tk >= 0 && j0 + 32 > len) bits[ch] &= seen_bits(p, gn, tk, j0 - len);
          }
        }
        mbar_wait(s_full + 8 * x, c & 1, abort_flag);
        tc_fence_after_sync();
        const uint32_t there = s_pages[(t0 + j) & 7];
        const bool dead = there != 0xffffffffu || own;
        const float* pos = s_pos + ((t0 + j) & 7) * 128;
        if (there != 0xffffffffu) {  // (rare) pages that do not exist
          const int rows = min(p.page_size, 128);
#pragma unroll
          for (int ch = 0; ch < 4; ++ch)
#pragma unroll 1
            for (int i = 0; i < 32; ++i)
              if (!(there >> ((ch * 32 + i) / rows) & 1)) bits[ch] &= ~(1u << i);
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        // A tile of new tokens takes every difference by itself (whole numbers, exact to 2^24), since a row may see the near keys alone
        // that a shared part of the bias would cancel with.
        float baseq = SLOPES && !own ? 0.25f * slope2 * (float)(k0 - my_pos) : 0.f;
        const float mine = SLOPES && own ? (float)(p.positions ? own_pos : my_pos - k0) : 0.f;
        auto complete = [&](int ch) {
          if (dead) {
            if (SLOPES) {
              const uint64_t less = f2(-mine, -mine), slope_p = f2(slope_r, slope_r);
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                const float4 f = own ? *reinterpret_cast<const float4*>(pos + ch * 32 + i)
                                     : make_float4((float)(ch * 32 + i), (float)(ch * 32 + i + 1), (float)(ch * 32 + i + 2), (float)(ch * 32 + i + 3));
                auto add = [&](int e, float p0, float p1) {
                  float v0, v1;
                  f2_unpack(f2_fma(slope_p, f2_add(f2(p0, p1), less), f2(__uint_as_float(s[ch][e]), __uint_as_float(s[ch][e + 1]))), v0, v1);
                  s[ch][e] = __float_as_uint(v0);
                  s[ch][e + 1] = __float_as_uint(v1);
                };
                add(i, f.x, f.y);
                add(i + 2, f.z, f.w);
              }
            }
            if (__any_sync(0xffffffffu, bits[ch] != 0xffffffffu)) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!(bits[ch] >> i & 1)) s[ch][i] = __float_as_uint(-INFINITY);
            }
#pragma unroll
            for (int i = 0; i < 32; i += 2) mx4[(i >> 1) & 3] = fmax3(mx4[(i >> 1) & 3], __uint_as_float(s[ch][i]), __uint_as_float(s[ch][i + 1]));
            __syncwarp();  // (the loads from tensor memory want the warp together)
            return;
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float v0 = __uint_as_float(s[ch][i]), v1 = __uint_as_float(s[ch][i + 1]);
            if (SLOPES) {
              v0 = fmaf((float)(ch * 32 + i), slope_r, v0);
              v1 = fmaf((float)(ch * 32 + i + 1), slope_r, v1);
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
        const float mx = fmaf(fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])), sl2q, baseq);  // sl2 > 0
        // Far from zero the rounding of the maximum, a 2^-24 of it, would be a factor that P cannot hold: there the logits are rounded
        // as their maximum was, and it is subtracted, before they are scaled.
        const bool far = mx > -INFINITY && fmaxf(fabsf(mx), fabsf(baseq)) >= 262144.f;
        auto subtract_far = [&] {
          if (!__any_sync(0xffffffffu, far)) return;
          const float msub = m_used == -INFINITY ? 0.f : m_used, back = 4.f / sl2;
          const uint64_t q2 = f2(sl2q, sl2q), b2 = f2(baseq, baseq), m2 = f2(-msub, -msub);
#pragma unroll
          for (int ch = 0; ch < 4; ++ch)
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              float v0, v1;
              f2_unpack(f2_add(f2_fma(f2(__uint_as_float(s[ch][i]), __uint_as_float(s[ch][i + 1])), q2, b2), m2), v0, v1);
              s[ch][i] = __float_as_uint(v0 * back);
              s[ch][i + 1] = __float_as_uint(v1 * back);
            }
          baseq = msub;
        };
        // ---- the reference maximum, from tile to tile: it moves only when the maximum has grown by more than 2^8 (exact: the row
        // sums carry the same reference)
        const float m_last = m_used;
        if (j > 0) {
          asm volatile("bar.sync %0, 256;" ::"r"(2 + (x ^ 1)) : "memory");
          m_used = __uint_as_float(ld_shared_flag(m_other));
          const float m_new = fmaxf(m_used, mx);
          if (__any_sync(0xffffffffu, m_new - m_used > 2.f || far)) {  // (from -inf: the difference is +inf, or NaN where both are)
            // O is stable behind the product of tile j - 1, which is the other stream's.  (The one two before it on that barrier,
            // tile j - 5, has completed: the other stream has waited for it ahead of its P of tile j - 3.)
            const int cp = co0 + ((j - 1) >> 1);
            mbar_wait(pv_bar(x ^ 1, cp), (cp >> 1) & 1, abort_flag);
            tc_fence_after_sync();
            const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(4.f * (m_used - m_new));
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
            subtract_far();
          }
        } else {
          m_used = mx;
          subtract_far();
        }
        if (j + 1 < n_kv) {
          st_shared_f32(m_own, m_used);
          asm volatile("bar.arrive %0, 256;" ::"r"(2 + x) : "memory");
        }
        if (c > 0) mbar_wait(pv_bar(x, c - 1), ((c - 1) >> 1) & 1, abort_flag);  // P has been read
        // ---- p = exp2(logit2 - m), row sum, P -> tensor memory (the A operand of O += P.V), rounded to the 16 bits of V
        const float msub = m_used == -INFINITY ? 0.f : m_used;
        l *= fast_exp2(4.f * (m_last - msub));  // (0 at the stream's first tile, where l is 0)
        uint64_t l2a = f2(0.f, 0.f), l2b = f2(0.f, 0.f);
        const float off = fminf(4.f * (baseq - msub), FLT_MAX) + kTileLift<T>;  // (finite: there may be no key, all -inf)
        const uint64_t nm = f2(off, off);
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {
          uint32_t pw[16];  // 32 keys = 16 packed words
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const uint64_t v = f2(__uint_as_float(s[ch][i]), __uint_as_float(s[ch][i + 1]));
            float a0, a1;
            f2_unpack(f2_fma(v, sl2p, nm), a0, a1);
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
      // ---- epilogue, this warpgroup's half of the columns.  The stream of the last tile knows its product to have completed (its
      // commit covers the ones before it, which the same thread issued); the other learns it from the warpgroups' barrier.
      c = c0 + ((n_kv + 1 - x) >> 1);
      co = co0 + ((n_kv + x) >> 1);
      const int xl = (n_kv - 1) & 1;  // stream of the last tile
      if (xl == x) mbar_wait(pv_bar(x, c - 1), ((c - 1) >> 1) & 1, abort_flag);
      float2* ml = reinterpret_cast<float2*>(smem + Cfg::OFF_ML) + (n & 1) * 256;
      ml[x * 128 + row] = make_float2(m_used, l);
      asm volatile("bar.sync 1, 256;" ::: "memory");  // both warpgroups
      tc_fence_after_sync();
      const float2 other = ml[(x ^ 1) * 128 + row];
      const float m = fmaxf(m_used, other.x), ms = m == -INFINITY ? 0.f : m;  // the last reference is the largest
      const float ls = l * fast_exp2(4.f * (m_used - ms)) + other.y * fast_exp2(4.f * (other.x - ms));
      const bool begins = sg->t0 == 0, whole = begins && t1 == sg->tiles, taken = s_taken[n & 7] == n + 1;
      const float inv = !whole ? 1.f : ls > 0.f ? 1.f / ls : ls == 0.f ? 0.f : ls;
      const int64_t slot = (int64_t)blockIdx.x * 2 + (begins ? 1 : 0);  // slot 1: the CTA in which the item begins
#pragma unroll 1
      for (int ch = 0; ch < TD / 64; ++ch) {
        const int col0 = x * (TD / 2) + ch * 32;
        uint32_t r[32];
        tmem_ld32(tO + col0, r);
        tmem_wait_ld(r);
        if (tk >= 0) {
          if (taken) {  // (rare) values that are not finite, for the rows that see their keys
            const int32_t* table = p.block_table + (int64_t)sg->b * p.table_stride;
            for (int key = max(len, sg->t0 * 128); key < min(keys, t1 * 128); ++key) {
              const int col = a.page_div.quot32(key), pg = table[col];
              if (pg < 0 || pg >= p.num_pages || !tree_sees(p, gn, tk, key - len)) continue;
              const T* v = reinterpret_cast<const T*>(p.value_cache) + pg * p.value_cache_stride[0] + (key - col * p.page_size) * p.value_cache_stride[1] +
                           sg->hg * p.value_cache_stride[2] + col0;
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
            float4* dst = reinterpret_cast<float4*>(a.part) + (slot * (TD / 4) + col0 / 4) * 128 + row;  // (columns / 4, rows, 4)
#pragma unroll
            for (int g = 0; g < 8; ++g)
              dst[g * 128] = make_float4(__uint_as_float(r[4 * g]), __uint_as_float(r[4 * g + 1]), __uint_as_float(r[4 * g + 2]), __uint_as_float(r[4 * g + 3]));
          }
        }
        __syncwarp();
      }
      if (x == 0 && tk >= 0) {
        if (!whole) a.ml[slot * 128 + row] = make_float2(m, ls);
        else if (p.lse) p.lse[(int64_t)gn * p.Hq + hd] = ls > 0.f ? fmaf(4.f * kLn2P, m, (fast_log2(ls) - kTileLift<T>) * kLn2P) : ls == 0.f ? -INFINITY : ls;
      }
      if (!whole && begins && threadIdx.x == 0) {
        a.desc[2 * blockIdx.x] = make_int4(sg->rt, sg->hg, sg->last_cta, 0);
        a.desc[2 * blockIdx.x + 1] = make_int4(sg->first, sg->tokens * a.G, 0, 0);
      }
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

// Joins the parts of the item that begins in CTA blockIdx.x, in the order of the CTAs: thread = row.  32 columns per block, or
// where few items are spread over many CTAs (SHARE = 4) 8 columns, and a quarter of the parts per thread (64 tokens over 11772
// keys, two heads, 74 parts each: 72 us a call with one thread per row, 27 so).
template <typename T, int TD, int SHARE>
__global__ void __launch_bounds__(128 * SHARE) paged_join_tile_kernel(const __grid_constant__ PagedArgs a) {
  constexpr int G = SHARE > 1 ? 2 : 8, U = SHARE > 1 ? 4 : 2;  // float4 of a thread; parts in flight
  __shared__ float4 s_acc[SHARE > 1 ? SHARE : 1][SHARE > 1 ? G : 1][SHARE > 1 ? 128 : 1];
  __shared__ float2 s_ml[SHARE > 1 ? SHARE : 1][SHARE > 1 ? 128 : 1];
  grid_dep_wait();
  const int4 d = a.desc[2 * blockIdx.x], e = a.desc[2 * blockIdx.x + 1];
  if (d.x < 0) return;
  const fb_paged_params& p = a.p;
  const int row = threadIdx.x & 127, share = threadIdx.x >> 7, gr = d.x * 128 + row, col0 = blockIdx.y * 4 * G, all = d.z - (int)blockIdx.x + 1;
  const int parts = (all - share + SHARE - 1) / SHARE;  // share, share + SHARE, ...
  auto slot_of = [&](int i) { return (int64_t)(blockIdx.x + i * SHARE + share) * 2 + (i * SHARE + share == 0 ? 1 : 0); };
  const bool live = gr < e.y;
  float m = -INFINITY, l = 0.f;
  float4 acc[G] = {};
  if (live && parts > 0) {
#pragma unroll 8
    for (int i = 0; i < parts; ++i) m = fmaxf(m, a.ml[slot_of(i) * 128 + row].x);
    const float ms = fmaxf(m, -FLT_MAX);
#pragma unroll U
    for (int i = 0; i < parts; ++i) {
      const float2 s = a.ml[slot_of(i) * 128 + row];
      const float f = fast_exp2(4.f * (s.x - ms));
      l = fmaf(s.y, f, l);
      const float4* src = reinterpret_cast<const float4*>(a.part) + (slot_of(i) * (TD / 4) + col0 / 4) * 128 + row;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float4 v = src[g * 128];
        acc[g] = make_float4(fmaf(v.x, f, acc[g].x), fmaf(v.y, f, acc[g].y), fmaf(v.z, f, acc[g].z), fmaf(v.w, f, acc[g].w));
      }
    }
  }
  if (SHARE > 1) {
#pragma unroll
    for (int g = 0; g < G; ++g) s_acc[share][g][row] = acc[g];
    s_ml[share][row] = make_float2(m, l);
    __syncthreads();
    if (share > 0) return;
    for (int x = 1; x < SHARE; ++x) m = fmaxf(m, s_ml[x][row].x);
    const float ms = fmaxf(m, -FLT_MAX);
    l = 0.f;
#pragma unroll
    for (int g = 0; g < G; ++g) acc[g] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int x = 0; x < SHARE; ++x) {
      const float2 s = s_ml[x][row];
      const float f = fast_exp2(4.f * (s.x - ms));
      l = fmaf(s.y, f, l);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float4 v = s_acc[x][g][row];
        acc[g] = make_float4(fmaf(v.x, f, acc[g].x), fmaf(v.y, f, acc[g].y), fmaf(v.z, f, acc[g].z), fmaf(v.w, f, acc[g].w));
      }
    }
  }
  if (!live) return;
  const int t = a.group_div.quot32(gr), h = d.y * a.G + gr - t * a.G, n = e.x + t;
  const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
  T* dst = reinterpret_cast<T*>(p.o) + (int64_t)n * p.o_stride[0] + h * p.o_stride[1] + col0;
  auto p2 = [&](float x, float y) { return l == 0.f ? 0u : Pack2<T>::pack(x * inv, y * inv); };
#pragma unroll
  for (int g = 0; g < G / 2; ++g)
    if (col0 + g * 8 < p.D)
      *reinterpret_cast<uint4*>(dst + g * 8) = make_uint4(p2(acc[2 * g].x, acc[2 * g].y), p2(acc[2 * g].z, acc[2 * g].w), p2(acc[2 * g + 1].x, acc[2 * g + 1].y),
                                                          p2(acc[2 * g + 1].z, acc[2 * g + 1].w));
  if (p.lse && blockIdx.y == 0) p.lse[(int64_t)n * p.Hq + h] = l > 0.f ? fmaf(4.f * kLn2P, m, (fast_log2(l) - kTileLift<T>) * kLn2P) : l == 0.f ? -INFINITY : l;
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
  if (const int rc = launch_pdl(kern, plan.ctas, kTileThreads, TileCfg<TD>::SMEM, st, tk, tv, a)) return rc;
  return plan.many_parts ? launch_pdl_2d(paged_join_tile_kernel<T, TD, 4>, dim3(plan.ctas, TD / 8), 512, st, a)
                         : launch_pdl_2d(paged_join_tile_kernel<T, TD, 1>, dim3(plan.ctas, TD / 32), 128, st, a);
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
  return p.dtype == FB_DTYPE_F16 ? go(__half()) : go(__nv_bfloat16());
}

}  // namespace fb
