// Attention over pages with few rows per key head (up to 32): decoding, and small trees or runs of drafted tokens.
//
// Bound by reading K and V once.  A warp works alone: it owns a head of the CTA's group and every WK-th tile of 16 keys, copies
// them into a ring of its own in shared memory (cp.async, so that what is in flight is bounded by shared memory and not by
// registers: 2 CTAs x 96 KB per SM), and keeps 16 or 32 query rows, the row maxima and sums and the output in registers.  The
// products are mma.sync m16n8k16: a tile of 16 keys and 16 rows is one fragment wide, S stays in the registers that P is fed
// from, and the tensor pipe is far from being the bound; a tcgen05 tile would spend 112 of its 128 rows on padding.  No
// barrier is needed between warps while a segment lasts; where a group has fewer heads than the CTA has warps, the warps of a
// head join their sums through shared memory at the segment's end.
#pragma once

#include <mutex>

#include "fb_paged.cuh"

namespace fb {

constexpr int kSplitWarps = 4;
constexpr int kSplitThreads = 32 * kSplitWarps;
constexpr int kSplitKT = 64;  // keys of a scheduled tile: four sub-tiles of 16

template <int TD>
struct SplitCfg {
  static constexpr int ROW = TD * 2;                                     // bytes of a key's row
  static constexpr int ST = TD == 128 ? 3 : 4;                           // ring stages
  static constexpr int HALF = 16 * ROW, STAGE = 2 * HALF, RING = ST * STAGE;  // K, then V
  static constexpr int SMEM = kSplitWarps * RING + kSplitWarps * ST * 4;
  static constexpr int CH = TD / 8;  // 16-byte chunks of a row
  // chunk c of key r: XOR-swizzled so that eight rows of one column of chunks fall on different banks
  __device__ static __forceinline__ uint32_t at(int r, int c) {
    return r * ROW + ((TD == 32 ? c ^ ((r >> 1) & 3) : c ^ (r & 7)) << 4);
  }
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// whether a 16-bit pair holds an infinity or a NaN
template <typename T>
__device__ __forceinline__ bool pair_not_finite(uint32_t w) {
  constexpr uint32_t E = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  return (w & E) == E || ((w >> 16) & E) == E;
}

enum { PAGED_PLAIN = 0, PAGED_SLOPES = 1, PAGED_FACTORS = 2 };

template <typename T, int TD, int MT, int BIAS>
__global__ void __launch_bounds__(kSplitThreads, split_ctas(TD, MT)) paged_split_kernel(const __grid_constant__ PagedArgs a, const int WH) {
  using Cfg = SplitCfg<TD>;
  constexpr int NM = MT / 16, KS = TD / 16, NT = TD / 8, ST = Cfg::ST;
  extern __shared__ __align__(1024) uint8_t smem[];
  const fb_paged_params& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, WK = kSplitWarps / WH, wh = warp / WK, wk = warp % WK;
  const uint32_t ring = smem_u32(smem) + warp * Cfg::RING;
  uint32_t* ring_ok = reinterpret_cast<uint32_t*>(smem + kSplitWarps * Cfg::RING) + warp * ST;  // keys of a stage that exist, as bits
  const int qr = lane >> 2, qc = 2 * (lane & 3);  // a fragment's row (and row + 8) and first column of this lane
  grid_dep_wait();
  if (threadIdx.x == 0) a.desc[2 * blockIdx.x].x = -1;
  PagedWalk<kSplitKT, MT, kSplitThreads> walk;
  walk.start(a, p.Hk / WH);

  Segment seg;
  while (walk.next(a, seg)) {
    const Request& rq = seg.r;
    const int hk = seg.hg * WH + wh, rows = rq.tokens * a.G - seg.rt * MT;  // rows of the request from this tile on
    const T* kbase = reinterpret_cast<const T*>(p.key_cache) + hk * p.key_cache_stride[2];
    const T* vbase = reinterpret_cast<const T*>(p.value_cache) + hk * p.value_cache_stride[2];
    const T* bbase = reinterpret_cast<const T*>(p.bias_cache) + (p.bias_heads > 1 ? hk * p.bias_cache_stride[2] : 0);
    const int32_t* table = p.block_table + (int64_t)min(seg.b, p.B - 1) * p.table_stride;
    const int tile_end = min(seg.t1 * 4, (rq.keys + 15) >> 4);

    // ---- copies: the pages of a tile's keys are looked up one tile ahead of their use (lane & 15 = key).  Where pages are whole
    // tiles one page serves all lanes, and a copy's address is one addition: half of the instructions that a tile of 64 columns
    // takes would otherwise go into addresses.
    const int c = lane % Cfg::CH, kr = lane / Cfg::CH;  // this lane's chunk, and its key in the first of a tile's copies
    const bool in = c * 8 < p.D;
    const int64_t kstep = (32 / Cfg::CH) * p.key_cache_stride[1], vstep = (32 / Cfg::CH) * p.value_cache_stride[1];
    const T *klane = kbase + kr * p.key_cache_stride[1] + (in ? c * 8 : 0), *vlane = vbase + kr * p.value_cache_stride[1] + (in ? c * 8 : 0);
    const uint32_t dst0 = ring + Cfg::at(kr, c);
    int page_next = -1, place_next = 0;
    auto look_up = [&](int tile) {
      const int j = tile * 16 + (a.whole_tiles ? 0 : lane & 15);
      page_next = -1;
      if (tile < tile_end && j < rq.keys) {
        const int col = a.page_div.quot32(j);
        place_next = j - col * p.page_size;
        page_next = table[col];
      }
    };
    auto fetch = [&](int tile, int stage) {
      if (tile < tile_end) {
        const int page = page_next, place = place_next;
        const uint32_t dst = ring + stage * Cfg::STAGE;
        if (a.whole_tiles && tile * 16 + 16 <= rq.keys && (uint32_t)page < (uint32_t)min(p.num_pages, (int64_t)0x7fffffff)) {
          look_up(tile + WK);
          if (lane == 0) ring_ok[stage] = 0xffffu;
          const T* k = klane + page * p.key_cache_stride[0] + place * p.key_cache_stride[1];
          const T* v = vlane + page * p.value_cache_stride[0] + place * p.value_cache_stride[1];
#pragma unroll
          for (int i = 0; i < TD / 16; ++i) {
            const uint32_t at = dst + Cfg::at(kr + i * (32 / Cfg::CH), c);
            cp_async16_zfill(at, k, in);
            cp_async16_zfill(at + Cfg::HALF, v, in);
            k += kstep;
            v += vstep;
          }
        } else {
          const int off = a.whole_tiles ? lane & 15 : 0;
          const bool there = tile * 16 + (lane & 15) < rq.keys, ok = there && page >= 0 && page < p.num_pages;
          if (there && !ok) paged_bad_index(p);
          const int64_t ko = ok ? page * p.key_cache_stride[0] + (place + off) * p.key_cache_stride[1] : 0;
          const int64_t vo = ok ? page * p.value_cache_stride[0] + (place + off) * p.value_cache_stride[1] : 0;
          const uint32_t okm = __ballot_sync(0xffffffffu, ok) & 0xffffu;
          if (lane == 0) ring_ok[stage] = okm;
          look_up(tile + WK);
#pragma unroll
          for (int i = 0; i < TD / 16; ++i) {
            const int key = kr + i * (32 / Cfg::CH);
            const int64_t k = __shfl_sync(0xffffffffu, ko, key), v = __shfl_sync(0xffffffffu, vo, key);
            const bool live = in && ((okm >> key) & 1);
            cp_async16_zfill(dst + Cfg::at(key, c), live ? kbase + k + c * 8 : kbase, live);
            cp_async16_zfill(dst + Cfg::HALF + Cfg::at(key, c), live ? vbase + v + c * 8 : vbase, live);
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // Factors of a tile's keys in the layout of the product's second operand (two columns a word), one tile ahead; their pages
    // two ahead.
    uint32_t kb[2][2] = {};
    int fpage[2] = {-1, -1}, fplace[2] = {};
    auto factor_pages = [&](int tile) {
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const int j = tile * 16 + nt * 8 + qr;
        fpage[nt] = -1;
        if (tile < tile_end && j < rq.keys) {
          const int col = a.page_div.quot32(j);
          fplace[nt] = j - col * p.page_size;
          fpage[nt] = table[col];
        }
      }
    };
    auto load_factors = [&](int r0, uint32_t (&f)[2][2]) {
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const bool ok = fpage[nt] >= 0 && fpage[nt] < p.num_pages;
        const uint16_t* src = reinterpret_cast<const uint16_t*>(bbase + (ok ? fpage[nt] * p.bias_cache_stride[0] + fplace[nt] * p.bias_cache_stride[1] : 0));
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int col = r0 + qc + x * 8;
          f[nt][x] = 0u;
          if (x == 1 && r0 + 8 >= p.R) continue;
          if (a.factor_words) {
            if (ok && col < p.R) f[nt][x] = *reinterpret_cast<const uint32_t*>(src + col);
          } else {
            if (ok && col < p.R) f[nt][x] = src[col];
            if (ok && col + 1 < p.R) f[nt][x] |= (uint32_t)src[col + 1] << 16;
          }
        }
      }
    };

    int fetched = seg.t0 * 4 + wk;
    look_up(fetched);
    if (BIAS == PAGED_FACTORS) factor_pages(fetched);

    // ---- query rows, as fragments of the products' first operand
    uint32_t q[NM][KS][4], qb[NM][4] = {};
    int row_tok[NM][2];               // token of the request, -1 for rows of padding
    float slope2[NM][2] = {}, m[NM][2], l[NM][2];
    int my_pos[NM][2] = {};
    const T* qbrow[NM][2] = {};
#pragma unroll
    for (int im = 0; im < NM; ++im)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = im * 16 + e * 8 + qr;
        const bool live = r < rows;
        const int gr = seg.rt * MT + r, t = live ? a.group_div.quot32(gr) : 0, h = hk * a.G + (live ? gr - t * a.G : 0), n = rq.first + t;
        row_tok[im][e] = live ? t : -1;
        m[im][e] = -INFINITY;
        l[im][e] = 0.f;
        const T* src = reinterpret_cast<const T*>(p.q) + (live ? n * p.q_stride[0] + h * p.q_stride[1] : 0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            q[im][ks][e + 2 * x] = live && ks * 16 + x * 8 < p.D ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + x * 8 + qc) : 0u;
        if (BIAS == PAGED_SLOPES && live) {
          slope2[im][e] = p.slopes[h] * kLog2eP;
          my_pos[im][e] = p.positions ? p.positions[n] : rq.len + t;
        }
        if (BIAS == PAGED_FACTORS) {
          qbrow[im][e] = live ? reinterpret_cast<const T*>(p.q_bias) + n * p.q_bias_stride[0] + h * p.q_bias_stride[1] : nullptr;
        }
      }
    auto load_qb = [&](int r0) {
#pragma unroll
      for (int im = 0; im < NM; ++im)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            uint32_t w = 0;
            const int c = r0 + x * 8 + qc;
            const uint16_t* src = reinterpret_cast<const uint16_t*>(qbrow[im][e]);
            if (src && c < p.R) w = src[c];
            if (src && c + 1 < p.R) w |= (uint32_t)src[c + 1] << 16;
            qb[im][e + 2 * x] = w;
          }
    };
    if (BIAS == PAGED_FACTORS) load_qb(0);

#pragma unroll
    for (int i = 0; i < ST - 1; ++i) {
      fetch(fetched, i);
      fetched += WK;
    }
    if (BIAS == PAGED_FACTORS) {
      load_factors(0, kb);
      factor_pages(seg.t0 * 4 + wk + WK);
    }

    float o[NM][NT][4];
#pragma unroll
    for (int im = 0; im < NM; ++im)
#pragma unroll
      for (int i = 0; i < NT; ++i) o[im][i][0] = o[im][i][1] = o[im][i][2] = o[im][i][3] = 0.f;

    int stage = 0, fill = ST - 1;
    for (int tile = seg.t0 * 4 + wk; tile < tile_end; tile += WK) {
      asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
      __syncwarp();  // every lane's copies have landed, and the stage read last has been read by all
      const uint32_t okm = ring_ok[stage];
      fetch(fetched, fill);
      fetched += WK;
      fill = fill + 1 == ST ? 0 : fill + 1;
      const uint32_t ks_base = ring + stage * Cfg::STAGE, vs_base = ks_base + Cfg::HALF;
      stage = stage + 1 == ST ? 0 : stage + 1;

      // ---- S = Q K^T
      float s[NM][2][4] = {};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if (TD > 32 && ks * 16 >= p.D) break;
        uint32_t b[4];
        ldsm4(ks_base + Cfg::at((lane >> 4) * 8 + (lane & 7), ks * 2 + ((lane >> 3) & 1)), b);
#pragma unroll
        for (int im = 0; im < NM; ++im) {
          mma16816<T>(s[im][0], q[im][ks], b[0], b[1]);
          mma16816<T>(s[im][1], q[im][ks], b[2], b[3]);
        }
      }
      float f[NM][2][4] = {};
      if (BIAS == PAGED_FACTORS) {
        uint32_t cur[2][2] = {{kb[0][0], kb[0][1]}, {kb[1][0], kb[1][1]}};
        load_factors(0, kb);
        factor_pages(tile + 2 * WK);
        for (int r0 = 0;;) {
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int im = 0; im < NM; ++im) mma16816<T>(f[im][nt], qb[im], cur[nt][0], cur[nt][1]);
          if (p.R <= 16 || (r0 += 16) >= p.R) break;
          // wider factors: loaded where they are used
          const int keep[4] = {fpage[0], fpage[1], fplace[0], fplace[1]};
          factor_pages(tile);
          load_factors(r0, cur);
          fpage[0] = keep[0], fpage[1] = keep[1], fplace[0] = keep[2], fplace[1] = keep[3];
          load_qb(r0);
        }
        if (p.R > 16) load_qb(0);
      }

      // ---- logits in log2 units; masks where the tile holds new tokens' keys or keys that do not exist
      const int j0 = tile * 16 + qc;
      const bool masked = okm != 0xffffu || tile * 16 + 16 > rq.len;
#pragma unroll
      for (int im = 0; im < NM; ++im)
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int e = i >> 1, j = j0 + nt * 8 + (i & 1);
            float v = s[im][nt][i] * a.scale_log2;
            if (BIAS == PAGED_SLOPES) {
              int pos = j;
              if (masked && p.positions && j >= rq.len && j < rq.keys) pos = p.positions[rq.first + j - rq.len];
              v = fmaf(slope2[im][e], (float)(pos - my_pos[im][e]), v);
            }
            if (BIAS == PAGED_FACTORS) v = fmaf(f[im][nt][i], kLog2eP, v);
            if (masked) {
              bool seen = (okm >> (j - tile * 16)) & 1;
              if (seen && j >= rq.len) seen = row_tok[im][e] >= 0 && tree_sees(p, rq.first + row_tok[im][e], row_tok[im][e], j - rq.len);
              if (!seen) v = -INFINITY;
            }
            s[im][nt][i] = v;
          }

      // ---- running maximum and sum, P as fragments
      uint32_t pf[NM][4];
      bool grown = false;
      float alpha[NM][2];
#pragma unroll
      for (int im = 0; im < NM; ++im)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(fmaxf(s[im][0][2 * e], s[im][0][2 * e + 1]), fmaxf(s[im][1][2 * e], s[im][1][2 * e + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          mx = fmaxf(mx, m[im][e]);
          grown |= mx > m[im][e];
          const float msub = fmaxf(mx, -FLT_MAX);  // no visible key yet: every exponential is zero
          alpha[im][e] = fast_exp2(m[im][e] - msub);
          m[im][e] = mx;
          const float p0 = fast_exp2(s[im][0][2 * e] - msub), p1 = fast_exp2(s[im][0][2 * e + 1] - msub);
          const float p2 = fast_exp2(s[im][1][2 * e] - msub), p3 = fast_exp2(s[im][1][2 * e + 1] - msub);
          l[im][e] = fmaf(l[im][e], alpha[im][e], (p0 + p1) + (p2 + p3));
          // the probabilities are rounded to the 16 bits of V: half a step of relative error each, what the result is rounded by
          pf[im][e] = Pack2<T>::pack(p0, p1);
          pf[im][2 + e] = Pack2<T>::pack(p2, p3);
        }
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int im = 0; im < NM; ++im)
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            o[im][i][0] *= alpha[im][0];
            o[im][i][1] *= alpha[im][0];
            o[im][i][2] *= alpha[im][1];
            o[im][i][3] *= alpha[im][1];
          }
      }

      // ---- O += P V.  A value that is not finite must not reach the rows that do not see its key (0 x inf): such a tile of new
      // tokens goes through a loop over its keys.
      bool odd = false;
      if (masked) {
        bool mine = false;
#pragma unroll
        for (int i = 0; i < TD / 16; ++i) {
          const uint4 w = *reinterpret_cast<const uint4*>(smem + warp * Cfg::RING + (vs_base - ring) + (i * 32 + lane) * 16);
          mine |= pair_not_finite<T>(w.x) || pair_not_finite<T>(w.y) || pair_not_finite<T>(w.z) || pair_not_finite<T>(w.w);
        }
        odd = __any_sync(0xffffffffu, mine);
      }
      if (!odd) {
#pragma unroll
        for (int np = 0; np < KS; ++np) {
          if (TD > 32 && np * 16 >= p.D) break;
          uint32_t b[4];
          ldsm4t(vs_base + Cfg::at(((lane >> 3) & 1) * 8 + (lane & 7), np * 2 + (lane >> 4)), b);
#pragma unroll
          for (int im = 0; im < NM; ++im) {
            mma16816<T>(o[im][2 * np], pf[im], b[0], b[1]);
            mma16816<T>(o[im][2 * np + 1], pf[im], b[2], b[3]);
          }
        }
      } else {
#pragma unroll 1
        for (int k = 0; k < 16; ++k) {
          const int src = (lane & ~3) | ((k & 7) >> 1);
          float pk[NM][2];
#pragma unroll
          for (int im = 0; im < NM; ++im)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t w = __shfl_sync(0xffffffffu, k < 8 ? pf[im][e] : pf[im][2 + e], src);
              const uint16_t h = (uint16_t)(k & 1 ? w >> 16 : w);
              pk[im][e] = to_f32(*reinterpret_cast<const T*>(&h));
            }
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            const uint32_t w = ld_shared_flag(vs_base + Cfg::at(k, i) + qc * 2);
            const T* v = reinterpret_cast<const T*>(&w);
            const float v0 = to_f32(v[0]), v1 = to_f32(v[1]);
#pragma unroll
            for (int im = 0; im < NM; ++im) {
              if (pk[im][0] != 0.f) {
                o[im][i][0] = fmaf(pk[im][0], v0, o[im][i][0]);
                o[im][i][1] = fmaf(pk[im][0], v1, o[im][i][1]);
              }
              if (pk[im][1] != 0.f) {
                o[im][i][2] = fmaf(pk[im][1], v0, o[im][i][2]);
                o[im][i][3] = fmaf(pk[im][1], v1, o[im][i][3]);
              }
            }
          }
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- the warp's sums: over the four lanes of a row, then over the warps of the head
#pragma unroll
    for (int im = 0; im < NM; ++im)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[im][e] += __shfl_xor_sync(0xffffffffu, l[im][e], 1);
        l[im][e] += __shfl_xor_sync(0xffffffffu, l[im][e], 2);
      }
    if (WK > 1) {
      float* mine = reinterpret_cast<float*>(smem + warp * Cfg::RING);  // (MT, TD) floats fit the ring, statistics behind them
      static_assert(MT * TD * 4 + MT * 8 <= Cfg::RING, "merge buffer");
      __syncwarp();
      if (wk > 0) {
#pragma unroll
        for (int im = 0; im < NM; ++im) {
#pragma unroll
          for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int x = 0; x < 4; ++x) mine[((im * NT + i) * 4 + x) * 32 + lane] = o[im][i][x];
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (qc == 0) reinterpret_cast<float2*>(mine + MT * TD)[im * 16 + e * 8 + qr] = make_float2(m[im][e], l[im][e]);
        }
      }
      __syncthreads();
      if (wk == 0) {
        for (int w = 1; w < WK; ++w) {
          const float* from = reinterpret_cast<const float*>(smem + (warp + w) * Cfg::RING);
#pragma unroll
          for (int im = 0; im < NM; ++im) {
            float fa[2], fb[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float2 s2 = reinterpret_cast<const float2*>(from + MT * TD)[im * 16 + e * 8 + qr];
              const float mn = fmaxf(m[im][e], s2.x), ms = fmaxf(mn, -FLT_MAX);
              fa[e] = fast_exp2(m[im][e] - ms);
              fb[e] = fast_exp2(s2.x - ms);
              m[im][e] = mn;
              l[im][e] = l[im][e] * fa[e] + s2.y * fb[e];
            }
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
              for (int x = 0; x < 4; ++x)
                o[im][i][x] = o[im][i][x] * fa[x >> 1] + from[((im * NT + i) * 4 + x) * 32 + lane] * fb[x >> 1];
          }
        }
      }
      __syncthreads();
    }
    const bool whole = seg.t0 == 0 && seg.t1 == seg.tiles;
    if (wk == 0) {
#pragma unroll
      for (int im = 0; im < NM; ++im)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = im * 16 + e * 8 + qr;
          if (whole) {
            const int t = row_tok[im][e];
            if (t < 0) continue;
            const int h = hk * a.G + (seg.rt * MT + r - t * a.G), n = rq.first + t;
            const float ls = l[im][e], inv = ls > 0.f ? 1.f / ls : ls == 0.f ? 0.f : ls;
            T* dst = reinterpret_cast<T*>(p.o) + n * p.o_stride[0] + h * p.o_stride[1];
#pragma unroll
            for (int i = 0; i < NT; ++i)
              if (i * 8 < p.D)
                *reinterpret_cast<uint32_t*>(dst + i * 8 + qc) =
                    ls == 0.f ? 0u : Pack2<T>::pack(o[im][i][2 * e] * inv, o[im][i][2 * e + 1] * inv);
            if (p.lse && qc == 0) p.lse[(int64_t)n * p.Hq + h] = ls > 0.f ? (m[im][e] + fast_log2(ls)) * kLn2P : ls == 0.f ? -INFINITY : ls;
          } else {
            // slot 1: the CTA in which the item begins; 0: the others
            const int64_t row = (((int64_t)blockIdx.x * 2 + (seg.t0 == 0 ? 1 : 0)) * WH + wh) * MT + r;
#pragma unroll
            for (int i = 0; i < NT; ++i)
              *reinterpret_cast<float2*>(a.part + row * TD + i * 8 + qc) = make_float2(o[im][i][2 * e], o[im][i][2 * e + 1]);
            if (qc == 0) a.ml[row] = make_float2(m[im][e], l[im][e]);
          }
        }
    }
    if (!whole && seg.t0 == 0 && threadIdx.x == 0) {
      a.desc[2 * blockIdx.x] = make_int4(seg.rt, seg.hg, seg.last_cta, 0);
      a.desc[2 * blockIdx.x + 1] = make_int4(rq.first, rq.tokens * a.G, 0, 0);
    }
  }
}

template <typename T, int TD, int MT, int BIAS>
int launch_paged_split_t(const PagedArgs& a, const PagedPlan& plan, cudaStream_t st) {
  auto kern = paged_split_kernel<T, TD, MT, BIAS>;
  static std::mutex mu;
  static bool attr_done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lk(mu);
    if (!attr_done[dev & 63]) {
      const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SplitCfg<TD>::SMEM);
      if (e != cudaSuccess) return (int)e;
      attr_done[dev & 63] = true;
    }
  }
  if (const int rc = launch_pdl(kern, plan.ctas, kSplitThreads, SplitCfg<TD>::SMEM, st, a, plan.WH)) return rc;
  return launch_paged_join<TD>(a, plan, st);
}

template <int TD>
int launch_paged_split(const PagedArgs& a, const PagedPlan& plan, cudaStream_t st) {
  auto by_bias = [&](auto t, auto mt) {
    using T = decltype(t);
    constexpr int MT = decltype(mt)::value;
    return a.p.slopes ? launch_paged_split_t<T, TD, MT, PAGED_SLOPES>(a, plan, st)
           : a.p.R    ? launch_paged_split_t<T, TD, MT, PAGED_FACTORS>(a, plan, st)
                      : launch_paged_split_t<T, TD, MT, PAGED_PLAIN>(a, plan, st);
  };
  auto by_rows = [&](auto t) {
    return plan.MT == 16 ? by_bias(t, std::integral_constant<int, 16>()) : by_bias(t, std::integral_constant<int, 32>());
  };
  return a.p.dtype == FB_DTYPE_F16 ? by_rows(__half()) : by_rows(__nv_bfloat16());
}

}  // namespace fb
