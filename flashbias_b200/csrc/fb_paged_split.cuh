// Attention over pages with few rows per key head (24 to 80 by their width): decoding, and small trees or runs of drafted tokens.
//
// Bound by reading K and V once.  A warp works alone: it owns a head of the CTA's group and every WK-th tile of 16 or 32 keys, copies
// them into a ring of its own in shared memory (cp.async, so that what is in flight is bounded by shared memory and not by
// registers: 2 CTAs x 96 KB per SM), and keeps 16 or 32 query rows, the row maxima and sums and the output in registers.  The
// products are mma.sync m16n8k16: a tile of 16 keys and 16 rows is one fragment wide, S stays in the registers that P is fed
// from, and the tensor pipe is far from being the bound; a tcgen05 tile would spend 112 of its 128 rows on padding.  No
// barrier is needed between warps while a segment lasts; where a group has fewer heads than the CTA has warps, the warps of a
// head join their sums through shared memory at the segment's end.
// 64 requests of up to 8192 tokens, H32-8 D128: 229 us (1356 MB, 5.9 TB/s).
//
// With few items (one or two requests of a few heads) latency is what counts, and the second launch half of it: CLUSTER gives
// every item to the CTAs of one cluster, which cut its key tiles into equal parts and join them through distributed shared
// memory (one token over 1000 keys, 8 heads: 10.6 us a call with the schedule and a join, 9.6 so).
#pragma once

#include <cooperative_groups.h>

#include <mutex>

#include "fb_paged.cuh"

namespace fb {

constexpr int kSplitWarps = 4;
constexpr int kSplitThreads = 32 * kSplitWarps;
constexpr int kSplitKT = 64;  // keys of a scheduled tile: several steps of a warp

template <int TD, int MT>
struct SplitCfg {
  static constexpr int KT = TD == 128 ? 16 : 32;                         // keys of a step
  static constexpr int ROW = TD * 2;                                     // bytes of a key's row
  static constexpr int ST = TD == 64 && MT == 16 ? 2 : 3;                // ring stages
  static constexpr int HALF = KT * ROW, STAGE = 2 * HALF, RING = ST * STAGE;  // K, then V
  static constexpr int F_ROW = 32, F_STAGE = KT * F_ROW;                 // factors: 16 columns, zeros behind the last
  static constexpr int OFF_F = kSplitWarps * RING, OFF_OK = OFF_F + kSplitWarps * ST * F_STAGE;
  static constexpr int smem(bool factors) { return factors ? OFF_OK + kSplitWarps * ST * 4 : OFF_F + kSplitWarps * ST * 4; }
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

// PAGED_FACTORS: up to 16 columns in rows that can be copied in pieces of 4, 8 or 16 bytes, beside the keys in the ring;
// PAGED_FACTORS_ANY: any others, read into registers.
enum { PAGED_PLAIN, PAGED_SLOPES, PAGED_FACTORS, PAGED_FACTORS_ANY };

// The parts of an item that the CTAs of a cluster hold (those of head wh in the registers of the warp with wk == 0), joined
// through distributed shared memory: every CTA writes some of the rows.  The parts lie in the rings of the warps that hold them.
template <typename T, int TD, int MT>
__device__ __forceinline__ void join_cluster(const PagedArgs& a, const Segment& seg, int hk, uint8_t* smem, int wh, int wk, int WH,
                                             const float (&o)[MT / 16][TD / 8][4], const float (&m)[MT / 16][2], const float (&l)[MT / 16][2]) {
  using Cfg = SplitCfg<TD, MT>;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  constexpr int LANES = TD / 4;  // of a row
  const fb_paged_params& p = a.p;
  const int lane = threadIdx.x & 31, qr = lane >> 2, qc = 2 * (lane & 3), step = Cfg::RING * (kSplitWarps / WH);
  float* mine = reinterpret_cast<float*>(smem + wh * step);  // (MT, TD), statistics behind
  __syncthreads();
  if (wk == 0) {
#pragma unroll
    for (int im = 0; im < MT / 16; ++im)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = im * 16 + e * 8 + qr;
#pragma unroll
        for (int i = 0; i < TD / 8; ++i) *reinterpret_cast<float2*>(mine + r * TD + i * 8 + qc) = make_float2(o[im][i][2 * e], o[im][i][2 * e + 1]);
        if (qc == 0) reinterpret_cast<float2*>(mine + MT * TD)[r] = make_float2(m[im][e], l[im][e]);
      }
  }
  cluster.sync();
  const int csize = (int)cluster.num_blocks(), col = (threadIdx.x % LANES) * 4;
  for (int i = (int)cluster.block_rank() * (kSplitThreads / LANES) + threadIdx.x / LANES; i < WH * MT; i += csize * (kSplitThreads / LANES)) {
    const int h_in = i / MT, r = i - h_in * MT, gr = seg.rt * MT + r;
    if (gr >= seg.r.tokens * a.G) continue;
    float* part = reinterpret_cast<float*>(smem + h_in * step);
    float mx = -INFINITY;
    for (int c = 0; c < csize; ++c) mx = fmaxf(mx, reinterpret_cast<const float2*>(cluster.map_shared_rank(part, c) + MT * TD)[r].x);
    const float ms = fmaxf(mx, -FLT_MAX);
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int c = 0; c < csize; ++c) {
      const float* from = cluster.map_shared_rank(part, c);
      const float2 s = reinterpret_cast<const float2*>(from + MT * TD)[r];
      const float4 v = *reinterpret_cast<const float4*>(from + r * TD + col);
      const float f = fast_exp2((s.x - ms) * kLog2eP);
      sum = fmaf(s.y, f, sum);
      acc = make_float4(fmaf(v.x, f, acc.x), fmaf(v.y, f, acc.y), fmaf(v.z, f, acc.z), fmaf(v.w, f, acc.w));
    }
    const int t = a.group_div.quot32(gr), h = (hk - wh + h_in) * a.G + gr - t * a.G, n = seg.r.first + t;
    const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;
    if (col < p.D)
      *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.o) + n * p.o_stride[0] + h * p.o_stride[1] + col) =
          sum == 0.f ? make_uint2(0u, 0u) : make_uint2(Pack2<T>::pack(acc.x * inv, acc.y * inv), Pack2<T>::pack(acc.z * inv, acc.w * inv));
    if (p.lse && col == 0) p.lse[(int64_t)n * p.Hq + h] = sum > 0.f ? fmaf(fast_log2(sum) - kSplitLift<T>, kLn2P, mx) : sum == 0.f ? -INFINITY : sum;
  }
  cluster.sync();  // the parts have been read
}

template <typename T, int TD, int MT, int BIAS, bool CLUSTER>
__global__ void __launch_bounds__(kSplitThreads, split_ctas(TD, MT)) paged_split_kernel(const __grid_constant__ PagedArgs a, const int WH) {
  using Cfg = SplitCfg<TD, MT>;
  constexpr int NM = MT / 16, KS = TD / 16, NT = TD / 8, ST = Cfg::ST, KT = Cfg::KT, NK = KT / 16, PER = kSplitKT / KT;
  constexpr uint32_t ALL = KT == 32 ? 0xffffffffu : 0xffffu;
  extern __shared__ __align__(1024) uint8_t smem[];
  const fb_paged_params& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, WK = kSplitWarps / WH, wh = warp / WK, wk = warp % WK;
  const uint32_t ring = smem_u32(smem) + warp * Cfg::RING;
  // keys of a stage that exist, as bits; the factors' ring
  uint32_t* ring_ok = reinterpret_cast<uint32_t*>(smem + (BIAS == PAGED_FACTORS ? Cfg::OFF_OK : Cfg::OFF_F)) + warp * ST;
  const uint32_t fring = smem_u32(smem) + Cfg::OFF_F + warp * ST * Cfg::F_STAGE;
  if (BIAS == PAGED_FACTORS) {
    for (int i = lane; i < ST * Cfg::F_STAGE / 16; i += 32) st_shared_v4(fring + i * 16, 0u, 0u, 0u, 0u);
    __syncwarp();
  }
  const int qr = lane >> 2, qc = 2 * (lane & 3);  // a fragment's row (and row + 8) and first column of this lane
  grid_dep_wait();
  if (!CLUSTER && threadIdx.x == 0) a.desc[2 * blockIdx.x].x = -1;
  // (a cluster walks whole items: one key tile each, as long as there are keys)
  PagedWalk<CLUSTER ? 0x7fffffff : kSplitKT, MT, kSplitThreads> walk;
  const int csize = CLUSTER ? (int)cooperative_groups::this_cluster().num_blocks() : 1, crank = CLUSTER ? (int)cooperative_groups::this_cluster().block_rank() : 0;
  walk.start(a, p.Hk / WH, blockIdx.x / csize, gridDim.x / csize);

  Segment seg;
  while (walk.next(a, seg)) {
    if (CLUSTER) {  // this CTA's part of the key tiles, possibly none
      const int64_t tiles = ((int64_t)seg.r.keys + kSplitKT - 1) / kSplitKT;
      seg.t0 = (int)(tiles * crank / csize);
      seg.t1 = (int)(tiles * (crank + 1) / csize);
    }
    const Request& rq = seg.r;
    const int hk = seg.hg * WH + wh, rows = rq.tokens * a.G - seg.rt * MT;  // rows of the request from this tile on
    const T* kbase = reinterpret_cast<const T*>(p.key_cache) + hk * p.key_cache_stride[2];
    const T* vbase = reinterpret_cast<const T*>(p.value_cache) + hk * p.value_cache_stride[2];
    const T* bbase = reinterpret_cast<const T*>(p.bias_cache) + (p.bias_heads > 1 ? hk * p.bias_cache_stride[2] : 0);
    const int32_t* table = p.block_table + (int64_t)min(seg.b, p.B - 1) * p.table_stride;
    const int tile_end = min(seg.t1 * PER, (rq.keys + KT - 1) / KT);

    // ---- copies: the pages of a tile's keys are looked up one tile ahead of their use (lane % KT = key).  Where pages are whole
    // runs of 16 keys one page serves a run, and a copy's address is one addition: half of the instructions that a tile of 64
    // columns takes would otherwise go into addresses.
    const int c = lane % Cfg::CH, kr = lane / Cfg::CH;  // this lane's chunk, and its key in the first of a tile's copies
    const bool in = c * 8 < p.D;
    const int64_t kstep = (32 / Cfg::CH) * p.key_cache_stride[1], vstep = (32 / Cfg::CH) * p.value_cache_stride[1];
    const T *klane = kbase + kr * p.key_cache_stride[1] + (in ? c * 8 : 0), *vlane = vbase + kr * p.value_cache_stride[1] + (in ? c * 8 : 0);
    int page_next = -1, place_next = 0;
    auto look_up = [&](int tile) {
      const int j = tile * KT + (a.whole_tiles ? lane & (KT - 16) : lane & (KT - 1));
      page_next = -1;
      if (tile < tile_end && j < rq.keys) {
        const int col = a.page_div.quot32(j);
        place_next = j - col * p.page_size;
        page_next = table[col];
      }
    };
    // the factors of the key lane % KT, whose page and place (or those of its run) this lane holds
    auto fetch_factors = [&](int stage, bool ok, int page, int place) {
      const char* src = reinterpret_cast<const char*>(bbase + (ok ? page * p.bias_cache_stride[0] + place * p.bias_cache_stride[1] : 0));
      const uint32_t dst = fring + stage * Cfg::F_STAGE + (lane & (KT - 1)) * Cfg::F_ROW, live = ok ? 0xffffffffu : 0u;
      if (KT == 16 && lane >= 16) return;
      if (a.factor_bytes == 16) {
        for (int i = 0; i < 2 * p.R; i += 16) asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst + i), "l"(src + i), "r"(live & 16u) : "memory");
      } else if (a.factor_bytes == 8) {
        for (int i = 0; i < 2 * p.R; i += 8) asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst + i), "l"(src + i), "r"(live & 8u) : "memory");
      } else {
        for (int i = 0; i < 2 * p.R; i += 4) asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + i), "l"(src + i), "r"(live & 4u) : "memory");
      }
    };
    auto fetch = [&](int tile, int stage) {
      if (tile < tile_end) {
        const int page = page_next, place = place_next;
        const uint32_t dst = ring + stage * Cfg::STAGE;
        if (a.whole_tiles && tile * KT + KT <= rq.keys && __all_sync(0xffffffffu, (uint32_t)page < a.pages32)) {
          look_up(tile + WK);
          if (lane == 0) ring_ok[stage] = ALL;
          if (BIAS == PAGED_FACTORS) fetch_factors(stage, true, page, place + (lane & 15));
#pragma unroll
          for (int h = 0; h < NK; ++h) {
            const int pg = NK > 1 ? __shfl_sync(0xffffffffu, page, h * 16) : page, pl = NK > 1 ? __shfl_sync(0xffffffffu, place, h * 16) : place;
            const T* k = klane + pg * p.key_cache_stride[0] + pl * p.key_cache_stride[1];
            const T* v = vlane + pg * p.value_cache_stride[0] + pl * p.value_cache_stride[1];
#pragma unroll
            for (int i = 0; i < TD / 16; ++i) {
              const uint32_t at = dst + Cfg::at(kr + i * (32 / Cfg::CH), c) + h * 16 * Cfg::ROW;
              cp_async16_zfill(at, k, in);
              cp_async16_zfill(at + Cfg::HALF, v, in);
              k += kstep;
              v += vstep;
            }
          }
        } else {
          const int off = a.whole_tiles ? lane & 15 : 0;
          const bool there = tile * KT + (lane & (KT - 1)) < rq.keys, ok = there && (uint32_t)page < a.pages32;
          if (there && !ok) paged_bad_index(p);
          const int64_t ko = ok ? page * p.key_cache_stride[0] + (place + off) * p.key_cache_stride[1] : 0;
          const int64_t vo = ok ? page * p.value_cache_stride[0] + (place + off) * p.value_cache_stride[1] : 0;
          const uint32_t okm = __ballot_sync(0xffffffffu, ok) & ALL;
          if (lane == 0) ring_ok[stage] = okm;
          look_up(tile + WK);
          if (BIAS == PAGED_FACTORS) fetch_factors(stage, ok, page, place + off);
#pragma unroll
          for (int i = 0; i < TD * NK / 16; ++i) {
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
    uint32_t kb[2 * NK][2] = {};
    int fpage[2 * NK], fplace[2 * NK];  // (of eight keys each)
    const uint16_t* const blane = reinterpret_cast<const uint16_t*>(bbase) + qc;
    auto factor_pages = [&](int tile) {
#pragma unroll
      for (int nt = 0; nt < 2 * NK; ++nt) {
        const int j = tile * KT + nt * 8 + qr;
        if ((nt & 1) && a.whole_tiles) {  // the run's other eight
          fpage[nt] = fpage[nt - 1];
          fplace[nt] = fplace[nt - 1] + 8;
          if (j >= rq.keys) fpage[nt] = -1;
          continue;
        }
        fpage[nt] = -1;
        fplace[nt] = 0;
        if (tile < tile_end && j < rq.keys) {
          const int col = a.page_div.quot32(j);
          fplace[nt] = j - col * p.page_size;
          fpage[nt] = table[col];
        }
      }
    };
    auto load_factors = [&](int r0, uint32_t (&f)[2 * NK][2]) {
#pragma unroll
      for (int nt = 0; nt < 2 * NK; ++nt) {
        const bool ok = (uint32_t)fpage[nt] < a.pages32;
        const uint16_t* src = blane + r0 + (ok ? fpage[nt] * p.bias_cache_stride[0] + fplace[nt] * p.bias_cache_stride[1] : 0);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int col = r0 + qc + x * 8;
          f[nt][x] = 0u;
          if (x == 1 && r0 + 8 >= p.R) continue;
          if (a.factor_words) {
            if (ok && col < p.R) f[nt][x] = *reinterpret_cast<const uint32_t*>(src + x * 8);
          } else {
            if (ok && col < p.R) f[nt][x] = src[x * 8];
            if (ok && col + 1 < p.R) f[nt][x] |= (uint32_t)src[x * 8 + 1] << 16;
          }
        }
      }
    };

    int fetched = seg.t0 * PER + wk;
    look_up(fetched);
    if (BIAS == PAGED_FACTORS_ANY) factor_pages(fetched);

    // ---- query rows, as fragments of the products' first operand
    uint32_t q[NM][KS][4], qb[NM][4] = {};
    int row_tok[NM][2];               // token of the request, -1 for rows of padding
    float slope[NM][2] = {}, m[NM][2], l[NM][2];
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
          slope[im][e] = p.slopes[h];
          my_pos[im][e] = p.positions ? p.positions[n] : rq.len + t;
        }
        if (BIAS >= PAGED_FACTORS) {
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
    if (BIAS >= PAGED_FACTORS) load_qb(0);

#pragma unroll
    for (int i = 0; i < ST - 1; ++i) {
      fetch(fetched, i);
      fetched += WK;
    }
    if (BIAS == PAGED_FACTORS_ANY) {
      load_factors(0, kb);
      factor_pages(seg.t0 * PER + wk + WK);
    }

    float o[NM][NT][4];
#pragma unroll
    for (int im = 0; im < NM; ++im)
#pragma unroll
      for (int i = 0; i < NT; ++i) o[im][i][0] = o[im][i][1] = o[im][i][2] = o[im][i][3] = 0.f;

    // lanes' addresses in a stage; the k-step or pair of column blocks i is an XOR of i << 5 away (rows begin at multiples of it)
    const uint32_t k_at = Cfg::at((lane >> 4) * 8 + (lane & 7), (lane >> 3) & 1), v_at = Cfg::at(((lane >> 3) & 1) * 8 + (lane & 7), lane >> 4);
    const uint32_t f_at = ((lane >> 4) * 8 + (lane & 7)) * Cfg::F_ROW + ((lane >> 3) & 1) * 16;
    int stage = 0, fill = ST - 1;
    for (int tile = seg.t0 * PER + wk; tile < tile_end; tile += WK) {
      asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
      __syncwarp();  // every lane's copies have landed, and the stage read last has been read by all
      const uint32_t okm = ring_ok[stage];
      fetch(fetched, fill);
      fetched += WK;
      fill = fill + 1 == ST ? 0 : fill + 1;
      const uint32_t ks_base = ring + stage * Cfg::STAGE, vs_base = ks_base + Cfg::HALF;
      stage = stage + 1 == ST ? 0 : stage + 1;

      // ---- S = Q K^T (columns beyond D hold zeros)
      float s[NM][2 * NK][4] = {};
#pragma unroll
      for (int h = 0; h < NK; ++h)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          uint32_t b[4];
          ldsm4((ks_base + h * 16 * Cfg::ROW + k_at) ^ (ks << 5), b);
#pragma unroll
          for (int im = 0; im < NM; ++im) {
            mma16816<T>(s[im][2 * h], q[im][ks], b[0], b[1]);
            mma16816<T>(s[im][2 * h + 1], q[im][ks], b[2], b[3]);
          }
        }
      float f[NM][2 * NK][4] = {};
      if (BIAS == PAGED_FACTORS) {
        const uint32_t fb = fring + (ks_base - ring) / Cfg::STAGE * Cfg::F_STAGE;
#pragma unroll
        for (int h = 0; h < NK; ++h) {
          uint32_t b[4];
          ldsm4(fb + h * 16 * Cfg::F_ROW + f_at, b);
#pragma unroll
          for (int im = 0; im < NM; ++im) {
            mma16816<T>(f[im][2 * h], qb[im], b[0], b[1]);
            mma16816<T>(f[im][2 * h + 1], qb[im], b[2], b[3]);
          }
        }
      }
      if (BIAS == PAGED_FACTORS_ANY) {
        uint32_t cur[2 * NK][2];
#pragma unroll
        for (int i = 0; i < 2 * NK; ++i) cur[i][0] = kb[i][0], cur[i][1] = kb[i][1];
        load_factors(0, kb);
        for (int r0 = 0;;) {
#pragma unroll
          for (int nt = 0; nt < 2 * NK; ++nt)
#pragma unroll
            for (int im = 0; im < NM; ++im) mma16816<T>(f[im][nt], qb[im], cur[nt][0], cur[nt][1]);
          if (p.R <= 16 || (r0 += 16) >= p.R) break;
          factor_pages(tile);  // wider factors: loaded where they are used
          load_factors(r0, cur);
          load_qb(r0);
        }
        if (p.R > 16) load_qb(0);
        factor_pages(tile + 2 * WK);
      }

      // ---- logits; masks where the tile holds new tokens' keys or keys that do not exist.  In their own units: in those of log2
      // what lies below -2.36e38 (a mask of the type's lowest value among the factors) would be -inf, a key that is not seen
      const int j0 = tile * KT + qc;
      const bool masked = okm != ALL || tile * KT + KT > rq.len;
      // keys of new tokens, whose position may lie anywhere: the difference is taken of whole numbers
      const bool moved = BIAS == PAGED_SLOPES && p.positions && tile * KT + KT > rq.len;
      if (moved) {
#pragma unroll
        for (int nt = 0; nt < 2 * NK; ++nt)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int j = j0 + nt * 8 + x, at = j >= rq.len && j < rq.keys ? p.positions[rq.first + j - rq.len] : j;
#pragma unroll
            for (int im = 0; im < NM; ++im)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                s[im][nt][2 * e + x] = fmaf(slope[im][e], (float)(at - my_pos[im][e]), s[im][nt][2 * e + x] * p.softmax_scale);
          }
      }
      if (!moved) {
#pragma unroll
        for (int im = 0; im < NM; ++im)
#pragma unroll
          for (int nt = 0; nt < 2 * NK; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float v = s[im][nt][i] * p.softmax_scale;
              if (BIAS == PAGED_SLOPES) v = fmaf(slope[im][i >> 1], (float)(j0 + nt * 8 + (i & 1) - my_pos[im][i >> 1]), v);
              if (BIAS >= PAGED_FACTORS) v += f[im][nt][i];
              s[im][nt][i] = v;
            }
      }
      if (masked) {
        const int td0 = tile * KT - rq.len;
#pragma unroll
        for (int im = 0; im < NM; ++im)
#pragma unroll
          for (int e = 0; e < 2; ++e) {  // what the row sees of the tile
            uint32_t bits = okm;
            if (row_tok[im][e] >= 0 && td0 + KT > 0) bits &= seen_bits(p, rq.first + row_tok[im][e], row_tok[im][e], td0);
#pragma unroll
            for (int nt = 0; nt < 2 * NK; ++nt)
#pragma unroll
              for (int x = 0; x < 2; ++x)
                if (!(bits >> (nt * 8 + qc + x) & 1)) s[im][nt][2 * e + x] = -INFINITY;
          }
      }

      // ---- running maximum and sum, P as fragments
      uint32_t pf[NM][NK][4];
      bool grown = false;
      float alpha[NM][2];
#pragma unroll
      for (int im = 0; im < NM; ++im)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = m[im][e];
#pragma unroll
          for (int nt = 0; nt < 2 * NK; ++nt) mx = fmax3(mx, s[im][nt][2 * e], s[im][nt][2 * e + 1]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          grown |= mx > m[im][e];
          const float msub = fmaxf(mx, -FLT_MAX);  // no visible key yet: every exponential is zero
          alpha[im][e] = fast_exp2((m[im][e] - msub) * kLog2eP);
          m[im][e] = mx;
          float sum = 0.f;
#pragma unroll
          for (int nt = 0; nt < 2 * NK; ++nt) {
            const float p0 = fast_exp2(fmaf(s[im][nt][2 * e] - msub, kLog2eP, kSplitLift<T>)),
                        p1 = fast_exp2(fmaf(s[im][nt][2 * e + 1] - msub, kLog2eP, kSplitLift<T>));
            sum += p0 + p1;
            // the probabilities are rounded to the 16 bits of V: half a step of relative error each, what the result is rounded by (an error
            // about a third larger than with 32 bits, in bf16); twice the products would carry a second part of P
            pf[im][nt >> 1][2 * (nt & 1) + e] = Pack2<T>::pack(p0, p1);
          }
          l[im][e] = fmaf(l[im][e], alpha[im][e], sum);
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

      // ---- O += P V.  A value that is not finite must not reach the rows that do not see its key (0 x inf), and must reach those
      // that do, however small their P: such a tile of new tokens goes through a loop over its keys.
      bool odd = false;
      if (masked) {
        bool mine = false;
#pragma unroll 4
        for (int i = 0; i < Cfg::HALF / 512; ++i) {
          const uint4 w = *reinterpret_cast<const uint4*>(smem + warp * Cfg::RING + (vs_base - ring) + (i * 32 + lane) * 16);
          mine |= pair_not_finite<T>(w.x) || pair_not_finite<T>(w.y) || pair_not_finite<T>(w.z) || pair_not_finite<T>(w.w);
        }
        odd = __any_sync(0xffffffffu, mine);
      }
      if (!odd) {
#pragma unroll
        for (int h = 0; h < NK; ++h)
#pragma unroll
          for (int np = 0; np < KS; ++np) {
            uint32_t b[4];
            ldsm4t((vs_base + h * 16 * Cfg::ROW + v_at) ^ (np << 5), b);
#pragma unroll
            for (int im = 0; im < NM; ++im) {
              mma16816<T>(o[im][2 * np], pf[im][h], b[0], b[1]);
              mma16816<T>(o[im][2 * np + 1], pf[im][h], b[2], b[3]);
            }
          }
      } else {
        uint32_t sees[NM][2];
#pragma unroll
        for (int im = 0; im < NM; ++im)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            sees[im][e] = row_tok[im][e] < 0 ? 0u : okm & seen_bits(p, rq.first + row_tok[im][e], row_tok[im][e], tile * KT - rq.len);
        auto add = [](float& acc, float pk, float v) { acc = fabsf(v) <= FLT_MAX ? fmaf(pk, v, acc) : acc + v; };
#pragma unroll 1
        for (int k = 0; k < KT; ++k) {
          const int src = (lane & ~3) | ((k & 7) >> 1), at = k >> 3;  // the fragment's lane and half
          float pk[NM][2];
#pragma unroll
          for (int im = 0; im < NM; ++im)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint32_t w = pf[im][0][e];
#pragma unroll
              for (int x = 1; x < 2 * NK; ++x)
                if (at == x) w = pf[im][x >> 1][2 * (x & 1) + e];
              w = __shfl_sync(0xffffffffu, w, src);
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
              if (sees[im][0] >> k & 1) {
                add(o[im][i][0], pk[im][0], v0);
                add(o[im][i][1], pk[im][0], v1);
              }
              if (sees[im][1] >> k & 1) {
                add(o[im][i][2], pk[im][1], v0);
                add(o[im][i][3], pk[im][1], v1);
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
              fa[e] = fast_exp2((m[im][e] - ms) * kLog2eP);
              fb[e] = fast_exp2((s2.x - ms) * kLog2eP);
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
    if constexpr (CLUSTER) {
      join_cluster<T, TD, MT>(a, seg, hk, smem, wh, wk, WH, o, m, l);
      continue;
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
            if (p.lse && qc == 0) p.lse[(int64_t)n * p.Hq + h] = ls > 0.f ? fmaf(fast_log2(ls) - kSplitLift<T>, kLn2P, m[im][e]) : ls == 0.f ? -INFINITY : ls;
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

template <typename T, int TD, int MT, int BIAS, bool CLUSTER>
int launch_paged_split_t(const PagedArgs& a, const PagedPlan& plan, cudaStream_t st) {
  auto kern = paged_split_kernel<T, TD, MT, BIAS, CLUSTER>;
  constexpr int SMEM = SplitCfg<TD, MT>::smem(BIAS == PAGED_FACTORS);
  static std::mutex mu;
  static bool attr_done[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> lk(mu);
    if (!attr_done[dev & 63]) {
      cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
      if (e == cudaSuccess && CLUSTER) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (e != cudaSuccess) return (int)e;
      attr_done[dev & 63] = true;
    }
  }
  if (!CLUSTER) {
    if (const int rc = launch_pdl(kern, plan.ctas, kSplitThreads, SMEM, st, a, plan.WH)) return rc;
    return launch_paged_join<TD>(a, plan, st);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(plan.ctas);
  cfg.blockDim = dim3(kSplitThreads);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = plan.cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, plan.WH);
  if (e == cudaSuccess) note_launch();
  return (int)e;
}

template <int TD>
int launch_paged_split(const PagedArgs& a, const PagedPlan& plan, cudaStream_t st) {
  auto by_bias = [&](auto t, auto mt) {
    using T = decltype(t);
    constexpr int MT = decltype(mt)::value;
    auto go = [&](auto bias) {
      constexpr int BIAS = decltype(bias)::value;
      return plan.cluster ? launch_paged_split_t<T, TD, MT, BIAS, true>(a, plan, st) : launch_paged_split_t<T, TD, MT, BIAS, false>(a, plan, st);
    };
    return a.p.slopes                ? go(std::integral_constant<int, PAGED_SLOPES>())
           : a.p.R && a.factor_bytes ? go(std::integral_constant<int, PAGED_FACTORS>())
           : a.p.R                   ? go(std::integral_constant<int, PAGED_FACTORS_ANY>())
                                     : go(std::integral_constant<int, PAGED_PLAIN>());
  };
  auto by_rows = [&](auto t) {
    return plan.MT == 16 ? by_bias(t, std::integral_constant<int, 16>()) : by_bias(t, std::integral_constant<int, 32>());
  };
  return a.p.dtype == FB_DTYPE_F16 ? by_rows(__half()) : by_rows(__nv_bfloat16());
}

}  // namespace fb
