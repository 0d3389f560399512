// Shared by the kernels of attention over pages: offsets and lengths as the device arrays hold them, and the schedule that
// cuts the work of a call into equal parts.
//
// The lengths live on the device and a call reads nothing back, so the grid cannot follow them.  Instead the key tiles of all
// (request, row tile, head group) items are numbered through, and CTA c of a fixed grid takes the numbers from c U / C to
// (c + 1) U / C: every CTA reads the same amount of K and V whatever the lengths are.  An item that spans several CTAs leaves
// unnormalised sums in the workspace, at most two per CTA, and a second small kernel joins them in the order of the CTAs.
#pragma once

#include <float.h>

#include <type_traits>

#include "fb_common.cuh"
#include "fb_internal.h"

namespace fb {

constexpr float kLog2eP = 1.4426950408889634f;
constexpr float kLn2P = 0.6931471805599453f;

// P is rounded to the 16 bits of V.  fp16 ends at 2^-24, and many keys of less than that beside a large one may be all of a row's
// result: there the probabilities, and the row's sum with them, are 2^15 times as large in the split kernel (which has them at most
// one) and 2^7 times in the tile kernel (2^8).
template <typename T>
constexpr float kSplitLift = std::is_same<T, __half>::value ? 15.f : 0.f;
template <typename T>
constexpr float kTileLift = std::is_same<T, __half>::value ? 7.f : 0.f;

// 16 bytes to shared memory; zeros, and nothing is read, where they do not exist
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16u : 0u) : "memory");
}

struct PagedArgs {
  fb_paged_params p;
  Div page_div, group_div;  // by page_size, by the query heads of a key head
  int G;                    // query heads of a key head
  int spread;               // more CTAs than this only if each has four key tiles: the parts of an item have to be joined again
  int whole_tiles;          // split kernel: pages are whole runs of 16 keys
  uint32_t pages32;         // num_pages, within 31 bits: what a page of the table is compared with
  int factor_words;         // split kernel: factor rows can be read two columns at a time
  int factor_bytes;         // split kernel: pieces in which a key's factors are copied; 0: not
  float scale_log2;         // tile kernel
  float* part;    // (CTAs, 2, heads of a group, rows of a tile, columns): sums of items that span CTAs
  float2* ml;     // the same without columns: maximum (tile kernel: in quarters of log2 units) and sum
  int4* desc;     // (CTAs, 2): the item that begins in a CTA and ends in another: row tile, head group, last CTA, -; first token,
                  // rows of the request; a row tile of -1: none
};

__device__ __forceinline__ void paged_bad_index(const fb_paged_params& p) {
  if (p.status) *reinterpret_cast<volatile int32_t*>(p.status) = FB_DEV_BAD_INDEX;
}

// Offsets within [0, N], whatever the device array holds.
__device__ __forceinline__ int cu_at(const fb_paged_params& p, int b) { return min(max(p.cu_tokens[b], 0), p.N); }

// A request as the kernels see it.  Two more than p.B: the tokens behind the last request and before the first one, as
// requests without keys, so that their rows are written.
struct Request {
  int first, tokens, len, keys;  // keys: cached and new ones, 0 where the request is not served
};
__device__ __forceinline__ Request request_at(const fb_paged_params& p, int b) {
  Request r;
  if (b >= p.B) {
    const int at = cu_at(p, b == p.B ? p.B : 0);
    r.first = b == p.B ? at : 0;
    r.tokens = b == p.B ? p.N - at : at;
    r.len = -1;
    r.keys = 0;
    return r;
  }
  const int c0 = p.cu_tokens[b], c1 = p.cu_tokens[b + 1];
  r.first = min(max(c0, 0), p.N);
  r.tokens = max(min(max(c1, 0), p.N) - r.first, 0);
  r.len = p.lens[b];
  if (c0 < 0 || c1 > p.N || c1 < c0) paged_bad_index(p);
  int64_t keys = r.len < 0 ? 0 : (int64_t)r.len + r.tokens;
  const int64_t room = (int64_t)p.table_width * p.page_size;
  if (keys > room) {
    paged_bad_index(p);
    keys = room;
  }
  r.keys = (int)keys;
  return r;
}

// One item of a request, and the part of its key tiles that a CTA takes.
struct Segment {
  int b, rt, hg;     // request, row tile, head group
  int t0, t1, tiles;  // key tiles [t0, t1) of `tiles`
  int last_cta;      // the CTA that holds the item's last tile
  Request r;
};

// 64-bit numbers that are 32 bits long almost always: their division is four times as long otherwise.
__device__ __forceinline__ int64_t quotient(int64_t n, int64_t d) {
  return ((n | d) >> 32) == 0 ? (int64_t)((uint32_t)n / (uint32_t)d) : n / d;
}

// Walks the segments of one CTA.  Every thread of the block calls it alike.
template <int KT, int MT, int THREADS>
struct PagedWalk {
  int64_t u, u1, pre;  // next number, end of the CTA's range, first number of request b
  int64_t total;
  int b, ngroups, ctas;
  Request r;

  __device__ __forceinline__ static int row_tiles(const PagedArgs& a, const Request& r) { return (int)(((int64_t)r.tokens * a.G + MT - 1) / MT); }
  __device__ __forceinline__ static int key_tiles(const Request& r) { return max((int)(((int64_t)r.keys + KT - 1) / KT), 1); }
  __device__ __forceinline__ static int64_t units(const PagedArgs& a, const Request& r, int ngroups) {
    return r.tokens ? (int64_t)row_tiles(a, r) * key_tiles(r) * ngroups : 0;
  }

  // Finds the request in which the range of CTA `me` of `n` begins: each thread adds up a run of requests, a scan over the threads.
  __device__ __forceinline__ void start(const PagedArgs& a, int groups, int me, int n) {
    __shared__ int64_t s_sum[THREADS / 32], s_pre;
    __shared__ int s_b;
    __shared__ Request s_r;
    ngroups = groups;
    const int nr = a.p.B + 2, per = (nr + THREADS - 1) / THREADS, b0 = threadIdx.x * per, b1 = min(b0 + per, nr);
    int64_t mine = 0;
    Request mr = {0, 0, -1, 0};  // the last of the run: all of it while there are fewer requests than threads
    for (int i = b0; i < b1; ++i) mine += units(a, mr = request_at(a.p, i), groups);
    int64_t x = mine;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) s_sum[warp] = x;
    if (threadIdx.x == 0) s_b = -1;
    __syncthreads();
    int64_t before = x - mine;
    total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) before += s_sum[w];
      total += s_sum[w];
    }
    // each of these has one number at least: an item's parts leave no gap
    ctas = (int)min(min((int64_t)n, total), max((int64_t)a.spread, total / 4));
    u = me < ctas ? quotient(me * total, ctas) : total;
    u1 = me < ctas ? quotient((me + 1) * total, ctas) : total;
    if (u < u1 && before <= u && u < before + mine) {
      int64_t at = before;
      int i = b0;
      for (; per > 1; ++i) {
        const int64_t k = units(a, mr = request_at(a.p, i), groups);
        if (u < at + k) break;
        at += k;
      }
      s_b = i;
      s_pre = at;
      s_r = mr;
    }
    __syncthreads();
    b = s_b;
    pre = s_pre;
    r = s_r;
  }

  __device__ __forceinline__ bool next(const PagedArgs& a, Segment& s) {
    if (u >= u1) return false;
    int64_t k;
    while (u >= pre + (k = units(a, r, ngroups))) {  // (ends: u lies below the sum of all)
      pre += k;
      r = request_at(a.p, ++b);
    }
    s.b = b;
    s.r = r;
    s.tiles = key_tiles(r);
    const int64_t local = u - pre, item = quotient(local, s.tiles);
    const int rts = row_tiles(a, r);
    s.hg = (int)quotient(item, rts);
    s.rt = (int)(item - (int64_t)s.hg * rts);
    s.t0 = (int)(local - item * s.tiles);
    s.t1 = (int)min((int64_t)s.tiles, s.t0 + (u1 - u));
    const int64_t end = pre + (item + 1) * s.tiles;  // CTA c holds number n if c U / C <= n: the last one for n = end - 1
    s.last_cta = (int)quotient(end * ctas - 1, total);
    u += s.t1 - s.t0;
    return true;
  }
};

// Whether drafted token td of the request is seen by token t (global token n).
__device__ __forceinline__ bool tree_sees(const fb_paged_params& p, int n, int t, int td) {
  if (!p.tree_mask) return td <= t;
  const int w = td >> 6;
  return w < p.mask_words && ((p.tree_mask[n * p.mask_stride + w] >> (td & 63)) & 1);
}

// The 32 keys from drafted token td0 on (negative: cached ones) that a row of token t (global token n) sees, as bits.
__device__ __forceinline__ uint32_t seen_bits(const fb_paged_params& p, int n, int t, int td0) {
  if (!p.tree_mask) return td0 > t ? 0u : t - td0 >= 31 ? 0xffffffffu : (2u << (t - td0)) - 1u;
  const int64_t* words = p.tree_mask + n * p.mask_stride;
  auto word = [&](int w) { return w < 0 ? ~0ull : w < p.mask_words ? (uint64_t)words[w] : 0ull; };
  const int w = td0 >> 6, s = td0 & 63;
  return (uint32_t)(s ? (word(w) >> s) | (word(w + 1) << (64 - s)) : word(w));
}

// ---- host side (fb_paged.cu, fb_paged_split_*.cu, fb_paged_tile_*.cu) ------------------------------------------------
// CTAs of the split kernel that an SM holds: three while their warps' output rows leave the registers for it
constexpr int split_ctas(int TD, int MT) { return TD < 128 && MT == 16 ? 3 : 2; }
struct PagedPlan {
  int kernel;  // FB_PAGED_*
  int TD, MT;  // columns and rows of a tile
  int WH;      // key heads of a group
  int ctas;
  int spread;       // of PagedArgs
  int cluster;      // split kernel: CTAs of an item, in one cluster; 0: the schedule
  bool many_parts;  // items are spread over more than eight CTAs on average, if they are as long as the table can hold
  size_t part_bytes, ml_bytes, desc_bytes;
};
int launch_paged_split_d32(const PagedArgs& a, const PagedPlan& plan, cudaStream_t st);
int launch_paged_split_d64(const PagedArgs& a, const PagedPlan& plan, cudaStream_t st);
int launch_paged_split_d128(const PagedArgs& a, const PagedPlan& plan, cudaStream_t st);
int launch_paged_tile_d64(const PagedArgs& a, const PagedPlan& plan, cudaStream_t st);
int launch_paged_tile_d128(const PagedArgs& a, const PagedPlan& plan, cudaStream_t st);

// Joins the parts of the item that begins in CTA blockIdx.x; TD / 4 lanes per row, the parts in the order of the CTAs.  Latency
// is all there is to it: what the rows need stands in the descriptor, and the first parts are on their way before the maximum
// is known.  ROWS: rows of a block; where few items are spread over many CTAs one, whose parts the block's lanes share (12 rows
// over 11772 keys, two heads, 148 parts each: 34 us a call with four rows per block).
constexpr int kJoinThreads = 128;  // (of 512 an SM holds one, and most have nothing to join)
template <typename T, int TD, int ROWS>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ PagedArgs a, const int WH, const int MT) {
  constexpr int LANES = TD / 4, U = 8, SHARE = kJoinThreads / LANES / ROWS;  // lanes of a row, parts in flight, groups of lanes of a row
  __shared__ float4 s_acc[SHARE > 1 ? kJoinThreads : 1];
  __shared__ float2 s_ml[SHARE > 1 ? SHARE : 1];
  grid_dep_wait();
  const int4 d = a.desc[2 * blockIdx.x], e = a.desc[2 * blockIdx.x + 1];
  if (d.x < 0) return;
  const fb_paged_params& p = a.p;
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES, share = SHARE > 1 ? group : 0;
  const int idx = blockIdx.y * ROWS + (SHARE > 1 ? 0 : group);
  const int wh = idx / MT, r = idx - wh * MT, gr = d.x * MT + r, all = d.z - (int)blockIdx.x + 1;
  if (gr >= e.y) return;  // (SHARE > 1: the whole block)
  const int64_t step = (int64_t)2 * WH * MT;  // rows of a CTA
  const int64_t row0 = blockIdx.x * step + (int64_t)(WH + wh) * MT + r, row1 = (int64_t)(blockIdx.x + 1) * step + (int64_t)wh * MT + r;
  // this group's parts: share, share + SHARE, ...
  const int parts = (all - share + SHARE - 1) / SHARE;
  auto row_of = [&](int i) { return i * SHARE + share == 0 ? row0 : row1 + (i * SHARE + share - 1) * step; };
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (parts > 0) {
    float4 v[U];
    float2 s[U];
    auto load = [&](int i0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t row = row_of(min(i0 + u, parts - 1));
        s[u] = a.ml[row];
        v[u] = reinterpret_cast<const float4*>(a.part + row * TD)[lane];
      }
    };
    load(0);
#pragma unroll
    for (int u = 0; u < U; ++u) m = fmaxf(m, s[u].x);
#pragma unroll 4
    for (int i = U; i < parts; ++i) m = fmaxf(m, a.ml[row_of(i)].x);
    const float ms = fmaxf(m, -FLT_MAX);
    for (int i0 = 0;;) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i0 + u >= parts) break;
        const float f = fast_exp2((s[u].x - ms) * kLog2eP);
        l = fmaf(s[u].y, f, l);
        acc = make_float4(fmaf(v[u].x, f, acc.x), fmaf(v[u].y, f, acc.y), fmaf(v[u].z, f, acc.z), fmaf(v[u].w, f, acc.w));
      }
      if ((i0 += U) >= parts) break;
      load(i0);
    }
  }
  if (SHARE > 1) {
    s_acc[threadIdx.x] = acc;
    if (lane == 0) s_ml[share] = make_float2(m, l);
    __syncthreads();
    if (share > 0) return;
    for (int g = 0; g < SHARE; ++g) m = fmaxf(m, s_ml[g].x);
    const float ms = fmaxf(m, -FLT_MAX);
    l = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int g = 0; g < SHARE; ++g) {
      const float f = fast_exp2((s_ml[g].x - ms) * kLog2eP);
      const float4 v = s_acc[g * LANES + lane];
      l = fmaf(s_ml[g].y, f, l);
      acc = make_float4(fmaf(v.x, f, acc.x), fmaf(v.y, f, acc.y), fmaf(v.z, f, acc.z), fmaf(v.w, f, acc.w));
    }
  }
  const int t = a.group_div.quot32(gr), h = (d.y * WH + wh) * a.G + gr - t * a.G, n = e.x + t;
  const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
  if (lane * 4 < p.D)  // D is a multiple of 8
    *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.o) + n * p.o_stride[0] + h * p.o_stride[1] + lane * 4) =
        l == 0.f ? make_uint2(0u, 0u) : make_uint2(Pack2<T>::pack(acc.x * inv, acc.y * inv), Pack2<T>::pack(acc.z * inv, acc.w * inv));
  if (p.lse && lane == 0) p.lse[(int64_t)n * p.Hq + h] = l > 0.f ? fmaf(fast_log2(l) - kSplitLift<T>, kLn2P, m) : l == 0.f ? -INFINITY : l;
}

// launch_pdl (fb_internal.h) with a grid of two dimensions and no dynamic shared memory
template <typename... P, typename... A>
int launch_pdl_2d(void (*kern)(P...), dim3 grid, unsigned block, cudaStream_t st, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...);
  if (e == cudaSuccess) note_launch();
  return (int)e;
}

// (an item may begin in any CTA and end in a later one)
template <int TD>
int launch_paged_join(const PagedArgs& a, const PagedPlan& plan, cudaStream_t st) {
  constexpr int ROWS = kJoinThreads / (TD / 4);
  auto go = [&](auto t, auto rows) {
    return launch_pdl_2d(paged_join_kernel<decltype(t), TD, decltype(rows)::value>, dim3(plan.ctas, plan.WH * plan.MT / decltype(rows)::value), kJoinThreads,
                         st, a, plan.WH, plan.MT);
  };
  auto by_parts = [&](auto t) {
    return plan.many_parts ? go(t, std::integral_constant<int, 1>()) : go(t, std::integral_constant<int, ROWS>());
  };
  return a.p.dtype == FB_DTYPE_F16 ? by_parts(__half()) : by_parts(__nv_bfloat16());
}

}  // namespace fb
