// Attention of the newest tokens of every request over its pages: one token (decoding), several, or a tree of drafted ones.
//
//   logit = scale q.k + slope (pos_key - pos_token)  |  + q_bias . bias_cache;   o = softmax(logit) v, statistics in fp32
//
// Bound by reading K and V of every request once while there are few rows per key head, by the products beyond.  Here: the
// shape-generic kernel, the choice of the kernel and the entry points.
#include "fb_paged.cuh"

namespace fb {

// ---- general kernel: any head_dim up to 128, any strides; one block per (token, head), keys over its warps ---------
template <typename T>
__global__ void __launch_bounds__(128) paged_general_kernel(const __grid_constant__ fb_paged_params p) {
  __shared__ float qs[128], qbs[256], s_acc[4][128], s_m[4], s_l[4];
  const int n = blockIdx.x / p.Hq, h = blockIdx.x % p.Hq, hk = h / (p.Hq / p.Hk);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int lo = 0, hi = p.B - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu_at(p, mid + 1) > n) hi = mid;
    else lo = mid + 1;
  }
  const Request rq = request_at(p, lo);
  const int first = rq.first, len = rq.len, t = n - first;
  const bool live = t >= 0 && t < rq.tokens && len >= 0;
  const int64_t keys = live ? rq.keys : 0;
  const int my_pos = live ? (p.positions ? p.positions[n] : len + t) : 0;
  const float slope = p.slopes ? p.slopes[h] : 0.f;
  const int64_t* words = p.tree_mask ? p.tree_mask + n * p.mask_stride : nullptr;
  const T* q = reinterpret_cast<const T*>(p.q) + n * p.q_stride[0] + h * p.q_stride[1];
  for (int c = threadIdx.x; c < p.D; c += 128) qs[c] = to_f32(q[c]) * p.softmax_scale;
  if (p.R) {
    const T* qb = reinterpret_cast<const T*>(p.q_bias) + n * p.q_bias_stride[0] + h * p.q_bias_stride[1];
    for (int c = threadIdx.x; c < p.R; c += 128) qbs[c] = to_f32(qb[c]);
  }
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int64_t j0 = warp * 32; j0 < keys; j0 += 128) {
    const int64_t j = j0 + lane;
    int page = -1, place = 0;
    if (j < keys) {
      const int col = (int)(j / p.page_size);
      place = (int)(j - (int64_t)col * p.page_size);
      page = p.block_table[lo * p.table_stride + col];
      if (page < 0 || page >= p.num_pages) {
        paged_bad_index(p);
        page = -1;
      }
    }
    const int td = (int)(j - len);
    bool seen = page >= 0;
    if (seen && td >= 0) seen = words ? (td >> 6) < p.mask_words && ((words[td >> 6] >> (td & 63)) & 1) : td <= t;
    float s = -INFINITY;
    if (seen) {
      const T* k = reinterpret_cast<const T*>(p.key_cache) + page * p.key_cache_stride[0] + place * p.key_cache_stride[1] + hk * p.key_cache_stride[2];
      s = 0.f;
      for (int c = 0; c < p.D; ++c) s = fmaf(qs[c], to_f32(k[c]), s);
      if (p.slopes) {
        const int pos = td >= 0 && p.positions ? p.positions[first + td] : (int)j;
        s = fmaf(slope, (float)(pos - my_pos), s);
      }
      if (p.R) {
        const T* kb = reinterpret_cast<const T*>(p.bias_cache) + page * p.bias_cache_stride[0] + place * p.bias_cache_stride[1] +
                      (p.bias_heads > 1 ? hk * p.bias_cache_stride[2] : 0);
        for (int c = 0; c < p.R; ++c) s = fmaf(qbs[c], to_f32(kb[c]), s);
      }
    }
    float mx = s;
#pragma unroll
    for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    mx = fmaxf(m, mx);
    const float msub = fmaxf(mx, -FLT_MAX), alpha = fast_exp2((m - msub) * kLog2eP);
    m = mx;
    const float e = seen ? fast_exp2((s - msub) * kLog2eP) : 0.f;
    l = l * alpha + e;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= alpha;
    for (uint32_t left = __ballot_sync(0xffffffffu, seen); left; left &= left - 1) {  // (what is not seen is not read)
      const int src = __ffs(left) - 1;
      const float pe = __shfl_sync(0xffffffffu, e, src);
      const T* v = reinterpret_cast<const T*>(p.value_cache) + (int64_t)__shfl_sync(0xffffffffu, page, src) * p.value_cache_stride[0] +
                   __shfl_sync(0xffffffffu, place, src) * p.value_cache_stride[1] + hk * p.value_cache_stride[2];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 32 * i < p.D) acc[i] = fmaf(pe, to_f32(v[lane + 32 * i]), acc[i]);
    }
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
  for (int i = 0; i < 4; ++i) s_acc[warp][lane + 32 * i] = acc[i];
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  __syncthreads();
  m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  const float msub = fmaxf(m, -FLT_MAX);
  l = 0.f;
  float o = 0.f;
  for (int w = 0; w < 4; ++w) {
    const float f = fast_exp2((s_m[w] - msub) * kLog2eP);
    l += s_l[w] * f;
    o += s_acc[w][threadIdx.x] * f;
  }
  if (threadIdx.x < p.D)
    reinterpret_cast<T*>(p.o)[n * p.o_stride[0] + h * p.o_stride[1] + threadIdx.x] = from_f32<T>(l > 0.f ? o / l : l == 0.f ? 0.f : l);
  if (p.lse && threadIdx.x == 0) p.lse[(int64_t)n * p.Hq + h] = l > 0.f ? fmaf(fast_log2(l), kLn2P, m) : l == 0.f ? -INFINITY : l;
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
// Rows of a call and places of a request: 31 bits, less what the last tile and the copies ahead of it count beyond them.
constexpr int64_t kMostPlaces = 0x7fff0000LL;

static int validate_paged(const fb_paged_params* p) {
  if (!p) return FB_EINVAL_NULL;
  if (p->N <= 0 || p->B <= 0 || p->B > kMostPlaces || p->Hq <= 0 || p->Hk <= 0 || p->Hq % p->Hk || (int64_t)p->N * p->Hq > kMostPlaces) return FB_EINVAL_SHAPE;
  if (p->D <= 0 || p->D > 128 || p->R < 0 || p->R > 256) return FB_EINVAL_SHAPE;
  if (p->dtype != FB_DTYPE_F16 && p->dtype != FB_DTYPE_BF16) return FB_EINVAL_DTYPE;
  if (p->page_size <= 0 || p->table_width <= 0 || p->num_pages <= 0 || (int64_t)p->table_width * p->page_size > kMostPlaces) return FB_EINVAL_PAGE;
  if (!p->q || !p->key_cache || !p->value_cache || !p->block_table || !p->lens || !p->cu_tokens || !p->o) return FB_EINVAL_NULL;
  if (p->R) {
    if (!p->q_bias || !p->bias_cache || p->slopes || (p->bias_heads != 1 && p->bias_heads != p->Hk)) return FB_EINVAL_BIAS;
  } else if (p->q_bias || p->bias_cache) {
    return FB_EINVAL_BIAS;
  }
  if (p->tree_mask && (p->mask_words <= 0 || p->mask_stride < 0)) return FB_EINVAL_MASK;
  if (p->table_stride < 0) return FB_EINVAL_STRIDE;
  for (int i = 0; i < 3; ++i) {
    if (p->key_cache_stride[i] < 0 || p->value_cache_stride[i] < 0 || p->bias_cache_stride[i] < 0) return FB_EINVAL_STRIDE;
    if (i < 2 && (p->q_stride[i] < 0 || p->q_bias_stride[i] < 0 || p->o_stride[i] < 0)) return FB_EINVAL_STRIDE;
  }
  return 0;
}

// The kernel of a call.  Rows that are whole aligned 16-byte chunks take the split kernel.
static PagedPlan plan_paged(const fb_paged_params* p) {
  PagedPlan plan = {};
  uintptr_t bits = reinterpret_cast<uintptr_t>(p->q) | reinterpret_cast<uintptr_t>(p->key_cache) | reinterpret_cast<uintptr_t>(p->value_cache) |
                   reinterpret_cast<uintptr_t>(p->o);
  for (int i = 0; i < 3; ++i) {
    bits |= (uintptr_t)(p->key_cache_stride[i] | p->value_cache_stride[i]) * 2;
    if (i < 2) bits |= (uintptr_t)(p->q_stride[i] | p->o_stride[i]) * 2;
  }
  const int G = p->Hq / p->Hk;
  if ((p->flags & FB_FLAG_FORCE_GENERAL) || p->D % 8 || (bits & 15)) return plan;
  const int64_t rows = ((int64_t)p->N * G + p->B - 1) / p->B;  // per request on average
  int dev = 0;
  cudaGetDevice(&dev);
  const int sms = device_sm_count(dev) > 0 ? device_sm_count(dev) : 148;
  // Many rows: 128 of them in a tcgen05 tile, if a tile of 128 keys is made of whole pages (or a page of whole tiles) that TMA can
  // address, and the scale may be taken out of a maximum.  Wide rows sooner, because the other kernel's work grows with the columns
  // and with every 32 rows, this one's hardly.  Tile / split kernel, us (rows on average, half as many more in the largest trees):
  // 128 columns, 18 rows (B16 T12 H16-8) over 100 keys 14.1 / 14.9, over 1000 28.4 / 26.7, over 8000 74.9 / 87.3; 26 rows 14.2 / 16.7,
  // 28.5 / 31.1, 75.7 / 103; 64 columns, 45 rows (T30) over 1000 keys 25.1 / 21.0, over 8000 61.8 / 66.8, 68 rows 25.4 / 24.0 and
  // 62.0 / 76.8; 32 columns, 68 rows 24.9 / 18.7 and 59.9 / 57.2, 90 rows 24.9 / 22.5 and 61.2 / 73.8.  The lines weigh a
  // few per cent over 1000 keys against a fifth over 8000.  Just below those of 128 and 64 columns the tile kernel would be ahead over
  // 8000 keys and behind over 1000; a line that follows the table's length, which the host knows, has not been measured, nor have
  // batches of very uneven requests, which the average sends to one kernel.
  const int few = p->D <= 32 ? 80 : p->D <= 64 ? 48 : 24;
  const bool tma = tma_compatible(p->key_cache, p->key_cache_stride[1], p->key_cache_stride[2], p->key_cache_stride[0], p->Hk, p->num_pages) &&
                   tma_compatible(p->value_cache, p->value_cache_stride[1], p->value_cache_stride[2], p->value_cache_stride[0], p->Hk, p->num_pages);
  if (rows > few && !(p->flags & FB_FLAG_PAGED_SPLIT) && tma && p->R == 0 && p->softmax_scale > 1e-20f && p->page_size % 8 == 0 && (128 % p->page_size == 0 || p->page_size % 128 == 0) &&
      p->num_pages < 0x7fffffffLL) {
    plan.kernel = FB_PAGED_TILE;
    plan.TD = p->D <= 64 ? 64 : 128;
    plan.MT = 128;
    plan.WH = 1;
    plan.ctas = sms;
  } else {
    plan.kernel = FB_PAGED_SPLIT;
    plan.TD = p->D <= 32 ? 32 : p->D <= 64 ? 64 : 128;
    plan.MT = rows <= 16 ? 16 : 32;
    plan.ctas = split_ctas(plan.TD, plan.MT) * sms;
    // Key heads of an item, each a warp's (or, with fewer than four, several warps').  Four share the walk and the table and read
    // the cache in the longest runs, and leave the fewest items; few items are cut in more parts, each with a beginning, an end and
    // a place in the join.  us for 4 / 2 / 1 heads, D128 H32-8 but for the second: B256 L300..500 67.8 / 68.6 / 89.6, of 32 columns
    // 19.6 / 23.3 / 32.1; B64 L1000 39.8 / 38.2 / 43.0, B16 L3000 43.3 / 35.3 / 35.3, B8 L4000 26.4 / 21.4 / 19.3.
    const int64_t each = (int64_t)p->B * ((rows + plan.MT - 1) / plan.MT) * p->Hk;
    plan.WH = p->Hk % 4 == 0 && each >= 4 * plan.ctas ? 4 : p->Hk % 2 == 0 && 2 * each > plan.ctas ? 2 : 1;
  }
  // items: row tiles (of every request at least one) times head groups
  const int64_t items = (int64_t)p->B * ((rows + plan.MT - 1) / plan.MT) * (p->Hk / plan.WH);
  plan.many_parts = items * 8 < plan.ctas;
  // 12 rows over 11772 keys, two heads: 18.6 us with all CTAs (184 with two tiles each), 14.5 with 92.  Where an item has no more
  // than 32 parts it is the other way about (one token over 1000 keys, 8 heads: 10.6 us with a tile per CTA, 12.5 with four).
  plan.spread = plan.kernel == FB_PAGED_SPLIT && items * 32 < plan.ctas ? (int)(items * 32) : plan.ctas;
  // Few items: each to a cluster of CTAs, 16 or 8 of them, no second launch.  Every row tile that the requests may have, and those
  // of tokens that no request owns, gets a cluster.  Limited to one CTA per SM (two waves of clusters of 16 came out of 256: one
  // token of two requests over 1000 keys 18.2 us, 11.2 with the schedule) and to tables of 8192 keys: a cluster has fewer CTAs
  // than the GPU (one token over 4000 keys, 8 heads, 12.2 us both ways, over 16000 21.4, with the schedule 17.7).
  const int64_t busy = ((int64_t)p->N * G / plan.MT + p->B) * (p->Hk / plan.WH), clusters = busy + 2 * (p->Hk / plan.WH);
  if (plan.kernel == FB_PAGED_SPLIT && plan.WH == 1 && (int64_t)p->table_width * p->page_size <= 8192 && busy * 8 <= sms) {
    plan.cluster = busy * 16 <= sms ? 16 : 8;
    plan.ctas = (int)clusters * plan.cluster;
    plan.spread = plan.ctas;
    return plan;
  }
  const size_t prows = (size_t)plan.ctas * 2 * plan.WH * plan.MT;
  plan.part_bytes = round256(prows * plan.TD * 4);
  plan.ml_bytes = round256(prows * 8);
  plan.desc_bytes = round256((size_t)plan.ctas * 32);
  return plan;
}

}  // namespace fb

using namespace fb;

extern "C" size_t fb_paged_params_size(void) { return sizeof(fb_paged_params); }

extern "C" int fb_paged_kernel(const fb_paged_params* p) {
  const int rc = validate_paged(p);
  return rc ? rc : plan_paged(p).kernel;
}

extern "C" size_t fb_paged_workspace_bytes(const fb_paged_params* p) {
  if (validate_paged(p)) return 0;
  const PagedPlan plan = plan_paged(p);
  return plan.part_bytes + plan.ml_bytes + plan.desc_bytes;
}

extern "C" int fb_paged_fwd(const fb_paged_params* p, void* cuda_stream) {
  if (const int rc = validate_paged(p)) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  const PagedPlan plan = plan_paged(p);
  if (plan.kernel != FB_PAGED_GENERAL) {
    const size_t need = plan.part_bytes + plan.ml_bytes + plan.desc_bytes;
    if (need && (!p->workspace || p->workspace_bytes < need || (reinterpret_cast<uintptr_t>(p->workspace) & 255))) return FB_EINVAL_WORKSPACE;
    PagedArgs a = {};
    a.p = *p;
    a.G = p->Hq / p->Hk;
    a.page_div = Div(p->page_size);
    a.group_div = Div(a.G);
    a.spread = plan.spread;
    a.whole_tiles = p->page_size % 16 == 0;
    a.pages32 = (uint32_t)(p->num_pages < 0x7fffffffLL ? p->num_pages : 0x7fffffffLL);
    if (p->R) {  // what the rows of the factors are aligned to
      const uintptr_t bits = reinterpret_cast<uintptr_t>(p->bias_cache) |
                             (uintptr_t)(p->bias_cache_stride[0] | p->bias_cache_stride[1] | (p->bias_heads > 1 ? p->bias_cache_stride[2] : 0) | p->R) * 2;
      a.factor_words = !(bits & 3);
      a.factor_bytes = p->R > 16 ? 0 : !(bits & 15) ? 16 : !(bits & 7) ? 8 : !(bits & 3) ? 4 : 0;
    }
    a.scale_log2 = p->softmax_scale * kLog2eP;
    uint8_t* ws = reinterpret_cast<uint8_t*>(p->workspace);
    a.part = reinterpret_cast<float*>(ws);
    a.ml = reinterpret_cast<float2*>(ws + plan.part_bytes);
    a.desc = reinterpret_cast<int4*>(ws + plan.part_bytes + plan.ml_bytes);
    if (plan.kernel == FB_PAGED_TILE) return plan.TD == 64 ? launch_paged_tile_d64(a, plan, st) : launch_paged_tile_d128(a, plan, st);
    return plan.TD == 32 ? launch_paged_split_d32(a, plan, st) : plan.TD == 64 ? launch_paged_split_d64(a, plan, st) : launch_paged_split_d128(a, plan, st);
  }
  const unsigned grid = (unsigned)(p->N * p->Hq);
  if (p->dtype == FB_DTYPE_F16) paged_general_kernel<__half><<<grid, 128, 0, st>>>(*p);
  else paged_general_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(*p);
  note_launch();
  return (int)cudaGetLastError();
}
