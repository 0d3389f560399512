// The plan of one serving step on the device: pages follow lengths, a stack of free pages follows the pages, and every new
// token gets its request, slot, position and the bits of its ancestors (the formulas stand at fb_plan_params).
//
// Bound by latency: a few kilobytes in and out, behind prefix sums over the requests.  One thread block, or one cluster of
// blocks when there are many tokens: the phases (count, give pages back, take pages, place tokens) are separated by barriers of
// the cluster, so the whole plan is a single launch.  Every block scans all requests by itself; the work behind the scans (pages,
// tokens) is spread over all threads of the cluster by flat index, found back by a search in the prefix sums.
// 64 requests of one token: 3.6 us a call in a graph; 256 trees of up to 64 tokens: 8.7.
#include <cooperative_groups.h>

#include "fb_common.cuh"
#include "fb_internal.h"

namespace fb {

constexpr int kPlanThreads = 1024, kPlanFewThreads = 128;
constexpr int kPlanMaxCluster = 8;  // blocks of a portable cluster
constexpr int kPlanMost = 0x7fff0000;  // tokens, requests: their counters go on by a cluster's threads, in 32 bits

// What a request asks for.  int64 where int32 inputs can pass 32 bits.
struct Ask {
  int len, held, need, tokens;
  bool valid;  // as far as the request alone tells, without the stack
};

// For each request of a chunk (as many as a block has threads).
template <int NT>
struct PlanShared {
  int64_t warp[2][32], total[2];
  int64_t pre[NT];   // exclusive prefix sums of the pages that are spread next
  int first[NT];     // the column where each request's part of them begins, -1: not served
  int cu[NT], len[NT];
  int taken;
};

__device__ __forceinline__ Ask plan_load(const fb_plan_params& p, int b) {
  Ask a = {0, 0, 0, 0, false};
  if (b >= p.B) return a;
  a.len = p.lens[b];
  a.tokens = p.new_lens[b];
  a.held = p.pages_held[b];
  return a;
}
// Completes what plan_load has read; the request's tokens begin at `tokens_before`.
__device__ __forceinline__ void plan_ask(const fb_plan_params& p, int b, int64_t tokens_before, Ask& a) {
  const int add = a.tokens;
  a.tokens = max(add, 0);
  const int64_t need = ((int64_t)a.len + a.tokens + p.page_size - 1) / p.page_size;
  const bool counted = a.held >= 0 && a.held <= p.table_width;
  a.valid = b < p.B && a.len >= 0 && add >= 0 && counted && need <= p.table_width && tokens_before + a.tokens <= p.num_tokens &&
            (!p.parents || a.tokens <= 64ll * p.mask_words);
  a.need = a.valid ? (int)need : a.held;
  if (!counted && p.status) *reinterpret_cast<volatile int32_t*>(p.status) = FB_DEV_BAD_INDEX;
}

// Exclusive prefix sums over the block of two values per thread, and their totals.
template <int NT>
__device__ __forceinline__ void block_scan(PlanShared<NT>& sh, int64_t& v0, int64_t& v1, int64_t& total0, int64_t& total1) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x0 = v0, x1 = v1;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y0 = __shfl_up_sync(0xffffffffu, x0, o), y1 = __shfl_up_sync(0xffffffffu, x1, o);
    if (lane >= o) x0 += y0, x1 += y1;
  }
  if (lane == 31) sh.warp[0][warp] = x0, sh.warp[1][warp] = x1;
  __syncthreads();
  if (warp < 2) {  // a warp per value
    const int64_t w = lane < NT / 32 ? sh.warp[warp][lane] : 0;
    int64_t z = w;
#pragma unroll
    for (int o = 1; o < NT / 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, z, o);
      if (lane >= o) z += y;
    }
    if (lane < NT / 32) sh.warp[warp][lane] = z - w;
    if (lane == NT / 32 - 1) sh.total[warp] = z;
  }
  __syncthreads();
  total0 = sh.total[0];
  total1 = sh.total[1];
  v0 = sh.warp[0][warp] + x0 - v0;
  v1 = sh.warp[1][warp] + x1 - v1;
  __syncthreads();
}

// The last i in [0, n) with pre[i] <= k.
__device__ __forceinline__ int find_part(const int64_t* pre, int n, int64_t k) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (pre[mid] <= k) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Pages given back: the k-th of the call goes to place top - 1 - k of the stack.
template <int NT>
__device__ __forceinline__ void push_pages(const fb_plan_params& p, PlanShared<NT>& sh, int base, int n, int64_t count, int64_t k0, int64_t top, int me,
                                           int nthreads) {
  for (int64_t k = me; k < count; k += nthreads) {
    const int i = find_part(sh.pre, n, k);
    const int64_t at = top - 1 - (k0 + k);
    if (at < p.stack_size) p.free_pages[at] = p.block_table[(base + i) * p.table_stride + sh.first[i] + (int)(k - sh.pre[i])];
    else if (p.status) *reinterpret_cast<volatile int32_t*>(p.status) = FB_DEV_BAD_INDEX;
  }
}
// Pages taken: the k-th of the call comes from place top - 1 - k.  (Read and written past L1: other blocks' writes.)
template <int NT>
__device__ __forceinline__ void pop_pages(const fb_plan_params& p, PlanShared<NT>& sh, int base, int n, int64_t count, int64_t k0, int64_t top, int me,
                                          int nthreads) {
  for (int64_t k = me; k < count; k += nthreads) {
    const int i = find_part(sh.pre, n, k);
    if (sh.first[i] < 0) continue;
    p.block_table[(base + i) * p.table_stride + sh.first[i] + (int)(k - sh.pre[i])] = __ldcg(p.free_pages + (top - 1 - (k0 + k)));
  }
}

// One new token: t-th of a request with `len` cached ones (-1: not served), whose first token is `first`.
__device__ __forceinline__ void place_token(const fb_plan_params& p, int n, int b, int first, int len) {
  int64_t slot = -1;
  const bool live = len >= 0;
  const int t = n - first;
  int pos = 0;
  if (live) {
    const uint32_t place = (uint32_t)(len + t), col = place / (uint32_t)p.page_size;  // (within the row: 31 bits)
    slot = (int64_t)__ldcg(p.block_table + b * p.table_stride + col) * p.page_size + (place - col * p.page_size);
    pos = p.parents ? len : (int)place;
  }
  if (p.parents) {
    int64_t* words = p.tree_mask + (int64_t)n * p.mask_words;
    int w = p.mask_words - 1;
    uint64_t bits = 0;
    // up the path: indices fall, so the walk ends
    for (int at = t; live && at >= 0;) {
      for (; w > (at >> 6); --w, bits = 0) words[w] = (int64_t)bits;
      bits |= 1ull << (at & 63);
      const int up = p.parents[first + at];
      if (up >= at) {
        if (p.status) *reinterpret_cast<volatile int32_t*>(p.status) = FB_DEV_BAD_INDEX;
        break;
      }
      if (up >= 0) ++pos;
      at = up;
    }
    for (; w >= 0; --w, bits = 0) words[w] = (int64_t)bits;
  }
  p.slots[n] = slot;
  p.positions[n] = pos;
}

// ONE: the requests fit one chunk, which is read once and kept in registers and shared memory.
template <int NT, bool ONE>
__global__ void __launch_bounds__(NT) paged_plan_kernel(const __grid_constant__ fb_plan_params p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ PlanShared<NT> sh;
  const int blocks = gridDim.x, rank = blockIdx.x, nthreads = blocks * NT, me = rank * NT + threadIdx.x;  // (the grid is one cluster)
  auto sync_all = [&] {
    if (blocks > 1) cluster.sync();
    else __syncthreads();
  };
  const int free_raw = *p.free_count;
  Ask a = plan_load(p, threadIdx.x);
  const int64_t free0 = min(max(free_raw, 0), p.stack_size);
  if (free0 != free_raw && threadIdx.x == 0 && p.status) *reinterpret_cast<volatile int32_t*>(p.status) = FB_DEV_BAD_INDEX;
  if (threadIdx.x == 0) sh.taken = 0;

  // ---- token offsets, pages that come back, pages that are missing
  int64_t given = 0, tokens = 0, avail = 0;
  for (int pass = ONE ? 1 : 0; pass < 2; ++pass) {  // (several chunks: the first pass counts what comes back)
    int64_t tok0 = 0, back0 = 0, more0 = 0;
    for (int base = 0; base < p.B; base += NT) {
      const int b = base + threadIdx.x, n = min(p.B - base, NT);
      if (!ONE) a = plan_load(p, b);
      int64_t before = max(a.tokens, 0), unused = 0, tot_tok, tot_unused, tot_back, tot_more;
      block_scan(sh, before, unused, tot_tok, tot_unused);
      before += tok0;
      plan_ask(p, b, before, a);
      const int back = max(a.held - a.need, 0), more = max(a.need - a.held, 0);
      int64_t pre_back = back, pre_more = more;
      block_scan(sh, pre_back, pre_more, tot_back, tot_more);
      if (pass == 1) {
        if (ONE) given = tot_back;
        avail = min(free0 + given, (int64_t)p.stack_size);
        const bool served = a.valid && (!more || more0 + pre_more + more <= avail);
        const int first = (int)min(before, (int64_t)p.num_tokens), len = served ? a.len : -1;
        if (b < p.B && rank == 0) {
          p.cu_tokens[b + 1] = (int)min(before + a.tokens, (int64_t)p.num_tokens);
          p.lens_out[b] = len;
          if (b == 0) p.cu_tokens[0] = 0;
        }
        if (served && more) atomicMax(&sh.taken, (int)(more0 + pre_more + more));
        sh.cu[threadIdx.x] = first;
        sh.len[threadIdx.x] = len;
        if (tot_back) {
          sh.pre[threadIdx.x] = pre_back;
          sh.first[threadIdx.x] = a.need;
          __syncthreads();
          push_pages(p, sh, base, n, tot_back, back0, free0 + given, me, nthreads);
          if (ONE && tot_more) sync_all();
          else __syncthreads();
        }
        if (ONE && tot_more) {
          sh.pre[threadIdx.x] = pre_more;
          sh.first[threadIdx.x] = served ? a.held : -1;
          __syncthreads();
          pop_pages(p, sh, base, n, tot_more, 0, avail, me, nthreads);
        }
      }
      tok0 += tot_tok;
      back0 += tot_back;
      more0 += tot_more;
    }
    given = back0;
    tokens = tok0;
  }
  sync_all();  // pages given back are on the stack; every block has read the state

  if (!ONE) {  // ---- pages taken, chunk by chunk
    int64_t tok0 = 0, more0 = 0;
    for (int base = 0; base < p.B; base += NT) {
      const int b = base + threadIdx.x, n = min(p.B - base, NT);
      a = plan_load(p, b);
      int64_t before = max(a.tokens, 0), unused = 0, tot_tok, tot_unused, tot_more;
      block_scan(sh, before, unused, tot_tok, tot_unused);
      plan_ask(p, b, tok0 + before, a);
      const int more = max(a.need - a.held, 0);
      int64_t pre_more = more;
      unused = 0;
      block_scan(sh, pre_more, unused, tot_more, tot_unused);
      sh.pre[threadIdx.x] = pre_more;
      sh.first[threadIdx.x] = a.valid && (!more || more0 + pre_more + more <= avail) ? a.held : -1;
      __syncthreads();
      pop_pages(p, sh, base, n, tot_more, more0, avail, me, nthreads);
      __syncthreads();
      tok0 += tot_tok;
      more0 += tot_more;
    }
    sync_all();
  }

  // ---- the tokens, and the state
  for (int n = me; n < p.num_tokens; n += nthreads) {
    int lo = 0, first = 0, len = -1;
    if (n < tokens) {
      int hi = p.B - 1;  // the last request whose tokens begin at or before n, of those that begin there the last
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if ((ONE ? sh.cu[mid] : p.cu_tokens[mid]) <= n) lo = mid;
        else hi = mid - 1;
      }
      first = ONE ? sh.cu[lo] : p.cu_tokens[lo];
      len = ONE ? sh.len[lo] : p.lens_out[lo];
    }
    place_token(p, n, lo, first, len);
  }
  if (rank == 0) {
    if (ONE) {
      if ((int)threadIdx.x < p.B && sh.len[threadIdx.x] >= 0) p.pages_held[threadIdx.x] = a.need;
    } else {
      for (int b = threadIdx.x; b < p.B; b += NT)
        if (p.lens_out[b] >= 0) p.pages_held[b] = (int)(((int64_t)p.lens_out[b] + max(p.new_lens[b], 0) + p.page_size - 1) / p.page_size);
    }
    if (threadIdx.x == 0) *p.free_count = (int)(avail - sh.taken);
  }
}

template <int NT, bool ONE>
static int launch_plan(const fb_plan_params& p, int blocks, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(NT);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = blocks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = blocks > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_plan_kernel<NT, ONE>, p);
  if (e == cudaSuccess) note_launch();
  return (int)e;
}

}  // namespace fb

using namespace fb;

extern "C" size_t fb_plan_params_size(void) { return sizeof(fb_plan_params); }

extern "C" int fb_paged_plan(const fb_plan_params* p, void* cuda_stream) {
  if (!p) return FB_EINVAL_NULL;
  if (p->B <= 0 || p->num_tokens < 0 || p->stack_size < 0 || p->B > kPlanMost || p->num_tokens > kPlanMost) return FB_EINVAL_SHAPE;
  if (p->page_size <= 0 || p->table_width <= 0 || (int64_t)p->table_width * p->page_size > 0x7fffffffLL) return FB_EINVAL_PAGE;
  if (p->table_stride < p->table_width) return FB_EINVAL_STRIDE;
  if (!p->block_table || !p->pages_held || !p->free_count || !p->lens || !p->new_lens || !p->cu_tokens || !p->lens_out) return FB_EINVAL_NULL;
  if (p->stack_size && !p->free_pages) return FB_EINVAL_NULL;
  if (p->num_tokens && (!p->positions || !p->slots)) return FB_EINVAL_NULL;
  if (p->parents && (!p->tree_mask || p->mask_words <= 0 || p->mask_words > 64)) return FB_EINVAL_MASK;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  // Few requests and tokens: a small block, whose barriers cost less (64 requests of one token: 10.0 us a call with 1024 threads
  // and the requests read in every phase).
  if (p->B <= kPlanFewThreads && p->num_tokens <= 4 * kPlanFewThreads) return launch_plan<kPlanFewThreads, true>(*p, 1, st);
  const int64_t want = ((int64_t)p->num_tokens + 2 * kPlanThreads - 1) / (2 * kPlanThreads);
  const int blocks = want < 1 ? 1 : want < kPlanMaxCluster ? (int)want : kPlanMaxCluster;
  return p->B <= kPlanThreads ? launch_plan<kPlanThreads, true>(*p, blocks, st) : launch_plan<kPlanThreads, false>(*p, blocks, st);
}
