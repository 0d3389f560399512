// The plan of one serving step on the device: pages follow lengths, a stack of free pages follows the pages, and every new
// token gets its request, slot, position and the bits of its ancestors (the formulas stand at fb_plan_params).
//
// Bound by latency: a few kilobytes in and out, behind prefix sums over the requests.  One thread block, or one cluster of
// blocks when there are many tokens: the phases (count, give pages back, take pages, place tokens) are separated by barriers of
// the cluster, so the whole plan is a single launch.  Every block scans all requests by itself; the work behind the scans (pages,
// tokens) is spread over all threads of the cluster by flat index, found back by a search in the prefix sums.
#include <cooperative_groups.h>

#include "fb_common.cuh"
#include "fb_internal.h"

namespace fb {

constexpr int kPlanThreads = 1024;
constexpr int kPlanChunk = kPlanThreads;  // requests scanned at a time
constexpr int kPlanMaxCluster = 8;        // blocks of a portable cluster

// What a request asks for.  int64 where int32 inputs can pass 32 bits.
struct Ask {
  int held, need, tokens;
  bool valid;  // as far as the request alone tells, without the stack
};

struct PlanShared {
  int64_t warp[3][32];
  int64_t total[3];
  int64_t pre[kPlanChunk + 1];  // exclusive prefix sums of what is spread next
  int first[kPlanChunk];        // and where each request's part begins
};

__device__ __forceinline__ Ask plan_ask(const fb_plan_params& p, int b, int64_t tokens_before) {
  Ask a;
  const int len = p.lens[b], add = p.new_lens[b];
  const int held = p.pages_held[b];
  a.tokens = max(add, 0);
  const int64_t all = (int64_t)len + a.tokens, need = (all + p.page_size - 1) / p.page_size;
  a.valid = len >= 0 && add >= 0 && held >= 0 && held <= p.table_width && need <= p.table_width &&
            tokens_before + a.tokens <= p.num_tokens && (!p.parents || a.tokens <= 64ll * p.mask_words);
  a.held = held;
  a.need = a.valid ? (int)need : held;
  if ((held < 0 || held > p.table_width) && p.status) *reinterpret_cast<volatile int32_t*>(p.status) = FB_DEV_BAD_INDEX;
  return a;
}

// Exclusive prefix sums over the block of one value per thread; the total in `total`.
__device__ __forceinline__ int64_t block_scan(PlanShared& sh, int slot, int64_t v, int64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) sh.warp[slot][warp] = x;
  __syncthreads();
  if (warp == 0) {
    const int64_t w = sh.warp[slot][lane];
    int64_t z = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, z, o);
      if (lane >= o) z += y;
    }
    sh.warp[slot][lane] = z - w;
    if (lane == 31) sh.total[slot] = z;
  }
  __syncthreads();
  total = sh.total[slot];
  const int64_t before = sh.warp[slot][warp] + x - v;
  __syncthreads();
  return before;
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

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const __grid_constant__ fb_plan_params p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ PlanShared sh;
  const int rank = cluster.block_rank(), nthreads = cluster.num_blocks() * kPlanThreads;
  const int me = rank * kPlanThreads + threadIdx.x;
  const int free0 = min(max(*p.free_count, 0), p.stack_size);

  // phase 1: token offsets, and pages that come back.  k-th page given back -> place free0 + given - 1 - k of the stack
  int64_t given = 0, tokens = 0;
  for (int pass = 0; pass < 2; ++pass) {
    int64_t tok0 = 0, back0 = 0;
    for (int base = 0; base < p.B; base += kPlanChunk) {
      const int b = base + threadIdx.x;
      const bool in = b < p.B;
      int64_t tot_tok, tot_back;
      const int add = in ? max(p.new_lens[b], 0) : 0;
      const int64_t before = tok0 + block_scan(sh, 0, add, tot_tok);
      Ask a = {0, 0, 0, false};
      if (in) a = plan_ask(p, b, before);
      const int back = a.held > a.need ? a.held - a.need : 0;
      const int64_t pre = block_scan(sh, 1, back, tot_back);
      if (pass == 1) {
        if (in && rank == 0) {
          const int64_t end = before + a.tokens;
          p.cu_tokens[b + 1] = (int)(end < p.num_tokens ? end : p.num_tokens);
          if (b == 0) p.cu_tokens[0] = 0;
        }
        sh.pre[threadIdx.x] = pre;
        sh.first[threadIdx.x] = a.need;
        __syncthreads();
        for (int64_t k = me; k < tot_back; k += nthreads) {
          const int i = find_part(sh.pre, kPlanChunk, k);
          const int64_t at = free0 + given - 1 - (back0 + k);
          const int col = sh.first[i] + (int)(k - sh.pre[i]);
          if (at < p.stack_size) p.free_pages[at] = p.block_table[(base + i) * p.table_stride + col];
          else if (p.status) *reinterpret_cast<volatile int32_t*>(p.status) = FB_DEV_BAD_INDEX;
        }
        __syncthreads();
      }
      tok0 += tot_tok;
      back0 += tot_back;
    }
    given = back0;
    tokens = tok0;
  }
  const int64_t avail = min(free0 + given, (int64_t)p.stack_size);
  cluster.sync();

  // phase 2: pages taken.  k-th page taken <- place avail - 1 - k
  int64_t taken = 0;
  {
    int64_t tok0 = 0, more0 = 0;
    for (int base = 0; base < p.B; base += kPlanChunk) {
      const int b = base + threadIdx.x;
      const bool in = b < p.B;
      int64_t tot_tok, tot_more;
      const int add = in ? max(p.new_lens[b], 0) : 0;
      const int64_t before = tok0 + block_scan(sh, 0, add, tot_tok);
      Ask a = {0, 0, 0, false};
      if (in) a = plan_ask(p, b, before);
      const int more = a.need > a.held ? a.need - a.held : 0;
      const int64_t pre = block_scan(sh, 1, more, tot_more);
      const bool served = a.valid && (!more || more0 + pre + more <= avail);
      sh.pre[threadIdx.x] = pre;
      sh.first[threadIdx.x] = served ? a.held : -1;
      if (in && rank == 0) p.lens_out[b] = served ? p.lens[b] : -1;
      // what has been taken when the last served request has its pages
      int64_t mine = served && more ? more0 + pre + more : 0;
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        const int64_t y = __shfl_xor_sync(0xffffffffu, mine, o);
        mine = y > mine ? y : mine;
      }
      if ((threadIdx.x & 31) == 0) sh.warp[2][threadIdx.x >> 5] = mine;
      __syncthreads();
      for (int w = 0; w < 32; ++w) taken = sh.warp[2][w] > taken ? sh.warp[2][w] : taken;
      for (int64_t k = me; k < tot_more; k += nthreads) {
        const int i = find_part(sh.pre, kPlanChunk, k);
        if (sh.first[i] < 0) continue;
        const int col = sh.first[i] + (int)(k - sh.pre[i]);
        p.block_table[(base + i) * p.table_stride + col] = p.free_pages[avail - 1 - (more0 + k)];
      }
      __syncthreads();
      tok0 += tot_tok;
      more0 += tot_more;
    }
  }
  cluster.sync();

  // phase 3: the tokens, and the state
  for (int n = me; n < p.num_tokens; n += nthreads) {
    int64_t slot = -1;
    int pos = 0, first = 0, t = 0;
    bool live = false;
    if (n < tokens) {
      int lo = 0, hi = p.B - 1;  // the request: the first b with cu[b + 1] > n
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (p.cu_tokens[mid + 1] > n) hi = mid;
        else lo = mid + 1;
      }
      const int len = p.lens_out[lo];
      if (len >= 0) {
        live = true;
        first = p.cu_tokens[lo];
        t = n - first;
        const uint32_t place = (uint32_t)(len + t), col = place / (uint32_t)p.page_size;  // (within the row: 31 bits)
        slot = (int64_t)p.block_table[lo * p.table_stride + col] * p.page_size + (place - col * p.page_size);
        pos = p.parents ? len : (int)place;
      }
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
  if (rank == 0) {
    for (int b = threadIdx.x; b < p.B; b += kPlanThreads)
      if (p.lens_out[b] >= 0) p.pages_held[b] = (int)(((int64_t)p.lens_out[b] + max(p.new_lens[b], 0) + p.page_size - 1) / p.page_size);
    if (threadIdx.x == 0) *p.free_count = (int)(avail - taken);
  }
}

}  // namespace fb

using namespace fb;

extern "C" size_t fb_plan_params_size(void) { return sizeof(fb_plan_params); }

extern "C" int fb_paged_plan(const fb_plan_params* p, void* cuda_stream) {
  if (!p) return FB_EINVAL_NULL;
  if (p->B <= 0 || p->num_tokens < 0 || p->stack_size < 0) return FB_EINVAL_SHAPE;
  if (p->page_size <= 0 || p->table_width <= 0 || (int64_t)p->table_width * p->page_size > 0x7fffffffLL) return FB_EINVAL_PAGE;
  if (p->table_stride < p->table_width) return FB_EINVAL_STRIDE;
  if (!p->block_table || !p->pages_held || !p->free_count || !p->lens || !p->new_lens || !p->cu_tokens || !p->lens_out) return FB_EINVAL_NULL;
  if (p->stack_size && !p->free_pages) return FB_EINVAL_NULL;
  if (p->num_tokens && (!p->positions || !p->slots)) return FB_EINVAL_NULL;
  if (p->parents && (!p->tree_mask || p->mask_words <= 0 || p->mask_words > 64)) return FB_EINVAL_MASK;
  // one block up to four tokens a thread
  const int64_t want = ((int64_t)p->num_tokens + 4 * kPlanThreads - 1) / (4 * kPlanThreads);
  const unsigned blocks = want < 1 ? 1 : want < kPlanMaxCluster ? (unsigned)want : kPlanMaxCluster;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.stream = reinterpret_cast<cudaStream_t>(cuda_stream);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = blocks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_plan_kernel, *p);
  if (e == cudaSuccess) note_launch();
  return (int)e;
}
