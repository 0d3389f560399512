// Norm of queries and keys per head with the rotation by position in the same pass, forward and backward, and the serving
// form that writes keys and values into the pages of a cache.
//
//   r = rsqrt(mean(x^2) + eps),  y = x r w,  (out_lo, out_hi) = (y_lo c - y_hi s, y_hi c + y_lo s)
//   g = rotation of dout by the opposite angle,  dw = sum over rows of g x r,  dx = r (w g - x r^2 mean(w g x))
//
// Bound by reading x (and dout) once and writing the result once.  The angle position * inv_freq is taken in 64 bits and
// reduced to a fraction of a turn before its sine and cosine are taken in 32, by the functions of the hardware: off by 2^-21, and the
// rounding of the fraction and of its product with 2 pi by half as much again.  Results of 16 bits do not show it (an eighth of a
// percent of a step of fp16); a term of a weight's gradient in fp32 carries it, several roundings of its own.  At position 1e6 a
// 32-bit product is off by up to 0.03 rad.  It costs one pair of
// functions per token and frequency, shared by the token's heads, so no table is kept.
#include "fb_rope.cuh"

namespace fb {

constexpr int kRopeWarps = 4;
constexpr int kRopeThreads = 32 * kRopeWarps;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ---- general kernels: any D up to 128, any strides; a warp per row ------------------------------------------------
template <typename T, bool APPEND>
__global__ void __launch_bounds__(kRopeThreads) rope_general_kernel(const __grid_constant__ fb_rope_params p) {
  __shared__ float2 turn[kRopeMaxD / 2];
  __shared__ float rows[kRopeWarps][kRopeMaxD];
  const int b = blockIdx.x / p.S, s = blockIdx.x % p.S;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = p.rot >> 1;
  if (threadIdx.x < half) turn[threadIdx.x] = rope_turn(p, b, s, threadIdx.x);
  __syncthreads();
  int64_t page = 0;
  int place = 0;
  const bool cached = APPEND && cache_place(p, s, page, place);
  float* row = rows[warp];
  for (int r = warp; r < p.Hq + p.Hk; r += kRopeWarps) {
    const bool is_q = r < p.Hq;
    const int h = is_q ? r : r - p.Hq;
    if (APPEND && !is_q && !cached) break;
    const int64_t* xs = is_q ? p.q_stride : p.k_stride;
    const T* x = reinterpret_cast<const T*>(is_q ? p.q : p.k) + b * xs[0] + h * xs[1] + s * xs[2];
    const void* w = is_q ? p.q_weight : p.k_weight;
    T* y;
    if (APPEND && !is_q) {
      y = reinterpret_cast<T*>(p.key_cache) + page * p.key_cache_stride[0] + place * p.key_cache_stride[1] + h * p.key_cache_stride[2];
    } else {
      const int64_t* ys = is_q ? p.q_out_stride : p.k_out_stride;
      y = reinterpret_cast<T*>(is_q ? p.q_out : p.k_out) + b * ys[0] + h * ys[1] + s * ys[2];
    }
    float ss = 0.f;
    for (int c = lane; c < p.D; c += 32) {
      const float v = to_f32(x[c]);
      row[c] = v;
      ss += v * v;
    }
    __syncwarp();
    if (w) {
      const float rr = rsqrtf(warp_sum(ss) / p.D + p.eps);
      for (int c = lane; c < p.D; c += 32) row[c] = row[c] * rr * load_scalar(w, p.weight_dtype, c);
      __syncwarp();
    }
    for (int i = lane; i < half; i += 32) {
      const int lo = p.interleaved ? 2 * i : i, hi = p.interleaved ? 2 * i + 1 : i + half;
      const float2 cs = turn[i];
      y[lo] = from_f32<T>(row[lo] * cs.x - row[hi] * cs.y);
      y[hi] = from_f32<T>(row[hi] * cs.x + row[lo] * cs.y);
    }
    for (int c = p.rot + lane; c < p.D; c += 32) y[c] = w ? from_f32<T>(row[c]) : x[c];  // (untouched values keep their bits)
    __syncwarp();
  }
  if constexpr (APPEND) {
    if (!cached) return;
    for (int i = threadIdx.x; i < p.Hk * p.D; i += kRopeThreads) {
      const int h = i / p.D, c = i - h * p.D;
      reinterpret_cast<T*>(p.value_cache)[page * p.value_cache_stride[0] + place * p.value_cache_stride[1] + h * p.value_cache_stride[2] + c] =
          reinterpret_cast<const T*>(p.v)[h * p.v_stride[1] + s * p.v_stride[2] + c];
    }
    for (int i = threadIdx.x; i < p.bias_heads * p.R; i += kRopeThreads) {
      const int h = i / p.R, c = i - h * p.R;
      reinterpret_cast<T*>(p.bias_cache)[page * p.bias_cache_stride[0] + place * p.bias_cache_stride[1] + h * p.bias_cache_stride[2] + c] =
          reinterpret_cast<const T*>(p.k_bias)[h * p.k_bias_stride[1] + s * p.k_bias_stride[2] + c];
    }
  }
}

// Partial sums of the weight gradients: (CTAs, 2, D) floats.
template <typename T>
__global__ void __launch_bounds__(kRopeThreads) rope_bwd_general_kernel(const __grid_constant__ fb_rope_params p, int64_t tokens) {
  __shared__ float2 turn[kRopeMaxD / 2];
  __shared__ float rows[kRopeWarps][2 * kRopeMaxD];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = p.rot >> 1;
  float* row = rows[warp];         // x
  float* grad = row + kRopeMaxD;   // dout, then g
  float dw[2][kRopeMaxD / 32] = {};
  for (int64_t tok = blockIdx.x; tok < tokens; tok += gridDim.x) {
    const int b = (int)(tok / p.S), s = (int)(tok % p.S);
    __syncthreads();
    if (threadIdx.x < half) turn[threadIdx.x] = rope_turn(p, b, s, threadIdx.x);
    __syncthreads();
    for (int r = warp; r < p.Hq + p.Hk; r += kRopeWarps) {
      const bool is_q = r < p.Hq;
      const int h = is_q ? r : r - p.Hq;
      const int64_t *xs = is_q ? p.q_stride : p.k_stride, *gs = is_q ? p.dq_out_stride : p.dk_out_stride,
                    *ds = is_q ? p.dq_stride : p.dk_stride;
      const T* x = reinterpret_cast<const T*>(is_q ? p.q : p.k) + b * xs[0] + h * xs[1] + s * xs[2];
      const T* go = reinterpret_cast<const T*>(is_q ? p.dq_out : p.dk_out) + b * gs[0] + h * gs[1] + s * gs[2];
      T* dx = reinterpret_cast<T*>(is_q ? p.dq : p.dk) + b * ds[0] + h * ds[1] + s * ds[2];
      const void* w = is_q ? p.q_weight : p.k_weight;
      for (int c = lane; c < p.D; c += 32) grad[c] = to_f32(go[c]);
      __syncwarp();
      for (int i = lane; i < half; i += 32) {
        const int lo = p.interleaved ? 2 * i : i, hi = p.interleaved ? 2 * i + 1 : i + half;
        const float2 cs = turn[i];
        const float gl = grad[lo], gh = grad[hi];
        grad[lo] = gl * cs.x + gh * cs.y;
        grad[hi] = gh * cs.x - gl * cs.y;
      }
      __syncwarp();
      if (!w) {
        for (int c = lane; c < p.D; c += 32) dx[c] = c < p.rot ? from_f32<T>(grad[c]) : go[c];
        __syncwarp();
        continue;
      }
      float ss = 0.f, sg = 0.f;
      for (int c = lane; c < p.D; c += 32) {
        const float v = to_f32(x[c]);
        row[c] = v;
        ss += v * v;
        sg += v * grad[c] * load_scalar(w, p.weight_dtype, c);
      }
      const float rr = rsqrtf(warp_sum(ss) / p.D + p.eps), mean = warp_sum(sg) / p.D;
#pragma unroll
      for (int j = 0; j < kRopeMaxD / 32; ++j) {
        const int c = lane + 32 * j;
        if (c >= p.D) break;
        const float xr = row[c] * rr;
        if (is_q) dw[0][j] += grad[c] * xr;
        else dw[1][j] += grad[c] * xr;
        dx[c] = from_f32<T>(rr * (load_scalar(w, p.weight_dtype, c) * grad[c] - xr * (rr * mean)));
      }
      __syncwarp();
    }
  }
  if (!p.workspace) return;
  float* part = reinterpret_cast<float*>(p.workspace) + (int64_t)blockIdx.x * 2 * p.D;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kRopeMaxD / 32; ++j) row[lane + 32 * j] = dw[t][j];
    __syncthreads();
    for (int c = threadIdx.x; c < p.D; c += kRopeThreads) {
      float v = 0.f;
      for (int w = 0; w < kRopeWarps; ++w) v += rows[w][c];
      part[t * p.D + c] = v;
    }
  }
}

// Adds up the blocks' partial sums in their order.  Block (32, 32): 32 columns of one weight, the partial sums spread over the
// other dimension.  Tensor t has `parts` of them, `step` floats apart, from t * first on.
struct WeightParts {
  int parts[2];
  int64_t first, step;
};
__global__ void __launch_bounds__(1024) rope_weight_kernel(const __grid_constant__ fb_rope_params p, const WeightParts q) {
  __shared__ float s[32][33];
  grid_dep_wait();
  const int c = blockIdx.x * 32 + threadIdx.x, t = blockIdx.y;
  const float* part = reinterpret_cast<const float*>(p.workspace) + t * q.first + c;
  float v = 0.f;
  if (c < p.D) {
#pragma unroll 8
    for (int i = threadIdx.y; i < q.parts[t]; i += 32) v += part[i * q.step];
  }
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y) return;
  v = 0.f;
  for (int i = 0; i < 32; ++i) v += s[i][threadIdx.x];
  void* out = t ? p.dk_weight : p.dq_weight;
  if (out && c < p.D) store_scalar(out, p.weight_dtype, c, v);
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
namespace {
bool negative(const int64_t (&s)[3]) { return s[0] < 0 || s[1] < 0 || s[2] < 0; }

int validate_rope(const fb_rope_params* p, bool backward = false) {
  if (!p) return FB_EINVAL_NULL;
  if (p->B <= 0 || p->S <= 0 || p->Hq < 0 || p->Hk < 0 || p->Hq + (int64_t)p->Hk <= 0 || p->Hq + (int64_t)p->Hk > 65536) return FB_EINVAL_SHAPE;
  if (p->D <= 0 || p->D > kRopeMaxD || (int64_t)p->B * p->S > 0x7fff0000LL) return FB_EINVAL_SHAPE;
  if (p->dtype != FB_DTYPE_F16 && p->dtype != FB_DTYPE_BF16) return FB_EINVAL_DTYPE;
  if (p->q_weight || p->k_weight) {
    if (p->weight_dtype != FB_DTYPE_F16 && p->weight_dtype != FB_DTYPE_BF16 && p->weight_dtype != FB_DTYPE_F32) return FB_EINVAL_DTYPE;
    if (!(p->eps >= 0.f)) return FB_EINVAL_SHAPE;
  }
  if (p->rot < 0 || p->rot > p->D || p->rot % 2) return FB_EINVAL_ROPE;
  if (p->rot) {
    if (!p->positions || !p->inv_freq || p->naxes < 1 || p->naxes > 4) return FB_EINVAL_ROPE;
    if (p->position_bits != 32 && p->position_bits != 64) return FB_EINVAL_DTYPE;
    if (p->freq_dtype != FB_DTYPE_F32 && p->freq_dtype != FB_DTYPE_F64) return FB_EINVAL_DTYPE;
    for (int i = 0; i < p->rot / 2; ++i)
      if (p->pair_axis[i] >= p->naxes) return FB_EINVAL_ROPE;
  }
  // (the backward reads q and k for the norm alone)
  if ((p->Hq && !p->q && (!backward || p->q_weight)) || (p->Hk && !p->k && (!backward || p->k_weight))) return FB_EINVAL_NULL;
  if (negative(p->q_stride) || negative(p->k_stride)) return FB_EINVAL_STRIDE;
  return 0;
}

int sm_count() {
  int dev = 0;
  cudaGetDevice(&dev);
  const int n = device_sm_count(dev);
  return n > 0 ? n : 148;
}

// The columns that a lane of the vector kernels reads at once (W of RopeLane): as long as the alignment of everything that the
// call touches and half of the rotated columns allow.  -1: the general kernel (odd D; neighbours that no word holds).  4001 tokens,
// 160 heads, weights, us forward / backward: D 20 by ones 47 / 71, by words with checks of each 39 / 52 (which cost D 80 with 20
// columns rotated 4 / 6 of 33 / 36, so W 2 has none); neighbours by words 39 / 49; D 19 by the general kernel 176 / 244.
int rope_run(const fb_rope_params* p, int what) {
  if ((p->flags & FB_FLAG_FORCE_GENERAL) || p->D % 2) return -1;
  const uintptr_t w = reinterpret_cast<uintptr_t>(p->q_weight) | reinterpret_cast<uintptr_t>(p->k_weight);
  uintptr_t bits = 0;
  auto add = [&](const void* ptr, const int64_t (&s)[3], bool used) {
    if (!used) return;
    bits |= reinterpret_cast<uintptr_t>(ptr) | (uintptr_t)(s[0] | s[1] | s[2]) * 2;
  };
  add(p->q, p->q_stride, p->Hq);
  add(p->k, p->k_stride, p->Hk);
  if (what != ROPE_BACKWARD) add(p->q_out, p->q_out_stride, p->Hq);
  if (what == ROPE_FORWARD) add(p->k_out, p->k_out_stride, p->Hk);
  if (what == ROPE_APPEND) {
    add(p->v, p->v_stride, true);
    add(p->key_cache, p->key_cache_stride, true);
    add(p->value_cache, p->value_cache_stride, true);
  }
  if (what == ROPE_BACKWARD) {
    add(p->dq_out, p->dq_out_stride, p->Hq);
    add(p->dk_out, p->dk_out_stride, p->Hk);
    add(p->dq, p->dq_stride, p->Hq);
    add(p->dk, p->dk_stride, p->Hk);
  }
  const bool chunks = p->D % 8 == 0 && !((bits | w) & 15);
  const bool words = !(bits & 3) && !(w & (p->weight_dtype == FB_DTYPE_F32 ? 7 : 3));
  if (p->interleaved) return chunks ? 8 : words ? 0 : -1;
  return chunks && p->rot % 8 == 0 ? 4 : words && p->D % 8 == 0 && p->rot % 4 == 0 ? 2 : 1;
}

// Warps of a token: few tokens are spread over more warps, up to two rows for a lane.  A share has its own angles and
// coefficients to take, five rows' worth, so no more shares than make two full GPUs.
int rope_split(const fb_rope_params* p) {
  const int G = rope_lanes(p->D), H = p->Hq > p->Hk ? p->Hq : p->Hk;
  const int64_t tokens = (int64_t)p->B * p->S, want = 48ll * sm_count();
  int split = 1;
  while (split * 2 * (32 / G) <= H && tokens * split < want) split *= 2;
  return split;
}
// Blocks of the backward; vector kernels: those of q, then those of k, each by its share of the rows.
struct BwdGrid {
  int q, all;
};
BwdGrid rope_bwd_grid(const fb_rope_params* p, int run) {
  const int64_t tokens = (int64_t)p->B * p->S;
  if (run < 0) {
    const int64_t most = 8ll * sm_count();
    return {0, (int)(tokens < most ? tokens : most)};
  }
  const int64_t most = (int64_t)rope_bwd_ctas(run) * sm_count(), each = (tokens * rope_split(p) + kRopeVWarps - 1) / kRopeVWarps;
  int64_t q = most * p->Hq / (p->Hq + p->Hk), k;
  q = !p->Hq ? 0 : q < 1 ? 1 : !p->Hk ? most : q > most - 1 ? most - 1 : q;
  k = p->Hk ? most - q : 0;
  if (q > each) q = each;
  if (k > each) k = each;
  return {(int)q, (int)(q + k)};
}
bool wants_weights(const fb_rope_params* p) { return p->dq_weight || p->dk_weight; }

void launch_rope_vector(const fb_rope_params& p, int what, int run, cudaStream_t st) {
  RopeV a = {};
  a.p = p;
  a.s_div = Div(p.S);
  a.tokens = p.B * p.S;
  a.split = rope_split(&p);
  a.run = run;
  const BwdGrid bwd = rope_bwd_grid(&p, run);
  a.q_ctas = bwd.q;
  const unsigned grid = what == ROPE_BACKWARD ? (unsigned)bwd.all : (unsigned)(((int64_t)a.tokens * a.split + kRopeVWarps - 1) / kRopeVWarps);
  if (p.dtype == FB_DTYPE_F16) launch_rope_t<__half>(a, what, grid, st);
  else launch_rope_t<__nv_bfloat16>(a, what, grid, st);
  note_launch();
}
}  // namespace

}  // namespace fb

using namespace fb;

extern "C" size_t fb_rope_params_size(void) { return sizeof(fb_rope_params); }

extern "C" int fb_norm_rope(const fb_rope_params* p, void* cuda_stream) {
  if (const int rc = validate_rope(p)) return rc;
  if ((p->Hq && !p->q_out) || (p->Hk && !p->k_out)) return FB_EINVAL_NULL;
  if (negative(p->q_out_stride) || negative(p->k_out_stride)) return FB_EINVAL_STRIDE;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  if (const int run = rope_run(p, ROPE_FORWARD); run >= 0) {
    launch_rope_vector(*p, ROPE_FORWARD, run, st);
    return (int)cudaGetLastError();
  }
  const unsigned grid = (unsigned)(p->B * p->S);
  if (p->dtype == FB_DTYPE_F16) rope_general_kernel<__half, false><<<grid, kRopeThreads, 0, st>>>(*p);
  else rope_general_kernel<__nv_bfloat16, false><<<grid, kRopeThreads, 0, st>>>(*p);
  note_launch();
  return (int)cudaGetLastError();
}

extern "C" size_t fb_norm_rope_bwd_workspace_bytes(const fb_rope_params* p) {
  if (validate_rope(p, true) || !wants_weights(p)) return 0;
  return round256((size_t)rope_bwd_grid(p, rope_run(p, ROPE_BACKWARD)).all * 2 * p->D * 4);
}

extern "C" int fb_norm_rope_bwd(const fb_rope_params* p, void* cuda_stream) {
  if (const int rc = validate_rope(p, true)) return rc;
  if ((p->Hq && (!p->dq_out || !p->dq)) || (p->Hk && (!p->dk_out || !p->dk))) return FB_EINVAL_NULL;
  if (negative(p->dq_out_stride) || negative(p->dk_out_stride) || negative(p->dq_stride) || negative(p->dk_stride)) return FB_EINVAL_STRIDE;
  if ((p->dq_weight && !p->q_weight) || (p->dk_weight && !p->k_weight)) return FB_EINVAL_NULL;
  fb_rope_params a = *p;
  const size_t need = fb_norm_rope_bwd_workspace_bytes(p);
  if (need && (!p->workspace || p->workspace_bytes < need || (reinterpret_cast<uintptr_t>(p->workspace) & 255))) return FB_EINVAL_WORKSPACE;
  if (!need) a.workspace = nullptr;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  const int run = rope_run(p, ROPE_BACKWARD);
  const BwdGrid grid = rope_bwd_grid(p, run);
  const int ctas = grid.all;
  const int64_t tokens = (int64_t)p->B * p->S;
  if (run >= 0) {
    launch_rope_vector(a, ROPE_BACKWARD, run, st);
  } else {
    if (p->dtype == FB_DTYPE_F16) rope_bwd_general_kernel<__half><<<ctas, kRopeThreads, 0, st>>>(a, tokens);
    else rope_bwd_general_kernel<__nv_bfloat16><<<ctas, kRopeThreads, 0, st>>>(a, tokens);
    note_launch();
  }
  if (need) {
    const WeightParts parts = run >= 0 ? WeightParts{{grid.q, ctas - grid.q}, (int64_t)grid.q * p->D, p->D} : WeightParts{{ctas, ctas}, p->D, 2 * p->D};
    cudaLaunchConfig_t cfg = {};  // (under the end of the first kernel)
    cfg.gridDim = dim3((p->D + 31) / 32, 2);
    cfg.blockDim = dim3(32, 32);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (const cudaError_t e = cudaLaunchKernelEx(&cfg, rope_weight_kernel, a, parts)) return (int)e;
    note_launch();
  }
  return (int)cudaGetLastError();
}

extern "C" int fb_paged_append(const fb_rope_params* p, void* cuda_stream) {
  if (const int rc = validate_rope(p)) return rc;
  if (p->B != 1 || !p->Hk) return FB_EINVAL_SHAPE;
  if ((p->Hq && !p->q_out) || !p->v || !p->key_cache || !p->value_cache || !p->slots) return FB_EINVAL_NULL;
  if (negative(p->q_out_stride) || negative(p->v_stride) || negative(p->key_cache_stride) || negative(p->value_cache_stride) || p->slot_stride < 0)
    return FB_EINVAL_STRIDE;
  if (p->slot_bits != 32 && p->slot_bits != 64) return FB_EINVAL_DTYPE;
  if (p->page_size <= 0 || p->num_pages <= 0) return FB_EINVAL_PAGE;
  if (p->R < 0 || p->R > 256) return FB_EINVAL_SHAPE;
  if (p->R) {
    if (!p->k_bias || !p->bias_cache || (p->bias_heads != 1 && p->bias_heads != p->Hk)) return FB_EINVAL_BIAS;
    if (negative(p->k_bias_stride) || negative(p->bias_cache_stride)) return FB_EINVAL_STRIDE;
  } else if (p->k_bias || p->bias_cache || p->bias_heads) {
    return FB_EINVAL_BIAS;
  }
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  if (const int run = rope_run(p, ROPE_APPEND); run >= 0) {
    launch_rope_vector(*p, ROPE_APPEND, run, st);
    return (int)cudaGetLastError();
  }
  if (p->dtype == FB_DTYPE_F16) rope_general_kernel<__half, true><<<p->S, kRopeThreads, 0, st>>>(*p);
  else rope_general_kernel<__nv_bfloat16, true><<<p->S, kRopeThreads, 0, st>>>(*p);
  note_launch();
  return (int)cudaGetLastError();
}
