// Norm of queries and keys per head with the rotation by position in the same pass, forward and backward, and the serving
// form that writes keys and values into the pages of a cache.
//
//   r = rsqrt(mean(x^2) + eps),  y = x r w,  (out_lo, out_hi) = (y_lo c - y_hi s, y_hi c + y_lo s)
//   g = rotation of dout by the opposite angle,  dw = sum over rows of g x r,  dx = r (w g - x r^2 mean(w g x))
//
// Bound by reading x (and dout) once and writing the result once.  The angle position * inv_freq is taken in 64 bits and
// reduced to a fraction of a turn before its sine and cosine are taken in 32 (by the functions of the hardware, off by 2^-21,
// an eighth of a percent of a step of fp16): at position 1e6 a 32-bit product is off by up to 0.03 rad.  It costs one pair of
// functions per token and frequency, shared by the token's heads, so no table is kept.
#include <type_traits>

#include "fb_common.cuh"
#include "fb_internal.h"

namespace fb {

constexpr int kRopeWarps = 4;
constexpr int kRopeThreads = 32 * kRopeWarps;
constexpr int kRopeMaxD = 128;
constexpr double kInv2Pi = 0.15915494309189533576888;
constexpr float k2Pi = 6.28318530717958647693f;

__device__ __forceinline__ float load_scalar(const void* p, int dtype, int i) {
  return dtype == FB_DTYPE_F32   ? reinterpret_cast<const float*>(p)[i]
         : dtype == FB_DTYPE_F16 ? __half2float(reinterpret_cast<const __half*>(p)[i])
                                 : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_scalar(void* p, int dtype, int i, float v) {
  if (dtype == FB_DTYPE_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dtype == FB_DTYPE_F16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
  else reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// (cos, sin) of the angle of pair `pr` at token (b, s)
__device__ __forceinline__ float2 rope_turn(const fb_rope_params& p, int b, int s, int pr) {
  const int64_t at = p.pair_axis[pr] * p.position_stride[0] + b * p.position_stride[1] + s * p.position_stride[2];
  const double pos = p.position_bits == 64 ? (double)reinterpret_cast<const int64_t*>(p.positions)[at]
                                           : (double)reinterpret_cast<const int32_t*>(p.positions)[at];
  const double f = p.freq_dtype == FB_DTYPE_F64 ? reinterpret_cast<const double*>(p.inv_freq)[pr]
                                                : (double)reinterpret_cast<const float*>(p.inv_freq)[pr];
  const double turns = pos * (f * kInv2Pi);
  float2 cs;
  __sincosf((float)(turns - rint(turns)) * k2Pi, &cs.y, &cs.x);  // within +-pi: off by 2^-21
  return cs;
}

// Where token s goes in the cache; false if nowhere.
__device__ __forceinline__ bool cache_place(const fb_rope_params& p, int s, int64_t& page, int& place) {
  const int64_t slot = p.slot_bits == 64 ? reinterpret_cast<const int64_t*>(p.slots)[s * p.slot_stride]
                                         : (int64_t) reinterpret_cast<const int32_t*>(p.slots)[s * p.slot_stride];
  if (slot < 0) return false;
  page = slot / p.page_size;
  place = (int)(slot - page * p.page_size);
  if (page < p.num_pages) return true;
  if (p.status) *reinterpret_cast<volatile int32_t*>(p.status) = FB_DEV_BAD_INDEX;
  return false;
}

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
        for (int c = lane; c < p.D; c += 32) dx[c] = from_f32<T>(grad[c]);
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

// ---- vector kernels: rows of whole aligned 16-byte chunks -----------------------------------------------------------
// A warp takes a token (or a share of its heads): G lanes (a power of two) share a row, 8 columns each, 32 / G rows side by
// side.  Issue slots and the latency of a row's sums are what holds the rows back, not HBM: a warp issues about 110
// instructions per 512 bytes (forward), at 6 warps per scheduler.  So all that depends on the column and the token alone
// (weight times cosine, weight of the partner times sine) is folded into two coefficients per column that serve all heads of
// the token, the address is one addition per row, and four rows (backward: two) are in flight per lane.
// A lane holds both halves of its pairs: where they are half of the rotated columns apart (PAIR 0) it reads two runs of four
// columns, where they are neighbours (1) one of eight.  Where the halves do not begin at a multiple of four (2) the other half
// comes through shared memory.
// B4 S4096 H32-8 D128 bf16, fp32 weights, us forward / backward: 64 (5.2 TB/s) / 117 (4.3 TB/s); with the other half by shuffle
// 72 / 143, with coefficients from shared memory for every row and rows found by division 329 together.  Arithmetic on packed
// pairs of fp32 issued as many instructions and was no faster; asking for the next token's rows ahead (L2) changed nothing.
constexpr int kRopeVWarps = 4;
constexpr int kRopeVThreads = 32 * kRopeVWarps;

struct RopeV {
  fb_rope_params p;
  Div s_div;
  int tokens;  // B S
  int split;   // warps of a token
  int q_ctas;  // backward: blocks that take rows of q, the others rows of k
};

template <typename T>
__device__ __forceinline__ void unpack_chunk(const uint4& raw, float (&x)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (std::is_same<T, __nv_bfloat16>::value) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack_chunk(const float (&y)[8]) {
  return make_uint4(Pack2<T>::pack(y[0], y[1]), Pack2<T>::pack(y[2], y[3]), Pack2<T>::pack(y[4], y[5]), Pack2<T>::pack(y[6], y[7]));
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// What a lane holds of every row: two runs of four columns, from c0 and c1 on.  PAIR 0: the first and the second halves of four
// pairs, or eight columns in a row behind the rotated ones.  PAIR 1, 2: eight columns in a row.
// FULL: the lanes' columns are those of the row, and all of them are rotated.
template <typename T, int G, int PAIR, bool FULL>
struct RopeLane {
  int c0, c1;
  bool in, turns;  // columns that exist; some of them rotated
  __device__ __forceinline__ RopeLane(const fb_rope_params& p) {
    const int part = (threadIdx.x & 31) % G;
    c0 = part * 8;
    in = FULL || c0 < p.D;
    turns = FULL || c0 < p.rot;
    if (!in) c0 = 0;  // (such a lane reads what exists and drops it)
    c1 = c0 + 4;
    if (PAIR == 0 && turns) {
      c0 = part * 4;
      c1 = c0 + (FULL ? 4 * G : p.rot >> 1);
    }
  }
  __device__ __forceinline__ uint4 load(const T* row) const {
    if (PAIR != 0) return __ldcs(reinterpret_cast<const uint4*>(row + c0));
    const uint2 a = __ldcs(reinterpret_cast<const uint2*>(row + c0)), b = __ldcs(reinterpret_cast<const uint2*>(row + c1));
    return make_uint4(a.x, a.y, b.x, b.y);
  }
  __device__ __forceinline__ void store(T* row, const uint4& w) const {
    if (PAIR != 0) {
      *reinterpret_cast<uint4*>(row + c0) = w;
    } else {
      *reinterpret_cast<uint2*>(row + c0) = make_uint2(w.x, w.y);
      *reinterpret_cast<uint2*>(row + c1) = make_uint2(w.z, w.w);
    }
  }
  // the weights of the columns (1 without weights)
  __device__ __forceinline__ void weights(const void* w, int dtype, float (&out)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = 1.f;
    if (!w || !in) return;
    if (dtype == FB_DTYPE_F32) {
      const float4 u = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(w) + c0), v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(w) + c1);
      out[0] = u.x; out[1] = u.y; out[2] = u.z; out[3] = u.w; out[4] = v.x; out[5] = v.y; out[6] = v.z; out[7] = v.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(w) + c0), v = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(w) + c1);
      if (dtype == FB_DTYPE_F16) unpack_chunk<__half>(make_uint4(u.x, u.y, v.x, v.y), out);
      else unpack_chunk<__nv_bfloat16>(make_uint4(u.x, u.y, v.x, v.y), out);
    }
  }
  // Coefficients of (own, partner's) value: out = a y + b y_partner, weights folded in if w; DIR -1: the opposite angle.
  // turn: cosines of the token's pairs, sines kRopeMaxD / 2 behind.
  template <int DIR>
  __device__ __forceinline__ void coefficients(const fb_rope_params& p, const void* w, const float* turn, float (&a)[8], float (&b)[8]) const {
    float wt[8];
    weights(w, p.weight_dtype, wt);
    if (PAIR == 0) {
      const float4 c4 = turns ? *reinterpret_cast<const float4*>(turn + c0) : make_float4(1.f, 1.f, 1.f, 1.f);
      const float4 s4 = turns ? *reinterpret_cast<const float4*>(turn + kRopeMaxD / 2 + c0) : make_float4(0.f, 0.f, 0.f, 0.f);
      const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = wt[i] * c[i];
        a[i + 4] = wt[i + 4] * c[i];
        b[i] = -DIR * (wt[i + 4] * s[i]);
        b[i + 4] = DIR * (wt[i] * s[i]);
      }
      return;
    }
    const int half = p.rot >> 1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = c0 + i;
      a[i] = wt[i];
      b[i] = 0.f;
      if (c < p.rot) {
        const bool lo = PAIR == 1 ? !(i & 1) : c < half;
        const float* t = turn + (PAIR == 1 ? c >> 1 : lo ? c : c - half);
        const float q = PAIR == 1 ? wt[i ^ 1] : w ? load_scalar(w, p.weight_dtype, lo ? c + half : c - half) : 1.f;
        a[i] = wt[i] * t[0];
        b[i] = (lo ? -DIR : DIR) * (q * t[kRopeMaxD / 2]);
      }
    }
  }
  // The partners of the values v of a row, times r: in the lane, or (PAIR 2) from the row's words in the warp's shared memory.
  __device__ __forceinline__ void partners(const fb_rope_params& p, const uint4& raw, const float (&v)[8], float r, uint4* stage,
                                           float (&vp)[8]) const {
    if (PAIR < 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) vp[i] = v[PAIR == 0 ? i ^ 4 : i ^ 1];
      return;
    }
    const int lane = threadIdx.x & 31, half = p.rot >> 1;
    stage[lane] = raw;
    __syncwarp();
    uint32_t e[4] = {};
    if (turns && !(half & 1)) {  // both columns of a word have their partners in one word
      const uint32_t* row = reinterpret_cast<const uint32_t*>(stage + lane - lane % G);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = c0 + 2 * i;
        if (c < p.rot) e[i] = row[(c < half ? c + half : c - half) >> 1];
      }
    } else if (turns) {
      const uint16_t* row = reinterpret_cast<const uint16_t*>(stage + lane - lane % G);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = c0 + i;
        if (c < p.rot) e[i >> 1] |= (uint32_t)row[c < half ? c + half : c - half] << (16 * (i & 1));
      }
    }
    __syncwarp();
    unpack_chunk<T>(make_uint4(e[0], e[1], e[2], e[3]), vp);
#pragma unroll
    for (int i = 0; i < 8; ++i) vp[i] *= r;
  }
};

// Cosines and sines of one token's pairs, by the warp, into its shared memory.
__device__ __forceinline__ void rope_turns(const fb_rope_params& p, int b, int s, float* turn) {
  __syncwarp();
  for (int pr = threadIdx.x & 31; pr < p.rot >> 1; pr += 32) {
    const float2 t = rope_turn(p, b, s, pr);
    turn[pr] = t.x;
    turn[kRopeMaxD / 2 + pr] = t.y;
  }
  __syncwarp();
}

template <typename T, int G, int PAIR, bool FULL, bool APPEND>
__global__ void __launch_bounds__(kRopeVThreads, 6) rope_vector_kernel(const __grid_constant__ RopeV a) {
  constexpr int SIDE = 32 / G, U = 4;
  __shared__ __align__(16) float turns[kRopeVWarps][kRopeMaxD];
  __shared__ uint4 stages[kRopeVWarps][PAIR == 2 ? 32 : 1];
  const fb_rope_params& p = a.p;
  const RopeLane<T, G, PAIR, FULL> me(p);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t gw = (int64_t)blockIdx.x * kRopeVWarps + warp;
  const int tok = (int)(gw / a.split), sub = (int)(gw - (int64_t)tok * a.split);
  if (tok >= a.tokens) return;
  const int b = a.s_div.quot32(tok), s = tok - b * p.S;
  int64_t page = 0;
  int place = 0;
  const bool cached = APPEND && cache_place(p, s, page, place);
  rope_turns(p, b, s, turns[warp]);
  const float inv_d = 1.f / p.D;

  // TENSOR 0: q, 1: k, 2: v (copied)
  auto rows_of = [&](auto tensor) {
    constexpr int X = decltype(tensor)::value;
    const int H = X == 0 ? p.Hq : p.Hk;
    const int h0 = sub * SIDE + lane / G, step = a.split * SIDE;
    if (sub * SIDE >= H) return;
    const int64_t* xs = X == 0 ? p.q_stride : X == 1 ? p.k_stride : p.v_stride;
    const T* x = reinterpret_cast<const T*>(X == 0 ? p.q : X == 1 ? p.k : p.v) + b * xs[0] + s * xs[2] + h0 * xs[1];
    const int64_t* os = X == 0 ? p.q_out_stride : p.k_out_stride;
    T* y = reinterpret_cast<T*>(X == 0 ? p.q_out : p.k_out) + b * os[0] + s * os[2];
    int64_t yh = os[1];
    if (APPEND && X > 0) {
      const int64_t* cs = X == 1 ? p.key_cache_stride : p.value_cache_stride;
      y = reinterpret_cast<T*>(X == 1 ? p.key_cache : p.value_cache) + page * cs[0] + place * cs[1];
      yh = cs[2];
    }
    y += h0 * yh;
    const int64_t xstep = step * xs[1], ystep = step * yh;
    const void* w = X == 0 ? p.q_weight : X == 1 ? p.k_weight : nullptr;
    const bool touched = FULL || w || me.turns;  // (untouched values keep their bits)
    float ca[8], cb[8];
    const T* const x0 = x - (lane / G) * xs[1];  // (the warp's first row exists)
    auto load = [&](uint4& raw, const T* src, bool live) {
      raw = me.load(live ? src : x0);
      if ((!FULL && !me.in) || !live) raw = make_uint4(0u, 0u, 0u, 0u);
    };
    auto finish = [&](const uint4& raw, T* dst, bool live) {
      uint4 out = raw;
      if (X < 2) {
        float v[8], vp[8], rr = 1.f;
        unpack_chunk<T>(raw, v);
        if (w) {
          float q = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) q = fmaf(v[i], v[i], q);
          rr = rsqrtf(fmaf(group_sum<G>(q), inv_d, p.eps));
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] *= rr;
        }
        if (FULL || p.rot) me.partners(p, raw, v, rr, stages[warp], vp);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= ca[i];
        if (me.turns) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = fmaf(vp[i], cb[i], v[i]);
        }
        if (touched) out = pack_chunk<T>(v);
      }
      if (live && me.in) me.store(dst, out);
    };
    int h = sub * SIDE;  // (of the warp's first row; the same in all lanes)
    uint4 raw[U];
    auto load_rows = [&](auto count) {
#pragma unroll
      for (int u = 0; u < decltype(count)::value; ++u) load(raw[u], x + u * xstep, true);
    };
    auto finish_rows = [&](auto count) {
      constexpr int N = decltype(count)::value;
      x += N * xstep;
#pragma unroll
      for (int u = 0; u < N; ++u) finish(raw[u], y + u * ystep, true);
      y += N * ystep;
      h += N * step;
    };
    const std::integral_constant<int, U> many;
    const std::integral_constant<int, U / 2> some;
    const bool whole = h + (U - 1) * step + SIDE <= H;
    if (whole) load_rows(many);
    if (X < 2) me.template coefficients<1>(p, w, turns[warp], ca, cb);  // under the first loads
    if (whole) {
      finish_rows(many);
      while (h + (U - 1) * step + SIDE <= H) {
        load_rows(many);
        finish_rows(many);
      }
    }
    if (h + (U / 2 - 1) * step + SIDE <= H) {
      load_rows(some);
      finish_rows(some);
    }
#pragma unroll 1
    for (; h < H; h += step, x += xstep, y += ystep) {
      const bool live = h + lane / G < H;
      load(raw[0], x, live);
      finish(raw[0], y, live);
    }
  };
  rows_of(std::integral_constant<int, 0>());
  if (APPEND && !cached) return;
  rows_of(std::integral_constant<int, 1>());
  if constexpr (APPEND) {
    rows_of(std::integral_constant<int, 2>());
    for (int i = sub * 32 + lane; i < p.bias_heads * p.R; i += a.split * 32) {
      const int h = i / p.R, c = i - h * p.R;
      reinterpret_cast<T*>(p.bias_cache)[page * p.bias_cache_stride[0] + place * p.bias_cache_stride[1] + h * p.bias_cache_stride[2] + c] =
          reinterpret_cast<const T*>(p.k_bias)[h * p.k_bias_stride[1] + s * p.k_bias_stride[2] + c];
    }
  }
}

// A block takes rows of one tensor, so that a lane keeps one set of weight sums: the first a.q_ctas blocks take q.
template <typename T, int G, int PAIR, bool FULL>
__global__ void __launch_bounds__(kRopeVThreads, 5) rope_bwd_vector_kernel(const __grid_constant__ RopeV a) {
  constexpr int SIDE = 32 / G, U = 2;
  __shared__ __align__(16) float turns[kRopeVWarps][kRopeMaxD];
  __shared__ uint4 stages[kRopeVWarps][PAIR == 2 ? 32 : 1];
  __shared__ float sums[kRopeVWarps * SIDE][G * 8 + 1];
  const fb_rope_params& p = a.p;
  const RopeLane<T, G, PAIR, FULL> me(p);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool is_q = (int)blockIdx.x < a.q_ctas;
  const int block = is_q ? blockIdx.x : blockIdx.x - a.q_ctas, blocks = is_q ? a.q_ctas : gridDim.x - a.q_ctas;
  const int H = is_q ? p.Hq : p.Hk;
  const int64_t *xs = is_q ? p.q_stride : p.k_stride, *gs = is_q ? p.dq_out_stride : p.dk_out_stride, *ds = is_q ? p.dq_stride : p.dk_stride;
  const T* x0 = reinterpret_cast<const T*>(is_q ? p.q : p.k);
  const T* g0 = reinterpret_cast<const T*>(is_q ? p.dq_out : p.dk_out);
  T* d0 = reinterpret_cast<T*>(is_q ? p.dq : p.dk);
  const void* w = is_q ? p.q_weight : p.k_weight;
  const bool touched = FULL || w || me.turns;
  float dw[8] = {}, wt[8];
  me.weights(w, p.weight_dtype, wt);
  const float inv_d = 1.f / p.D;
  const int64_t nwarps = (int64_t)a.tokens * a.split;
  for (int64_t gw = (int64_t)block * kRopeVWarps + warp; gw < nwarps; gw += (int64_t)blocks * kRopeVWarps) {
    const int tok = (int)(gw / a.split), sub = (int)(gw - (int64_t)tok * a.split);
    const int h0 = sub * SIDE + lane / G, step = a.split * SIDE;
    if (sub * SIDE >= H) continue;
    const int b = a.s_div.quot32(tok), s = tok - b * p.S;
    const T* x = x0 + b * xs[0] + s * xs[2] + h0 * xs[1];
    const T* g = g0 + b * gs[0] + s * gs[2] + h0 * gs[1];
    T* d = d0 + b * ds[0] + s * ds[2] + h0 * ds[1];
    const int64_t xstep = step * xs[1], gstep = step * gs[1], dstep = step * ds[1];
    float ca[8], cb[8];
    uint4 xr[U], gr[U];
    const T *const gfirst = g - (lane / G) * gs[1], *const xfirst = x - (lane / G) * xs[1];  // (the warp's first row exists)
    auto load = [&](int u, const T* gsrc, const T* xsrc, bool live) {
      gr[u] = me.load(live ? gsrc : gfirst);
      if (w) xr[u] = me.load(live ? xsrc : xfirst);
      if ((!FULL && !me.in) || !live) xr[u] = gr[u] = make_uint4(0u, 0u, 0u, 0u);
    };
    auto finish = [&](int u, T* dst, bool live) {
      uint4 out = gr[u];
      float v[8], vp[8];
      unpack_chunk<T>(gr[u], v);
      if (FULL || p.rot) me.partners(p, gr[u], v, 1.f, stages[warp], vp);
      if (me.turns) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fmaf(vp[i], cb[i], v[i] * ca[i]);
      }
      if (w) {
        float x8[8], q = 0.f, t = 0.f;
        unpack_chunk<T>(xr[u], x8);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          q = fmaf(x8[i], x8[i], q);
          t = fmaf(v[i] * wt[i], x8[i], t);
        }
        const float rr = rsqrtf(fmaf(group_sum<G>(q), inv_d, p.eps)), k = -rr * (rr * (group_sum<G>(t) * inv_d));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float xn = x8[i] * rr;
          dw[i] = fmaf(v[i], xn, dw[i]);
          v[i] = fmaf(xn, k, v[i] * (wt[i] * rr));
        }
      }
      if (touched) out = pack_chunk<T>(v);
      if (live && me.in) me.store(dst, out);
    };
    int h = sub * SIDE;  // (of the warp's first row; the same in all lanes)
    if (h + (U - 1) * step + SIDE <= H) {
#pragma unroll
      for (int u = 0; u < U; ++u) load(u, g + u * gstep, x + u * xstep, true);
    }
    rope_turns(p, b, s, turns[warp]);  // under the first loads
    me.template coefficients<-1>(p, nullptr, turns[warp], ca, cb);
    for (bool first = true; h + (U - 1) * step + SIDE <= H; h += U * step, first = false) {
      if (!first) {
#pragma unroll
        for (int u = 0; u < U; ++u) load(u, g + u * gstep, x + u * xstep, true);
      }
      g += U * gstep;
      x += U * xstep;
#pragma unroll
      for (int u = 0; u < U; ++u) finish(u, d + u * dstep, true);
      d += U * dstep;
    }
#pragma unroll 1
    for (; h < H; h += step, g += gstep, x += xstep, d += dstep) {
      const bool live = h + lane / G < H;
      load(0, g, x, live);
      finish(0, d, live);
    }
  }
  if (!p.workspace) return;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (me.in) sums[warp * SIDE + lane / G][i < 4 ? me.c0 + i : me.c1 + i - 4] = dw[i];
  __syncthreads();
  for (int c = threadIdx.x; c < p.D; c += kRopeVThreads) {
    float v = 0.f;
#pragma unroll 4
    for (int r = 0; r < kRopeVWarps * SIDE; ++r) v += sums[r][c];
    reinterpret_cast<float*>(p.workspace)[(int64_t)blockIdx.x * p.D + c] = v;
  }
}

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
namespace {
bool negative(const int64_t (&s)[3]) { return s[0] < 0 || s[1] < 0 || s[2] < 0; }

int validate_rope(const fb_rope_params* p) {
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
  if ((p->Hq && !p->q) || (p->Hk && !p->k)) return FB_EINVAL_NULL;
  if (negative(p->q_stride) || negative(p->k_stride)) return FB_EINVAL_STRIDE;
  return 0;
}

int sm_count() {
  int dev = 0;
  cudaGetDevice(&dev);
  const int n = device_sm_count(dev);
  return n > 0 ? n : 148;
}

// Warps of a token: few tokens are spread over more warps, up to two rows for a lane.  A share has its own angles and
// coefficients to take, five rows' worth, so no more shares than make two full GPUs.
int rope_split(const fb_rope_params* p) {
  const int G = p->D <= 8 ? 1 : p->D <= 16 ? 2 : p->D <= 32 ? 4 : p->D <= 64 ? 8 : 16, H = p->Hq > p->Hk ? p->Hq : p->Hk;
  const int64_t tokens = (int64_t)p->B * p->S, want = 48ll * sm_count();
  int split = 1;
  while (split * 2 * (32 / G) <= H && tokens * split < want) split *= 2;
  return split;
}
// Blocks of the backward; vector kernels: those of q, then those of k, each by its share of the rows.
struct BwdGrid {
  int q, all;
};
BwdGrid rope_bwd_grid(const fb_rope_params* p, bool vector) {
  const int64_t tokens = (int64_t)p->B * p->S;
  if (!vector) {
    const int64_t most = 8ll * sm_count();
    return {0, (int)(tokens < most ? tokens : most)};
  }
  const int64_t most = 5ll * sm_count(), each = (tokens * rope_split(p) + kRopeVWarps - 1) / kRopeVWarps;
  int64_t q = most * p->Hq / (p->Hq + p->Hk), k;
  q = !p->Hq ? 0 : q < 1 ? 1 : !p->Hk ? most : q > most - 1 ? most - 1 : q;
  k = p->Hk ? most - q : 0;
  if (q > each) q = each;
  if (k > each) k = each;
  return {(int)q, (int)(q + k)};
}
bool wants_weights(const fb_rope_params* p) { return p->dq_weight || p->dk_weight; }

enum { ROPE_FORWARD, ROPE_BACKWARD, ROPE_APPEND };
// Rows of whole aligned chunks of 16 bytes in everything that the call touches.
bool rope_vector(const fb_rope_params* p, int what) {
  if ((p->flags & FB_FLAG_FORCE_GENERAL) || p->D % 8) return false;
  uintptr_t bits = reinterpret_cast<uintptr_t>(p->q_weight) | reinterpret_cast<uintptr_t>(p->k_weight);
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
  return !(bits & 15);
}

template <typename T, int G, int PAIR, bool FULL>
void launch_rope_v(const RopeV& a, int what, unsigned grid, cudaStream_t st) {
  if (what == ROPE_FORWARD) rope_vector_kernel<T, G, PAIR, FULL, false><<<grid, kRopeVThreads, 0, st>>>(a);
  else if (what == ROPE_APPEND) rope_vector_kernel<T, G, PAIR, FULL, true><<<grid, kRopeVThreads, 0, st>>>(a);
  else rope_bwd_vector_kernel<T, G, PAIR, FULL><<<grid, kRopeVThreads, 0, st>>>(a);
}
template <typename T, int G>
void launch_rope_g(const RopeV& a, int what, unsigned grid, cudaStream_t st) {
  if constexpr (G >= 8) {
    if (a.p.D == 8 * G && a.p.rot == a.p.D)
      return a.p.interleaved ? launch_rope_v<T, G, 1, true>(a, what, grid, st) : launch_rope_v<T, G, 0, true>(a, what, grid, st);
  }
  if (a.p.interleaved) launch_rope_v<T, G, 1, false>(a, what, grid, st);
  else if (a.p.rot % 8 == 0) launch_rope_v<T, G, 0, false>(a, what, grid, st);
  else launch_rope_v<T, G, 2, false>(a, what, grid, st);
}
template <typename T>
void launch_rope_t(const RopeV& a, int what, unsigned grid, cudaStream_t st) {
  if (a.p.D <= 8) launch_rope_g<T, 1>(a, what, grid, st);
  else if (a.p.D <= 16) launch_rope_g<T, 2>(a, what, grid, st);
  else if (a.p.D <= 32) launch_rope_g<T, 4>(a, what, grid, st);
  else if (a.p.D <= 64) launch_rope_g<T, 8>(a, what, grid, st);
  else launch_rope_g<T, 16>(a, what, grid, st);
}
void launch_rope_vector(const fb_rope_params& p, int what, cudaStream_t st) {
  RopeV a = {};
  a.p = p;
  a.s_div = Div(p.S);
  a.tokens = p.B * p.S;
  a.split = rope_split(&p);
  const BwdGrid bwd = rope_bwd_grid(&p, true);
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
  if (rope_vector(p, ROPE_FORWARD)) {
    launch_rope_vector(*p, ROPE_FORWARD, st);
    return (int)cudaGetLastError();
  }
  const unsigned grid = (unsigned)(p->B * p->S);
  if (p->dtype == FB_DTYPE_F16) rope_general_kernel<__half, false><<<grid, kRopeThreads, 0, st>>>(*p);
  else rope_general_kernel<__nv_bfloat16, false><<<grid, kRopeThreads, 0, st>>>(*p);
  note_launch();
  return (int)cudaGetLastError();
}

extern "C" size_t fb_norm_rope_bwd_workspace_bytes(const fb_rope_params* p) {
  if (validate_rope(p) || !wants_weights(p)) return 0;
  return round256((size_t)rope_bwd_grid(p, rope_vector(p, ROPE_BACKWARD)).all * 2 * p->D * 4);
}

extern "C" int fb_norm_rope_bwd(const fb_rope_params* p, void* cuda_stream) {
  if (const int rc = validate_rope(p)) return rc;
  if ((p->Hq && (!p->dq_out || !p->dq)) || (p->Hk && (!p->dk_out || !p->dk))) return FB_EINVAL_NULL;
  if (negative(p->dq_out_stride) || negative(p->dk_out_stride) || negative(p->dq_stride) || negative(p->dk_stride)) return FB_EINVAL_STRIDE;
  if ((p->dq_weight && !p->q_weight) || (p->dk_weight && !p->k_weight)) return FB_EINVAL_NULL;
  fb_rope_params a = *p;
  const size_t need = fb_norm_rope_bwd_workspace_bytes(p);
  if (need && (!p->workspace || p->workspace_bytes < need || (reinterpret_cast<uintptr_t>(p->workspace) & 255))) return FB_EINVAL_WORKSPACE;
  if (!need) a.workspace = nullptr;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(cuda_stream);
  const bool vector = rope_vector(p, ROPE_BACKWARD);
  const BwdGrid grid = rope_bwd_grid(p, vector);
  const int ctas = grid.all;
  const int64_t tokens = (int64_t)p->B * p->S;
  if (vector) {
    launch_rope_vector(a, ROPE_BACKWARD, st);
  } else {
    if (p->dtype == FB_DTYPE_F16) rope_bwd_general_kernel<__half><<<ctas, kRopeThreads, 0, st>>>(a, tokens);
    else rope_bwd_general_kernel<__nv_bfloat16><<<ctas, kRopeThreads, 0, st>>>(a, tokens);
    note_launch();
  }
  if (need) {
    const WeightParts parts = vector ? WeightParts{{grid.q, ctas - grid.q}, (int64_t)grid.q * p->D, p->D} : WeightParts{{ctas, ctas}, p->D, 2 * p->D};
    rope_weight_kernel<<<dim3((p->D + 31) / 32, 2), dim3(32, 32), 0, st>>>(a, parts);
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
  if (rope_vector(p, ROPE_APPEND)) {
    launch_rope_vector(*p, ROPE_APPEND, st);
    return (int)cudaGetLastError();
  }
  if (p->dtype == FB_DTYPE_F16) rope_general_kernel<__half, true><<<p->S, kRopeThreads, 0, st>>>(*p);
  else rope_general_kernel<__nv_bfloat16, true><<<p->S, kRopeThreads, 0, st>>>(*p);
  note_launch();
  return (int)cudaGetLastError();
}
