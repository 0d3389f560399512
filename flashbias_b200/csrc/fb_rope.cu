// Norm of queries and keys per head with the rotation by position in the same pass, forward and backward, and the serving
// form that writes keys and values into the pages of a cache.
//
//   r = rsqrt(mean(x^2) + eps),  y = x r w,  (out_lo, out_hi) = (y_lo c - y_hi s, y_hi c + y_lo s)
//   g = rotation of dout by the opposite angle,  dw = sum over rows of g x r,  dx = r (w g - x r^2 mean(w g x))
//
// Bound by reading x (and dout) once and writing the result once.  The angle position * inv_freq is taken in 64 bits and
// reduced to a fraction of a turn before its sine and cosine are taken in 32: at position 1e6 a 32-bit product is off by up to
// 0.03 rad.  It costs one pair of functions per token and frequency, shared by the token's heads, so no table is kept.
#include "fb_common.cuh"
#include "fb_internal.h"

namespace fb {

constexpr int kRopeWarps = 4;
constexpr int kRopeThreads = 32 * kRopeWarps;
constexpr int kRopeMaxD = 128;
constexpr double kInv2Pi = 0.15915494309189533576888;

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
  sincospif(2.f * (float)(turns - rint(turns)), &cs.y, &cs.x);
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

// Partial sums of the weight gradients: (CTAs, 2, D) floats, added up in the order of the CTAs by rope_weight_kernel.
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

// Block (32, 32): 32 columns of one weight, the partial sums spread over the other dimension.
__global__ void __launch_bounds__(1024) rope_weight_kernel(const __grid_constant__ fb_rope_params p, int parts) {
  __shared__ float s[32][33];
  grid_dep_wait();
  const int c = blockIdx.x * 32 + threadIdx.x, t = blockIdx.y;
  float v = 0.f;
  if (c < p.D)
    for (int i = threadIdx.y; i < parts; i += 32) v += reinterpret_cast<const float*>(p.workspace)[((int64_t)i * 2 + t) * p.D + c];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y) return;
  v = 0.f;
  for (int i = 0; i < 32; ++i) v += s[i][threadIdx.x];
  void* out = t ? p.dk_weight : p.dq_weight;
  if (out && c < p.D) store_scalar(out, p.weight_dtype, c, v);
}

// ---- vector kernels: rows of whole aligned 16-byte chunks, pairs that are whole chunks apart (or inside one) -------
// G lanes (a power of two) share a row, 8 columns each; a block takes a run of tokens, all their heads.  The columns of a lane
// are the same in every row, so its norm weights stay in registers; the angles of the block's tokens are taken once, into
// shared memory; the other half of a pair comes from the lane that holds it, as 16-bit words.  Two rows per lane are in flight,
// with 8 warps and 4 blocks per SM 64 KB.
constexpr int kRopeVThreads = 256;
constexpr int kRopeMaxTokens = 8;  // of a block at a time
constexpr int kRopeUnroll = 2;

struct RopeV {
  fb_rope_params p;
  Div s_div, hq_div, hk_div;
  int tokens;   // B S
  int run;      // tokens of a block at a time
};

template <typename T>
__device__ __forceinline__ void unpack_chunk(const uint4& w, float (&x)[8]) {
  const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
}
template <typename T>
__device__ __forceinline__ uint4 pack_chunk(const float (&y)[8]) {
  return make_uint4(Pack2<T>::pack(y[0], y[1]), Pack2<T>::pack(y[2], y[3]), Pack2<T>::pack(y[4], y[5]), Pack2<T>::pack(y[6], y[7]));
}
__device__ __forceinline__ uint4 shfl_chunk(const uint4& w, int lane) {
  return make_uint4(__shfl_sync(0xffffffffu, w.x, lane), __shfl_sync(0xffffffffu, w.y, lane), __shfl_sync(0xffffffffu, w.z, lane),
                    __shfl_sync(0xffffffffu, w.w, lane));
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What a lane holds of every row: 8 columns from col on, its partner's lane, its place among the pairs.
template <int G, bool IL>
struct RopeLane {
  int part, col, partner, pair0;
  float sign;  // of the partner's term: out = y c + sign * y_partner s
  bool in, turns;
  __device__ __forceinline__ RopeLane(const fb_rope_params& p) {
    const int lane = threadIdx.x & 31, hc = p.rot >> 4;
    part = lane % G;
    col = part * 8;
    in = col < p.D;
    turns = col < p.rot;
    const bool lo = part < hc;
    partner = IL || !turns ? lane : lo ? lane + hc : lane - hc;
    pair0 = IL ? col / 2 : lo ? col : col - 8 * hc;
    sign = lo ? -1.f : 1.f;
  }
  __device__ __forceinline__ void weights(const void* w, int dtype, int c0, float (&out)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = w && in ? load_scalar(w, dtype, c0 + i) : 1.f;
  }
  __device__ __forceinline__ int partner_col() const { return (partner % G) * 8; }
  // rotates y (and the partner's yp) by the pairs' (cos, sin); DIR -1: by the opposite angle
  template <int DIR>
  __device__ __forceinline__ void rotate(const float2* turn, float (&y)[8], const float (&yp)[8]) const {
    if (!turns) return;
    if (IL) {
      const float4 t0 = reinterpret_cast<const float4*>(turn + pair0)[0], t1 = reinterpret_cast<const float4*>(turn + pair0)[1];
      const float c[4] = {t0.x, t0.z, t1.x, t1.z}, s[4] = {t0.y * DIR, t0.w * DIR, t1.y * DIR, t1.w * DIR};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float lo = y[2 * i], hi = y[2 * i + 1];
        y[2 * i] = lo * c[i] - hi * s[i];
        y[2 * i + 1] = hi * c[i] + lo * s[i];
      }
    } else {
      const float k = sign * DIR;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 t = reinterpret_cast<const float4*>(turn + pair0)[i];
        y[2 * i] = y[2 * i] * t.x + yp[2 * i] * (k * t.y);
        y[2 * i + 1] = y[2 * i + 1] * t.z + yp[2 * i + 1] * (k * t.w);
      }
    }
  }
};

// (cos, sin) of the tokens tok0 .. tok0 + n - 1, by all threads of the block
__device__ __forceinline__ void rope_turns(const RopeV& a, int tok0, int n, float2 (*turn)[kRopeMaxD / 2]) {
  const int half = a.p.rot >> 1;
  for (int i = threadIdx.x; i < n * half; i += kRopeVThreads) {
    const int t = i / half, pr = i - t * half, b = a.s_div.quot32(tok0 + t);
    turn[t][pr] = rope_turn(a.p, b, tok0 + t - b * a.p.S, pr);
  }
}

template <typename T, int G, bool IL, bool APPEND>
__global__ void __launch_bounds__(kRopeVThreads) rope_vector_kernel(const __grid_constant__ RopeV a) {
  constexpr int ROWS = kRopeVThreads / G;  // side by side
  __shared__ __align__(16) float2 turn[kRopeMaxTokens][kRopeMaxD / 2];
  __shared__ int64_t s_page[kRopeMaxTokens];
  __shared__ int s_place[kRopeMaxTokens];
  const fb_rope_params& p = a.p;
  const RopeLane<G, IL> me(p);
  const int slot = threadIdx.x / G, tok0 = blockIdx.x * a.run, ntok = min(a.run, a.tokens - tok0);
  if (APPEND && threadIdx.x < ntok) {
    int64_t page = -1;
    int place = 0;
    if (!cache_place(p, tok0 + threadIdx.x, page, place)) page = -1;
    s_page[threadIdx.x] = page;
    s_place[threadIdx.x] = place;
  }
  rope_turns(a, tok0, ntok, turn);
  __syncthreads();

  // TENSOR 0: q, 1: k, 2: v (copied)
  auto rows_of = [&](auto tensor) {
    constexpr int X = decltype(tensor)::value;
    const int H = X == 0 ? p.Hq : p.Hk, rows = ntok * H;
    const Div& div = X == 0 ? a.hq_div : a.hk_div;
    const int64_t* xs = X == 0 ? p.q_stride : X == 1 ? p.k_stride : p.v_stride;
    const T* x = reinterpret_cast<const T*>(X == 0 ? p.q : X == 1 ? p.k : p.v);
    const void* w = X == 0 ? p.q_weight : X == 1 ? p.k_weight : nullptr;
    float wt[8], wp[8];
    if (X < 2) {
      me.weights(w, p.weight_dtype, me.col, wt);
      me.weights(w, p.weight_dtype, me.partner_col(), wp);
    }
    for (int r0 = 0; r0 < rows; r0 += ROWS * kRopeUnroll) {
      uint4 raw[kRopeUnroll];
      T* dst[kRopeUnroll];
      int tk[kRopeUnroll];
#pragma unroll
      for (int u = 0; u < kRopeUnroll; ++u) {
        const int r = r0 + u * ROWS + slot;
        dst[u] = nullptr;
        raw[u] = make_uint4(0u, 0u, 0u, 0u);
        tk[u] = 0;
        if (r < rows && me.in) {
          const int t = div.quot32(r), h = r - t * H, tok = tok0 + t, b = a.s_div.quot32(tok), s = tok - b * p.S;
          tk[u] = t;
          if (APPEND && X > 0) {
            if (s_page[t] >= 0) {
              const int64_t* cs = X == 1 ? p.key_cache_stride : p.value_cache_stride;
              dst[u] = reinterpret_cast<T*>(X == 1 ? p.key_cache : p.value_cache) + s_page[t] * cs[0] + s_place[t] * cs[1] + h * cs[2] + me.col;
            }
          } else {
            const int64_t* os = X == 0 ? p.q_out_stride : p.k_out_stride;
            dst[u] = reinterpret_cast<T*>(X == 0 ? p.q_out : p.k_out) + b * os[0] + h * os[1] + s * os[2] + me.col;
          }
          if (dst[u]) raw[u] = __ldcs(reinterpret_cast<const uint4*>(x + b * xs[0] + h * xs[1] + s * xs[2] + me.col));
        }
      }
#pragma unroll
      for (int u = 0; u < kRopeUnroll; ++u) {
        uint4 out = raw[u];
        if (X < 2) {
          float y[8], yp[8];
          unpack_chunk<T>(raw[u], y);
          float rr = 1.f;
          if (w) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(y[i], y[i], ss);
            rr = rsqrtf(group_sum<G>(ss) / p.D + p.eps);
          }
          if (!IL && p.rot) unpack_chunk<T>(shfl_chunk(raw[u], me.partner), yp);
          if (w) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              y[i] = y[i] * rr * wt[i];
              if (!IL) yp[i] = yp[i] * rr * wp[i];
            }
          }
          me.template rotate<1>(turn[tk[u]], y, yp);
          if (w || me.turns) out = pack_chunk<T>(y);  // (untouched values keep their bits)
        }
        if (dst[u]) *reinterpret_cast<uint4*>(dst[u]) = out;
      }
    }
  };
  rows_of(std::integral_constant<int, 0>());
  rows_of(std::integral_constant<int, 1>());
  if constexpr (APPEND) {
    rows_of(std::integral_constant<int, 2>());
    const int per = p.bias_heads * p.R;
    for (int i = threadIdx.x; i < ntok * per; i += kRopeVThreads) {
      const int t = i / per, h = (i - t * per) / p.R, c = i - t * per - h * p.R;
      if (s_page[t] < 0) continue;
      reinterpret_cast<T*>(p.bias_cache)[s_page[t] * p.bias_cache_stride[0] + s_place[t] * p.bias_cache_stride[1] + h * p.bias_cache_stride[2] + c] =
          reinterpret_cast<const T*>(p.k_bias)[h * p.k_bias_stride[1] + (tok0 + t) * p.k_bias_stride[2] + c];
    }
  }
}

template <typename T, int G, bool IL>
__global__ void __launch_bounds__(kRopeVThreads) rope_bwd_vector_kernel(const __grid_constant__ RopeV a) {
  constexpr int ROWS = kRopeVThreads / G;
  __shared__ __align__(16) float2 turn[kRopeMaxTokens][kRopeMaxD / 2];
  __shared__ float sums[ROWS][G * 8 + 1];
  const fb_rope_params& p = a.p;
  const RopeLane<G, IL> me(p);
  const int slot = threadIdx.x / G;
  float dw[2][8] = {};
  for (int tok0 = blockIdx.x * a.run; tok0 < a.tokens; tok0 += gridDim.x * a.run) {
    const int ntok = min(a.run, a.tokens - tok0);
    __syncthreads();
    rope_turns(a, tok0, ntok, turn);
    __syncthreads();
    auto rows_of = [&](auto tensor) {
      constexpr int X = decltype(tensor)::value;
      const int H = X == 0 ? p.Hq : p.Hk, rows = ntok * H;
      const Div& div = X == 0 ? a.hq_div : a.hk_div;
      const int64_t *xs = X == 0 ? p.q_stride : p.k_stride, *gs = X == 0 ? p.dq_out_stride : p.dk_out_stride,
                    *ds = X == 0 ? p.dq_stride : p.dk_stride;
      const void* w = X == 0 ? p.q_weight : p.k_weight;
      float wt[8];
      me.weights(w, p.weight_dtype, me.col, wt);
      for (int r0 = 0; r0 < rows; r0 += ROWS * kRopeUnroll) {
        uint4 xr[kRopeUnroll], gr[kRopeUnroll];
        T* dst[kRopeUnroll];
        int tk[kRopeUnroll];
#pragma unroll
        for (int u = 0; u < kRopeUnroll; ++u) {
          const int r = r0 + u * ROWS + slot;
          dst[u] = nullptr;
          tk[u] = 0;
          xr[u] = gr[u] = make_uint4(0u, 0u, 0u, 0u);
          if (r < rows && me.in) {
            const int t = div.quot32(r), h = r - t * H, tok = tok0 + t, b = a.s_div.quot32(tok), s = tok - b * p.S;
            tk[u] = t;
            gr[u] = __ldcs(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(X == 0 ? p.dq_out : p.dk_out) + b * gs[0] + h * gs[1] + s * gs[2] + me.col));
            if (w) xr[u] = __ldcs(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(X == 0 ? p.q : p.k) + b * xs[0] + h * xs[1] + s * xs[2] + me.col));
            dst[u] = reinterpret_cast<T*>(X == 0 ? p.dq : p.dk) + b * ds[0] + h * ds[1] + s * ds[2] + me.col;
          }
        }
#pragma unroll
        for (int u = 0; u < kRopeUnroll; ++u) {
          float g[8], gp[8];
          uint4 out = gr[u];
          unpack_chunk<T>(gr[u], g);
          if (!IL && p.rot) unpack_chunk<T>(shfl_chunk(gr[u], me.partner), gp);
          me.template rotate<-1>(turn[tk[u]], g, gp);
          if (w) {
            float x[8], ss = 0.f, sg = 0.f;
            unpack_chunk<T>(xr[u], x);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              ss = fmaf(x[i], x[i], ss);
              sg = fmaf(x[i] * g[i], wt[i], sg);
            }
            const float rr = rsqrtf(group_sum<G>(ss) / p.D + p.eps), mean = rr * (group_sum<G>(sg) / p.D);
            if (dst[u]) {
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float xn = x[i] * rr;
                dw[X][i] = fmaf(g[i], xn, dw[X][i]);
                g[i] = rr * (wt[i] * g[i] - xn * mean);
              }
            }
          }
          if (w || me.turns) out = pack_chunk<T>(g);
          if (dst[u]) *reinterpret_cast<uint4*>(dst[u]) = out;
        }
      }
    };
    rows_of(std::integral_constant<int, 0>());
    rows_of(std::integral_constant<int, 1>());
  }
  if (!p.workspace) return;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[slot][me.col + i] = dw[t][i];
    __syncthreads();
    for (int c = threadIdx.x; c < p.D; c += kRopeVThreads) {
      float v = 0.f;
      for (int r = 0; r < ROWS; ++r) v += sums[r][c];
      reinterpret_cast<float*>(p.workspace)[((int64_t)blockIdx.x * 2 + t) * p.D + c] = v;
    }
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

// Tokens of a block at a time: enough blocks for four on every SM first, then longer runs.
int rope_run(const fb_rope_params* p) {
  const int64_t run = (int64_t)p->B * p->S / (4ll * sm_count());
  return run < 1 ? 1 : run > kRopeMaxTokens ? kRopeMaxTokens : (int)run;
}
int rope_bwd_ctas(const fb_rope_params* p, bool vector) {
  const int run = vector ? rope_run(p) : 1;
  const int64_t most = (vector ? 4ll : 8ll) * sm_count(), runs = ((int64_t)p->B * p->S + run - 1) / run;
  return (int)(runs < most ? runs : most);
}
bool wants_weights(const fb_rope_params* p) { return p->dq_weight || p->dk_weight; }

enum { ROPE_FORWARD, ROPE_BACKWARD, ROPE_APPEND };
// Rows of whole aligned chunks of 16 bytes in everything that the call touches, pairs inside a chunk or whole chunks apart.
bool rope_vector(const fb_rope_params* p, int what) {
  if ((p->flags & FB_FLAG_FORCE_GENERAL) || p->D % 8 || p->rot % (p->interleaved ? 8 : 16)) return false;
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
  return !(bits & 15);
}

template <typename T, int G, bool IL>
void launch_rope_v(const RopeV& a, int what, unsigned grid, cudaStream_t st) {
  if (what == ROPE_FORWARD) rope_vector_kernel<T, G, IL, false><<<grid, kRopeVThreads, 0, st>>>(a);
  else if (what == ROPE_APPEND) rope_vector_kernel<T, G, IL, true><<<grid, kRopeVThreads, 0, st>>>(a);
  else rope_bwd_vector_kernel<T, G, IL><<<grid, kRopeVThreads, 0, st>>>(a);
}
template <typename T, int G>
void launch_rope_g(const RopeV& a, int what, unsigned grid, cudaStream_t st) {
  if (a.p.interleaved) launch_rope_v<T, G, true>(a, what, grid, st);
  else launch_rope_v<T, G, false>(a, what, grid, st);
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
  a.hq_div = Div(p.Hq > 0 ? p.Hq : 1);
  a.hk_div = Div(p.Hk > 0 ? p.Hk : 1);
  a.tokens = p.B * p.S;
  a.run = rope_run(&p);
  const unsigned grid = what == ROPE_BACKWARD ? (unsigned)rope_bwd_ctas(&p, true) : (unsigned)((a.tokens + (int64_t)a.run - 1) / a.run);
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
  return round256((size_t)rope_bwd_ctas(p, rope_vector(p, ROPE_BACKWARD)) * 2 * p->D * 4);
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
  const int ctas = rope_bwd_ctas(p, vector);
  const int64_t tokens = (int64_t)p->B * p->S;
  if (vector) {
    launch_rope_vector(a, ROPE_BACKWARD, st);
  } else {
    if (p->dtype == FB_DTYPE_F16) rope_bwd_general_kernel<__half><<<ctas, kRopeThreads, 0, st>>>(a, tokens);
    else rope_bwd_general_kernel<__nv_bfloat16><<<ctas, kRopeThreads, 0, st>>>(a, tokens);
    note_launch();
  }
  if (need) {
    rope_weight_kernel<<<dim3((p->D + 31) / 32, 2), dim3(32, 32), 0, st>>>(a, ctas);
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
