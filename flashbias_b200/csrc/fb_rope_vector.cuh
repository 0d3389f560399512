// Rotary passes, a few lanes to a row (instantiated in fb_rope_f16.cu and fb_rope_bf16.cu).
#pragma once

#include <type_traits>

#include "fb_rope.cuh"

namespace fb {

// A warp takes a token (or a share of its heads): G lanes share a row, 8 columns each, 32 / G rows side by side.  Issue slots
// and the latency of a row's sums are what holds the rows back, not HBM: a warp issues about 110 instructions per 512 bytes
// (forward), at 6 warps per scheduler.  So all that depends on the column and the token alone (weight times cosine, weight of
// the partner times sine) is folded into two coefficients per column that serve all heads of the token, the address is one
// addition per row, and four rows (backward: two) are in flight per lane.
// A lane holds both halves of its pairs: where they are half of the rotated columns apart it reads pairs of runs, where they
// are neighbours eight columns in a row (by twos, where rows are no whole aligned chunks of 16 bytes).  G is what a row has of chunks where that makes room for one more row.
// B4 S4096 H32-8 D128 bf16, fp32 weights, us forward / backward: 64 (5.2 TB/s) / 114 (4.4 TB/s); with the other half by shuffle
// 72 / 143, with coefficients from shared memory for every row and rows found by division 329 together.  Arithmetic on packed
// pairs of fp32 issued as many instructions and was no faster; asking for the next token's rows ahead (L2) changed nothing.
// The append of 16384 tokens, 32 + 8 + 8 heads of 128 and factors: 76 us (5.3 TB/s).
// 4001 tokens, H25-25 D80 fp16 with weights (64 MB each way, from a cold L2): 30.7 / 43.9, with 16 lanes a row 36.9 / 62.5;
// without weights and 20 columns rotated 32.8 / 35.9, with 16 lanes and the other half through shared memory 41.0 / 59.4.

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
// Sum over the G lanes of a row; the G are 32 / G groups from lane 0 on.  Where G is no power of two: over its cosets of an odd
// factor, then over them (5 shuffles for 10 lanes, 4 for 9 and 5, 3 for 6, 2 for 3).
template <int G>
__device__ __forceinline__ float group_sum(float v) {
  if constexpr ((G & (G - 1)) == 0) {
#pragma unroll
    for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  } else {
    constexpr int ODD = G % 5 == 0 ? 5 : 3, REST = G / ODD;  // lanes part, part + ODD, part + 2 ODD ... make a coset
    const int lane = threadIdx.x & 31, part = lane % G;
    auto ring = [&](float x, int by) { return __shfl_sync(0xffffffffu, x, lane + (part + by < G ? by : by - G)); };
    const float v0 = v;
#pragma unroll
    for (int j = 1; j < REST; ++j) v += ring(v0, j * ODD);
    const float v1 = v;
#pragma unroll
    for (int j = 1; j < ODD; ++j) v += ring(v1, j);
    return v;
  }
}
template <int N>
__device__ __forceinline__ void load_floats(const float* p, float* out) {
  if constexpr (N == 4) {
    const float4 u = *reinterpret_cast<const float4*>(p);
    out[0] = u.x; out[1] = u.y; out[2] = u.z; out[3] = u.w;
  } else if constexpr (N == 2) {
    const float2 u = *reinterpret_cast<const float2*>(p);
    out[0] = u.x; out[1] = u.y;
  } else {
    out[0] = *p;
  }
}

// What a lane holds of every row: up to eight columns, in runs of W, from col[] on.  W 4, 2, 1: runs 2j and 2j + 1 are the two
// halves of W pairs, or neighbours behind the rotated columns.  W 8, 0 (pairs are neighbours): eight columns in a row, read at
// once or (0) by twos.
// FULL: the lanes' columns are those of the row, and all of them are rotated.
template <typename T, int G, int W, bool FULL>
struct RopeLane {
  static constexpr bool NEAR = W == 8 || W == 0, PARTIAL = W < 2;  // PARTIAL: rows may end inside a lane's columns
  static constexpr int RUNS = NEAR ? 1 : 8 / W, SIDE = 32 / G;
  int col[RUNS];
  int row;     // of the SIDE rows that a warp holds side by side
  int have;    // values, two of a word together; 8 or 0 where not PARTIAL
  bool in;     // any
  bool turns;  // some of them are rotated
  __device__ __forceinline__ RopeLane(const fb_rope_params& p) {
    const int lane = threadIdx.x & 31, part = lane % G, half = p.rot >> 1;
    const bool mine = SIDE * G == 32 || lane < SIDE * G;
    row = mine ? lane / G : 0;
    // (whole pairs of runs come first: where a row ends inside the last lane's columns that lane lacks its last ones)
    have = FULL ? 8 : !mine ? 0 : max(0, min(8, p.D - part * 8));
    in = FULL || have > 0;
    if constexpr (NEAR) {
      col[0] = in ? part * 8 : 0;  // (a lane without columns reads what exists and drops it)
      turns = FULL || (in && col[0] < p.rot);
    } else {
#pragma unroll
      for (int j = 0; j < RUNS / 2; ++j) {
        const int u = (part * (RUNS / 2) + j) * W;
        const bool exists = FULL || (PARTIAL ? 2 * W * j < have : in);
        col[2 * j] = !exists ? 0 : FULL || u < half ? u : 2 * u;
        col[2 * j + 1] = !exists ? 0 : u < half || FULL ? u + (FULL ? 4 * G : half) : 2 * u + W;
      }
      turns = FULL || (in && part * 4 < half);
    }
  }
  __device__ __forceinline__ int column(int i) const {
    if constexpr (NEAR) return col[0] + i;
    else return col[i / W] + i % W;
  }
  // whether value i of the lane is rotated
  __device__ __forceinline__ bool turned(const fb_rope_params& p, int i) const {
    if constexpr (FULL) return true;
    else if constexpr (NEAR) return turns && col[0] + i < p.rot;
    else if constexpr (W == 4) return turns;
    else return turns && (!PARTIAL || i < have) && col[i / (2 * W) * 2] < p.rot >> 1;
  }
  __device__ __forceinline__ uint4 load(const T* src) const {
    if constexpr (W == 8) {
      return __ldcs(reinterpret_cast<const uint4*>(src + col[0]));
    } else if constexpr (W == 4) {
      const uint2 a = __ldcs(reinterpret_cast<const uint2*>(src + col[0])), b = __ldcs(reinterpret_cast<const uint2*>(src + col[1]));
      return make_uint4(a.x, a.y, b.x, b.y);
    } else if constexpr (W == 1) {
      auto one = [&](int j) { return (uint32_t)__ldcs(reinterpret_cast<const uint16_t*>(src + col[j])); };
      auto word = [&](int j) { return 2 * j < have ? one(2 * j) | one(2 * j + 1) << 16 : 0u; };
      return make_uint4(word(0), word(1), word(2), word(3));
    } else {
      auto word = [&](int j) { return !PARTIAL || 2 * j < have ? __ldcs(reinterpret_cast<const uint32_t*>(src + column(2 * j))) : 0u; };
      return make_uint4(word(0), word(1), word(2), word(3));
    }
  }
  __device__ __forceinline__ void store(T* dst, const uint4& v) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if constexpr (W == 8) {
      *reinterpret_cast<uint4*>(dst + col[0]) = v;
    } else if constexpr (W == 4) {
      *reinterpret_cast<uint2*>(dst + col[0]) = make_uint2(v.x, v.y);
      *reinterpret_cast<uint2*>(dst + col[1]) = make_uint2(v.z, v.w);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (PARTIAL && 2 * j >= have) continue;
        if constexpr (W == 1) {
          *reinterpret_cast<uint16_t*>(dst + col[2 * j]) = (uint16_t)w[j];
          *reinterpret_cast<uint16_t*>(dst + col[2 * j + 1]) = (uint16_t)(w[j] >> 16);
        } else {
          *reinterpret_cast<uint32_t*>(dst + column(2 * j)) = w[j];
        }
      }
    }
  }
  // the weights of the columns (1 without weights)
  __device__ __forceinline__ void weights(const void* w, int dtype, float (&out)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = 1.f;
    if (!w || !in) return;
    if (dtype == FB_DTYPE_F32) {
      constexpr int N = W == 0 ? 2 : W < 4 ? W : 4;
#pragma unroll
      for (int i = 0; i < 8; i += N)
        if (!PARTIAL || i < have) load_floats<N>(reinterpret_cast<const float*>(w) + column(i), out + i);
      return;
    }
    const uint4 raw = load(reinterpret_cast<const T*>(w));  // (both 16-bit types have the size of T)
    if (dtype == FB_DTYPE_F16) unpack_chunk<__half>(raw, out);
    else unpack_chunk<__nv_bfloat16>(raw, out);
  }
  // Coefficients of (own, partner's) value: out = a y + b y_partner, weights folded in if w; DIR -1: the opposite angle.
  // turn: cosines of the token's pairs, sines kRopeMaxD / 2 behind.
  template <int DIR>
  __device__ __forceinline__ void coefficients(const fb_rope_params& p, const void* w, const float* turn, float (&a)[8], float (&b)[8]) const {
    float wt[8];
    weights(w, p.weight_dtype, wt);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      a[i] = wt[i];
      b[i] = 0.f;
    }
    // N pairs at a time: the first of value i, its second value STEP on
    constexpr int N = W == 8 ? 4 : W == 0 ? 1 : W, STEP = NEAR ? 1 : W;
#pragma unroll
    for (int i = 0; i < 8; i += 2 * N) {
      float c[N], s[N];
      if (!turned(p, i)) continue;
      const int pr = NEAR ? column(i) >> 1 : column(i);
      load_floats<N>(turn + pr, c);
      load_floats<N>(turn + kRopeMaxD / 2 + pr, s);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int lo = i + (NEAR ? 2 * e : e), hi = lo + STEP;
        if (W == 8 && !turned(p, lo)) continue;
        a[lo] = wt[lo] * c[e];
        a[hi] = wt[hi] * c[e];
        b[lo] = -DIR * (wt[hi] * s[e]);
        b[hi] = DIR * (wt[lo] * s[e]);
      }
    }
  }
  // The rotation of a row by those coefficients; values that are not rotated are left with their own factor alone.
  __device__ __forceinline__ void rotate(const fb_rope_params& p, float (&v)[8], const float (&a)[8], const float (&b)[8]) const {
    constexpr int OTHER = NEAR ? 1 : W;
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = v[i] * a[i];
    if (turns) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (turned(p, i)) o[i] = fmaf(v[i ^ OTHER], b[i], o[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = o[i];
  }
  // A result, with the bits of what was neither rotated nor multiplied by a weight left as they were.
  __device__ __forceinline__ uint4 pack(const fb_rope_params& p, const uint4& raw, const float (&v)[8], bool weighted) const {
    if (FULL) return pack_chunk<T>(v);
    if (!weighted && !turns) return raw;
    uint4 out = pack_chunk<T>(v);
    if (W != 4 && !weighted) {  // (a word is rotated or not as a whole)
      if (!turned(p, 0)) out.x = raw.x;
      if (!turned(p, 2)) out.y = raw.y;
      if (!turned(p, 4)) out.z = raw.z;
      if (!turned(p, 6)) out.w = raw.w;
    }
    return out;
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

template <typename T, int G, int W, bool FULL, bool APPEND>
__global__ void __launch_bounds__(kRopeVThreads, W <= 2 ? 4 : 6) rope_vector_kernel(const __grid_constant__ RopeV a) {
  constexpr int SIDE = 32 / G, U = W == 1 ? 2 : 4;
  __shared__ __align__(16) float turns[kRopeVWarps][kRopeMaxD];
  const fb_rope_params& p = a.p;
  const RopeLane<T, G, W, FULL> me(p);
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
    const int h0 = sub * SIDE + me.row, step = a.split * SIDE;
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
    float ca[8], cb[8];
    const T* const x0 = x - me.row * xs[1];  // (the warp's first row exists)
    auto load = [&](uint4& raw, const T* src, bool live) {
      raw = me.load(live ? src : x0);
      if ((!FULL && !me.in) || !live) raw = make_uint4(0u, 0u, 0u, 0u);
    };
    auto finish = [&](const uint4& raw, T* dst, bool live) {
      uint4 out = raw;
      if (X < 2) {
        float v[8];
        unpack_chunk<T>(raw, v);
        if (w) {
          float q = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) q = fmaf(v[i], v[i], q);
          const float rr = rsqrtf(fmaf(group_sum<G>(q), inv_d, p.eps));
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] *= rr;
        }
        me.rotate(p, v, ca, cb);
        out = me.pack(p, raw, v, w);
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
      const bool live = h + me.row < H;
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
template <typename T, int G, int W, bool FULL>
__global__ void __launch_bounds__(kRopeVThreads, rope_bwd_ctas(W)) rope_bwd_vector_kernel(const __grid_constant__ RopeV a) {
  constexpr int SIDE = 32 / G, U = 2;
  __shared__ __align__(16) float turns[kRopeVWarps][kRopeMaxD];
  __shared__ float sums[kRopeVWarps * SIDE][G * 8 + 1];
  const fb_rope_params& p = a.p;
  const RopeLane<T, G, W, FULL> me(p);
  const int warp = threadIdx.x >> 5;
  const bool is_q = (int)blockIdx.x < a.q_ctas;
  const int block = is_q ? blockIdx.x : blockIdx.x - a.q_ctas, blocks = is_q ? a.q_ctas : gridDim.x - a.q_ctas;
  const int H = is_q ? p.Hq : p.Hk;
  const int64_t *xs = is_q ? p.q_stride : p.k_stride, *gs = is_q ? p.dq_out_stride : p.dk_out_stride, *ds = is_q ? p.dq_stride : p.dk_stride;
  const T* x0 = reinterpret_cast<const T*>(is_q ? p.q : p.k);
  const T* g0 = reinterpret_cast<const T*>(is_q ? p.dq_out : p.dk_out);
  T* d0 = reinterpret_cast<T*>(is_q ? p.dq : p.dk);
  const void* w = is_q ? p.q_weight : p.k_weight;
  float dw[8] = {}, wt[8];
  me.weights(w, p.weight_dtype, wt);
  const float inv_d = 1.f / p.D;
  const int64_t nwarps = (int64_t)a.tokens * a.split;
  for (int64_t gw = (int64_t)block * kRopeVWarps + warp; gw < nwarps; gw += (int64_t)blocks * kRopeVWarps) {
    const int tok = (int)(gw / a.split), sub = (int)(gw - (int64_t)tok * a.split);
    const int h0 = sub * SIDE + me.row, step = a.split * SIDE;
    if (sub * SIDE >= H) continue;
    const int b = a.s_div.quot32(tok), s = tok - b * p.S;
    const T* x = x0 + b * xs[0] + s * xs[2] + h0 * xs[1];
    const T* g = g0 + b * gs[0] + s * gs[2] + h0 * gs[1];
    T* d = d0 + b * ds[0] + s * ds[2] + h0 * ds[1];
    const int64_t xstep = step * xs[1], gstep = step * gs[1], dstep = step * ds[1];
    float ca[8], cb[8];
    uint4 xr[U], gr[U];
    const T *const gfirst = g - me.row * gs[1], *const xfirst = x - me.row * xs[1];  // (the warp's first row exists)
    auto load = [&](int u, const T* gsrc, const T* xsrc, bool live) {
      gr[u] = me.load(live ? gsrc : gfirst);
      if (w) xr[u] = me.load(live ? xsrc : xfirst);
      if ((!FULL && !me.in) || !live) xr[u] = gr[u] = make_uint4(0u, 0u, 0u, 0u);
    };
    auto finish = [&](int u, T* dst, bool live) {
      float v[8];
      unpack_chunk<T>(gr[u], v);
      me.rotate(p, v, ca, cb);
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
      if (live && me.in) me.store(dst, me.pack(p, gr[u], v, w));
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
      const bool live = h + me.row < H;
      load(0, g, x, live);
      finish(0, d, live);
    }
  }
  if (!p.workspace) return;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < me.have) sums[warp * SIDE + me.row][me.column(i)] = dw[i];
  __syncthreads();
  for (int c = threadIdx.x; c < p.D; c += kRopeVThreads) {
    float v = 0.f;
#pragma unroll 4
    for (int r = 0; r < kRopeVWarps * SIDE; ++r) v += sums[r][c];
    reinterpret_cast<float*>(p.workspace)[(int64_t)blockIdx.x * p.D + c] = v;
  }
}

// ---- host side
template <typename T, int G, int W, bool FULL>
void launch_rope_v(const RopeV& a, int what, unsigned grid, cudaStream_t st) {
  if (what == ROPE_FORWARD) rope_vector_kernel<T, G, W, FULL, false><<<grid, kRopeVThreads, 0, st>>>(a);
  else if (what == ROPE_APPEND) rope_vector_kernel<T, G, W, FULL, true><<<grid, kRopeVThreads, 0, st>>>(a);
  else rope_bwd_vector_kernel<T, G, W, FULL><<<grid, kRopeVThreads, 0, st>>>(a);
}
template <typename T, int G>
void launch_rope_g(const RopeV& a, int what, unsigned grid, cudaStream_t st) {
  if constexpr (G == 8 || G == 16) {
    if (a.run >= 4 && a.p.D == 8 * G && a.p.rot == a.p.D)
      return a.run == 8 ? launch_rope_v<T, G, 8, true>(a, what, grid, st) : launch_rope_v<T, G, 4, true>(a, what, grid, st);
  }
  switch (a.run) {
    case 8: return launch_rope_v<T, G, 8, false>(a, what, grid, st);
    case 0: return launch_rope_v<T, G, 0, false>(a, what, grid, st);
    case 4: return launch_rope_v<T, G, 4, false>(a, what, grid, st);
    case 2: return launch_rope_v<T, G, 2, false>(a, what, grid, st);
    default: return launch_rope_v<T, G, 1, false>(a, what, grid, st);
  }
}
template <typename T>
void launch_rope_t(const RopeV& a, int what, unsigned grid, cudaStream_t st) {
  switch (rope_lanes(a.p.D)) {
    case 4: return launch_rope_g<T, 4>(a, what, grid, st);
    case 5: return launch_rope_g<T, 5>(a, what, grid, st);
    case 6: return launch_rope_g<T, 6>(a, what, grid, st);
    case 8: return launch_rope_g<T, 8>(a, what, grid, st);
    case 9: return launch_rope_g<T, 9>(a, what, grid, st);
    case 10: return launch_rope_g<T, 10>(a, what, grid, st);
    default: return launch_rope_g<T, 16>(a, what, grid, st);
  }
}
}  // namespace fb
