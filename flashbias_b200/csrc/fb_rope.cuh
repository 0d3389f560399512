// What the rope kernels share: angles, places in a cache, and the arguments of the vector kernels.
#pragma once

#include "fb_common.cuh"
#include "fb_internal.h"

namespace fb {

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
  __sincosf((float)(turns - rint(turns)) * k2Pi, &cs.y, &cs.x);  // within +-pi: off by 2^-21, half as much again by the argument's roundings
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

// ---- vector kernels (fb_rope_vector.cuh) ----------------------------------------------------------------------------
constexpr int kRopeVWarps = 4;
constexpr int kRopeVThreads = 32 * kRopeVWarps;

struct RopeV {
  fb_rope_params p;
  Div s_div;
  int tokens;  // B S
  int split;   // warps of a token
  int run;     // W of RopeLane
  int q_ctas;  // backward: blocks that take rows of q, the others rows of k
};

enum { ROPE_FORWARD, ROPE_BACKWARD, ROPE_APPEND };
// Lanes of a row.  As many as it has chunks where that lets a warp hold more rows than the next power of two does.
inline int rope_lanes(int D) {
  const int n = (D + 7) / 8;
  for (int g : {4, 5, 6, 8, 9, 10})
    if (n <= g) return g;
  return 16;
}
// Blocks of the backward per SM: short runs take more registers.
constexpr int rope_bwd_ctas(int run) { return run <= 2 ? 4 : 5; }
template <typename T>
void launch_rope_t(const RopeV& a, int what, unsigned grid, cudaStream_t st);  // fb_rope_f16.cu, fb_rope_bf16.cu
}  // namespace fb
