// Rows of logits: loads by wavefronts, and reductions over them.
#pragma once

#include "kernels.hpp"

namespace aios {

constexpr int kLpUnroll = 4;                  // 8-logit loads in flight per lane
constexpr int kLpBatch = 64 * 8 * kLpUnroll;  // logits per wavefront and batch

// Eight consecutive logits, aligned to their own size only.
__device__ __forceinline__ void lp_load8(const bf16* p, float (&f)[8]) {
  typedef uint16_t u16x8 __attribute__((ext_vector_type(8), aligned(2)));
  const uint4 v = __builtin_bit_cast(uint4, *reinterpret_cast<const u16x8*>(p));
  f[0] = lo_bf16(v.x); f[1] = hi_bf16(v.x); f[2] = lo_bf16(v.y); f[3] = hi_bf16(v.y);
  f[4] = lo_bf16(v.z); f[5] = hi_bf16(v.z); f[6] = lo_bf16(v.w); f[7] = hi_bf16(v.w);
}
__device__ __forceinline__ void lp_load8(const float* p, float (&f)[8]) {
  typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
  const f32x4u a = *reinterpret_cast<const f32x4u*>(p);
  const f32x4u b = *reinterpret_cast<const f32x4u*>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[i] = a[i];
    f[4 + i] = b[i];
  }
}

// Reductions over the wavefront: DPP within 16-lane rows, lane swaps across.
template <int CTRL>
__device__ __forceinline__ uint32_t lp_dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ float lp_wave_max(float x) {
  x = vmax(x, __uint_as_float(lp_dpp<0xB1>(__float_as_uint(x))));
  x = vmax(x, __uint_as_float(lp_dpp<0x4E>(__float_as_uint(x))));
  x = vmax(x, __uint_as_float(lp_dpp<0x141>(__float_as_uint(x))));
  x = vmax(x, __uint_as_float(lp_dpp<0x140>(__float_as_uint(x))));
  return xrow_max(x);
}
__device__ __forceinline__ uint32_t lp_wave_max_u(uint32_t x) {
  x = max(x, lp_dpp<0xB1>(x));
  x = max(x, lp_dpp<0x4E>(x));
  x = max(x, lp_dpp<0x141>(x));
  x = max(x, lp_dpp<0x140>(x));
  const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max((uint32_t)r[0], (uint32_t)r[1]);
  const auto t = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max((uint32_t)t[0], (uint32_t)t[1]);
}
__device__ __forceinline__ float lp_wave_sum(float x) { return xrow_sum(row16_sum(x)); }

// A lane's share of a batch: logits i0 + 512 u + e (u < 4, e < 8) below end, the
// others -inf.
template <typename T>
__device__ __forceinline__ void lp_load_batch(const T* x, int b0, int end, float (&f)[kLpUnroll][8]) {
  const int i0 = b0 + (threadIdx.x & 63) * 8;
  if (b0 + kLpBatch <= end) {
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) lp_load8(x + i0 + u * 512, f[u]);
  } else {
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      const int i = i0 + u * 512;
      if (i + 8 <= end) {
        lp_load8(x + i, f[u]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[u][e] = i + e < end ? (float)x[i + e] : kNegInf;
      }
    }
  }
}

}  // namespace aios
