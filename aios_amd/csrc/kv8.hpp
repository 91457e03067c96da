// The 8-bit KV cache's numbers.
//
// A row (one head's D values of one token) with largest finite magnitude a is
// held as e4m3 codes c_i = rne(x_i / s), s = 2^e with the smallest e >= -110
// for which a <= 448 s (448 is e4m3's largest value).  Both sides of that
// division are exact but for the one rounding to e4m3 (2^-4 relative): s is a
// power of two, and since e4m3 is a floating type a scale with a mantissa
// would win no precision (only the smallest values of a row fall into e4m3's
// subnormals one binade earlier).  c * s has 4 significant bits and an
// exponent from -119 on, so it is exact in bf16, which is what the attention
// kernels multiply: the cache's rounding is the only one that K takes, and V's
// scale needs no rounding either.
//
// A row that holds a NaN or an infinity gets a NaN scale (those elements'
// codes are 0): a token with a NaN K or V scale makes every output that
// attends to it NaN and, since its score is NaN and its V row is not, no
// other output.
#pragma once

#include "engine.hpp"

namespace aios {

constexpr int kKv8MinExp = -110;

// The exponent of a row's scale from its largest finite |x| as fp32 bits.
__device__ __forceinline__ int kv8_exp(uint32_t amax_bits) {
  const int x = (int)(amax_bits >> 23) - 127;  // floor(log2 a); -127 for 0 and subnormals
  const int e = x - 8 + ((amax_bits & 0x7fffffu) > 0x600000u);  // 448 = 1.75 * 2^8
  return max(e, kKv8MinExp);
}
__device__ __forceinline__ float kv8_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The magnitude bits (fp32) of a bf16 if finite, else 0; bad: set if not.
__device__ __forceinline__ uint32_t kv8_mag(uint32_t bits16, bool& bad) {
  const uint32_t m = bits16 & 0x7fffu;
  const bool fin = m < 0x7f80u;
  bad = bad || !fin;
  return fin ? m << 16 : 0u;
}

// Codes of two / four values (fp32), the first in the low byte; non-finite -> 0.
__device__ __forceinline__ uint32_t kv8_codes2(float a, float b, float inv) {
  a = __builtin_isfinite(a) ? a * inv : 0.f;
  b = __builtin_isfinite(b) ? b * inv : 0.f;
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu;
}

// E codes (two per word's low half) to dst, aligned to E & -E bytes.
template <int E>
__device__ __forceinline__ void kv8_store_codes(uint8_t* dst, const uint32_t (&q)[E / 2]) {
  if constexpr (E == 8) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
  } else if constexpr (E == 4) {
    *reinterpret_cast<uint32_t*>(dst) = q[0] | q[1] << 16;
  } else {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) reinterpret_cast<uint16_t*>(dst)[i] = (uint16_t)q[i];
  }
}

// bf16 bits of a row's scale.
__device__ __forceinline__ uint32_t kv8_scale_bits(int e, bool bad) {
  return bad ? 0x7fc0u : (uint32_t)(e + 127) << 7;
}

// The scales of a record as the kernels apply them: K's is NaN if either is,
// V's is 1 in place of a NaN.
__device__ __forceinline__ void kv8_scales(uint32_t rec, float& ks, float& vs) {
  const float v = hi_bf16(rec);
  ks = fmaf(v, 0.f, lo_bf16(rec));
  vs = v == v ? v : 1.f;
}

// Four codes as bf16 times a power of two (exact).
__device__ __forceinline__ uint2 kv8_dequant4(uint32_t codes, float scale) {
  uint2 r;
  r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false));
  r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true));
  return r;
}
__device__ __forceinline__ bf16x8 kv8_dequant8(uint32_t lo, uint32_t hi, float scale) {
  const uint2 a = kv8_dequant4(lo, scale), b = kv8_dequant4(hi, scale);
  return __builtin_bit_cast(bf16x8, make_uint4(a.x, a.y, b.x, b.y));
}

// Max over a 16-lane row of the wavefront (every lane receives it).
__device__ __forceinline__ uint32_t row16_max_u(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xB1, 0xF, 0xF, false));
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4E, 0xF, 0xF, false));
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x141, 0xF, 0xF, false));
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x140, 0xF, 0xF, false));
}

// Raw buffer descriptor over `bytes` bytes from p: loads past the end return
// zeros, which is how page ids outside the pool and positions past a range
// read all-zero rows.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t kv8_rsrc(const void* p, int64_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, (short)0,
                                           (int)(bytes < 0xffffffffll ? bytes : 0xffffffffll),
                                           kBufferWord3);
}

// One kv-head of a layer's cache: rows at offset page * tok_b, scale records
// at page * 4; page n_pages (any larger id is clamped to it) reads zeros.
struct Kv8Head {
  __amdgpu_buffer_rsrc_t k, v, s;
  uint32_t tok_b, n_pages;

  __device__ __forceinline__ Kv8Head(const Kv8Layer& c, int h, int D)
      : k(kv8_rsrc(c.k + (int64_t)h * D, rows_bytes(c, D))),
        v(kv8_rsrc(c.v + (int64_t)h * D, rows_bytes(c, D))),
        s(kv8_rsrc(c.scales + (int64_t)h * c.num_pages, c.num_pages * 4)),
        tok_b((uint32_t)c.tok_bytes),
        n_pages((uint32_t)c.num_pages) {}
  static __device__ __forceinline__ int64_t rows_bytes(const Kv8Layer& c, int D) {
    return c.num_pages > 0 ? (c.num_pages - 1) * (int64_t)c.tok_bytes + D : 0;
  }
  __device__ __forceinline__ uint32_t page(int32_t id, bool live) const {
    return live ? min((uint32_t)id, n_pages) : n_pages;
  }
  __device__ __forceinline__ uint32_t row(uint32_t page) const { return __umul24(page, tok_b); }
};

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ u32x4 load_b128(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0));
}
__device__ __forceinline__ u32x2 load_b64(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, 0));
}
__device__ __forceinline__ uint32_t load_b32(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  return (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, (int)off, 0, 0);
}

}  // namespace aios
