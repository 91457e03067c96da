// Quantising append into the 8-bit KV cache (numbers in kv8.hpp).
#include "kv8.hpp"

namespace aios {
namespace {

// One 16-lane row of a wavefront per (token, kv-head): each lane holds E = D /
// 16 values of the K row and of the V row, the row's largest magnitude takes
// four DPP steps, and both scales go out as one record.  (A lane's share of a
// row stays in registers between the maximum and the rounding: one read, one
// write.)  Bound: bandwidth behind the launch; 4,096 tokens of 8 x 128 6.9 us,
// 3.7 TB/s; 8 tokens of 2 x 96 2.0 us, a launch.
template <int D>
__global__ __launch_bounds__(256) void kv8_append_kernel(
    Kv8Layer c, int32_t hkv, const int32_t* __restrict__ out_loc, const bf16* __restrict__ k,
    int64_t k_stride, const bf16* __restrict__ v, int64_t v_stride, int64_t n_tokens) {
  constexpr int E = D / 16;
  constexpr int W = E / 2;
  const int l16 = threadIdx.x & 15;
  const int64_t total = n_tokens * hkv;
  const int64_t item = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  if (item >= total) return;
  const int64_t t = item / hkv;
  const int32_t h = (int32_t)(item - t * hkv);
  const int64_t slot = out_loc[t];
  if (slot < 0 || slot >= c.num_pages) return;
  uint32_t x[2][W];
  const uint32_t* kp = reinterpret_cast<const uint32_t*>(k + t * k_stride + h * D + l16 * E);
  const uint32_t* vp = reinterpret_cast<const uint32_t*>(v + t * v_stride + h * D + l16 * E);
#pragma unroll
  for (int i = 0; i < W; ++i) {
    x[0][i] = kp[i];
    x[1][i] = vp[i];
  }
  uint32_t rec = 0;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    bool bad = false;
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < W; ++i)
      a = max(a, max(kv8_mag(x[w][i] & 0xffffu, bad), kv8_mag(x[w][i] >> 16, bad)));
    a = row16_max_u(a);
    const bool row_bad = row16_max_u(bad ? 1u : 0u) != 0;
    const int e = kv8_exp(a);
    const float inv = kv8_pow2(-e);
    uint8_t* dst = (w ? c.v : c.k) + slot * c.tok_bytes + h * D + l16 * E;
    uint32_t q[W];
#pragma unroll
    for (int i = 0; i < W; ++i) q[i] = kv8_codes2(lo_bf16(x[w][i]), hi_bf16(x[w][i]), inv);
    kv8_store_codes<E>(dst, q);
    rec |= kv8_scale_bits(e, row_bad) << (16 * w);
  }
  if (l16 == 0) c.scales[h * c.num_pages + slot] = rec;
}

// qk_norm_rope_append_kernel (model_ops.hip) with the 8-bit cache: a 16-lane
// row of a wavefront per (token, head), E = D / 16 dims a lane; q heads are
// normalised, rotated and stored as bf16, k heads the same and then quantised
// from those bf16 values, v heads quantised as they come.  One wavefront per
// token and four heads: with two of them in a workgroup, or eight heads a
// wavefront, a prompt took as long or up to 20% more (1,024 tokens of 32q/8kv x
// 128: 8.6 / 9.4 / 10.4 us; 4,096: 24.1 / 23.0 / 24.9, 3.8 TB/s).
template <int D>
__global__ __launch_bounds__(64) void qk_norm_rope_append8_kernel(
    const bf16* __restrict__ qkv, int64_t stride, int hq, int hkv, const bf16* __restrict__ qw,
    const bf16* __restrict__ kw, const float* __restrict__ cos_t,
    const float* __restrict__ sin_t, int64_t table_rows, const int32_t* __restrict__ positions,
    bf16* __restrict__ q_out, Kv8Layer cache, const int32_t* __restrict__ out_loc, float eps) {
  constexpr int E = D / 16;
  constexpr int W = E / 2;
  const int lane = threadIdx.x & 63;
  const int l16 = lane & 15;
  const int heads = hq + 2 * hkv;
  const int head = blockIdx.y * 4 + (lane >> 4);
  const int64_t t = blockIdx.x;
  const int64_t pos = min(max((int64_t)positions[t], (int64_t)0), table_rows - 1);
  const int64_t slot = out_loc[t];
  uint32_t x[W];
  const bf16* src = qkv + t * stride + (int64_t)min(head, heads - 1) * D + l16 * E;
#pragma unroll
  for (int i = 0; i < W; ++i) x[i] = reinterpret_cast<const uint32_t*>(src)[i];
  float c[E], s[E];
  const float* cr = cos_t + pos * D + l16 * E;
  const float* sr = sin_t + pos * D + l16 * E;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    c[i] = round_bf16(cr[i]);
    s[i] = round_bf16(sr[i]);
  }
  const bool first_half = l16 < 8;
  const bool slot_ok = slot >= 0 && slot < cache.num_pages;
  const bool is_q = head < hq;
  const bool is_v = head >= hq + hkv;
  const int hh = is_q ? head : is_v ? head - hq - hkv : head - hq;
  uint32_t y[W];
#pragma unroll
  for (int i = 0; i < W; ++i) y[i] = x[i];
  if (__ballot(!is_v) != 0) {  // (not four V heads)
    const uint32_t* wp = reinterpret_cast<const uint32_t*>((is_q ? qw : kw) + l16 * E);
    float v[E], wv[E];
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const uint32_t b = wp[i];
      v[2 * i] = lo_bf16(x[i]);
      v[2 * i + 1] = hi_bf16(x[i]);
      wv[2 * i] = lo_bf16(b);
      wv[2 * i + 1] = hi_bf16(b);
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) ss = fmaf(v[i], v[i], ss);
    const float inv = rsqrtf(row16_sum(ss) / (float)D + eps);
    float xn[E], pn[E];
#pragma unroll
    for (int i = 0; i < E; ++i) xn[i] = round_bf16(v[i] * inv * wv[i]);
#pragma unroll
    for (int i = 0; i < E; ++i)  // lane l16 ^ 8
      pn[i] = __int_as_float(
          __builtin_amdgcn_update_dpp(0, __float_as_int(xn[i]), 0x128, 0xF, 0xF, false));
#pragma unroll
    for (int i = 0; i < W; ++i) {
      float o[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int e = 2 * i + j;
        const float rot = first_half ? -pn[e] : pn[e];
        o[j] = round_bf16(round_bf16(xn[e] * c[e]) + round_bf16(rot * s[e]));
      }
      if (!is_v) y[i] = pack_bf16x2(o[0], o[1]);
    }
  }
  // (the row maxima below are taken by every lane: no lane has left yet)
  bool bad = false;
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < W; ++i)
    a = max(a, max(kv8_mag(y[i] & 0xffffu, bad), kv8_mag(y[i] >> 16, bad)));
  a = row16_max_u(a);
  const bool row_bad = row16_max_u(bad ? 1u : 0u) != 0;
  if (head >= heads) return;
  if (is_q) {
    uint32_t* dst = reinterpret_cast<uint32_t*>(q_out + (t * hq + hh) * D + l16 * E);
#pragma unroll
    for (int i = 0; i < W; ++i) dst[i] = y[i];
    return;
  }
  if (!slot_ok) return;
  const int e = kv8_exp(a);
  const float inv = kv8_pow2(-e);
  uint32_t q[W];
#pragma unroll
  for (int i = 0; i < W; ++i) q[i] = kv8_codes2(lo_bf16(y[i]), hi_bf16(y[i]), inv);
  kv8_store_codes<E>((is_v ? cache.v : cache.k) + slot * cache.tok_bytes + hh * D + l16 * E, q);
  if (l16 == 0)
    reinterpret_cast<uint16_t*>(cache.scales + hh * cache.num_pages + slot)[is_v ? 1 : 0] =
        (uint16_t)kv8_scale_bits(e, row_bad);
}

}  // namespace

namespace {
template <int D>
hipError_t rope_append8_d(const void* qkv, int64_t stride, int64_t tokens, int hq, int hkv,
                          const void* qw, const void* kw, const float* cos_t, const float* sin_t,
                          int64_t table_rows, const int32_t* positions, void* q_out,
                          const Kv8Layer& c, const int32_t* out_loc, float eps,
                          hipStream_t stream) {
  hipLaunchKernelGGL(qk_norm_rope_append8_kernel<D>,
                     dim3((unsigned)tokens, (unsigned)(hq + 2 * hkv + 3) / 4), dim3(64), 0, stream,
                     static_cast<const bf16*>(qkv), stride, hq, hkv, static_cast<const bf16*>(qw),
                     static_cast<const bf16*>(kw), cos_t, sin_t, table_rows, positions,
                     static_cast<bf16*>(q_out), c, out_loc, eps);
  return hipGetLastError();
}
}  // namespace

hipError_t qk_norm_rope_append8(const void* qkv, int64_t stride, int64_t tokens, int hq, int hkv,
                                int D, const void* qw, const void* kw, const float* cos_t,
                                const float* sin_t, int64_t table_rows, const int32_t* positions,
                                void* q_out, const Kv8Layer& c, const int32_t* out_loc, float eps,
                                hipStream_t stream) {
  if (tokens == 0) return hipSuccess;
#define AIOS_ROPE8(DD)                                                                         \
  return rope_append8_d<DD>(qkv, stride, tokens, hq, hkv, qw, kw, cos_t, sin_t, table_rows,    \
                            positions, q_out, c, out_loc, eps, stream)
  switch (D) {
    case 64: AIOS_ROPE8(64);
    case 96: AIOS_ROPE8(96);
    case 128: AIOS_ROPE8(128);
    default: return hipErrorInvalidValue;
  }
#undef AIOS_ROPE8
}

hipError_t kv8_append(const Kv8Layer& c, int D, const int32_t* out_loc, const void* k,
                      int64_t k_stride, const void* v, int64_t v_stride, int64_t n_tokens,
                      hipStream_t stream) {
  const int32_t hkv = c.tok_bytes / D;
  const int64_t blocks = (n_tokens * hkv + 15) / 16;
  if (blocks == 0) return hipSuccess;
  if (blocks > 0x7fffffffll) return hipErrorInvalidValue;
  const dim3 grid((unsigned)blocks), block(256);
  const bf16* kb = static_cast<const bf16*>(k);
  const bf16* vb = static_cast<const bf16*>(v);
#define AIOS_KV8(DD)                                                                            \
  hipLaunchKernelGGL(kv8_append_kernel<DD>, grid, block, 0, stream, c, hkv, out_loc, kb, k_stride, \
                     vb, v_stride, n_tokens)
  switch (D) {
    case 64: AIOS_KV8(64); break;
    case 96: AIOS_KV8(96); break;
    case 128: AIOS_KV8(128); break;
    default: return hipErrorInvalidValue;
  }
#undef AIOS_KV8
  return hipGetLastError();
}

}  // namespace aios
