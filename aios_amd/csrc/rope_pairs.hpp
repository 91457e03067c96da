// Rotation on load in a decode suffix item, shared by the bf16 and the 8-bit
// cache's decode kernels.
#pragma once

#include "engine.hpp"

namespace aios {

// Rotation on load in a suffix item, in the pair layout: eight lanes per row
// (row 8 p + lane / 8 in pass p: the item's G query rows, then the new
// token's K row), lane c = lane % 8 holding the P = D / 16 pairs (i, i + D/2)
// for i in [P c, P c + P).  Each pair is rotated by the lane that holds both
// of its dims and a row's sum of squares takes three DPP steps, so a lane
// normalises and rotates 2 P elements per pass (12 at D = 96) with no
// partner exchange; in the 16-row tile layout (one query row per lane of a
// 16-lane group, G of its 16 rows live) a lane took 4 D / 16 of them plus
// the K row's.  The rows go to the wavefront's staging area in LDS as bf16
// and are read back as query fragments and as the K row's 16-byte chunks.
// Arithmetic and roundings are those of qk_norm8 / qk_rope8.
template <int D, int G>
struct RopePairs {
  static constexpr int P = D / 16;  // pairs per lane
  static constexpr int W = P / 2;   // 32-bit words per half row per lane
  static constexpr int ROWS = G + 1;
  static constexpr int NPASS = (ROWS + 7) / 8;
  static constexpr int STAGE_BYTES = (ROWS * D * 2 + 15) / 16 * 16;
  static_assert(P % 2 == 0, "whole words per half row");
  uint32_t x[NPASS][2][W], w[NPASS][2][W], c[NPASS][2][W], s[NPASS][2][W];

  // q0: the item's first query row, kn: the new K row (a valid row of D
  // bf16 either way), qw / kw: norm weights, cr / sr: the table rows of the
  // position.  Lanes past the last row load query row 0 again (not used):
  // the loads carry no branch.
  __device__ __forceinline__ void load(const bf16* q0, const bf16* kn, const bf16* qw,
                                       const bf16* kw, const bf16* cr, const bf16* sr) {
    const int lane = threadIdx.x & 63;
    const int c8 = lane & 7;
#pragma unroll
    for (int ps = 0; ps < NPASS; ++ps) {
      const int r = ps * 8 + (lane >> 3);
      const bool isk = r == G;
      const bf16* xs = isk ? kn : q0 + (r < G ? r : 0) * D;
      const bf16* ws = isk ? kw : qw;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int off = hf * (D / 2) + P * c8;
        const uint32_t* xp = reinterpret_cast<const uint32_t*>(xs + off);
        const uint32_t* wp = reinterpret_cast<const uint32_t*>(ws + off);
        const uint32_t* cp = reinterpret_cast<const uint32_t*>(cr + off);
        const uint32_t* sp = reinterpret_cast<const uint32_t*>(sr + off);
#pragma unroll
        for (int i = 0; i < W; ++i) {
          x[ps][hf][i] = xp[i];
          w[ps][hf][i] = wp[i];
          c[ps][hf][i] = cp[i];
          s[ps][hf][i] = sp[i];
        }
      }
    }
  }

  // Once the loads have landed: the rotated rows into stage ([ROWS][D] bf16).
  __device__ __forceinline__ void finish(uint8_t* stage, float eps) const {
    const int lane = threadIdx.x & 63;
    const int c8 = lane & 7;
#pragma unroll
    for (int ps = 0; ps < NPASS; ++ps) {
      const int r = ps * 8 + (lane >> 3);
      float xl[P], xh[P];
#pragma unroll
      for (int i = 0; i < W; ++i) {
        xl[2 * i] = lo_bf16(x[ps][0][i]);
        xl[2 * i + 1] = hi_bf16(x[ps][0][i]);
        xh[2 * i] = lo_bf16(x[ps][1][i]);
        xh[2 * i + 1] = hi_bf16(x[ps][1][i]);
      }
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < P; ++i) ss = fmaf(xl[i], xl[i], ss);
#pragma unroll
      for (int i = 0; i < P; ++i) ss = fmaf(xh[i], xh[i], ss);
      ss = row8_sum(ss);
      const float inv = rsqrtf(ss / (float)D + eps);
      uint32_t yl[W], yh[W];
#pragma unroll
      for (int i = 0; i < W; ++i) {
        float ol[2], oh[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t wl = w[ps][0][i], wh = w[ps][1][i];
          const uint32_t cl = c[ps][0][i], ch = c[ps][1][i];
          const uint32_t sl = s[ps][0][i], sh = s[ps][1][i];
          const float nl = round_bf16(xl[2 * i + k] * inv * (k ? hi_bf16(wl) : lo_bf16(wl)));
          const float nh = round_bf16(xh[2 * i + k] * inv * (k ? hi_bf16(wh) : lo_bf16(wh)));
          ol[k] = round_bf16(round_bf16(nl * (k ? hi_bf16(cl) : lo_bf16(cl))) +
                             round_bf16(-nh * (k ? hi_bf16(sl) : lo_bf16(sl))));
          oh[k] = round_bf16(round_bf16(nh * (k ? hi_bf16(ch) : lo_bf16(ch))) +
                             round_bf16(nl * (k ? hi_bf16(sh) : lo_bf16(sh))));
        }
        yl[i] = pack_bf16x2(ol[0], ol[1]);
        yh[i] = pack_bf16x2(oh[0], oh[1]);
      }
      if (r < ROWS) {
        uint32_t* dl = reinterpret_cast<uint32_t*>(stage + (r * D + P * c8) * 2);
        uint32_t* dh = reinterpret_cast<uint32_t*>(stage + (r * D + D / 2 + P * c8) * 2);
#pragma unroll
        for (int i = 0; i < W; ++i) {
          dl[i] = yl[i];
          dh[i] = yh[i];
        }
      }
    }
  }
};

}  // namespace aios
