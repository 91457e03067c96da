// Paged decode over the 8-bit KV cache: shared-prefix cascade, per-row items
// and the log-sum-exp combine, with the new token's quantising append and its
// q/k norm + rotation inside the main launch (attn_decode.hip's scheme).
//
//   * prefix workgroups: the 128-row tile engine (engine8.hpp) over one chunk
//     of the shared prefix;
//   * row items: positions of the rows' own pages for one kv-head, the four
//     wavefronts taking 32-position sub-tiles round-robin (RowEngine8 below):
//     one row, whole, or one of the equal parts of a longer row (more of them
//     the longer it is).
#include "engine8.hpp"
#include "rope_pairs.hpp"

namespace aios {
namespace {

// Byte slot of 16-code chunk c of token t's V row in a wavefront's LDS tile
// (rows of D bytes): rotated so that the 32 rows a transpose read takes at
// one chunk spread over the banks (D = 128, 64: every 16-byte bank group
// twice; D = 96: at most three times).
template <int D>
__device__ __forceinline__ int v8_slot(int t, int c) {
  constexpr int CPR = D / 16;
  const int rot = D == 128 ? t >> 1 : D == 64 ? t >> 2 : t >> 3;
  return (c + rot) % CPR;
}

// A wavefront's math on 32 positions for one 16-row MFMA tile whose first G
// rows are the item's query heads.
//   S^T = K Q^T: lane (l16, lg) of token tile tt holds K[tt * 16 + l16] at the
//     dims qdim(s, lg) .. + 7 of k-step s, straight from its own global loads:
//     a 16-byte load holds the dims of two k-steps, and Q is loaded in the
//     same order, so K never passes through LDS;
//   O^T += V^T P^T: V goes to LDS as codes (rows of D bytes) and comes back
//     transposed by ds_read_b64_tr_b8: 8 positions of one dim per lane, in the
//     order of the lane's own scores; V's scales multiply P (before its one
//     rounding to bf16), so its codes are converted unscaled.
template <int D, int G>
struct RowEngine8 {
  static constexpr int KS = D / 32;   // k-steps of S^T
  static constexpr int DT = D / 16;   // 16-dim tiles of O^T
  static constexpr int K16 = D / 64;  // 16-byte K loads per token tile
  static constexpr int K8 = (D % 64) / 32;
  static constexpr int NV = D / 32;   // 16-byte V loads
  static constexpr int CH = D / 16;
  static constexpr int V_BYTES = 32 * D;
  static constexpr int TILE_BYTES = V_BYTES + 32 * 4;  // V codes, V scales

  struct Ids {
    int32_t k[2], v[NV];
  };
  struct Regs {
    u32x4 k16[2][K16];
    u32x2 k8[2][K8 ? K8 : 1];
    u32x4 v[NV];
    uint32_t rec[2];
  };

  bf16x8 qf[KS];
  f32x4 o[DT];
  float m_run, nm, ls;

  static __device__ __forceinline__ int qdim(int s, int lg) {
    if (s < 2 * K16) return (s >> 1) * 64 + lg * 16 + (s & 1) * 8;
    return K16 * 64 + (s - 2 * K16) * 32 + lg * 8;
  }

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    m_run = kNegInf;
    nm = 0.f;
    ls = 0.f;
  }
  // q: the lane's query row (16-byte aligned, in memory or LDS)
  __device__ __forceinline__ void load_q(const bf16* q, bool ok) {
    const int lg = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const bf16x8 f = *reinterpret_cast<const bf16x8*>(q + qdim(s, lg));
      qf[s] = ok ? f : bf16x8{};
    }
  }

  static __device__ __forceinline__ int v_tok(int j) { return (j * 64 + (threadIdx.x & 63)) / CH; }

  // Page ids of positions kv0 ..; those past `last` read its entry.
  static __device__ __forceinline__ void ids(const int32_t* idx, int kv0, int last, Ids& r) {
    const int l16 = threadIdx.x & 15;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) r.k[tt] = idx[min(kv0 + tt * 16 + l16, last)];
#pragma unroll
    for (int j = 0; j < NV; ++j) r.v[j] = idx[min(kv0 + v_tok(j), last)];
  }
  // Positions in [kv0, end) but `skip` (the new token, whose rows come from
  // registers); the others read zeros.
  static __device__ __forceinline__ void load(const Kv8Head& hd, const Ids& i, int kv0, int end,
                                              int skip, Regs& r) {
    const int lane = threadIdx.x & 63;
    const int l16 = lane & 15, lg = lane >> 4;
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const int pos = kv0 + tt * 16 + l16;
      const uint32_t pg = hd.page(i.k[tt], pos < end && pos != skip);
      const uint32_t off = hd.row(pg);
      r.rec[tt] = load_b32(hd.s, pg * 4);
#pragma unroll
      for (int c = 0; c < K16; ++c) r.k16[tt][c] = load_b128(hd.k, off + c * 64 + lg * 16);
#pragma unroll
      for (int c = 0; c < K8; ++c) r.k8[tt][c] = load_b64(hd.k, off + K16 * 64 + c * 32 + lg * 8);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int ch = j * 64 + lane;
      const int t = ch / CH;
      const int pos = kv0 + t;
      const uint32_t pg = hd.page(i.v[j], pos < end && pos != skip);
      r.v[j] = load_b128(hd.v, hd.row(pg) + (ch - t * CH) * 16);
    }
  }

  // V codes and scales to the wavefront's tile (its LDS accesses complete in
  // order, so its own reads behind them need no wait).
  static __device__ __forceinline__ void store_v(uint8_t* tile, const Regs& r) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int ch = j * 64 + lane;
      const int t = ch / CH;
      *reinterpret_cast<u32x4*>(tile + t * D + v8_slot<D>(t, ch - t * CH) * 16) = r.v[j];
    }
    float ks, vs;
    kv8_scales(lane < 16 ? r.rec[0] : r.rec[1], ks, vs);
    if (lane < 32) reinterpret_cast<float*>(tile + V_BYTES)[lane] = vs;
  }

  // S^T of the sub-tile: st[tt] register i = row l16, position tt * 16 + lg * 4 + i.
  __device__ __forceinline__ void scores(const Regs& r, f32x4 (&st)[2]) const {
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      float ks, vs;
      kv8_scales(r.rec[tt], ks, vs);
      st[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < K16; ++c) {
        const u32x4 w = r.k16[tt][c];
        st[tt] = mfma16x16x32(kv8_dequant8(w[0], w[1], ks), qf[2 * c], st[tt]);
        st[tt] = mfma16x16x32(kv8_dequant8(w[2], w[3], ks), qf[2 * c + 1], st[tt]);
      }
#pragma unroll
      for (int c = 0; c < K8; ++c) {
        const u32x2 w = r.k8[tt][c];
        st[tt] = mfma16x16x32(kv8_dequant8(w[0], w[1], ks), qf[2 * K16 + c], st[tt]);
      }
    }
  }

  // Softmax and O^T of the sub-tile whose V is in the wavefront's LDS tile.
  __device__ __forceinline__ void update(const uint8_t* tile, const f32x4 (&st)[2], int kv0, int end,
                                         float scale_log2) {
    const int lane = threadIdx.x & 63;
    const int l16 = lane & 15, lg = lane >> 4;
    // V^T: group lg reads the 8 positions of its lanes' scores, each row's 16
    // bytes by two lanes.
    const int rr = l16 >> 1;
    const int tv = rr < 4 ? lg * 4 + rr : 16 + lg * 4 + rr - 4;
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    i32x2 va[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      va[dt] = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
          (AIOS_LDS i32x2*)(tile + tv * D + v8_slot<D>(tv, dt) * 16 + (l16 & 1) * 8));
    const f32x4 s0 = *reinterpret_cast<const f32x4*>(tile + V_BYTES + lg * 16);
    const f32x4 s1 = *reinterpret_cast<const f32x4*>(tile + V_BYTES + 64 + lg * 16);

    // Online softmax of row l16 (lanes l16 + 16 k hold its scores), reference
    // moved only by more than kRescaleSlack.
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = st[0][i];
      x[4 + i] = st[1][i];
    }
    if (__builtin_expect(kv0 + 32 > end, 0)) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (kv0 + (i >> 2) * 16 + lg * 4 + (i & 3) >= end) x[i] = kNegInf;
    }
    float mx = vmax(vmax(vmax(x[0], x[1]), vmax(x[2], x[3])),
                    vmax(vmax(x[4], x[5]), vmax(x[6], x[7])));
    mx = xrow_max(mx) * scale_log2;
    const bool need = mx > m_run + kRescaleSlack;
    if (__builtin_amdgcn_ballot_w64(need)) {
      const float al = need ? fast_exp2(m_run - mx) : 1.f;
      ls *= al;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= al;
      m_run = need ? mx : m_run;
      nm = need ? -mx : nm;
    }
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = fast_exp2(fmaf(x[i], scale_log2, nm));
    ls += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] *= s0[i];
      p[4 + i] *= s1[i];
    }
    const bf16x8 pb = __builtin_bit_cast(
        bf16x8, make_uint4(pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]),
                           pack_bf16x2(p[4], p[5]), pack_bf16x2(p[6], p[7])));
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      o[dt] = mfma16x16x32(kv8_dequant8((uint32_t)va[dt][0], (uint32_t)va[dt][1], 1.f), pb, o[dt]);
  }
};

// fp16 pair, nearest even.
__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
}
// Power of two that brings magnitudes up to mx below 4 (2: bits of its inverse).
__device__ __forceinline__ float part_scale(float mx, float& inverse) {
  const uint32_t ex = min(max(__float_as_uint(mx) >> 23 & 255u, 1u), 253u);
  inverse = __uint_as_float(ex << 23);
  return __uint_as_float((254u - ex) << 23);
}

__device__ __forceinline__ float lse_of(float l, float m) {
  return l > 0.f ? m + fast_log2(l) : l == 0.f ? kNegInf : l;
}

// ---------------------------------------------------------------------------
// prefix part
template <int D, int G, bool ROPE>
__device__ __forceinline__ void decode8_prefix_part(uint8_t* lds, const Decode8Args& a, int wg) {
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int hl = lane >> 5;
  const int mg = wg / a.prefix_units;
  const int unit = wg % a.prefix_units;
  const int h = unit % a.num_kv_heads;
  const int chunk = unit / a.num_kv_heads;

  TileEngine32<D, false> eng;
  eng.min_limit = 0x7fffffff;
  const int m = mg * 128 + wave * 32 + (lane & 31);
  const bool ok = m < a.m_rows;
  const int b = m / G;
  const int g = m - b * G;
  const bf16* qr = a.q + (int64_t)b * a.q_tok_stride + (int64_t)(h * G + g) * D;
  const int kv_begin = chunk * a.chunk_len;
  const int kv_end = min(a.prefix_len, kv_begin + a.chunk_len);
  const bool active = mg * 128 + wave * 32 < a.m_rows;
  run_tile8<D, false>(eng, lds, a.kv, h, a.indices, kv_begin, kv_end, a.scale_log2,
                      [&] {
                        if constexpr (ROPE) {
                          const int64_t pos = ok ? (int64_t)a.positions[b] : 0;
                          const int64_t rrow = min(max(pos, (int64_t)0), a.rope_rows - 1);
                          eng.load_q_rope(qr, ok, a.q_norm, a.rope_cos + rrow * D,
                                          a.rope_sin + rrow * D, a.norm_eps);
                        } else {
                          eng.load_q(qr, ok);
                        }
                      },
                      active);
  const float l_tot = eng.l_run;
  const float inv = l_tot > 0.f ? 1.f / l_tot : l_tot * 0.f;
  float mx = 0.f;
#pragma unroll
  for (int nt = 0; nt < D / 32; ++nt)
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      eng.o[nt][i] *= inv;
      mx = fmaxf(mx, fabsf(eng.o[nt][i]));
    }
  mx = xor32_max(mx);
  if (!ok) return;
  float unscale;
  const float sc = part_scale(mx, unscale);
  // (the lane pair swaps halves so that each lane stores 16 bytes: see
  // decode_prefix_part)
#pragma unroll
  for (int nt = 0; nt < D / 32; ++nt)
#pragma unroll
    for (int jp = 0; jp < 2; ++jp) {
      const int j0 = 2 * jp, j1 = j0 + 1;
      uint2 g0, g1;
      g0.x = pack_f16x2(eng.o[nt][4 * j0] * sc, eng.o[nt][4 * j0 + 1] * sc);
      g0.y = pack_f16x2(eng.o[nt][4 * j0 + 2] * sc, eng.o[nt][4 * j0 + 3] * sc);
      g1.x = pack_f16x2(eng.o[nt][4 * j1] * sc, eng.o[nt][4 * j1 + 1] * sc);
      g1.y = pack_f16x2(eng.o[nt][4 * j1 + 2] * sc, eng.o[nt][4 * j1 + 3] * sc);
      const uint2 snd = hl ? g0 : g1;
      const auto rx = __builtin_amdgcn_permlane32_swap(snd.x, snd.x, false, false);
      const auto ry = __builtin_amdgcn_permlane32_swap(snd.y, snd.y, false, false);
      const uint2 rcv = hl ? make_uint2(rx[0], ry[0]) : make_uint2(rx[1], ry[1]);
      const uint4 v = hl ? make_uint4(rcv.x, rcv.y, g1.x, g1.y) : make_uint4(g0.x, g0.y, rcv.x, rcv.y);
      *reinterpret_cast<uint4*>(a.parts.o +
                                a.parts.o_index(D, h, chunk, m, nt * 32 + 16 * jp + 8 * hl)) = v;
    }
  if (hl == 0) a.parts.ls[a.parts.ls_index(h, chunk, m)] = make_float2(lse_of(l_tot, eng.m_run), unscale);
}

// ---------------------------------------------------------------------------
// row items
template <int D, int G>
struct Item8 {
  using E = RowEngine8<D, G>;
  using RP = RopePairs<D, G>;
  static constexpr int NW = kEngineThreads / 64;
  static constexpr int MERGE_BYTES = D / 16 * 64 * 16 + 2 * 16 * 4;
  static constexpr int WAVE_BYTES = MERGE_BYTES > E::TILE_BYTES ? MERGE_BYTES : E::TILE_BYTES;
  static constexpr int STAGE_BYTES = RP::STAGE_BYTES;
  static constexpr int LDS_BYTES = NW * (WAVE_BYTES + STAGE_BYTES);
};

// A row's new token as the cache holds it: two values of K and of V per lane
// (lanes below D / 2).
template <int D>
struct NewToken {
  uint32_t code[2];  // K, V
  uint32_t rec;
  bool in_pool;      // the row's last page id is: the token is attended to

  static __device__ __forceinline__ bool mine() { return (int)(threadIdx.x & 63) < D / 2; }

  // kr, vr: the token's rows, 4-byte aligned, in memory or LDS
  __device__ __forceinline__ void quantize(const bf16* kr, const bf16* vr) {
    const int lane = threadIdx.x & 63;
    uint32_t x[2] = {0u, 0u};
    if (mine()) {
      x[0] = reinterpret_cast<const uint32_t*>(kr)[lane];
      x[1] = reinterpret_cast<const uint32_t*>(vr)[lane];
    }
    rec = 0;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      bool bad = false;
      uint32_t m = max(kv8_mag(x[w] & 0xffffu, bad), kv8_mag(x[w] >> 16, bad));
      m = row16_max_u(m);
      m = __float_as_uint(xrow_max(__uint_as_float(m)));
      const bool row_bad = __builtin_amdgcn_ballot_w64(bad) != 0;
      const int e = kv8_exp(m);
      code[w] = kv8_codes2(lo_bf16(x[w]), hi_bf16(x[w]), kv8_pow2(-e));
      rec |= kv8_scale_bits(e, row_bad) << (16 * w);
    }
  }
  __device__ __forceinline__ void write(const Kv8Layer& kv, int h, int64_t slot) const {
    const int lane = threadIdx.x & 63;
    if (mine()) {
      const int64_t off = slot * (int64_t)kv.tok_bytes + h * D + lane * 2;
      *reinterpret_cast<uint16_t*>(kv.k + off) = (uint16_t)code[0];
      *reinterpret_cast<uint16_t*>(kv.v + off) = (uint16_t)code[1];
    }
    if (lane == 0) kv.scales[(int64_t)h * kv.num_pages + slot] = rec;
  }
  // In place of position tl of a sub-tile's registers, by way of the token's
  // V row of the wavefront's LDS tile (K's codes first, then V's).
  template <class E>
  __device__ __forceinline__ void put(uint8_t* tile, int tl, typename E::Regs& r) const {
    const int lane = threadIdx.x & 63;
    const int l16 = lane & 15, lg = lane >> 4;
    uint8_t* row = tile + tl * D;
    if (mine()) reinterpret_cast<uint16_t*>(row)[lane] = (uint16_t)code[0];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
      const bool at = l16 + 16 * tt == tl;
      if (at) r.rec[tt] = rec;
#pragma unroll
      for (int c = 0; c < E::K16; ++c) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(row + c * 64 + lg * 16);
        if (at) r.k16[tt][c] = w;
      }
#pragma unroll
      for (int c = 0; c < E::K8; ++c) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(row + E::K16 * 64 + c * 32 + lg * 8);
        if (at) r.k8[tt][c] = w;
      }
    }
    if (mine()) reinterpret_cast<uint16_t*>(row)[lane] = (uint16_t)code[1];
#pragma unroll
    for (int j = 0; j < E::NV; ++j) {
      const int ch = j * 64 + lane;
      const int t = ch / E::CH;
      const u32x4 w = *reinterpret_cast<const u32x4*>(row + (ch - t * E::CH) * 16);
      if (t == tl) r.v[j] = w;
    }
  }
};

// Positions [s_begin, s_end) of row b for kv-head h, as part `part` of the row
// (or its output); kv_len positions with page ids idx.  own_parts: of a split
// row, the parts of its own positions (it goes to the combine with the state).
template <int D, int G, bool ROPE>
__device__ __forceinline__ void decode8_rows(uint8_t* lds, const Decode8Args& a, int b, int h,
                                             const int32_t* idx, int kv_len, int s_begin, int s_end,
                                             int part, int own_parts) {
  using I = Item8<D, G>;
  using E = typename I::E;
  using RP = typename I::RP;
  constexpr int NW = I::NW;
  constexpr int DT = D / 16;
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int l16 = lane & 15;
  const int lg = lane >> 4;
  uint8_t* buf = lds + wave * I::WAVE_BYTES;
  uint8_t* stage = lds + NW * I::WAVE_BYTES + wave * I::STAGE_BYTES;
  const bool append = a.out_loc != nullptr;
  const int t_new = append ? kv_len - 1 : -1;

  E eng;
  eng.reset();
  const Kv8Head hd(a.kv, h, D);
  const bf16* qrow0 = a.q + (int64_t)b * a.q_tok_stride + (int64_t)(h * G) * D;
  const bf16* kn = append ? a.k_new + (int64_t)b * a.k_new_stride + (int64_t)h * D : nullptr;
  const bf16* vn = append ? a.v_new + (int64_t)b * a.v_new_stride + (int64_t)h * D : nullptr;
  const int kv0_first = s_begin + wave * kSubTok;
  if (kv0_first < s_end) {
    typename E::Regs r;
    typename E::Ids id;
    constexpr int STEP = NW * kSubTok;
    // The wavefront whose sub-tile holds the new token.
    const bool has_new = t_new >= s_begin && t_new < s_end &&
                         ((t_new - s_begin) / kSubTok & (NW - 1)) == wave;
    E::ids(idx, kv0_first, s_end - 1, id);
    E::load(hd, id, kv0_first, s_end, t_new, r);
    E::ids(idx, kv0_first + STEP, s_end - 1, id);
    if constexpr (ROPE) {
      const int64_t pos = (int64_t)a.positions[b];
      const int64_t rrow = min(max(pos, (int64_t)0), a.rope_rows - 1);
      RP rp;
      rp.load(qrow0, kn, a.q_norm, a.k_norm, a.rope_cos + rrow * D, a.rope_sin + rrow * D);
      rp.finish(stage, a.norm_eps);
      eng.load_q(reinterpret_cast<const bf16*>(stage) + min(l16, G - 1) * D, l16 < G);
    } else {
      eng.load_q(qrow0 + (int64_t)min(l16, G - 1) * D, l16 < G);
    }
    // The new token's rows are quantised here (K rotated from the staging
    // area) and written to page out_loc[b]; code and rec keep them for its
    // sub-tile.  (Nothing in the loop below may load or store memory but the
    // sub-tiles ahead: loads and stores complete in order, and behind a branch
    // that may hold others the compiler waits for all of them.)
    NewToken<D> nt;
    if (has_new) {
      const bf16* kr = ROPE ? reinterpret_cast<const bf16*>(stage) + G * D : kn;
      const int64_t slot = a.out_loc[b];
      nt.quantize(kr, vn);
      nt.in_pool = (uint32_t)idx[t_new] < hd.n_pages;
      if (slot >= 0 && slot < a.kv.num_pages) nt.write(a.kv, h, slot);
    }
    // One set of registers per sub-tile: K is used up by the scores and V by
    // its LDS store, so the next sub-tile's loads go out ahead of the softmax
    // and the O^T update, and three workgroups fit a unit.
    for (int kv0 = kv0_first; kv0 < s_end; kv0 += STEP) {
      if (has_new && nt.in_pool && kv0 <= t_new && t_new < kv0 + kSubTok)
        nt.template put<E>(buf, t_new - kv0, r);
      f32x4 st[2];
      E::store_v(buf, r);
      eng.scores(r, st);
      // (past the item's end: zeros, without a memory access)
      E::load(hd, id, kv0 + STEP, s_end, t_new, r);
      E::ids(idx, kv0 + 2 * STEP, s_end - 1, id);
      __builtin_amdgcn_sched_barrier(0);
      eng.update(buf, st, kv0, s_end, a.scale_log2);
    }
  }
  eng.ls = xrow_sum(eng.ls);

  // The G x D rows o / l of one state through LDS, in the destination's order.
  auto write_rows = [&](const f32x4 (&acc)[DT], float l_tot, float m, uint8_t* stage_buf, int part,
                        bool final) {
    const float inv = l_tot > 0.f ? 1.f / l_tot : l_tot * 0.f;
    float sc = inv, unscale = 1.f;
    if (!final) {
      float mx = 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, fabsf(acc[dt][i]));
      // (rows past G are zero or unused; a row's four lanes share its scale)
      sc *= part_scale(xrow_max(mx) * inv, unscale);
    }
    uint16_t* srows = reinterpret_cast<uint16_t*>(stage_buf);
    if (l16 < G) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const f32x4 v = acc[dt] * sc;
        const int e = final ? l16 * D + dt * 16 + lg * 4 : (dt * G + l16) * 16 + lg * 4;
        *reinterpret_cast<uint2*>(srows + e) =
            final ? make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]))
                  : make_uint2(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]));
      }
    }
    constexpr int NCH = G * D / 8;
    for (int c = lane; c < NCH; c += 64) {
      const uint4 v = reinterpret_cast<const uint4*>(srows)[c];
      if (final) {
        *reinterpret_cast<uint4*>(a.out + ((int64_t)b * a.num_qo_heads + h * G) * D + c * 8) = v;
      } else {
        const int dt = c * 8 / (G * 16);
        const int r = c * 8 - dt * G * 16;
        *reinterpret_cast<uint4*>(a.parts.o + a.parts.o_index(D, h, part, b * G + r / 16,
                                                             dt * 16 + (r & 15))) = v;
      }
    }
    if (!final && lg == 0 && l16 < G)
      a.parts.ls[a.parts.ls_index(h, part, b * G + l16)] =
          make_float2(lse_of(l_tot, m), __uint_as_float(__float_as_uint(unscale) | (uint32_t)own_parts));
  };

  if (a.wave_parts) {
    write_rows(eng.o, eng.ls, eng.m_run, buf, part + wave, false);
    return;
  }

  // The four wavefronts' states, merged by the first one.
  f32x4* so = reinterpret_cast<f32x4*>(buf);
  float* sm = reinterpret_cast<float*>(buf + DT * 64 * 16);
  float* sl = sm + 16;
  if (wave > 0) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) so[dt * 64 + lane] = eng.o[dt];
    if (lg == 0) {
      sm[l16] = eng.m_run;
      sl[l16] = eng.ls;
    }
  }
  __syncthreads();
  if (wave > 0) return;
  float mw[NW], lw[NW];
  mw[0] = eng.m_run;
  lw[0] = eng.ls;
  float mx = mw[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) {
    const float* smw = reinterpret_cast<const float*>(lds + w * I::WAVE_BYTES + DT * 64 * 16);
    mw[w] = smw[l16];
    lw[w] = smw[16 + l16];
    mx = fmaxf(mx, mw[w]);
  }
  float f[NW];
  float l_tot = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    f[w] = (mw[w] == kNegInf) ? lw[w] * 0.f : fast_exp2(mw[w] - mx);
    l_tot += lw[w] * f[w];
  }
  f32x4 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    acc[dt] = eng.o[dt] * f[0];
#pragma unroll
    for (int w = 1; w < NW; ++w)
      acc[dt] += reinterpret_cast<const f32x4*>(lds + w * I::WAVE_BYTES)[dt * 64 + lane] * f[w];
  }
  write_rows(acc, l_tot, mx, buf, part, a.final_out != 0);
}

// A row's own positions in equal parts of at most `most` (split: how many, and
// the length of each but the last), longer ones where that would be more than
// max_parts.
__device__ __forceinline__ int row_parts(int own, int most, int max_parts) {
  return min((int)(((uint32_t)max(own, 0) + (uint32_t)most - 1u) / (uint32_t)most), max_parts);
}
// The next longer split of a batch whose rows have more parts than its list
// (the lengths are the device's: rows may have outgrown the plan's); the last
// one leaves every row whole, and the list has a part for every row.
__device__ __forceinline__ int longer_split(int most) {
  return most < (1 << 30) ? most * 2 : 0x7fffffff;
}
__device__ __forceinline__ int row_part_len(int own, int parts) {
  return ((own + parts - 1) / parts + kSubTok - 1) / kSubTok * kSubTok;
}
// The sum of the lanes' n up to each one.
__device__ __forceinline__ int scan_add(int n) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    const int v = __shfl_up(n, k);
    if (lane >= k) n += v;
  }
  return n;
}
// The parts of all rows (uniform).
__device__ __forceinline__ int parts_of_all(const Decode8Args& a, int most, int max_parts) {
  int n = 0;
  for (int i = threadIdx.x & 63; i < a.batch; i += 64)
    n += row_parts(a.cu_k[i + 1] - a.cu_k[i] - a.prefix_len, most, max_parts);
  return __builtin_amdgcn_readlane(scan_add(n), 63);
}

// The by-value arguments behind an item's first loads, asked for with the row's
// bounds: used only here, the compiler loads them behind the wait for those (a
// memory round trip more ahead of the page ids and K/V).
__device__ __forceinline__ void args_with_bounds(const Decode8Args& a) {
  asm volatile("" ::"s"(a.kv.k), "s"(a.kv.v), "s"(a.kv.scales), "s"(a.kv.num_pages),
               "s"(a.kv.tok_bytes), "s"(a.q), "s"(a.q_tok_stride), "s"(a.k_new), "s"(a.v_new),
               "s"(a.k_new_stride), "s"(a.v_new_stride), "s"(a.scale_log2));
}

template <int D, int G, bool ROPE>
__device__ __forceinline__ void decode8_item(uint8_t* lds, const Decode8Args& a, int item) {
  int h, b, base, kv_len, s_begin, s_end, part = a.parts.n_chunks, own_parts = 0;
  if (!a.split) {
    h = item % a.num_kv_heads;
    b = item / a.num_kv_heads;
    base = a.cu_k[b];
    kv_len = a.cu_k[b + 1] - base;
    args_with_bounds(a);
    s_begin = a.prefix_len;
    s_end = kv_len;
  } else {
    // Part w of head h's list of all rows' parts, found from the lengths: lane
    // i counts the parts of row i.  (Parts side by side are one row's: heads
    // side by side read one page's rows from eight XCDs at once, 5 to 10% less
    // bandwidth.)
    const int lane = threadIdx.x & 63;
    h = item / a.n_splits;
    int w = item - h * a.n_splits;
    const int max_parts = a.parts.n_parts - a.parts.n_chunks;
    int most = a.split_len;
    // (the parts of more rows than lanes are counted ahead)
    if (a.batch > 64)
      while (parts_of_all(a, most, max_parts) > a.n_splits) most = longer_split(most);
    int own = 0, at = 0, n = 0, i = 0;
    for (int b0 = 0;; b0 += 64) {
      if (b0 >= a.batch) return;  // (fewer parts than the plan's longest rows have)
      i = b0 + lane;
      at = a.cu_k[min(i, a.batch)];
      own = a.cu_k[min(i + 1, a.batch)];
      args_with_bounds(a);
      own = i < a.batch ? own - at - a.prefix_len : 0;
      n = row_parts(own, most, max_parts);
      int sum = scan_add(n);
      if (a.batch <= 64 && __builtin_expect(__builtin_amdgcn_readlane(sum, 63) > a.n_splits, 0)) {
        do {
          most = longer_split(most);
          n = row_parts(own, most, max_parts);
          sum = scan_add(n);
        } while (__builtin_amdgcn_readlane(sum, 63) > a.n_splits);
      }
      const uint64_t past = __builtin_amdgcn_ballot_w64(sum > w);
      if (past) {
        const int src = __ffsll((unsigned long long)past) - 1;
        b = b0 + src;
        base = __builtin_amdgcn_readlane(at, src);
        own = __builtin_amdgcn_readlane(own, src);
        n = __builtin_amdgcn_readlane(n, src);
        w -= __builtin_amdgcn_readlane(sum, src) - n;
        break;
      }
      w -= __builtin_amdgcn_readlane(sum, 63);
    }
    own_parts = n;
    const int len = row_part_len(own, n);
    kv_len = own + a.prefix_len;
    s_begin = a.prefix_len + w * len;
    s_end = min(kv_len, s_begin + len);
    part += w;
  }
  decode8_rows<D, G, ROPE>(lds, a, b, h, a.indices + base, kv_len, s_begin, s_end, part,
                           own_parts);
}

template <int D, int G>
constexpr int decode8_lds(bool prefix) {
  constexpr int a = Stage8<D>::LDS_BYTES, b = Item8<D, G>::LDS_BYTES;
  return prefix && a > b ? a : b;
}

// The fields that come before a workgroup's first memory access lead the kernel
// arguments as scalars: with kernel-argument preloading they are in SGPRs at
// wave start (14 dwords of them), where a by-value struct takes a memory round
// trip ahead of the page ids.  The copies in Decode8Args are overridden with them.
// n_parts_flags: parts of a row, of the prefix among them (8 bits each), then
// the three flags.
__host__ __device__ inline int32_t parts_flags(const Decode8Args& a) {
  return a.parts.n_parts | a.parts.n_chunks << 8 | a.split << 16 | a.final_out << 17 |
         a.wave_parts << 18;
}

// Bound: with few bytes the chain launch - row bounds - page ids - K/V - math -
// states, with many the bandwidth of 128-byte rows.  32q/8kv x 128: 24 rows on a
// shared 4,096 8.7 us; 16 rows of 5,191 to 8,192 on scattered pages 53 us, 4.3
// TB/s (all 8,192 on pages in order: 57 us, 4.8 TB/s); one row of 16,001 of
// 16q/8kv 10.7 us, 3.1 TB/s; 8 rows of 24 + 16 of 8q/2kv x 96 5.2 us.  With the
// norm and rotation inside (ROPE), both launches without / with: the 24 rows 12.3 /
// 15.2 us, the 16 57.8 / 59.2, the one 13.9 / 14.9, the 8 5.2 / 5.8.
//
// PREFIX: the launch has prefix workgroups (first: they carry most bytes);
// without them the row items' smaller LDS lets more workgroups share a unit.
template <int D, int G, bool ROPE, bool PREFIX>
__global__ __launch_bounds__(kEngineThreads) __attribute__((amdgpu_waves_per_eu(PREFIX ? 2 : 3, PREFIX ? 2 : 8))) void decode8_main_kernel(
    const int32_t* __restrict__ indices, const int32_t* __restrict__ cu_k,
    const int32_t* __restrict__ out_loc, int32_t prefix_wgs, int32_t prefix_len, int32_t chunk_len,
    int32_t num_kv_heads, int32_t n_parts_flags, int32_t split_len, int32_t n_splits,
    int32_t batch, Decode8Args args) {
  __shared__ __align__(16) uint8_t lds[decode8_lds<D, G>(PREFIX)];
  Decode8Args a = args;
  a.indices = indices;
  a.cu_k = cu_k;
  a.out_loc = out_loc;
  a.prefix_wgs = prefix_wgs;
  a.prefix_len = PREFIX ? prefix_len : 0;
  a.chunk_len = chunk_len;
  a.num_kv_heads = num_kv_heads;
  a.num_qo_heads = num_kv_heads * G;
  a.parts.n_parts = n_parts_flags & 255;
  a.parts.n_chunks = n_parts_flags >> 8 & 255;
  a.prefix_units = a.parts.n_chunks * num_kv_heads;
  a.split = n_parts_flags >> 16 & 1;
  a.final_out = n_parts_flags >> 17 & 1;
  a.wave_parts = n_parts_flags >> 18 & 1;
  a.split_len = split_len;
  a.n_splits = n_splits;
  a.batch = batch;
  const int wg = blockIdx.x;
  if constexpr (PREFIX) {
    if (wg < a.prefix_wgs) {
      decode8_prefix_part<D, G, ROPE>(lds, a, wg);
      return;
    }
    decode8_item<D, G, ROPE>(lds, a, wg - a.prefix_wgs);
  } else {
    decode8_item<D, G, ROPE>(lds, a, wg);
  }
}

// ---------------------------------------------------------------------------
// combine: one workgroup per (row, kv-head); weight of part j for query row g
// 2^(lse_j - m) / sum_i 2^(lse_i - m) times the inverse of the part's scale.
// The states are asked for together with the weights' inputs (one memory round
// trip instead of two): a thread's first kBatch parts, all of them for up to 32
// parts of 4 heads x 128.  Bound: that trip and the launch, 2.8 to 3.5 us.
constexpr int kComb8Threads = 256;
constexpr int kComb8MaxParts = 64;
constexpr int kComb8Batch = 8;

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) x = fmaxf(x, __shfl_xor(x, k));
  return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) x += __shfl_xor(x, k);
  return x;
}

template <int D, int G>
__global__ __launch_bounds__(kComb8Threads) void decode8_combine_kernel(
    const float2* __restrict__ states, const _Float16* __restrict__ po_base,
    const int32_t* __restrict__ cu_k, bf16* __restrict__ out, int32_t n_parts_flags, int32_t rows,
    int32_t num_kv_heads, int32_t prefix_len) {
  constexpr int E8 = G * D / 8;  // 8-dim elements per part
  static_assert(E8 <= kComb8Threads, "one element per thread per part");
  constexpr int R = kComb8Threads / E8;  // threads sharing one element
  constexpr int NW = kComb8Threads / 64;
  constexpr int WP = kComb8MaxParts + 1;
  typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
  __shared__ float w_s[G * WP];
  __shared__ f32x4 red[2][kComb8Threads];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int b = blockIdx.x / num_kv_heads;
  const int h = blockIdx.x - b * num_kv_heads;
  Parts8 parts;
  parts.n_parts = n_parts_flags & 255;
  parts.n_chunks = n_parts_flags >> 8 & 255;
  parts.rows = rows;
  const bool split = n_parts_flags >> 16 & 1;
  const int last = parts.n_parts - 1;
  const int e = tid % E8;
  const int r = min(tid / E8, R - 1);  // (threads past R * E8 repeat another one's work)
  const int g = (e >> 1) % G;
  const int d = e / (2 * G) * 16 + (e & 1) * 8;
  const int64_t part_stride = (int64_t)(D / 16) * rows * 16;
  const _Float16* po = po_base + parts.o_index(D, h, 0, b * G + g, d);
  constexpr int LG = (G + NW - 1) / NW;  // query rows per wavefront
  float2 ls[LG];
#pragma unroll
  for (int i = 0; i < LG; ++i)
    ls[i] = states[parts.ls_index(h, min(lane, last), b * G + min(wave + i * NW, G - 1))];
  f16x8 v[kComb8Batch];
#pragma unroll
  for (int i = 0; i < kComb8Batch; ++i)
    v[i] = *reinterpret_cast<const f16x8*>(po + (int64_t)min(r + i * R, last) * part_stride);
  int np = parts.n_parts;  // (parts behind them were not written)
  if (split) {
    // (as the main launch counted them: see Parts8)
    const int own = __builtin_amdgcn_readlane(__float_as_int(ls[0].y), parts.n_chunks) & 127;
    np = parts.n_chunks + (cu_k[b + 1] - cu_k[b] > prefix_len ? own : 0);
  }
#pragma unroll
  for (int i = 0; i < LG; ++i) {
    if (wave + i * NW >= G) break;
    const float x = lane < np ? ls[i].x : kNegInf;
    const float mx = wave_max(x);
    const float w = fast_exp2(x - (mx == kNegInf ? 0.f : mx));
    const float den = wave_sum(w);
    const float unscale = __uint_as_float(__float_as_uint(ls[i].y) & 0xff800000u);
    w_s[(wave + i * NW) * WP + lane] = (den > 0.f ? w / den : den * 0.f) * (lane < np ? unscale : 0.f);
  }
  __syncthreads();
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
  auto add = [&](const f16x8& x, int j) {
    const float w = w_s[g * WP + j];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = fmaf((float)x[i], w, acc[i]);
  };
#pragma unroll
  for (int i = 0; i < kComb8Batch; ++i)
    if (r + i * R < np) add(v[i], r + i * R);
  for (int j = r + kComb8Batch * R; j < np; j += R)
    add(*reinterpret_cast<const f16x8*>(po + (int64_t)j * part_stride), j);
  f32x4 acc0 = f32x4{acc[0], acc[1], acc[2], acc[3]}, acc1 = f32x4{acc[4], acc[5], acc[6], acc[7]};
  if (R > 1) {
    red[0][tid] = acc0;
    red[1][tid] = acc1;
    __syncthreads();
    if (tid < E8)
      for (int rr = 1; rr < R; ++rr) {
        acc0 += red[0][rr * E8 + e];
        acc1 += red[1][rr * E8 + e];
      }
  }
  if (tid < E8)
    *reinterpret_cast<uint4*>(out + ((int64_t)b * num_kv_heads * G + h * G + g) * D + d) =
        make_uint4(pack_bf16x2(acc0[0], acc0[1]), pack_bf16x2(acc0[2], acc0[3]),
                   pack_bf16x2(acc1[0], acc1[1]), pack_bf16x2(acc1[2], acc1[3]));
}

template <int D, int G, bool ROPE, bool PREFIX>
void main_launch(const Decode8Args& a, hipStream_t s) {
  hipLaunchKernelGGL((decode8_main_kernel<D, G, ROPE, PREFIX>),
                     dim3(a.prefix_wgs + a.suffix_items), dim3(kEngineThreads), 0, s, a.indices,
                     a.cu_k, a.out_loc, a.prefix_wgs, a.prefix_len, a.chunk_len,
                     a.num_kv_heads, parts_flags(a), a.split_len, a.n_splits, a.batch, a);
}

template <int D, int G>
hipError_t main_dg(const Decode8Args& a, hipStream_t s) {
  if (a.prefix_wgs + a.suffix_items == 0) return hipSuccess;
  if (a.n_splits < 1 || a.parts.n_parts > kComb8MaxParts || a.num_qo_heads != a.num_kv_heads * G)
    return hipErrorInvalidValue;
  const bool rope = a.q_norm != nullptr;
  if (a.prefix_wgs > 0) {
    if (rope) main_launch<D, G, true, true>(a, s);
    else main_launch<D, G, false, true>(a, s);
  } else {
    if (rope) main_launch<D, G, true, false>(a, s);
    else main_launch<D, G, false, false>(a, s);
  }
  return hipGetLastError();
}

template <int D, int G>
hipError_t combine_dg(const Decode8Args& a, hipStream_t s) {
  const dim3 grid(a.batch * a.num_kv_heads);
  if (grid.x == 0) return hipSuccess;
  if (a.parts.n_parts > kComb8MaxParts) return hipErrorInvalidValue;
  hipLaunchKernelGGL((decode8_combine_kernel<D, G>), grid, dim3(kComb8Threads), 0, s, a.parts.ls,
                     a.parts.o, a.cu_k, a.out, parts_flags(a), a.parts.rows, a.num_kv_heads,
                     a.prefix_len);
  return hipGetLastError();
}

template <int D>
hipError_t by_group(const Decode8Args& a, bool main, hipStream_t s) {
  switch (a.group) {
    case 1: return main ? main_dg<D, 1>(a, s) : combine_dg<D, 1>(a, s);
    case 2: return main ? main_dg<D, 2>(a, s) : combine_dg<D, 2>(a, s);
    case 3: return main ? main_dg<D, 3>(a, s) : combine_dg<D, 3>(a, s);
    case 4: return main ? main_dg<D, 4>(a, s) : combine_dg<D, 4>(a, s);
    case 6: return main ? main_dg<D, 6>(a, s) : combine_dg<D, 6>(a, s);
    case 8: return main ? main_dg<D, 8>(a, s) : combine_dg<D, 8>(a, s);
    default: return hipErrorInvalidValue;
  }
}

hipError_t by_head(int D, const Decode8Args& a, bool main, hipStream_t s) {
  switch (D) {
    case 64: return by_group<64>(a, main, s);
    case 96: return by_group<96>(a, main, s);
    case 128: return by_group<128>(a, main, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_decode8_main(int D, const Decode8Args& a, hipStream_t s) {
  return by_head(D, a, true, s);
}
hipError_t launch_decode8_combine(int D, const Decode8Args& a, hipStream_t s) {
  return by_head(D, a, false, s);
}

}  // namespace aios
