// Log probabilities of given tokens over rows of logits, with the entropy of
// each row and its most likely alternatives.
//
// With m the row's maximum, d_i = x_i - m, Z = sum e^d_i, T = sum e^d_i d_i:
//   logprob(t) = d_t - ln Z       entropy = ln Z - T / Z
// One pass over the row: a thread keeps (m, Z, T) of its elements, moving all
// three to a new maximum m' by delta = m - m': Z' = Z e^delta, T' = (T + Z
// delta) e^delta.  Elements are subtracted from m before they are scaled for
// the exponential, so their error does not grow with |m|; d is held at -200 or
// more, where e^d is 0 in fp32, so that an excluded id (-inf, or the type's
// lowest value) adds 0 to both sums.  Bound: the logits, read once from HBM.
//
// Alternatives: the pass keeps the maximum of every 32 logits (a lane's share of
// a wavefront's batch), an order-preserving key of 4 bytes.  Afterwards the
// top-th largest of a wavefront's thread maxima is a lower limit that at least
// `top` logits reach; the few groups whose maximum reaches it are read again
// and their candidates ranked (equal logits: the lower id first).  Rows where
// too many logits reach the limit (equal ones, or fewer possible ids than
// alternatives) are streamed once more with a list per wavefront.
#include "kernels.hpp"

namespace aios {
namespace {

constexpr int kLpUnroll = 4;                       // 8-logit loads in flight per lane
constexpr int kLpBatch = 64 * 8 * kLpUnroll;       // logits per wavefront and batch
constexpr int kLpThreads = 256;
constexpr int kLpMergeThreads = 512;
constexpr int kLpWholeRow = 2 * 4 * kLpBatch;      // rows up to this are not split
constexpr int kLpMaxSegments = 64;                 // one per lane in the merge
constexpr int kLpCap = 128;                        // candidates that one wavefront ranks
constexpr int kLpMaxGroups = 8192;                 // group maxima in LDS
constexpr int kLpListCap = 512;                    // groups read again, and their candidates
constexpr float kLpLowest = -3.402823466e38f;      // maximum of no elements
constexpr float kLpMinD = -200.f;
static_assert(kLogprobMaxTop + 64 <= kLpCap, "64 more fit behind the kept ones");

// one: 1 where the maximum's own term is not in z (it is then the only term
// above 1/2, and ln Z = ln(1 + z) keeps what rounding next to 1 would lose).
struct LpState {
  float m, z, t, one;
};

// Order-preserving bits of a logit: larger is better, NaN best (all NaNs
// alike), -0 as +0.  Never 0.
__device__ __forceinline__ uint32_t lp_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  if (x != x) return 0xffc00000u;
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lp_unkey(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

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

// (z, t) of reference m relative to m_new >= m.
__device__ __forceinline__ void lp_move(float& z, float& t, float m, float m_new) {
  const float dl = vmax(m - m_new, kLpMinD);
  const float f = fast_exp2(dl * kLog2e);
  t = (t + z * dl) * f;
  z *= f;
}

// The 64-bit word of lane j (uniform) on every lane.
__device__ __forceinline__ uint64_t lp_lane(uint64_t x, int j) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), j) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)x, j);
}

// The best `top` of `count` <= kLpCap distinct keys at e -> get(e), by one
// wavefront: put(rank, key) for each.  Every key is compared with all of them
// out of the lanes' registers (a key takes two lane reads and a comparison).
template <typename Get, typename Put>
__device__ __forceinline__ void lp_rank(int count, int top, Get&& get, Put&& put) {
  const int lane = threadIdx.x & 63;
  constexpr int N = kLpCap / 64;
  uint64_t mine[N];
  int rank[N];
#pragma unroll
  for (int e = 0; e < N; ++e) {
    mine[e] = e * 64 + lane < count ? get(e * 64 + lane) : 0;
    rank[e] = 0;
  }
#pragma unroll
  for (int g = 0; g < N; ++g) {
    const int m = min(count - g * 64, 64);
    for (int j = 0; j < m; ++j) {
      const uint64_t k = lp_lane(mine[g], j);
#pragma unroll
      for (int e = 0; e < N; ++e) rank[e] += k > mine[e];
    }
  }
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (mine[e] != 0 && rank[e] < top) put(rank[e], mine[e]);
}

// A wavefront's candidates: buf[0 .. count), of which the best `top` are kept
// in descending order.  Every lane has the same count and limit.
struct LpTop {
  uint64_t* buf;
  int count;
  uint32_t limit;  // a logit is a candidate if its key is above
  int top;

  // Keeps the best `top`; returns the last kept one's key (0 while fewer).
  __device__ __forceinline__ uint64_t prune() {
    __builtin_amdgcn_wave_barrier();
    uint64_t last = 0;
    lp_rank(count, top, [&](int e) { return buf[e]; },
            [&](int r, uint64_t k) {
              buf[r] = k;
              if (r == top - 1) last = k;
            });
    __builtin_amdgcn_wave_barrier();
    count = min(count, top);
    const uint64_t who = __builtin_amdgcn_ballot_w64(last != 0);
    return who ? lp_lane(last, __ffsll((unsigned long long)who) - 1) : 0;
  }
  __device__ __forceinline__ void push(bool want, uint32_t key, uint32_t id) {
    const uint64_t who = __builtin_amdgcn_ballot_w64(want);
    if (want)
      buf[count + __popcll(who & ((1ull << (threadIdx.x & 63)) - 1))] =
          ((uint64_t)key << 32) | (uint32_t)~id;
    count += __popcll(who);
  }
};

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

// The state of elements [begin, end) of one row by the whole workgroup, in st
// on every thread; put(batch, key) gets every batch's maximum of the lane.
// Of a row with one likely id (Z < 2) the sums are small beside its term 1,
// and every addition to that term would round them at 2^-24: the thread that
// holds it has its logits summed again without it, by all threads.
template <int NT, typename T, typename Put>
__device__ __forceinline__ void lp_segment(const T* x, int begin, int end, bool want_max,
                                           LpState& st, LpState* wst, Put&& put) {
  constexpr int kLpThreads = NT, kLpWaves = NT / 64, kLpSegment = kLpWaves * kLpBatch;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float m = kLpLowest, z = 0.f, t = 0.f;
  for (int b0 = begin + wave * kLpBatch; b0 < end; b0 += kLpSegment) {
    float f[kLpUnroll][8];
    lp_load_batch(x, b0, end, f);
    float bm = kNegInf;
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u)
      bm = vmax(bm, vmax(vmax(vmax(f[u][0], f[u][1]), vmax(f[u][2], f[u][3])),
                         vmax(vmax(f[u][4], f[u][5]), vmax(f[u][6], f[u][7]))));
    if (want_max) put(b0 / kLpBatch, lp_key(bm));
    const float m_new = vmax(m, bm);
    lp_move(z, t, m, m_new);
    m = m_new;
    float bz = 0.f, bt = 0.f;
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      float uz = 0.f, ut = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = vmax(f[u][e] - m, kLpMinD);
        const float p = fast_exp2(d * kLog2e);
        uz += p;
        ut = fmaf(p, d, ut);
      }
      bz += uz;
      bt += ut;
    }
    z += bz;
    t += bt;
  }
  // the wavefront's sums relative to its maximum, then the workgroup's
  const float m0 = m, wm = lp_wave_max(m);
  lp_move(z, t, m, wm);
  float z1 = lp_wave_sum(z), t1 = lp_wave_sum(t);
  if (lane == 0) wst[wave] = LpState{wm, z1, t1, 0.f};
  __syncthreads();
  float gm = wst[0].m;
#pragma unroll
  for (int w = 1; w < kLpWaves; ++w) gm = vmax(gm, wst[w].m);
  float gz = 0.f, gt = 0.f;
#pragma unroll
  for (int w = 0; w < kLpWaves; ++w) {
    float wz = wst[w].z, wt = wst[w].t;
    lp_move(wz, wt, wst[w].m, gm);
    gz += wz;
    gt += wt;
  }
  st = LpState{gm, gz, gt, 0.f};
  if (gz < 2.f && gm > kLpLowest) {  // (the maximum is then one element's)
    __syncthreads();
    if (m0 == gm) wst[kLpWaves].t = __int_as_float((int)threadIdx.x);
    __syncthreads();
    const int ow = __float_as_int(wst[kLpWaves].t);
    lp_move(z, t, wm, gm);
    if ((int)threadIdx.x == ow) z = t = 0.f;
    const int rounds = (end - begin + kLpSegment - 1) / kLpSegment;
    const int own0 = begin + (ow >> 6) * kLpBatch + (ow & 63) * 8;
    for (int k = threadIdx.x; k < rounds * 32; k += kLpThreads) {
      const int64_t i = (int64_t)own0 + (int64_t)(k >> 5) * kLpSegment + (k >> 3 & 3) * 512 + (k & 7);
      if (i >= end) continue;
      const float d = vmax((float)x[i] - gm, kLpMinD);
      const float p = d < 0.f ? fast_exp2(d * kLog2e) : 0.f;
      z += p;
      t = fmaf(p, d, t);
    }
    z1 = lp_wave_sum(z);
    t1 = lp_wave_sum(t);
    if (lane == 0) wst[wave] = LpState{gm, z1, t1, 0.f};
    __syncthreads();
    gz = gt = 0.f;
#pragma unroll
    for (int w = 0; w < kLpWaves; ++w) {
      gz += wst[w].z;
      gt += wst[w].t;
    }
    st = LpState{gm, gz, gt, 1.f};
  }
}

// LDS of the selection: group maxima, then candidates.
template <int NT>
struct LpSelect {
  uint32_t group[kLpMaxGroups];
  uint64_t cand[NT / 64 * kLpCap];
  uint32_t list[kLpListCap];
  uint32_t wave_limit[NT / 64];
  int32_t n_list, n_cand;
};

// Batches per group: r consecutive ones of one wavefront (1 up to kLpMaxGroups
// * 32 logits).
template <int NT>
__device__ __forceinline__ int lp_rounds(int vocab) {
  return (vocab + NT / 64 * kLpBatch - 1) / (NT / 64 * kLpBatch);
}
template <int NT>
__device__ __forceinline__ int lp_groups_per(int vocab) {
  return (lp_rounds<NT>(vocab) * NT + kLpMaxGroups - 1) / kLpMaxGroups;
}

// put(rank, key) for the best `top` of n keys at e -> get(e), by the whole
// workgroup (0: no key).
template <int NT, typename Get, typename Put>
__device__ __forceinline__ void lp_rank_all(int n, int top, Get&& get, Put&& put) {
  for (int e = threadIdx.x; e < n; e += NT) {
    const uint64_t c = get(e);
    if (c == 0) continue;
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) rank += get(j) > c;
    if (rank < top) put(rank, c);
  }
}

// The `top` largest logits of a row, put(rank, key) for each, by the whole
// workgroup; sh.group holds the maxima of n_groups groups (and a barrier lies
// behind their writes).
template <int NT, typename T, typename Put>
__device__ __forceinline__ void lp_select(LpSelect<NT>& sh, const T* x, int vocab, int top,
                                          int n_groups, int r, Put&& put) {
  constexpr int NW = NT / 64;
  constexpr int CAP = NW * kLpCap < kLpListCap ? NW * kLpCap : kLpListCap;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint32_t mine = 0;
  for (int i = tid; i < n_groups; i += NT) mine = max(mine, sh.group[i]);
  // the largest value that at least `top` threads' maxima reach: by the largest
  // remaining one at a time (about 100 cycles each), from 12 on by all
  // comparisons
  uint32_t v;
  if (top < 12) {
    uint32_t left = mine;
    int reached = 0;
    do {
      v = lp_wave_max_u(left);
      reached += __popcll(__builtin_amdgcn_ballot_w64(left == v));
      if (left == v) left = 0;
    } while (reached < top && v != 0);
  } else {
    int reach = 0;
#pragma unroll 16
    for (int j = 0; j < 64; ++j) reach += (uint32_t)__builtin_amdgcn_readlane((int)mine, j) >= mine;
    v = lp_wave_max_u(reach >= top ? mine : 0u);
  }
  if (lane == 0) sh.wave_limit[wave] = v;
  if (tid == 0) sh.n_list = sh.n_cand = 0;
  __syncthreads();
  uint32_t limit = sh.wave_limit[0];
#pragma unroll
  for (int w = 1; w < NW; ++w) limit = max(limit, sh.wave_limit[w]);
  if (mine >= limit) {
    for (int i = tid; i < n_groups; i += NT)
      if (sh.group[i] >= limit) {
        const int at = atomicAdd(&sh.n_list, 1);
        if (at < kLpListCap) sh.list[at] = (uint32_t)i;
      }
  }
  __syncthreads();
  const int n_list = sh.n_list;
  if (n_list <= kLpListCap) {
    // one logit of a group per thread and round, two rounds in flight
    for (int l0 = tid >> 5; l0 < n_list; l0 += 2 * (NT / 32)) {
      const int k = tid & 31;
      for (int q = 0; q < r; ++q) {
        float xv[2];
        int64_t id[2];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int l = l0 + p * (NT / 32);
          const int g = (int)sh.list[l < n_list ? l : l0];
          const int gw = g >> 6;
          const int b = NW * (gw / NW * r + q) + gw % NW;
          id[p] = (int64_t)b * kLpBatch + (g & 63) * 8 + (k >> 3) * 512 + (k & 7);
          if (l >= n_list) id[p] = vocab;
          xv[p] = (float)x[id[p] < vocab ? id[p] : 0];
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const uint32_t key = lp_key(xv[p]);
          if (id[p] < vocab && key >= limit) {
            const int at = atomicAdd(&sh.n_cand, 1);
            if (at < CAP) sh.cand[at] = ((uint64_t)key << 32) | (uint32_t)~(uint32_t)id[p];
          }
        }
      }
    }
  }
  __syncthreads();
  const int n = sh.n_cand;
  if (n_list <= kLpListCap && n <= CAP) {
    if (n <= 64) {
      if (wave == 0) lp_rank(n, top, [&](int e) { return sh.cand[e]; }, put);
    } else {
      lp_rank_all<NT>(n, top, [&](int e) { return sh.cand[e]; }, put);
    }
    return;
  }
  // Streamed: every wavefront keeps the best of its batches, 64 logits at a
  // time in the order of their ids (so that behind a kept list only larger
  // values count), then the lists are joined.
  __syncthreads();
  LpTop best{sh.cand + wave * kLpCap, 0, limit ? limit - 1u : 0u, top};  // (no key is 0)
  for (int64_t b0 = wave * kLpBatch; b0 < vocab; b0 += NW * kLpBatch) {
    const int end = (int)min((int64_t)vocab, b0 + kLpBatch);
    for (int i0 = (int)b0; i0 < end; i0 += 64) {
      const int i = i0 + lane;
      const uint32_t key = i < end ? lp_key((float)x[i]) : 0u;
      if (__builtin_amdgcn_ballot_w64(key > best.limit) == 0) continue;
      best.push(key > best.limit, key, (uint32_t)i);
      if (best.count > kLpCap - 64) {
        const uint64_t last = best.prune();
        if (last != 0) best.limit = max(best.limit, (uint32_t)(last >> 32));
      }
    }
  }
  best.prune();
  for (int e = best.count + lane; e < top; e += 64) best.buf[e] = 0;
  __syncthreads();
  lp_rank_all<NT>(NW * top, top, [&](int e) { return sh.cand[e / top * kLpCap + e % top]; }, put);
}

// A row's token and its logit (NaN outside the vocabulary), asked for before the
// row's sums: two dependent loads, 2 us of a short row behind them.
template <typename T>
__device__ __forceinline__ float lp_token(const LogprobArgs& a, int64_t row, const T* x) {
  const int64_t tok = a.tokens[row];
  const bool ok = tok >= 0 && tok < a.vocab;
  const float v = (float)x[ok ? tok : 0];
  return ok ? v : __builtin_nanf("");
}

__device__ __forceinline__ void lp_finish(const LogprobArgs& a, int64_t row, float x_tok, double m,
                                          double z, double t, double ones, double& ln_z) {
  // Z = z + ones.  (No finite maximum: every element -inf leaves 0; a NaN or
  // +inf leaves NaN.)
  ln_z = ones > 0.0 ? log1p(z + (ones - 1.0)) : z > 0.0 ? log(z) : __builtin_nan("");
  if (threadIdx.x == 0) {
    a.logprobs[row] = (float)((double)x_tok - m - ln_z);
    a.entropies[row] = (float)(ln_z - t / (z + ones));
  }
}

__device__ __forceinline__ void lp_write_top(const LogprobArgs& a, int64_t row, double m,
                                             double ln_z, int rank, uint64_t key) {
  a.top_ids[row * a.top + rank] = (int64_t)(uint32_t)~(uint32_t)key;
  a.top_logprobs[row * a.top + rank] = (float)((double)lp_unkey((uint32_t)(key >> 32)) - m - ln_z);
}

// Segment s of row r (SPLIT: its state and maxima to the workspace).  2,048 rows
// of 151,936 bf16 logits 117 us, 5.3 TB/s, with one alternative 119 to 123; 5
// rows of 10,007 fp32 4.2 us, with 8 alternatives 8.0, by the chain of the
// selection.
template <typename T, bool SPLIT>
__global__ __launch_bounds__(kLpThreads) void logprob_kernel(LogprobArgs a, int32_t segs,
                                                             int32_t seg_len, LpState* states,
                                                             uint32_t* keys) {
  constexpr int NT = kLpThreads;
  __shared__ LpState wst[NT / 64 + 1];
  const int lane = threadIdx.x & 63;
  LpState st;
  if constexpr (SPLIT) {
    const int64_t row = blockIdx.x / segs;
    const int s = (int)(blockIdx.x - row * segs);
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
    const int begin = s * seg_len;
    const int batches = (a.vocab + kLpBatch - 1) / kLpBatch;
    uint32_t* out = keys + row * batches * 64;
    lp_segment<NT>(x, begin, min(a.vocab, begin + seg_len), a.top > 0, st, wst,
                   [&](int b, uint32_t key) { out[b * 64 + lane] = key; });
    if (threadIdx.x == 0) states[row * segs + s] = st;
  } else {
    __shared__ LpSelect<NT> sh;
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
    const float x_tok = lp_token(a, row, x);
    const int r = lp_groups_per<NT>(a.vocab);
    const int wave = threadIdx.x >> 6;
    const int rounds = lp_rounds<NT>(a.vocab);
    const int n_groups = (rounds + r - 1) / r * NT;
    // (a wavefront without a batch in the last round leaves its group empty)
    if (a.top > 0 && (rounds - 1) % r == 0 &&
        ((int64_t)(rounds - 1) * (NT / 64) + wave) * kLpBatch >= a.vocab)
      sh.group[(rounds - 1) / r * NT + threadIdx.x] = 0;
    lp_segment<NT>(x, 0, a.vocab, a.top > 0, st, wst, [&](int b, uint32_t key) {
      const int j = b / (NT / 64);
      uint32_t& g = sh.group[j / r * NT + threadIdx.x];
      g = j % r == 0 ? key : max(g, key);
    });
    double ln_z;
    lp_finish(a, row, x_tok, (double)st.m, (double)st.z, (double)st.t, (double)st.one, ln_z);
    if (a.top > 0)
      lp_select(sh, x, a.vocab, a.top, n_groups, r,
                [&](int rank, uint64_t k) { lp_write_top(a, row, (double)st.m, ln_z, rank, k); });
  }
}

// One workgroup per row: lane s of every wavefront takes segment s's sums (in
// 64 bits: exact references, one rounding at the end).  24 rows of 151,936 bf16
// logits, both launches: 7.2 us, with 5 alternatives 13.2 (their chain: maxima,
// limit, second read, ranks), with 20 18.7.
template <typename T>
__global__ __launch_bounds__(kLpMergeThreads) void logprob_merge_kernel(LogprobArgs a, int32_t segs,
                                                                        const LpState* states,
                                                                        const uint32_t* keys) {
  constexpr int NT = kLpMergeThreads;
  __shared__ LpSelect<NT> sh;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  const LpState st = lane < segs ? states[row * segs + lane] : LpState{kLpLowest, 0.f, 0.f, 0.f};
  const float x_tok = lp_token(a, row, x);
  const int r = lp_groups_per<NT>(a.vocab);
  const int batches = (a.vocab + kLpBatch - 1) / kLpBatch;
  const int n_groups = (lp_rounds<NT>(a.vocab) + r - 1) / r * NT;
  if (a.top > 0) {
    const uint32_t* in = keys + row * batches * 64;
    constexpr int N = kLpMaxGroups / NT;  // groups of a thread, their loads in flight together
    uint32_t key[N] = {};
    for (int q = 0; q < r; ++q) {
      uint32_t v[N];
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const int64_t at = ((int64_t)k * r + q) * NT + tid;  // batch * 64 + lane
        v[k] = at < (int64_t)batches * 64 ? in[at] : 0u;
      }
#pragma unroll
      for (int k = 0; k < N; ++k) key[k] = max(key[k], v[k]);
    }
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (k * NT < n_groups) sh.group[k * NT + tid] = key[k];
  }
  const float m = lp_wave_max(st.m);
  const double d = fmax((double)st.m - (double)m, -800.0);
  const double f = exp(d);
  // (terms left out of a segment's z stay apart where they are the row's)
  double one = d == 0.0 ? (double)st.one : 0.0;
  const double zs = (double)st.z + ((double)st.one - one);
  double z = zs * f, t = ((double)st.t + zs * d) * f;
  // (a NaN or +inf maximum: fmax dropped it)
  if (!__builtin_isfinite(m)) z = one = __builtin_nan("");
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) {
    z += __shfl_xor(z, k);
    t += __shfl_xor(t, k);
    one += __shfl_xor(one, k);
  }
  double ln_z;
  lp_finish(a, row, x_tok, (double)m, z, t, one, ln_z);
  if (a.top == 0) return;
  __syncthreads();
  lp_select(sh, x, a.vocab, a.top, n_groups, r,
            [&](int rank, uint64_t k) { lp_write_top(a, row, (double)m, ln_z, rank, k); });
}

template <typename T>
hipError_t launch(const LogprobArgs& a, int32_t segs, void* workspace, hipStream_t s) {
  const dim3 block(kLpThreads);
  if (segs <= 1) {
    hipLaunchKernelGGL((logprob_kernel<T, false>), dim3((unsigned)a.rows), block, 0, s, a, 1,
                       a.vocab, nullptr, nullptr);
    return hipGetLastError();
  }
  const int32_t seg_len = ((a.vocab + segs - 1) / segs + kLpBatch - 1) / kLpBatch * kLpBatch;
  LpState* states = static_cast<LpState*>(workspace);
  uint32_t* keys = reinterpret_cast<uint32_t*>(states + a.rows * segs);
  hipLaunchKernelGGL((logprob_kernel<T, true>), dim3((unsigned)(a.rows * segs)), block, 0, s, a,
                     segs, seg_len, states, keys);
  hipLaunchKernelGGL(logprob_merge_kernel<T>, dim3((unsigned)a.rows), dim3(kLpMergeThreads), 0, s, a,
                     segs, states, keys);
  return hipGetLastError();
}

}  // namespace

int32_t logprob_segments(int64_t rows, int32_t vocab, int32_t cus) {
  const int64_t want = (2ll * cus + rows - 1) / rows;
  int64_t n = vocab <= kLpWholeRow ? 1 : (vocab + 4 * kLpBatch - 1) / (4 * kLpBatch);
  if (n > want) n = want;
  if (n > kLpMaxSegments) n = kLpMaxSegments;
  if (n <= 1) return 1;
  // (no empty segments behind the rounding of their length)
  const int64_t len = ((vocab + n - 1) / n + kLpBatch - 1) / kLpBatch * kLpBatch;
  return (int32_t)((vocab + len - 1) / len);
}

int64_t logprob_workspace(int64_t rows, int32_t vocab, int32_t segments, int32_t top) {
  if (segments <= 1) return 0;
  const int64_t batches = (vocab + kLpBatch - 1) / kLpBatch;
  return rows * (segments * (int64_t)sizeof(LpState) + (top > 0 ? batches * 64 * 4 : 0));
}

hipError_t token_logprobs(const LogprobArgs& a, int32_t segments, void* workspace,
                          hipStream_t stream) {
  return a.elem_bytes == 2 ? launch<bf16>(a, segments, workspace, stream)
                           : launch<float>(a, segments, workspace, stream);
}

}  // namespace aios
