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
// Alternatives: each wavefront keeps the candidates that can still be among
// its `top` largest in LDS, as 64-bit keys (order-preserving value bits, then
// ~id: equal logits go to the lower id).  The first batch sets a lower limit,
// the top-th largest of the lanes' maxima, below which nothing is kept; a
// batch whose maximum does not pass the limit costs one comparison per lane.
#include "kernels.hpp"

namespace aios {
namespace {

constexpr int kLpThreads = 256;
constexpr int kLpWaves = kLpThreads / 64;
constexpr int kLpUnroll = 4;                       // 8-logit loads in flight per lane
constexpr int kLpBatch = 64 * 8 * kLpUnroll;       // logits per wavefront and batch
constexpr int kLpSegment = kLpWaves * kLpBatch;    // one batch of a workgroup
constexpr int kLpMaxSegments = 64;                 // one per lane in the merge
constexpr int kLpCap = 128;                        // candidates of a wavefront
constexpr float kLpLowest = -3.402823466e38f;      // maximum of no elements
constexpr float kLpMinD = -200.f;
static_assert(kLogprobMaxTop + 64 <= kLpCap, "a round of pushes fits behind the kept ones");

struct LpState {
  float m, z, t, pad;
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

__device__ __forceinline__ float lp_wave_max(float x) {
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) x = vmax(x, __shfl_xor(x, k));
  return x;
}
__device__ __forceinline__ float lp_wave_sum(float x) {
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) x += __shfl_xor(x, k);
  return x;
}

// (z, t) of reference m relative to m_new >= m.
__device__ __forceinline__ void lp_move(float& z, float& t, float m, float m_new) {
  const float dl = vmax(m - m_new, kLpMinD);
  const float f = fast_exp2(dl * kLog2e);
  t = (t + z * dl) * f;
  z *= f;
}

// A wavefront's candidates: buf[0 .. count), of which those of rank < top are
// kept in descending order.  Every lane has the same count.
struct LpTop {
  uint64_t* buf;
  int count;
  uint32_t limit;  // a logit is a candidate if its key is above
  int top;

  // Keeps the best `top`; returns the last kept one's key (0 while fewer).
  __device__ __forceinline__ uint64_t prune() {
    const int lane = threadIdx.x & 63;
    __builtin_amdgcn_wave_barrier();
    uint64_t mine[kLpCap / 64];
    int rank[kLpCap / 64];
#pragma unroll
    for (int e = 0; e < kLpCap / 64; ++e) {
      mine[e] = e * 64 + lane < count ? buf[e * 64 + lane] : 0;
      rank[e] = 0;
    }
    for (int j = 0; j < count; ++j) {
      const uint64_t k = buf[j];
#pragma unroll
      for (int e = 0; e < kLpCap / 64; ++e) rank[e] += k > mine[e];
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int e = 0; e < kLpCap / 64; ++e)
      if (mine[e] != 0 && rank[e] < top) buf[rank[e]] = mine[e];
    __builtin_amdgcn_wave_barrier();
    count = min(count, top);
    return count == top ? buf[top - 1] : 0;
  }

  __device__ __forceinline__ void push(bool want, uint32_t key, uint32_t id) {
    const uint64_t who = __builtin_amdgcn_ballot_w64(want);
    if (who == 0) return;
    if (count > kLpCap - 64) {
      // (the limit stays one below the last kept value: later rounds of the
      // same batch may hold that value at a lower id)
      const uint64_t last = prune();
      if (last != 0) limit = max(limit, (uint32_t)(last >> 32) - 1u);
    }
    const int lane = threadIdx.x & 63;
    if (want)
      buf[count + __popcll(who & ((1ull << lane) - 1))] = ((uint64_t)key << 32) | (uint32_t)~id;
    count += __popcll(who);
  }
};

// The state of elements [begin, end) of one row: every thread of the workgroup
// takes part; the result is in st and, if top > 0, cand[0 .. top) (missing
// ones 0), valid for wavefront 0 after the call.
template <typename T>
__device__ __forceinline__ void lp_segment(const T* x, int begin, int end, int top, LpState& st,
                                           uint64_t* cand, LpState* wst) {
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  float m = kLpLowest, z = 0.f, t = 0.f;
  LpTop best{cand + wave * kLpCap, 0, 0u, top};
  bool first = true;
  for (int b0 = begin + wave * kLpBatch; b0 < end; b0 += kLpWaves * kLpBatch) {
    float f[kLpUnroll][8];
    const int i0 = b0 + lane * 8;
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
    float bm = kNegInf;
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u)
      bm = vmax(bm, vmax(vmax(vmax(f[u][0], f[u][1]), vmax(f[u][2], f[u][3])),
                         vmax(vmax(f[u][4], f[u][5]), vmax(f[u][6], f[u][7]))));
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

    if (top > 0) {
      const uint32_t bk = lp_key(bm);
      if (first) {
        // limit: the top-th largest of the lanes' maxima (lanes without an
        // element hold the key of -inf, which is below or at every other)
        best.buf[lane] = ((uint64_t)bk << 32) | (uint32_t)(63 - lane);
        __builtin_amdgcn_wave_barrier();
        const uint64_t mine = best.buf[lane];
        int rank = 0;
        for (int j = 0; j < 64; ++j) rank += best.buf[j] > mine;
        __builtin_amdgcn_wave_barrier();
        const uint64_t at = __builtin_amdgcn_ballot_w64(rank == top - 1);
        best.limit = (uint32_t)__shfl((int)bk, __ffsll((unsigned long long)at) - 1) - 1u;
        first = false;
      }
      if (__builtin_amdgcn_ballot_w64(bk > best.limit) != 0) {
        const int before = best.count;
#pragma unroll
        for (int u = 0; u < kLpUnroll; ++u)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int id = i0 + u * 512 + e;
            const uint32_t k = lp_key(f[u][e]);
            best.push(k > best.limit && id < end, k, (uint32_t)id);
          }
        // every later id of this wavefront is higher, so from here on only
        // larger values than the last kept one count
        if (best.count > before || best.count >= top) {
          const uint64_t last = best.prune();
          if (last != 0) best.limit = max(best.limit, (uint32_t)(last >> 32));
        }
      }
    }
  }
  if (top > 0) {
    if (best.count > 0) best.prune();
    __builtin_amdgcn_wave_barrier();
    for (int e = best.count + lane; e < top; e += 64) best.buf[e] = 0;
  }
  // the wavefront's sums relative to its maximum
  const float wm = lp_wave_max(m);
  lp_move(z, t, m, wm);
  z = lp_wave_sum(z);
  t = lp_wave_sum(t);
  if (lane == 0) wst[wave] = LpState{wm, z, t, 0.f};
  __syncthreads();
  // the workgroup's
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
}

// The best `top` of n keys (0: none) in descending order: f(rank, key).
template <typename F>
__device__ __forceinline__ void lp_ranked(const uint64_t* keys, int n, int pitch, int per, int top,
                                          F&& f) {
  // entry e is keys[e / per * pitch + e % per]
  for (int e = threadIdx.x; e < n; e += kLpThreads) {
    const uint64_t mine = keys[e / per * pitch + e % per];
    if (mine == 0) continue;
    int rank = 0;
    for (int g = 0; g < n / per; ++g)
      for (int j = 0; j < per; ++j) rank += keys[g * pitch + j] > mine;
    if (rank < top) f(rank, mine);
  }
}

template <typename T>
__device__ __forceinline__ void lp_finish(const LogprobArgs& a, int64_t row, const T* x, double m,
                                          double z, double t, double& ln_z) {
  // (no finite maximum: every element -inf leaves z = 0; a NaN or +inf leaves NaN)
  ln_z = z > 0.0 ? log(z) : __builtin_nan("");
  if (threadIdx.x == 0) {
    const int64_t tok = a.tokens[row];
    const bool ok = tok >= 0 && tok < a.vocab;
    const double d = ok ? (double)(float)x[tok] - m : __builtin_nan("");
    a.logprobs[row] = (float)(d - ln_z);
    a.entropies[row] = (float)(ln_z - t / z);
  }
}

__device__ __forceinline__ void lp_write_top(const LogprobArgs& a, int64_t row, double m,
                                             double ln_z, int rank, uint64_t key) {
  a.top_ids[row * a.top + rank] = (int64_t)(uint32_t)~(uint32_t)key;
  a.top_logprobs[row * a.top + rank] = (float)((double)lp_unkey((uint32_t)(key >> 32)) - m - ln_z);
}

// Segment s of row r (segs > 1: its state to the workspace).
template <typename T>
__global__ __launch_bounds__(kLpThreads) void logprob_kernel(LogprobArgs a, int32_t segs,
                                                             int32_t seg_len, LpState* states,
                                                             uint64_t* keys) {
  __shared__ uint64_t cand[kLpWaves * kLpCap];
  __shared__ LpState wst[kLpWaves];
  const int64_t row = blockIdx.x / segs;
  const int s = (int)(blockIdx.x - row * segs);
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  const int begin = s * seg_len;
  const int end = min(a.vocab, begin + seg_len);
  LpState st;
  lp_segment(x, begin, end, a.top, st, cand, wst);
  const int n = kLpWaves * a.top;
  if (segs > 1) {
    const int64_t slot = row * segs + s;
    if (threadIdx.x == 0) states[slot] = st;
    uint64_t* out = keys + slot * a.top;
    // (a segment with fewer elements than `top` leaves 0 behind them)
    const int have = min(a.top, end - begin);
    for (int e = threadIdx.x; e < a.top; e += kLpThreads)
      if (e >= have) out[e] = 0;
    lp_ranked(cand, n, kLpCap, a.top, a.top, [&](int rank, uint64_t k) { out[rank] = k; });
    return;
  }
  double ln_z;
  lp_finish(a, row, x, (double)st.m, (double)st.z, (double)st.t, ln_z);
  lp_ranked(cand, n, kLpCap, a.top, a.top,
            [&](int rank, uint64_t k) { lp_write_top(a, row, (double)st.m, ln_z, rank, k); });
}

template <typename T>
__global__ __launch_bounds__(kLpThreads) void logprob_merge_kernel(LogprobArgs a, int32_t segs,
                                                                   const LpState* states,
                                                                   const uint64_t* keys) {
  __shared__ uint64_t cand[kLpMaxSegments * kLogprobMaxTop];
  const int64_t row = blockIdx.x;
  const int n = segs * a.top;
  for (int e = threadIdx.x; e < n; e += kLpThreads) cand[e] = keys[row * n + e];
  float m = kLpLowest;
  for (int s = 0; s < segs; ++s) m = vmax(m, states[row * segs + s].m);
  double z = 0.0, t = 0.0;
  for (int s = 0; s < segs; ++s) {
    const LpState st = states[row * segs + s];
    // (in 64 bits: exact references, one rounding at the end)
    const double d = fmax((double)st.m - (double)m, -800.0);
    const double f = d == 0.0 ? 1.0 : exp(d);
    t += ((double)st.t + (double)st.z * d) * f;
    z += (double)st.z * f;
  }
  double ln_z;
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  lp_finish(a, row, x, (double)m, z, t, ln_z);
  __syncthreads();
  if (a.top > 0)
    lp_ranked(cand, n, a.top, a.top, a.top,
              [&](int rank, uint64_t k) { lp_write_top(a, row, (double)m, ln_z, rank, k); });
}

template <typename T>
hipError_t launch(const LogprobArgs& a, int32_t segs, void* workspace, hipStream_t s) {
  const int32_t seg_len = ((a.vocab + segs - 1) / segs + 511) / 512 * 512;
  LpState* states = static_cast<LpState*>(workspace);
  uint64_t* keys = reinterpret_cast<uint64_t*>(states + (segs > 1 ? a.rows * segs : 0));
  hipLaunchKernelGGL(logprob_kernel<T>, dim3((unsigned)(a.rows * segs)), dim3(kLpThreads), 0, s, a,
                     segs, seg_len, states, keys);
  if (segs > 1)
    hipLaunchKernelGGL(logprob_merge_kernel<T>, dim3((unsigned)a.rows), dim3(kLpThreads), 0, s, a,
                       segs, states, keys);
  return hipGetLastError();
}

}  // namespace

int32_t logprob_segments(int64_t rows, int32_t vocab, int32_t cus) {
  const int64_t want = (2ll * cus + rows - 1) / rows;
  int64_t most = (vocab + kLpSegment - 1) / kLpSegment;
  if (most > kLpMaxSegments) most = kLpMaxSegments;
  int64_t n = want < most ? want : most;
  if (n < 1) n = 1;
  // (no empty segments behind the rounding of their length)
  const int64_t len = ((vocab + n - 1) / n + 511) / 512 * 512;
  return (int32_t)((vocab + len - 1) / len);
}

int64_t logprob_workspace(int64_t rows, int32_t segments, int32_t top) {
  return segments > 1 ? rows * segments * ((int64_t)sizeof(LpState) + 8 * top) : 0;
}

hipError_t token_logprobs(const LogprobArgs& a, int32_t segments, void* workspace,
                          hipStream_t stream) {
  return a.elem_bytes == 2 ? launch<bf16>(a, segments, workspace, stream)
                           : launch<float>(a, segments, workspace, stream);
}

}  // namespace aios
