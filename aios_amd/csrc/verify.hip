// Verification of drafted tokens against the target's probabilities, from given
// random numbers.
//
// A request is a tree of nodes: node 0 is decided, node i > 0 a draft behind its
// parent.  With p the target's distribution behind node v (at its temperature)
// and q the one that v's children were drawn from, the children are tried in the
// order of their indices.  Child x is accepted if u q(x) < p(x); if not, p becomes
// max(p - q, 0), normalised, for the next.  Written with sums over the vocabulary
//   F(l) = sum max(p - l q, 0),
// what p has become behind j rejected children is max(p - l_j q, 0) / F(l_j) with
//   l_0 = 0, F(l_0) = 1, l_{j+1} = l_j + F(l_j)
// (max(p_j - q, 0) = max(p - l_j q - F_j q, 0) / F_j), so one number stands for it,
// and the test is u F(l_j) q(x) < p(x) - l_j q(x).  Children without a q count as
// drawn with certainty: a rejected one is removed from p, F is what is left.
// The added token is the first id whose cumulative weight, in id order, exceeds
// u times the total.
//
// Which id a number falls on is decided by sums of up to 10^5 terms, so these are
// held in 64 bits, and the exponentials of their terms are taken with the
// exponent's rounding error added back: what remains are errors of 2^-24 a term
// with no common sign.  A common factor, such as a rounded reciprocal of a sum,
// would move every border between two ids the same way.
//
// Every node's outcome (the accepted child, or none) is independent of the way
// that leads to it, so the passes over the vocabulary run for all nodes at once:
//   stats  maximum and sums of the rows of nodes with children, by segments
//   join   those sums together, the first tests; F(1) where the first child of
//          several is rejected, by segments
//   walk   the other tests, the path, and the added token's weights by batches of
//          2048 ids (a leaf's row is read here only)
//   pick   the added token
// Bound: the rows, read once from HBM (those of F(1) and of the last node again).
#include "logits.hpp"

namespace aios {
namespace {

constexpr int kVNodes = kVerifyMaxNodes;
constexpr int kVThreads = 256;
static_assert(kVNodes <= kVThreads, "a node per thread");
constexpr int kVSpan = kVThreads / 64 * kLpBatch;  // logits of a workgroup's round
constexpr int kVMaxSegments = 64;                  // one per lane where they are joined
constexpr double kLn2 = 0.69314718055994530942;

// Sums of one segment of a row relative to its maximum m: s of exp((x - m) / T),
// s1 of exp(x - m); best: the first id at the maximum.
struct VPart {
  double s, s1;
  float m;
  int32_t best;
};
// A node: its rows' sums, relative to the maxima m (target) and mq (draft).
constexpr int kVNone = -1;    // next: no child is accepted
constexpr int kVOpen = -2;    // the first one is rejected, F(1) decides on the second
constexpr int kVMore = -3;    // (walk) F(lambda) is needed for the next
constexpr int kVSummed = 1;   // flags: m, s, s1 are set (the node has children)
constexpr int kVBad = 2;      // the target's row has no finite maximum
constexpr int kVBadDraft = 4;
struct VNode {
  double s, s1, sq;
  float m, mq;
  int32_t next, flags, best, pad;
};
// The last accepted node's row, as the pick needs it.
struct VLast {
  double s1;        // of the row (not of a leaf's)
  float m, mq, khi, klo;
  int32_t node;     // -1: nothing to pick
  int32_t flags;    // kVSummed: m is set
};
// A batch of that row, relative to m: the weights' sum, p's, and s1's terms.
struct VBatch {
  double w, p, s1;
  float m;
  int32_t best;
};

struct VScale {  // log2(e) / T in two floats
  float hi, lo;
};

// exp(d / T), d <= 0: the product's rounding error is added back.
__device__ __forceinline__ float vexp(float d, VScale c) {
  const float t = d * c.hi;
  const float r = fmaf(d, c.lo, fmaf(d, c.hi, -t));
  const float e = fast_exp2(t);
  return t > -150.f ? fmaf(e, r * (float)kLn2, e) : 0.f;
}
__device__ __forceinline__ double vexp64(double d, double inv_t) {
  return d * inv_t > -1000.0 ? exp(d * inv_t) : 0.0;
}

__device__ __forceinline__ double wave_sum64(double x) {
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) x += __shfl_xor(x, i);
  return x;
}
__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) x = min(x, __shfl_xor(x, i));
  return x;
}
__device__ __forceinline__ bool finite_max(float m) { return m > kNegInf && m < __builtin_inff(); }

// The request of a node (workgroup-uniform), or -1, with its first node and size.
__device__ __forceinline__ int locate(const VerifyArgs& a, int64_t node, int64_t& first, int& n) {
  int r = 0;
  for (int t0 = 0; t0 < a.batch; t0 += kVThreads) {
    const int t = t0 + threadIdx.x;
    r += __syncthreads_count(t < a.batch && a.cu[t + 1] <= node);
  }
  if (r >= a.batch) return -1;
  first = a.cu[r];
  const int64_t size = (int64_t)a.cu[r + 1] - first;
  n = (int)(size < kVNodes ? size : kVNodes);
  return first >= 0 && first <= node && node < first + n && first + n <= a.total ? r : -1;
}

// A draft's random number; one that is not below 1 accepts nothing.
__device__ __forceinline__ double number(float u) { return u < 1.f ? u : __builtin_inf(); }

template <typename T>
__device__ __forceinline__ const T* row_of(const void* x, int64_t stride, int64_t node) {
  return static_cast<const T*>(x) + node * stride;
}

// -- stats ---------------------------------------------------------------------

// One workgroup per (node, segment) and row kind (the target's, then the drafts').
template <typename T, bool GREEDY>
__global__ __launch_bounds__(kVThreads) void verify_stats_kernel(VerifyArgs a, VPart* parts) {
  __shared__ double ss[4], ss1[4];
  __shared__ float sm[4];
  __shared__ int sb[4];
  const int seg = blockIdx.x % a.segments;
  const int64_t rest = blockIdx.x / a.segments;
  const int which = rest >= a.total;
  const int64_t node = rest - which * a.total;
  int64_t first;
  int n;
  if (locate(a, node, first, n) < 0) return;
  const int i = (int)(node - first), tid = threadIdx.x;
  if (!__syncthreads_or(tid > i && tid < n && a.parents[first + tid] == i)) return;
  const T* x = which ? row_of<T>(a.draft, a.draft_stride, node) : row_of<T>(a.logits, a.stride, node);
  const VScale c = which ? VScale{a.dhi, a.dlo} : VScale{a.thi, a.tlo};
  const double inv_t = which ? a.inv_dt : a.inv_t;
  const bool same = which || a.inv_t == 1.0;  // (no second sum)
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int begin = seg * a.seg_len, end = min(a.vocab, begin + a.seg_len);
  float m = kNegInf;
  double s = 0, s1 = 0;
  int best = 0x7fffffff;
  for (int b0 = begin + wave * kLpBatch; b0 < end; b0 += kVSpan) {
    float f[kLpUnroll][8];
    lp_load_batch(x, b0, end, f);
    float bm = kNegInf;
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u)
      bm = vmax(bm, vmax(vmax(vmax(f[u][0], f[u][1]), vmax(f[u][2], f[u][3])),
                         vmax(vmax(f[u][4], f[u][5]), vmax(f[u][6], f[u][7]))));
    const float m_new = vmax(m, lp_wave_max(bm));
    if (m_new != m) {  // (uniform; also for a NaN)
      s *= vexp64((double)m - m_new, inv_t);
      if constexpr (!GREEDY) s1 *= vexp64((double)m - m_new, 1.0);
      m = m_new;
      best = 0x7fffffff;
    }
    const float mu = m == kNegInf ? 0.f : m;
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      float us = 0.f, us1 = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = f[u][e] - mu;
        if constexpr (GREEDY) {
          us += fast_exp2(d * kLog2e);
          if (f[u][e] == m)
            best = min(best, b0 + u * 512 + (tid & 63) * 8 + e);
        } else {
          us += vexp(d, c);
          if (!same) us1 += fast_exp2(d * kLog2e);
        }
      }
      s += us;
      s1 += us1;
    }
  }
  s = wave_sum64(s);
  if constexpr (GREEDY) best = wave_min(best);
  else if (!same) s1 = wave_sum64(s1);
  if ((tid & 63) == 0) {
    ss[wave] = s;
    ss1[wave] = s1;
    sm[wave] = m;
    sb[wave] = best;
  }
  __syncthreads();
  if (tid == 0) {
    VPart p;
    p.m = vmax(vmax(sm[0], sm[1]), vmax(sm[2], sm[3]));
    p.s = p.s1 = 0;
    p.best = 0x7fffffff;
    const float mu = p.m == kNegInf ? 0.f : p.m;
    for (int w = 0; w < 4; ++w) {
      const double d = (double)sm[w] - mu;
      p.s += ss[w] * vexp64(d, GREEDY ? 1.0 : inv_t);
      p.s1 += ss1[w] * vexp64(d, 1.0);
      if (sm[w] == p.m) p.best = min(p.best, sb[w]);
    }
    if (GREEDY || same) p.s1 = p.s;
    parts[(node * (a.draft ? 2 : 1) + which) * a.segments + seg] = p;
  }
}

// A row's sums from its segments, by one wavefront (every lane has them).
__device__ __forceinline__ VPart join(const VPart* parts, int n, double inv_t) {
  const int lane = threadIdx.x & 63;
  VPart p = {0, 0, kNegInf, 0x7fffffff};
  if (lane < n) p = parts[lane];
  VPart r;
  r.m = lp_wave_max(p.m);
  const float mu = r.m == kNegInf ? 0.f : r.m;
  r.s = wave_sum64(p.s * vexp64((double)p.m - mu, inv_t));
  r.s1 = wave_sum64(p.s1 * vexp64((double)p.m - mu, 1.0));
  r.best = wave_min(p.m == r.m ? p.best : 0x7fffffff);
  return r;
}

// -- weights of a batch ----------------------------------------------------------

// A row whose added token is drawn: w = p - k q (drawn drafts; k = lambda S_p /
// S_q, so that both are in units of p's exponentials), relative to m.
struct VRow {
  const void* x;
  const void* q;
  float m, mq, khi, klo;
  bool own_max;  // m is not known: each batch takes its own
};

// Weights and p of the lane's logits of batch b0; returns the batch's reference.
// skip(id): removed ids' weights are 0.
template <typename T, bool DRAWN>
__device__ __forceinline__ float batch_weights(const VerifyArgs& a, const VRow& r, int b0,
                                               const int64_t* gone, int n_gone,
                                               float (&w)[kLpUnroll][8], double& p, double& s1) {
  float f[kLpUnroll][8];
  lp_load_batch(static_cast<const T*>(r.x), b0, a.vocab, f);
  float m = r.m;
  if (r.own_max) {
    m = kNegInf;
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) m = vmax(m, f[u][e]);
    m = lp_wave_max(m);
  }
  const float mu = m == kNegInf ? 0.f : m;
  const VScale c = {a.thi, a.tlo}, cd = {a.dhi, a.dlo};
  p = s1 = 0;
#pragma unroll
  for (int u = 0; u < kLpUnroll; ++u) {
    float up = 0.f, us1 = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = f[u][e] - mu;
      w[u][e] = vexp(d, c);
      up += w[u][e];
      if (r.own_max) us1 += fast_exp2(d * kLog2e);
    }
    p += up;
    s1 += us1;
  }
  if constexpr (DRAWN) {
    if (r.khi != 0.f) {  // (uniform)
      lp_load_batch(static_cast<const T*>(r.q), b0, a.vocab, f);
#pragma unroll
      for (int u = 0; u < kLpUnroll; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float q = vexp(f[u][e] - r.mq, cd);
          w[u][e] = fmaxf(fmaf(-q, r.klo, fmaf(-q, r.khi, w[u][e])), 0.f);
        }
    }
  }
  for (int j = 0; j < n_gone; ++j) {
    const int64_t off = gone[j] - b0;
    if (off < 0 || off >= kLpBatch) continue;  // (uniform)
    const int at = (int)off - (threadIdx.x & 63) * 8;
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (at == u * 512 + e) w[u][e] = 0.f;
  }
  return m;
}

// lambda S_p / S_q in two floats.
__device__ __forceinline__ void split_k(double k, float& hi, float& lo) {
  hi = (float)k;
  lo = (float)(k - (double)hi);
}

// Sum of max(p - l q, 0) over [begin, end), in units of p's exponentials, by the
// whole workgroup (every thread has it).
template <typename T>
__device__ __forceinline__ double residual_sum(const VerifyArgs& a, VRow r, int begin, int end,
                                               double* sh) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  double sum = 0;
  for (int b0 = begin + wave * kLpBatch; b0 < end; b0 += kVSpan) {
    float w[kLpUnroll][8];
    double p, s1;
    batch_weights<T, true>(a, r, b0, nullptr, 0, w, p, s1);
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) s += w[u][e];
      sum += s;
    }
  }
  sum = wave_sum64(sum);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[wave] = sum;
  __syncthreads();
  return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

// -- join ------------------------------------------------------------------------

// One workgroup per node, or (drawn drafts) per (node, segment).
template <typename T, bool DRAWN, bool GREEDY>
__global__ __launch_bounds__(kVThreads) void verify_join_kernel(VerifyArgs a, const VPart* parts,
                                                                VNode* nodes, double* f1) {
  __shared__ VPart sp[2];
  __shared__ double sh[4];
  __shared__ double kp[kVNodes], kq[kVNodes];
  __shared__ int64_t ktok[kVNodes];
  __shared__ double ku[kVNodes];
  __shared__ int kid[kVNodes];
  __shared__ int s_next, s_wave[4];
  const int segs = DRAWN ? a.segments : 1;
  const int seg = blockIdx.x % segs;
  const int64_t node = blockIdx.x / segs;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int64_t first = 0;
  int n = 0;
  if (locate(a, node, first, n) < 0) {
    if (tid == 0 && seg == 0) {  // behind the last request, or past the nodes of one
      a.accepted[node] = 0;
      a.logprobs[node] = __builtin_nanf("");
    }
    return;
  }
  const int i = (int)(node - first);
  const int par = tid < n ? a.parents[first + tid] : -1;
  const bool is_kid = tid > i && tid < n && par == i;
  const uint64_t who = __builtin_amdgcn_ballot_w64(is_kid);
  if (lane == 0) s_wave[wave] = __popcll(who);
  if (i == 0 && seg == 0 && tid > 0 && tid < n && (par < 0 || par >= tid))
    a.logprobs[first + tid] = __builtin_nanf("");
  __syncthreads();
  int base = 0, k = 0;
  for (int w = 0; w < 4; ++w) {
    if (w < wave) base += s_wave[w];
    k += s_wave[w];
  }
  if (k == 0) {
    if (tid == 0 && seg == 0) nodes[node] = VNode{0, 0, 0, 0.f, 0.f, kVNone, 0, 0, 0};
    return;
  }
  const VPart* mine = parts + node * (DRAWN ? 2 : 1) * a.segments;
  if (wave == 0) {
    const VPart p = join(mine, a.segments, GREEDY ? 1.0 : a.inv_t);
    if (lane == 0) sp[0] = p;
  } else if (DRAWN && wave == 1) {
    const VPart p = join(mine + a.segments, a.segments, a.inv_dt);
    if (lane == 0) sp[1] = p;
  }
  __syncthreads();
  const VPart p = sp[0], q = DRAWN ? sp[1] : VPart{};
  const bool bad = !finite_max(p.m), bad_draft = DRAWN && !finite_max(q.m);
  if (is_kid) {
    const int j = base + __popcll(who & ((1ull << lane) - 1));
    const int64_t tok = a.tokens[first + tid];
    const bool in = tok >= 0 && tok < a.vocab;
    const float x = in ? (float)row_of<T>(a.logits, a.stride, node)[tok] : kNegInf;
    kid[j] = tid;
    ktok[j] = tok;
    ku[j] = GREEDY ? 0.0 : number(a.uniforms[first + tid]);
    kp[j] = bad || !in ? 0.0 : vexp64((double)x - p.m, a.inv_t) / p.s;
    if constexpr (DRAWN) {
      const float y = in ? (float)row_of<T>(a.draft, a.draft_stride, node)[tok] : kNegInf;
      kq[j] = bad_draft || !in ? 0.0 : vexp64((double)y - q.m, a.inv_dt) / q.s;
    }
    if (seg == 0)
      a.logprobs[first + tid] =
          bad || !in ? __builtin_nanf("") : (float)(((double)x - p.m) - log(p.s1));
  }
  __syncthreads();
  if (tid == 0) {
    int next = kVNone;
    if (bad || bad_draft) {
    } else if (GREEDY) {
      for (int j = 0; j < k && next < 0; ++j)
        if (ktok[j] == p.best) next = kid[j];
    } else if (DRAWN) {
      if (ku[0] * kq[0] < kp[0]) next = kid[0];
      else if (k > 1) next = kVOpen;
    } else {
      double left = 1.0;
      for (int j = 0; j < k && next < 0; ++j) {
        double pj = kp[j];
        for (int l = 0; l < j; ++l)
          if (ktok[l] == ktok[j]) pj = 0.0;
        if (ku[j] * left < pj) next = kid[j];
        left -= pj;
      }
    }
    s_next = next;
    if (seg == 0)
      nodes[node] = VNode{p.s, p.s1, q.s, p.m, q.m, next,
                          kVSummed | (bad ? kVBad : 0) | (bad_draft ? kVBadDraft : 0),
                          p.best, 0};
  }
  if constexpr (DRAWN) {
    __syncthreads();
    if (s_next != kVOpen) return;  // (uniform)
    VRow r = {row_of<T>(a.logits, a.stride, node), row_of<T>(a.draft, a.draft_stride, node),
              p.m, q.m, 0.f, 0.f, false};
    split_k(p.s / q.s, r.khi, r.klo);
    const int begin = seg * a.seg_len;
    const double f = residual_sum<T>(a, r, begin, min(a.vocab, begin + a.seg_len), sh);
    if (tid == 0) f1[node * a.segments + seg] = f / p.s;
  }
}

// -- walk ------------------------------------------------------------------------

// Inclusive sums over the workgroup's threads, in their order.
__device__ __forceinline__ double block_scan(double x, double* sh, double& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) {
    const double y = __shfl_up(x, i);
    if (lane >= i) x += y;
  }
  __syncthreads();
  if (lane == 63) sh[wave] = x;
  __syncthreads();
  double base = 0;
  total = 0;
  for (int w = 0; w < 4; ++w) {
    if (w < wave) base += sh[w];
    total += sh[w];
  }
  return base + x;
}

// The added token of one request from its row's batches, by the whole workgroup.
template <typename T, bool DRAWN, bool GREEDY>
__device__ __forceinline__ void pick(const VerifyArgs& a, int req, const VLast& l, const VRow& r,
                                     const VBatch* batches, const int64_t* gone, int n_gone,
                                     int64_t first) {
  __shared__ double sh[4];
  __shared__ float shm[4];
  __shared__ int si[4];
  __shared__ double s_base;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int nb = (a.vocab + kLpBatch - 1) / kLpBatch;
  float m = l.m;
  double s1 = l.s1;
  if (r.own_max) {
    m = kNegInf;
    for (int b = tid; b < nb; b += kVThreads) m = vmax(m, batches[b].m);
    m = lp_wave_max(m);
    if (lane == 0) shm[wave] = m;
    __syncthreads();
    m = vmax(vmax(shm[0], shm[1]), vmax(shm[2], shm[3]));
    if (!finite_max(m)) {  // (uniform)
      if (tid == 0) {
        a.next_tokens[req] = -1;
        a.logprobs[first] = __builtin_nanf("");
      }
      return;
    }
    s1 = 0;
    for (int b = tid; b < nb; b += kVThreads)
      s1 += batches[b].s1 * vexp64((double)batches[b].m - m, 1.0);
    double total;
    block_scan(s1, sh, total);
    s1 = total;
  }
  if constexpr (GREEDY) {
    int best = 0x7fffffff;
    for (int b = tid; b < nb; b += kVThreads)
      if (batches[b].m == m) best = min(best, batches[b].best);
    best = wave_min(best);
    if (lane == 0) si[wave] = best;
    __syncthreads();
    if (tid == 0) {
      a.next_tokens[req] = min(min(si[0], si[1]), min(si[2], si[3]));
      a.logprobs[first] = (float)-log(s1);
    }
    return;
  }
  // weights of batch b in the row's units; without any mass left, p's own
  auto scale = [&](int b) {
    return r.own_max ? vexp64((double)batches[b].m - m, a.inv_t) : 1.0;
  };
  auto sum = [&](int b, bool residual) {
    return b < nb ? (residual ? batches[b].w : batches[b].p) * scale(b) : 0.0;
  };
  bool residual = true;
  double total = 0;
  for (int t = 0; t < 2; ++t) {
    total = 0;
    for (int b0 = 0; b0 < nb; b0 += kVThreads) {
      double part;
      block_scan(sum(b0 + tid, residual), sh, part);
      total += part;
    }
    if (total > 0) break;  // (uniform)
    residual = false;
  }
  const double target = (double)a.uniforms[first] * total;
  // the first batch past the target, or the last one with any weight
  double base = 0;
  int at = 0x7fffffff, last = -1;
  for (int b0 = 0; b0 < nb; b0 += kVThreads) {
    const double x = sum(b0 + tid, residual);
    double part;
    const double cum = base + block_scan(x, sh, part);
    const int hit = wave_min(cum > target && x > 0 ? b0 + tid : 0x7fffffff);
    const int any = -wave_min(x > 0 ? -(b0 + tid) : 0x7fffffff);
    __syncthreads();
    if (lane == 0) {
      si[wave] = hit;
      shm[wave] = __int_as_float(any);
    }
    __syncthreads();
    at = min(min(si[0], si[1]), min(si[2], si[3]));
    for (int w = 0; w < 4; ++w) last = max(last, __float_as_int(shm[w]));
    if (at != 0x7fffffff) {
      if (b0 + tid == at) s_base = cum - x;
      break;  // (uniform)
    }
    base += part;
  }
  const bool found = at != 0x7fffffff;
  if (!found) at = last;
  __syncthreads();
  if (wave != 0) return;
  // inside the batch: eight logits a lane, 512 at a time
  float w[kLpUnroll][8];
  double p, unused;
  VRow one = r;
  if (!residual) one.khi = one.klo = 0.f;
  const float bm = batch_weights<T, DRAWN>(a, one, at * kLpBatch, gone, residual ? n_gone : 0, w, p,
                                           unused);
  const double f = scale(at);
  double run = found ? s_base : 0.0;
  int got = 0x7fffffff, tail = -1;
#pragma unroll
  for (int u = 0; u < kLpUnroll; ++u) {
    double s = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) s += w[u][e];
    s *= f;
    double inc = s;
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) {
      const double y = __shfl_up(inc, i);
      if (lane >= i) inc += y;
    }
    double c = run + (inc - s);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int id = at * kLpBatch + u * 512 + lane * 8 + e;
      c += w[u][e] * f;
      if (w[u][e] > 0.f) {
        tail = id;
        if (found && c > target) got = min(got, id);
      }
    }
    run += __shfl(inc, 63);
  }
  got = wave_min(got);
  tail = -wave_min(-tail);
  const int id = got != 0x7fffffff ? got : tail;
  if (lane == 0) {
    a.next_tokens[req] = id;
    const float x = (float)static_cast<const T*>(r.x)[id];
    a.logprobs[first] = (float)(((double)x - m) - log(s1));
  }
}

// Tokens of a node's children, in gone (drafts without a distribution: all of
// them are rejected where the token is added).  Returns their number.
__device__ __forceinline__ int rejected(const VerifyArgs& a, int64_t first, int n, int v,
                                        int64_t* gone, int* count) {
  const int tid = threadIdx.x;
  if (tid == 0) *count = 0;
  __syncthreads();
  if (tid > v && tid < n && a.parents[first + tid] == v)
    gone[atomicAdd(count, 1)] = a.tokens[first + tid];
  __syncthreads();
  return *count;  // (their order does not matter)
}

// A workgroup per (request, round of batches): the path, found by every one of
// them, and its share of the batches; with one a request also the added token.
template <typename T, bool DRAWN, bool GREEDY>
__global__ __launch_bounds__(kVThreads) void verify_walk_kernel(VerifyArgs a, const VNode* nodes,
                                                                const double* f1, VLast* lasts,
                                                                VBatch* batches) {
  __shared__ int par[kVNodes], next[kVNodes], tries[kVNodes];
  __shared__ double lam[kVNodes], mass[kVNodes];
  __shared__ uint8_t on_path[kVNodes];
  __shared__ int64_t gone[kVNodes];
  __shared__ int s_v, s_count, s_gone;
  __shared__ double sh[4];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wgs = a.walk_wgs;
  const int c = blockIdx.x % wgs, req = blockIdx.x / wgs;
  const int64_t first = a.cu[req];
  const int64_t size = (int64_t)a.cu[req + 1] - first;
  const int n = (int)(size < kVNodes ? size : kVNodes);
  if (n <= 0 || first < 0 || first + n > a.total) {
    if (c == 0 && tid == 0) {
      a.counts[req] = 0;
      a.last[req] = -1;
      a.next_tokens[req] = -1;
      lasts[req].node = -1;
    }
    return;
  }
  if (tid < n) {
    const VNode& v = nodes[first + tid];
    par[tid] = a.parents[first + tid];
    next[tid] = v.next;
    on_path[tid] = 0;
    if constexpr (DRAWN) {
      lam[tid] = 1.0;  // (behind one rejected child)
      double f = 0;
      if (v.next == kVOpen)
        for (int s = 0; s < a.segments; ++s) f += f1[(first + tid) * a.segments + s];
      mass[tid] = f;
      tries[tid] = 1;
    }
  }
  __syncthreads();
  // Tests of node v's next child against what p has become (mass, lam): sets
  // next[v] to the child, kVNone, or kVMore where F is needed again.
  auto test = [&](int v) {
    const VNode& nd = nodes[first + v];
    int left = tries[v];
    for (int i = v + 1; i < n; ++i) {
      if (par[i] != v) continue;
      if (left > 0) {
        --left;
        continue;
      }
      if (tries[v] < 0) {  // (the tested child was not the last one)
        next[v] = kVMore;
        tries[v] = -tries[v];
        return;
      }
      const int64_t tok = a.tokens[first + i];
      double p = 0, q = 0;
      if (tok >= 0 && tok < a.vocab) {
        p = vexp64((double)(float)row_of<T>(a.logits, a.stride, first + v)[tok] - nd.m, a.inv_t) /
            nd.s;
        q = vexp64((double)(float)row_of<T>(a.draft, a.draft_stride, first + v)[tok] - nd.mq,
                   a.inv_dt) / nd.sq;
      }
      if (number(a.uniforms[first + i]) * mass[v] * q < p - lam[v] * q) {
        next[v] = i;
        return;
      }
      lam[v] += mass[v];
      tries[v] = -(tries[v] + 1);
      left = 0;
    }
    next[v] = kVNone;
  };
  if constexpr (DRAWN) {
    if (tid < n && next[tid] == kVOpen) test(tid);
    __syncthreads();
  }
  if (tid == 0) {
    s_v = 0;
    s_count = 0;
    on_path[0] = 1;
  }
  __syncthreads();
  for (;;) {
    if (tid == 0) {
      int v = s_v, k = s_count;
      while (next[v] >= 0) {
        v = next[v];
        on_path[v] = 1;
        ++k;
      }
      s_v = v;
      s_count = k;
    }
    __syncthreads();
    const int v = s_v;
    if (!DRAWN || next[v] != kVMore) break;  // (uniform)
    if constexpr (DRAWN) {
      // a third child or later: F at its lambda, by this workgroup alone
      const VNode& nd = nodes[first + v];
      VRow r = {row_of<T>(a.logits, a.stride, first + v),
                row_of<T>(a.draft, a.draft_stride, first + v), nd.m, nd.mq, 0.f, 0.f, false};
      split_k(lam[v] * (nd.s / nd.sq), r.khi, r.klo);
      const double f = residual_sum<T>(a, r, 0, a.vocab, sh) / nd.s;
      if (tid == 0) {
        mass[v] = f;
        test(v);
      }
      __syncthreads();
    }
  }
  const int v = s_v;
  const VNode nd = nodes[first + v];
  if (c == 0) {
    if (tid < n) a.accepted[first + tid] = on_path[tid];
    if (tid == 0) {
      a.counts[req] = s_count;
      a.last[req] = v;
    }
  }
  const bool summed = (nd.flags & kVSummed) != 0;
  if ((nd.flags & kVBad) != 0 || (GREEDY && summed)) {
    if (c == 0 && tid == 0) {
      const bool bad = (nd.flags & kVBad) != 0;
      a.next_tokens[req] = bad ? -1 : nd.best;
      a.logprobs[first] = bad ? __builtin_nanf("") : (float)-log(nd.s1);
      lasts[req].node = -1;
    }
    return;
  }
  VLast l = {nd.s1, nd.m, nd.mq, 0.f, 0.f, v, nd.flags};
  if (DRAWN && summed && (nd.flags & kVBadDraft) == 0)
    split_k(lam[v] * (nd.s / nd.sq), l.khi, l.klo);
  VRow r = {row_of<T>(a.logits, a.stride, first + v),
            DRAWN ? row_of<T>(a.draft, a.draft_stride, first + v) : nullptr, l.m, l.mq, l.khi,
            l.klo, !summed};
  const int n_gone = !DRAWN && !GREEDY && summed ? rejected(a, first, n, v, gone, &s_gone) : 0;
  const int nb = (a.vocab + kLpBatch - 1) / kLpBatch;
  VBatch* mine = batches + (int64_t)req * nb;
  for (int b = c * 4 + wave; b < nb; b += wgs * 4) {
    float w[kLpUnroll][8];
    VBatch out;
    out.best = 0x7fffffff;
    if constexpr (GREEDY) {
      float f[kLpUnroll][8];
      lp_load_batch(static_cast<const T*>(r.x), b * kLpBatch, a.vocab, f);
      float m = kNegInf;
#pragma unroll
      for (int u = 0; u < kLpUnroll; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) m = vmax(m, f[u][e]);
      m = lp_wave_max(m);
      const float mu = m == kNegInf ? 0.f : m;
      double s = 0;
      int best = 0x7fffffff;
#pragma unroll
      for (int u = 0; u < kLpUnroll; ++u) {
        float us = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          us += fast_exp2((f[u][e] - mu) * kLog2e);
          if (f[u][e] == m) best = min(best, b * kLpBatch + u * 512 + lane * 8 + e);
        }
        s += us;
      }
      out.w = out.p = 0;
      out.s1 = wave_sum64(s);
      out.m = m;
      out.best = wave_min(best);
    } else {
      double p, s1;
      out.m = batch_weights<T, DRAWN>(a, r, b * kLpBatch, gone, n_gone, w, p, s1);
      double sum = 0;
#pragma unroll
      for (int u = 0; u < kLpUnroll; ++u) {
        float us = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) us += w[u][e];
        sum += us;
      }
      out.w = wave_sum64(sum);
      out.p = wave_sum64(p);
      out.s1 = wave_sum64(s1);
    }
    if (lane == 0) mine[b] = out;
  }
  if (wgs > 1) {
    if (c == 0 && tid == 0) lasts[req] = l;
    return;
  }
  __threadfence_block();
  __syncthreads();
  pick<T, DRAWN, GREEDY>(a, req, l, r, mine, gone, n_gone, first);
}

// -- pick ------------------------------------------------------------------------

template <typename T, bool DRAWN, bool GREEDY>
__global__ __launch_bounds__(kVThreads) void verify_pick_kernel(VerifyArgs a, const VLast* lasts,
                                                                const VBatch* batches) {
  __shared__ int64_t gone[kVNodes];
  __shared__ int s_gone;
  const int req = blockIdx.x;
  const VLast l = lasts[req];
  if (l.node < 0) return;
  const int64_t first = a.cu[req];
  const int64_t size = (int64_t)a.cu[req + 1] - first;
  const int n = (int)(size < kVNodes ? size : kVNodes);
  const bool summed = (l.flags & kVSummed) != 0;
  VRow r = {row_of<T>(a.logits, a.stride, first + l.node),
            DRAWN ? row_of<T>(a.draft, a.draft_stride, first + l.node) : nullptr, l.m, l.mq, l.khi,
            l.klo, !summed};
  const int n_gone = !DRAWN && !GREEDY && summed ? rejected(a, first, n, l.node, gone, &s_gone) : 0;
  const int nb = (a.vocab + kLpBatch - 1) / kLpBatch;
  pick<T, DRAWN, GREEDY>(a, req, l, r, batches + (int64_t)req * nb, gone, n_gone, first);
}

struct Layout {
  int32_t segments, seg_len, walk_wgs;
  int64_t parts, nodes, f1, lasts, batches, bytes;
};

Layout layout(int32_t batch, int64_t total, int32_t vocab, bool drawn) {
  Layout l;
  const int32_t spans = (vocab + kVSpan - 1) / kVSpan;
  const int32_t rounds = (spans + kVMaxSegments - 1) / kVMaxSegments;
  l.seg_len = rounds * kVSpan;
  l.segments = (vocab + l.seg_len - 1) / l.seg_len;
  l.walk_wgs = l.segments;
  const int64_t nb = (vocab + kLpBatch - 1) / kLpBatch;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t p = at;
    at += (bytes + 15) / 16 * 16;
    return p;
  };
  l.parts = take(total * (drawn ? 2 : 1) * l.segments * (int64_t)sizeof(VPart));
  l.nodes = take(total * (int64_t)sizeof(VNode));
  l.f1 = take(drawn ? total * l.segments * 8 : 0);
  l.lasts = take(batch * (int64_t)sizeof(VLast));
  l.batches = take(batch * nb * (int64_t)sizeof(VBatch));
  l.bytes = at;
  return l;
}

template <typename T, bool DRAWN, bool GREEDY>
hipError_t run(VerifyArgs a, const Layout& l, char* ws, hipStream_t s) {
  VPart* parts = reinterpret_cast<VPart*>(ws + l.parts);
  VNode* nodes = reinterpret_cast<VNode*>(ws + l.nodes);
  double* f1 = reinterpret_cast<double*>(ws + l.f1);
  VLast* lasts = reinterpret_cast<VLast*>(ws + l.lasts);
  VBatch* batches = reinterpret_cast<VBatch*>(ws + l.batches);
  const dim3 block(kVThreads);
  const int64_t rows = a.total * (DRAWN ? 2 : 1) * l.segments;
  if (a.total > 0) {
    hipLaunchKernelGGL((verify_stats_kernel<T, GREEDY>), dim3((uint32_t)rows), block, 0, s, a,
                       parts);
    hipLaunchKernelGGL((verify_join_kernel<T, DRAWN, GREEDY>),
                       dim3((uint32_t)(a.total * (DRAWN ? l.segments : 1))), block, 0, s, a, parts,
                       nodes, f1);
  }
  hipLaunchKernelGGL((verify_walk_kernel<T, DRAWN, GREEDY>),
                     dim3((uint32_t)((int64_t)a.batch * l.walk_wgs)), block, 0, s, a, nodes, f1,
                     lasts, batches);
  if (l.walk_wgs > 1)
    hipLaunchKernelGGL((verify_pick_kernel<T, DRAWN, GREEDY>), dim3((uint32_t)a.batch), block, 0, s,
                       a, lasts, batches);
  return hipGetLastError();
}

template <typename T>
hipError_t run_t(const VerifyArgs& a, const Layout& l, char* ws, bool greedy, hipStream_t s) {
  if (greedy) return run<T, false, true>(a, l, ws, s);
  return a.draft ? run<T, true, false>(a, l, ws, s) : run<T, false, false>(a, l, ws, s);
}

}  // namespace

int64_t verify_workspace(int32_t batch, int64_t total, int32_t vocab, bool drawn) {
  return layout(batch, total, vocab, drawn).bytes;
}

bool verify_fits(int32_t batch, int64_t total, int32_t vocab, bool drawn) {
  const Layout l = layout(batch, total, vocab, drawn);
  return total * 2 * l.segments < 0x7fffffffll && (int64_t)batch * l.walk_wgs < 0x7fffffffll;
}

hipError_t verify_drafts(VerifyArgs a, double temperature, double draft_temperature,
                         void* workspace, hipStream_t s) {
  const bool greedy = temperature == 0.0;
  if (greedy) a.draft = nullptr;
  const Layout l = layout(a.batch, a.total, a.vocab, a.draft != nullptr);
  auto split = [](double t, double& inv, float& hi, float& lo) {
    inv = t > 0 ? 1.0 / t : 1.0;
    const double c = 1.4426950408889634074 * inv;
    hi = (float)c;
    lo = (float)(c - (double)hi);
  };
  split(temperature, a.inv_t, a.thi, a.tlo);
  split(draft_temperature, a.inv_dt, a.dhi, a.dlo);
  a.segments = l.segments;
  a.seg_len = l.seg_len;
  a.walk_wgs = l.walk_wgs;
  char* ws = static_cast<char*>(workspace);
  return a.elem_bytes == 2 ? run_t<bf16>(a, l, ws, greedy, s) : run_t<float>(a, l, ws, greedy, s);
}

}  // namespace aios
