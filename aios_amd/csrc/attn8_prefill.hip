// Varlen causal prefill and extension over the 8-bit KV cache: the tiles,
// order and KV split of attn_prefill.hip on the staging of engine8.hpp.
#include "engine8.hpp"

namespace aios {
namespace {

// bf16 output row from the lane's half of o.
template <int D>
__device__ __forceinline__ void store_row(const TileEngine32<D, true>& eng, float inv, bf16* row) {
  bf16* po = row + 4 * ((threadIdx.x & 63) >> 5);
#pragma unroll
  for (int nt = 0; nt < D / 32; ++nt)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint2 packed;
      packed.x = pack_bf16x2(eng.o[nt][4 * j] * inv, eng.o[nt][4 * j + 1] * inv);
      packed.y = pack_bf16x2(eng.o[nt][4 * j + 2] * inv, eng.o[nt][4 * j + 3] * inv);
      *reinterpret_cast<uint2*>(po + nt * 32 + 8 * j) = packed;
    }
}

__device__ __forceinline__ float inv_or_zero(float l) { return l > 0.f ? 1.f / l : l * 0.f; }

// Both kernels take the arguments that a workgroup needs before its first page
// ids as leading scalars: preloaded into SGPRs, where a by-value struct takes a
// memory round trip.  PrefillArgs' own copies are overridden with them.
__device__ __forceinline__ PrefillArgs with_scalars(PrefillArgs a, const int32_t* cu_q,
                                                    const int32_t* cu_k, const int32_t* indices,
                                                    int32_t num_kv_heads, int32_t batch,
                                                    int32_t q_tiles, int32_t q_tile, int32_t group,
                                                    int32_t n_parts, int32_t part_sub,
                                                    int32_t part_rows) {
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.indices = indices;
  a.num_kv_heads = num_kv_heads;
  a.num_qo_heads = num_kv_heads * group;
  a.batch = batch;
  a.q_tiles = q_tiles;
  a.q_tile = q_tile;
  a.group = group;
  a.n_parts = n_parts;
  a.part_sub = part_sub;
  a.part_rows = part_rows;
  return a;
}

// One workgroup of NT threads per (tile of NT / 2 MFMA rows, kv-head), a row tile
// per wavefront.  Bound: the math, two wavefronts a SIMD, and the conversion,
// which takes 55 VALU instructions a wavefront and step of 64 positions with four
// wavefronts to share it and half of that with eight.  4,096 tokens of 32q/8kv x
// 128 150 - 153 us, 901 - 919 TFLOP/s (bf16 cache, whose K/V come to LDS without
// passing through registers: 150 - 158); with four wavefronts 172.  Eight share one
// barrier and need longer ranges and more tiles to pay (prefill8_wide, api.hip).
// Fewer tiles than two a unit leave a SIMD one wavefront and nothing beside its
// chain: seven requests of 301 to 204 tokens on 517, 12q/4kv x 64, 19.5 us.
template <int D, int NT>
__global__ __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(2, 2))) void prefill8_kernel(
    const int32_t* __restrict__ cu_q, const int32_t* __restrict__ cu_k,
    const int32_t* __restrict__ indices, int32_t num_kv_heads, int32_t batch, int32_t q_tiles,
    int32_t q_tile, int32_t group, int32_t n_parts, int32_t part_sub, int32_t part_rows,
    PrefillArgs args, Kv8Layer kv) {
  const PrefillArgs a = with_scalars(args, cu_q, cu_k, indices, num_kv_heads, batch, q_tiles,
                                     q_tile, group, n_parts, part_sub, part_rows);
  __shared__ __align__(16) uint8_t lds[Stage8<D, NT>::LDS_BYTES];
  const int lane = threadIdx.x & 63;
  const int wave = threadIdx.x >> 6;
  const int G = a.group;
  const int flat = blockIdx.x;
  const int h = flat % a.num_kv_heads;
  const int rest = flat / a.num_kv_heads;
  const int r = rest % a.batch;
  const int qt = a.q_tiles - 1 - rest / a.batch;
  const int q_start = a.cu_q[r];
  const int q_len = a.cu_q[r + 1] - q_start;
  if (qt * a.q_tile >= q_len) return;
  const int kv_base = a.cu_k[r];
  const int kv_len = a.cu_k[r + 1] - kv_base;
  const int cached = kv_len - q_len;
  const int q_hi = min(q_len, (qt + 1) * a.q_tile);

  TileEngine32<D, true> eng;
  const int m = wave * 32 + (lane & 31);
  const int i = qt * a.q_tile + m / G;
  const int g = m - (m / G) * G;
  const bool ok = (m < a.q_tile * G) && (i < q_len);
  const bf16* qr = a.q + (int64_t)(q_start + i) * a.q_tok_stride + (int64_t)(h * G + g) * D;
  const int64_t out_off = ((int64_t)(q_start + i) * a.num_qo_heads + (h * G + g)) * D;
  eng.limit = cached + i;
  const int m0 = __builtin_amdgcn_readfirstlane(wave * 32);
  eng.min_limit = cached + qt * a.q_tile + m0 / G;  // (of the wavefront)
  const bool active = m0 < a.q_tile * G && qt * a.q_tile + m0 / G < q_len;
  run_tile8<D, true, NT>(eng, lds, kv, h, a.indices + kv_base, 0, min(kv_len, cached + q_hi),
                         a.scale_log2, [&] { eng.load_q(qr, ok); }, active);
  if (ok) store_row<D>(eng, inv_or_zero(eng.l_run), a.out + out_off);
}

// The parts of a tile of `rows` MFMA rows over kv positions (prefill_parts):
// one, written directly, where it has more rows than the plan gave its parts
// room for.
__device__ __forceinline__ PrefillParts tile_parts8(const PrefillArgs& a, int rows, int kv) {
  return prefill_parts(kv, a.part_sub, rows <= a.part_rows ? a.n_parts : 1);
}

template <int D>
__device__ __forceinline__ int64_t part_o8(const PrefillArgs& a, int64_t part, int dg, int m) {
  return ((part * (D / 8) + dg) * a.part_rows + m) * 8;
}

// One part of a tile's KV range per workgroup (prefill_split_kernel's scheme:
// tiles of at most 64 rows share a part's sub-tiles over their wavefronts, which
// merge their states at the end).  Bound: few workgroups by the chain of steps
// (0.6 - 1 us each), many by bandwidth: 8 tokens of 32q/8kv x 128 on 4,091
// positions, with the combine, one request of 6 13.5 us, eight 26.4 us (2.6
// TB/s), sixteen 37.8 us (3.7 TB/s).
template <int D>
__global__ __launch_bounds__(kEngineThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void prefill8_split_kernel(
    const int32_t* __restrict__ cu_q, const int32_t* __restrict__ cu_k,
    const int32_t* __restrict__ indices, int32_t num_kv_heads, int32_t batch, int32_t q_tiles,
    int32_t q_tile, int32_t group, int32_t n_parts, int32_t part_sub, int32_t part_rows,
    PrefillArgs args, Kv8Layer kv) {
  const PrefillArgs a = with_scalars(args, cu_q, cu_k, indices, num_kv_heads, batch, q_tiles,
                                     q_tile, group, n_parts, part_sub, part_rows);
  using S = Stage8<D>;
  using T = typename S::T;
  constexpr int kMl = 4 * 32 * 8;  // (m, l) of the four wavefronts' rows
  __shared__ __align__(16) uint8_t lds[S::LDS_BYTES + kMl];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int G = a.group;
  const int flat = blockIdx.x;
  const int h = flat % a.num_kv_heads;
  int rest = flat / a.num_kv_heads;
  const int r = rest % a.batch;
  rest /= a.batch;
  const int qt = a.q_tiles - 1 - rest % a.q_tiles;
  const int s = rest / a.q_tiles;
  const int q_start = a.cu_q[r];
  const int q_len = a.cu_q[r + 1] - q_start;
  if (qt * a.q_tile >= q_len) return;
  const int kv_base = a.cu_k[r];
  const int kv_len = a.cu_k[r + 1] - kv_base;
  const int cached = kv_len - q_len;
  const int q_hi = min(q_len, (qt + 1) * a.q_tile);
  const int kv_hi = min(kv_len, cached + q_hi);
  const int rows = (q_hi - qt * a.q_tile) * G;
  const PrefillParts pp = tile_parts8(a, rows, kv_hi);
  if (s >= pp.n) return;
  const int kv_begin = s * pp.per * kSubTok;
  const int kv_end = min(kv_hi, kv_begin + pp.per * kSubTok);

  const int nr = rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
  const int rt = wave & (nr - 1);
  const int share = nr == 4 ? 0 : nr == 2 ? wave >> 1 : wave;
  const int m = rt * 32 + (lane & 31);
  const int i = qt * a.q_tile + m / G;
  const int g = m - (m / G) * G;
  const bool ok = m < rows;
  const int hl = lane >> 5;
  const bf16* qr = a.q + (int64_t)(q_start + i) * a.q_tok_stride + (int64_t)(h * G + g) * D;

  TileEngine32<D, true> eng;
  eng.limit = cached + i;
  eng.min_limit = cached + qt * a.q_tile;
  const int64_t slot = ((int64_t)r * a.q_tiles + qt) * a.num_kv_heads + h;
  const int64_t part = slot * a.n_parts + s;
  bf16* out_row = a.out + ((int64_t)(q_start + i) * a.num_qo_heads + (h * G + g)) * D;

  if (nr == 4) {
    run_tile8<D, true>(eng, lds, kv, h, a.indices + kv_base, kv_begin, kv_end, a.scale_log2,
                       [&] { eng.load_q(qr, ok); }, rt * 32 < rows);
    if (!ok) return;
    if (pp.n == 1) {
      store_row<D>(eng, inv_or_zero(eng.l_run), out_row);
      return;
    }
#pragma unroll
    for (int nt = 0; nt < D / 32; ++nt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4*>(a.part_o + part_o8<D>(a, part, nt * 4 + j, m) + 4 * hl) =
            f32x4{eng.o[nt][4 * j], eng.o[nt][4 * j + 1], eng.o[nt][4 * j + 2],
                  eng.o[nt][4 * j + 3]};
    if (hl == 0) a.part_ml[part * a.part_rows + m] = make_float2(eng.m_run, eng.l_run);
    return;
  }

  // Few rows: the wavefronts share the two sub-tiles of every step.  With one
  // row tile the second pair of wavefronts takes the odd steps.
  eng.reset();
  const auto lo = eng.lane_offsets(lds);
  S st(kv, h, a.indices + kv_base, kv_begin, kv_end);
  const int n = st.steps();
  if (n <= 2) {
    // (the usual part: both steps staged, then one barrier)
    typename S::Regs r0, r1;
    typename S::Ids i0, i1;
    st.ids(0, i0);
    st.ids(1, i1);
    st.load(0, i0, r0);
    st.load(1, i1, r1);
    eng.load_q(qr, ok);
    st.store(lds, 0, r0);
    st.store(lds, 1, r1);
    lds_barrier();
    const int n_sub = (kv_end - kv_begin + kSubTok - 1) / kSubTok;
    for (int it = share; it < n_sub; it += 4 / nr)
      eng.compute_at(lo, (uint32_t)(it * T::SUB_BYTES), kv_begin + it * kSubTok, kv_end,
                     a.scale_log2);
  } else {
    // (two sub-tiles a step, each for the wavefronts whose turn it is)
    st.template stream<1>(
        lds, [&] { eng.load_q(qr, ok); },
        [&](auto sb, int kv0) {
          if (((kv0 - kv_begin) / kSubTok & (4 / nr - 1)) == share)
            eng.template compute_at<decltype(sb)::value>(lo, 0, kv0, kv_end, a.scale_log2);
        },
        true);
  }

  static_assert(T::SUB_BYTES == 32 * D * 4, "a row tile's fp32 o fills one sub-tile");
  lds_barrier();  // every wavefront is done with K/V
  float* so = reinterpret_cast<float*>(lds + wave * T::SUB_BYTES);
  float2* sml = reinterpret_cast<float2*>(lds + S::LDS_BYTES);  // [wave][32]
#pragma unroll
  for (int nt = 0; nt < D / 32; ++nt)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<f32x4*>(so + ((nt * 4 + j) * 32 + (lane & 31)) * 8 + 4 * hl) =
          f32x4{eng.o[nt][4 * j], eng.o[nt][4 * j + 1], eng.o[nt][4 * j + 2], eng.o[nt][4 * j + 3]};
  if (hl == 0) sml[wave * 32 + (lane & 31)] = make_float2(eng.m_run, eng.ol[0]);
  __syncthreads();
  const int nrow = nr * 32;
  for (int e = threadIdx.x; e < nrow * (D / 8); e += kEngineThreads) {
    const int dg = e / nrow;
    const int row = e - dg * nrow;
    if (row >= rows) continue;
    const int w0 = row >> 5;  // the row tile; its shares are wavefronts w0 + k * nr
    float mx = kNegInf;
    for (int w = w0; w < 4; w += nr) mx = vmax(mx, sml[w * 32 + (row & 31)].x);
    const float mu = mx == kNegInf ? 0.f : mx;
    f32x4 acc0 = f32x4{0.f, 0.f, 0.f, 0.f}, acc1 = acc0;
    float l = 0.f;
    for (int w = w0; w < 4; w += nr) {
      const float2 ml = sml[w * 32 + (row & 31)];
      const float f = fast_exp2(ml.x - mu);
      l += ml.y * f;
      const f32x4* po = reinterpret_cast<const f32x4*>(lds + w * T::SUB_BYTES) +
                        (dg * 32 + (row & 31)) * 2;
      acc0 += po[0] * f;
      acc1 += po[1] * f;
    }
    if (pp.n == 1) {
      const float inv = inv_or_zero(l);
      acc0 *= inv;
      acc1 *= inv;
      const int qi = q_start + qt * a.q_tile + row / G;
      bf16* po = a.out + ((int64_t)qi * a.num_qo_heads + h * G + row % G) * D + dg * 8;
      *reinterpret_cast<uint4*>(po) =
          make_uint4(pack_bf16x2(acc0[0], acc0[1]), pack_bf16x2(acc0[2], acc0[3]),
                     pack_bf16x2(acc1[0], acc1[1]), pack_bf16x2(acc1[2], acc1[3]));
    } else {
      f32x4* po = reinterpret_cast<f32x4*>(a.part_o + part_o8<D>(a, part, dg, row));
      po[0] = acc0;
      po[1] = acc1;
      if (dg == 0) a.part_ml[part * a.part_rows + row] = make_float2(mx, l);
    }
  }
}

template <typename Kernel>
hipError_t launch(Kernel kernel, int wgs, int threads, const PrefillArgs& a, const Kv8Layer& kv,
                  hipStream_t s) {
  if (wgs == 0) return hipSuccess;
  hipLaunchKernelGGL(kernel, dim3(wgs), dim3(threads), 0, s, a.cu_q, a.cu_k, a.indices,
                     a.num_kv_heads, a.batch, a.q_tiles, a.q_tile, a.group, a.n_parts, a.part_sub,
                     a.part_rows, a, kv);
  return hipGetLastError();
}

template <int D>
hipError_t launch_whole(const PrefillArgs& a, const Kv8Layer& kv, hipStream_t s) {
  const int tiles = a.q_tiles * a.num_kv_heads * a.batch;
  const int rows = a.q_tile * a.group;
  if (rows > 256) return hipErrorInvalidValue;
  return rows > 128 ? launch(prefill8_kernel<D, 512>, tiles, 512, a, kv, s)
                    : launch(prefill8_kernel<D, 256>, tiles, 256, a, kv, s);
}

}  // namespace

hipError_t launch_prefill8(int D, const PrefillArgs& a, const Kv8Layer& kv, hipStream_t s) {
  switch (D) {
    case 64: return launch_whole<64>(a, kv, s);
    case 96: return launch_whole<96>(a, kv, s);
    case 128: return launch_whole<128>(a, kv, s);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_prefill8_split(int D, const PrefillArgs& a, const Kv8Layer& kv, hipStream_t s) {
  const int wgs = a.q_tiles * a.num_kv_heads * a.batch * a.n_parts;
  hipError_t e = hipErrorInvalidValue;
  switch (D) {
    case 64: e = launch(prefill8_split_kernel<64>, wgs, kEngineThreads, a, kv, s); break;
    case 96: e = launch(prefill8_split_kernel<96>, wgs, kEngineThreads, a, kv, s); break;
    case 128: e = launch(prefill8_split_kernel<128>, wgs, kEngineThreads, a, kv, s); break;
  }
  return e == hipSuccess && wgs > 0 ? launch_prefill_combine(D, a, s) : e;
}

}  // namespace aios
