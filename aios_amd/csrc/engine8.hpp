// The 128-row tile engine over the 8-bit KV cache: TileEngine32's math on
// sub-tiles that are dequantised on their way into LDS.
//
// A 256-thread workgroup owns one kv-head, one KV range and up to 128 query
// rows.  Every thread loads 16-code chunks of K and V rows (and their scale
// record) into registers, a step of 64 positions ahead or more, turns them
// into bf16 (exact, kv8.hpp) and writes them to LDS in TileEngine32's layout:
// the conversion runs once for the four wavefronts that read the tile, and its
// math and results are those of the bf16 engine on a cache that holds the
// same values.  Two step slots alternate, so one barrier per step separates a
// slot's writers from its readers.
#pragma once

#include "kv8.hpp"

namespace aios {

constexpr int kStep8 = 64;  // KV positions per step: two sub-tiles

// NT: threads of the workgroup.
template <int D, int NT = kEngineThreads>
struct Stage8 {
  using T = KVTile<D, true>;
  static constexpr int CH = D / 16;                    // 16-code chunks of a row
  static constexpr int TPP = NT >= 64 * CH ? 64 : 32;  // positions per pass of the threads
  static constexpr int NTHR = TPP * CH;                // threads that load (192 of 256 at D = 96)
  static constexpr int NP = kStep8 / TPP;              // passes per step
  static constexpr int STEP_BYTES = 2 * T::SUB_BYTES;
  static constexpr int LDS_BYTES = 2 * STEP_BYTES;
  static_assert(NTHR <= NT, "one chunk per thread and pass");

  struct Ids {
    int32_t id[NP];
  };
  struct Regs {
    u32x4 k[NP], v[NP];
    uint32_t rec[NP];
  };

  const int32_t* idx;
  int begin, end;  // KV positions
  Kv8Head head;
  int tok;         // the thread's position in a pass
  uint32_t coff;   // its chunk's byte offset in a row
  bool loads;
  uint32_t dk[2], dv[2];  // its chunk's two bf16 chunks in a sub-tile

  __device__ __forceinline__ Stage8(const Kv8Layer& kv, int h, const int32_t* idx_, int begin_,
                                    int end_)
      : idx(idx_), begin(begin_), end(end_), head(kv, h, D) {
    const int tid = threadIdx.x;
    loads = tid < NTHR;
    tok = loads ? tid / CH : 0;
    const int c = loads ? tid - tok * CH : 0;
    coff = (uint32_t)c * 16;
    const int tl = tok & 31;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      dk[i] = (uint32_t)(tl * T::ROWB + T::k_slot(tl, 2 * c + i) * 16);
      dv[i] = (uint32_t)(T::SUB_KB + tl * T::ROWB + T::v_slot(tl, 2 * c + i) * 16);
    }
  }
  __device__ __forceinline__ int steps() const { return (end - begin + kStep8 - 1) / kStep8; }

  // Page ids of step s (positions past the range read its last entry).
  __device__ __forceinline__ void ids(int s, Ids& r) const {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int pos = begin + s * kStep8 + p * TPP + tok;
      r.id[p] = idx[min(pos, end - 1)];
    }
  }
  __device__ __forceinline__ void load(int s, const Ids& i, Regs& r) const {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int pos = begin + s * kStep8 + p * TPP + tok;
      const uint32_t pg = head.page(i.id[p], pos < end && loads);
      const uint32_t off = head.row(pg) + coff;
      r.rec[p] = load_b32(head.s, pg * 4);
      r.k[p] = load_b128(head.k, off);
      r.v[p] = load_b128(head.v, off);
    }
  }
  // Dequantised into step slot `slot`.
  __device__ __forceinline__ void store(uint8_t* lds, int slot, const Regs& r) const {
    if (!loads) return;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      float ks, vs;
      kv8_scales(r.rec[p], ks, vs);
      const int sub = NP == 1 ? tok >> 5 : p;
      uint8_t* buf = lds + slot * STEP_BYTES + sub * T::SUB_BYTES;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        *reinterpret_cast<bf16x8*>(buf + dk[i]) =
            kv8_dequant8(r.k[p][2 * i], r.k[p][2 * i + 1], ks);
        *reinterpret_cast<bf16x8*>(buf + dv[i]) =
            kv8_dequant8(r.v[p][2 * i], r.v[p][2 * i + 1], vs);
      }
    }
  }

  // A range of at most two steps, in flight at once: runs pipe(ready), where
  // ready(i) returns once sub-tile i (byte offset i * SUB_BYTES) is in LDS, to
  // be called for every sub-tile in order.
  template <typename QLoad, typename Pipe>
  __device__ __forceinline__ void resident(uint8_t* lds, QLoad&& qload, Pipe&& pipe, bool active) {
    const bool act = __builtin_amdgcn_readfirstlane((int)active) != 0;
    const bool second = end - begin > kStep8;
    Regs r0, r1;
    Ids i0, i1;
    ids(0, i0);
    ids(1, i1);
    qload();
    load(0, i0, r0);
    load(1, i1, r1);  // (past the range: zeros, without a memory access)
    auto ready = [&](int sub) {
      if (sub == 0) {
        store(lds, 0, r0);
        lds_barrier();
      } else if (sub == 2) {
        store(lds, 1, r1);
        lds_barrier();
      }
    };
    if (act) {
      pipe(ready);
    } else {
      ready(0);
      if (second) ready(2);
    }
  }

  // Runs math(sb, kv0) on every sub-tile of the range (sb: its byte offset in
  // lds, a constant); `qload()` issues the Q loads behind the first loads.  AHEAD: steps in
  // flight.  One (the prefill, whose math of a step outlasts a load) needs one
  // set of registers, used up by the step's LDS store; two put both steps of a
  // short range in flight at once.
  template <int AHEAD, typename QLoad, typename Math>
  __device__ __forceinline__ void stream(uint8_t* lds, QLoad&& qload, Math&& math, bool active) {
    const int n = steps();
    if (n <= 0) return;
    const bool act = __builtin_amdgcn_readfirstlane((int)active) != 0;
    Regs r0, r1;
    Ids i0, i1;
    ids(0, i0);
    if constexpr (AHEAD == 2) ids(1, i1);
    load(0, i0, r0);
    qload();
    if constexpr (AHEAD == 2) load(1, i1, r1);  // (past the range: zeros, without a memory access)
    ids(AHEAD, i0);
    if constexpr (AHEAD == 2) ids(3, i1);
    auto step = [&](int s, Regs& r, Ids& i, auto slot) {
      constexpr uint32_t SB = decltype(slot)::value * STEP_BYTES;
      store(lds, slot, r);
      // (unconditional, past the range without a memory access: behind a
      // branch around loads the compiler waits for all that are in flight)
      load(s + AHEAD, i, r);
      ids(s + 2 * AHEAD, i);
      lds_barrier();  // the slot is written; every wavefront is done with the other one's readers
      if (act) {
        const int kv0 = begin + s * kStep8;
        math(std::integral_constant<uint32_t, SB>{}, kv0);
        if (kv0 + kSubTok < end)
          math(std::integral_constant<uint32_t, SB + T::SUB_BYTES>{}, kv0 + kSubTok);
      }
    };
    // (both slots written out: offsets in the LDS reads' offset fields)
    for (int s = 0; s < n; s += 2) {
      step(s, r0, i0, std::integral_constant<int, 0>{});
      if (s + 1 >= n) break;
      if constexpr (AHEAD == 1) step(s + 1, r0, i0, std::integral_constant<int, 1>{});
      else step(s + 1, r1, i1, std::integral_constant<int, 1>{});
    }
  }
};

// TileEngine32 over range [kv_begin, kv_end) of the 8-bit cache.
template <int D, bool CAUSAL, int NT = kEngineThreads, typename QLoad>
__device__ __forceinline__ void run_tile8(TileEngine32<D, CAUSAL>& eng, uint8_t* lds,
                                          const Kv8Layer& kv, int h, const int32_t* idx,
                                          int kv_begin, int kv_end, float scale_log2,
                                          QLoad&& qload, bool active) {
  eng.reset();
  const auto lo = eng.lane_offsets(lds);
  Stage8<D, NT> st(kv, h, idx, kv_begin, kv_end);
  auto stream = [&] {
    st.template stream<CAUSAL ? 1 : 2>(
        lds, qload,
        [&](auto sb, int kv0) {
          eng.template compute_at<decltype(sb)::value>(lo, 0, kv0, kv_end, scale_log2);
        },
        active);
  };
  if constexpr (CAUSAL) {
    stream();
  } else {
    // (a shared prefix's usual chunk: the engine's pipelined math)
    auto pipe = [&](auto n) {
      st.resident(
          lds, qload,
          [&](auto&& ready) {
            eng.template pipe_n<decltype(n)::value>(lo, ready, kv_begin, kv_end, scale_log2);
          },
          active);
    };
    switch ((kv_end - kv_begin + kSubTok - 1) / kSubTok) {
      case 1: pipe(std::integral_constant<int, 1>{}); break;
      case 2: pipe(std::integral_constant<int, 2>{}); break;
      case 3: pipe(std::integral_constant<int, 3>{}); break;
      case 4: pipe(std::integral_constant<int, 4>{}); break;
      default: stream();
    }
  }
  if constexpr (CAUSAL) eng.l_run = eng.ol[0];
  else eng.l_run = xor32_sum(eng.ls);
}

}  // namespace aios
