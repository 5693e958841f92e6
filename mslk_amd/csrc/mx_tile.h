// Tile of a product of two MXFP4 matrices for gfx950 (formats: mx.h): Y[m, n] = sum_k X[m, k] W[n, k].
//
// One workgroup (a WM x WN grid of wavefronts) makes a BM x BN tile of sums.
//
// Steps.  K is consumed 256 values (128 bytes of a row) at a time, copied global -> LDS by the 128-bit DMA load (gemm_tile.h) into a
// ring of NS stages.  Eight 16-byte chunks make a row of 128 bytes in LDS, one chunk being one block of 32 values; they are permuted
// by swz_x() / swz_w() so that the lanes which are served together touch different banks, and since the DMA cannot scatter inside a
// wave the permutation is applied to the global side.
// Scales.  A row's scales of two steps are 16 bytes.  They travel by the same DMA, every second step, into a ring of their own, 16
// bytes per row.  (Loaded into registers instead, the compiler's wait for them would be one for the DMA loads too, which it does
// not know of; and a lane's load would touch a line per row.)
// Products.  v_mfma_scale_f32_32x32x64_f8f6f4, W first: lane (i = l & 31, h = l >> 5) gives row i's chunk 4 h + j to product j of a
// step, and the four bytes of its scales of the step are those of chunks 4 h ... 4 h + 3: the instruction picks byte j.  Any order of
// K would do that both operands share; this one needs neither shifts nor shuffles of scales.  Out of registers and on quantized normal
// numbers these run at 6.66 PFLOP/s, 16x16x128 at 5.96 (on zeros 9.89 and 6.63: the limit on numbers is power).
// Rows of W in a fragment.  A lane receives, of 32 rows of the fragment, rows 8 q + 4 h + r (q, r = 0 ... 3).  Fragment 2 T + t of a
// wave reads LDS rows 64 T + 16 q + 8 h + 4 t + r, so that the two fragments of a pair give a lane eight neighbouring rows: 16 bytes
// of a row of Y, stored as they are.
// GATED: a tile has BN / 2 columns; its LDS rows with t = 0 are filled from the gate's rows of W, those with t = 1 from the rows N
// further, so a lane holds both factors of its columns.
#pragma once
#include <type_traits>

#include "gemm_tile.h"
#include "mx.h"

namespace mslk_amd {

constexpr int kMxStep = 128;          // bytes of a row per step
constexpr int kMxStepValues = 256;

// NS stages: NS - 1 steps are in flight while one is multiplied.
template <int BM_, int BN_, int WM_, int WN_, int NS_>
struct MxShape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, NS = NS_;
  static constexpr int NW = WM * WN, NTHREADS = NW * 64;
  static constexpr int FM = BM / WM / 32, FN = BN / WN / 32;        // fragments of 32 rows per wave
  static constexpr int X_BYTES = BM * kMxStep, W_BYTES = BN * kMxStep;
  static constexpr int LX = BM / 8 / NW, LW = BN / 8 / NW;          // DMA loads per wave and step
  // scales of two steps: DMA loads per wave (the rows of X, then of W, 64 rows a load; the last ones may have none)
  static constexpr int LS = ((BM + BN) / 64 + NW - 1) / NW;
  static constexpr int S_BYTES = LS * NW * 1024;
  // A pair's place is taken again by the pair S_STAGES further, NS - 1 steps before that begins and after the last step of this one.
  static constexpr int S_STAGES = (NS + 2) / 2;
  static constexpr int LDS_BYTES = NS * (X_BYTES + W_BYTES) + S_STAGES * S_BYTES;
  static_assert(BM % (32 * WM) == 0 && BN % (64 * WN) == 0 && BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && (BM + BN) % 32 == 0, "whole fragments and loads");
  static_assert(LDS_BYTES <= 160 * 1024, "LDS of a CU");
};

// What a tile reads: first rows of its operands, valid rows (>= 1), steps [0, steps) of which the last has `last_chunks` blocks.
struct MxOperands {
  const uint8_t *x, *w, *xs, *ws;
  int rows_x, rows_w;       // rows_w: of the gate's rows, if gated
  uint32_t ld;              // bytes between rows of x and of w
  int x_pitch, w_pitch;     // between rows of scales
  uint32_t up, up_scale;    // gated: bytes from a gate's row of codes / scales to its partner
  int steps, last_chunks;
};

MSLK_AMD_DEVINL int swz_x(int row) { return (row >> 1) & 7; }
MSLK_AMD_DEVINL int swz_w(int row) { return ((row >> 1) & 1) | (((row >> 3) & 3) << 1); }

MSLK_AMD_DEVINL v8i mx_operand(v4i a) { return v8i{a[0], a[1], a[2], a[3], 0, 0, 0, 0}; }

template <typename TS, bool GATED>
struct MxTile {
  uint32_t x_off[TS::LX], w_off[TS::LW];   // of this lane's chunk of a load, step 0
  uint32_t s_off[TS::LS];                  // of this lane's 16 bytes of scales, relative to xs or ws
  bool s_is_w[TS::LS];                     // which of the two (the same in every lane of a wave)
  MxOperands o;

  MSLK_AMD_DEVINL static int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

  // Row of W (of the tile's) that LDS row r holds, and whether it is one of the second half.
  MSLK_AMD_DEVINL static int w_row(int r, bool& up) {
    up = false;
    if constexpr (!GATED) return r;
    up = (r >> 2) & 1;
    // within a wave's 64 rows: q, h, r as above; column 16 h + 4 q + r, so that a lane's columns of a pair are neighbours
    return (r >> 6) * 32 + ((r >> 3) & 1) * 16 + ((r >> 4) & 3) * 4 + (r & 3);
  }

  MSLK_AMD_DEVINL void init(const MxOperands& operands) {
    o = operands;
    o.x = uniform_ptr(o.x);
    o.w = uniform_ptr(o.w);
    o.xs = uniform_ptr(o.xs);
    o.ws = uniform_ptr(o.ws);
    const int lane = threadIdx.x & 63, wave = wave_id();
#pragma unroll
    for (int i = 0; i < TS::LX; ++i) {   // rows beyond the valid ones read the last valid one again: their sums are not stored
      const int r = (wave * TS::LX + i) * 8 + (lane >> 3);
      x_off[i] = (uint32_t)min(r, o.rows_x - 1) * o.ld + (((lane & 7) ^ swz_x(r)) << 4);
    }
#pragma unroll
    for (int i = 0; i < TS::LW; ++i) {
      const int r = (wave * TS::LW + i) * 8 + (lane >> 3);
      bool up;
      const int row = min(w_row(r, up), o.rows_w - 1);
      w_off[i] = (uint32_t)row * o.ld + (up ? o.up : 0u) + (((lane & 7) ^ swz_w(r)) << 4);
    }
#pragma unroll
    for (int i = 0; i < TS::LS; ++i) {
      const int first = (wave * TS::LS + i) * 64;   // in the list of rows of X, then of W
      const int r = min(first + lane, TS::BM + TS::BN - 1);
      // (with BM = 32 the first load has rows of both: s_is_w is then that of the lane)
      s_is_w[i] = r >= TS::BM;
      bool up;
      const int row = s_is_w[i] ? min(w_row(r - TS::BM, up), o.rows_w - 1) : min(r, o.rows_x - 1);
      s_off[i] = s_is_w[i] ? (uint32_t)row * (uint32_t)o.w_pitch + (up ? o.up_scale : 0u) : (uint32_t)row * (uint32_t)o.x_pitch;
    }
  }

  MSLK_AMD_DEVINL static char* x_stage(char* lds, int i) { return lds + i * TS::X_BYTES; }
  MSLK_AMD_DEVINL static char* w_stage(char* lds, int i) { return lds + TS::NS * TS::X_BYTES + i * TS::W_BYTES; }
  MSLK_AMD_DEVINL static char* s_stage(char* lds, int i) { return lds + TS::NS * (TS::X_BYTES + TS::W_BYTES) + i * TS::S_BYTES; }

  // The loads of step kt into stage `at`; of the scales, too, where a pair of steps begins.
  MSLK_AMD_DEVINL void issue(char* lds, int kt, int at) {
    const int lane = threadIdx.x & 63, wave = wave_id();
    if ((kt & 1) == 0) {
      char* dst = s_stage(lds, (kt >> 1) % TS::S_STAGES);
#pragma unroll
      for (int i = 0; i < TS::LS; ++i) {
        if constexpr (TS::BM % 64 == 0) {
          dma16((__builtin_amdgcn_readfirstlane((int)s_is_w[i]) ? o.ws : o.xs) + (kt >> 1) * 16, s_off[i], dst + (wave * TS::LS + i) * 1024);
        } else {   // one base for lanes of both: the 64-bit difference does not fit the offset, so two loads share the instruction slot
          if (s_is_w[i]) dma16(o.ws + (kt >> 1) * 16, s_off[i], dst + (wave * TS::LS + i) * 1024);
          else dma16(o.xs + (kt >> 1) * 16, s_off[i], dst + (wave * TS::LS + i) * 1024);
        }
      }
    }
    const uint8_t *x = o.x + (int64_t)kt * kMxStep, *w = o.w + (int64_t)kt * kMxStep;
    char *xd = x_stage(lds, at) + wave * TS::LX * 1024, *wd = w_stage(lds, at) + wave * TS::LW * 1024;
    const bool whole = kt + 1 < o.steps || o.last_chunks == 8;
    if (whole) {
#pragma unroll
      for (int i = 0; i < TS::LX; ++i) dma16(x, x_off[i], xd + i * 1024);
#pragma unroll
      for (int i = 0; i < TS::LW; ++i) dma16(w, w_off[i], wd + i * 1024);
    } else {   // the last blocks of the rows: chunks behind them become zeros.  (Each load has lanes with chunk 0, so each is issued.)
#pragma unroll
      for (int i = 0; i < TS::LX; ++i) {
        const int r = (wave * TS::LX + i) * 8 + (lane >> 3);
        if (((lane & 7) ^ swz_x(r)) < o.last_chunks) dma16(x, x_off[i], xd + i * 1024);
        else *reinterpret_cast<uint4*>(xd + i * 1024 + lane * 16) = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < TS::LW; ++i) {
        const int r = (wave * TS::LW + i) * 8 + (lane >> 3);
        if (((lane & 7) ^ swz_w(r)) < o.last_chunks) dma16(w, w_off[i], wd + i * 1024);
        else *reinterpret_cast<uint4*>(wd + i * 1024 + lane * 16) = make_uint4(0, 0, 0, 0);
      }
    }
  }

  // At most `PENDING` of this wave's youngest loads are in flight and its LDS accesses are done; then the workgroup's barrier.
  template <int PENDING>
  MSLK_AMD_DEVINL static void wait_and_barrier() {
    static_assert(PENDING >= 0 && PENDING < 64, "vmcnt is a 6-bit counter");
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | (PENDING & 15) | ((PENDING >> 4) << 14));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }

  template <int J, int FM>
  MSLK_AMD_DEVINL static void multiply(const v4i& wf, const v4i (&xf)[FM], uint32_t sw, const uint32_t (&sx)[FM], v16f (&acc)[FM]) {
#pragma unroll
    for (int tm = 0; tm < FM; ++tm)
      acc[tm] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(wf), mx_operand(xf[tm]), acc[tm], 4, 4, J, (int)sw, J, (int)sx[tm]);
  }

  // LDS row of W that lane i of fragment tn of this wave holds
  MSLK_AMD_DEVINL static int frag_row_w(int wn, int tn, int i) {
    return wn * (TS::BN / TS::WN) + (tn >> 1) * 64 + (tn & 1) * 4 + (i & 3) + (i >> 2) * 8;
  }

  // acc = the tile's sums.  Ends with a barrier: LDS is free.
  MSLK_AMD_DEVINL void run(char* lds, v16f (&acc)[TS::FN][TS::FM]) {
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int wm = wave / TS::WN, wn = wave % TS::WN;
    const int i = lane & 31, h = lane >> 5;
#pragma unroll
    for (int tn = 0; tn < TS::FN; ++tn)
#pragma unroll
      for (int tm = 0; tm < TS::FM; ++tm)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[tn][tm][r] = 0.f;
    constexpr int D = TS::NS - 1, PER = TS::LX + TS::LW;
    // In flight behind the loads of a step when its turn comes: those of the D - 1 steps after it, and of the scales of at least
    // (D - 1) / 2 pairs (a pair's scales go in front of its first step's codes).
    constexpr int PENDING = (D - 1) * PER + (D - 1) / 2 * TS::LS;
    for (int kt = 0; kt < D && kt < o.steps; ++kt) issue(lds, kt, kt);
    int at = 0;
    for (int kt = 0; kt < o.steps; ++kt) {
      if (kt + D - 1 < o.steps) wait_and_barrier<PENDING>();
      else wait_and_barrier<0>();
      // the stage of step kt - 1, which everybody has left, takes step kt + D
      if (kt + D < o.steps) issue(lds, kt + D, at == 0 ? TS::NS - 1 : at - 1);
      const char *xb = x_stage(lds, at), *wb = w_stage(lds, at), *sb = s_stage(lds, (kt >> 1) % TS::S_STAGES) + (kt & 1) * 8 + h * 4;
      uint32_t sx[TS::FM], sw[TS::FN];
#pragma unroll
      for (int tm = 0; tm < TS::FM; ++tm)
        sx[tm] = *reinterpret_cast<const uint32_t*>(sb + (wm * (TS::BM / TS::WM) + tm * 32 + i) * 16);
#pragma unroll
      for (int tn = 0; tn < TS::FN; ++tn) sw[tn] = *reinterpret_cast<const uint32_t*>(sb + (TS::BM + frag_row_w(wn, tn, i)) * 16);
      auto product = [&](auto j) {
        constexpr int J = decltype(j)::value;
        v4i xf[TS::FM];
#pragma unroll
        for (int tm = 0; tm < TS::FM; ++tm) {
          const int r = wm * (TS::BM / TS::WM) + tm * 32 + i;
          xf[tm] = *reinterpret_cast<const v4i*>(xb + r * kMxStep + (((4 * h + J) ^ swz_x(r)) << 4));
        }
#pragma unroll
        for (int tn = 0; tn < TS::FN; ++tn) {
          const int r = frag_row_w(wn, tn, i);
          const v4i wf = *reinterpret_cast<const v4i*>(wb + r * kMxStep + (((4 * h + J) ^ swz_w(r)) << 4));
          multiply<J, TS::FM>(wf, xf, sw[tn], sx, acc[tn]);
        }
      };
      product(std::integral_constant<int, 0>{});
      product(std::integral_constant<int, 1>{});
      product(std::integral_constant<int, 2>{});
      product(std::integral_constant<int, 3>{});
      at = at + 1 == TS::NS ? 0 : at + 1;
    }
    wait_and_barrier<0>();
  }
};

}  // namespace mslk_amd
