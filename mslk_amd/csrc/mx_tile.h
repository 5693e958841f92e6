// Tile of a product of two MXFP4 matrices for gfx950 (formats: mx.h): Y[m, n] = sum_k X[m, k] W[n, k].
//
// One workgroup (a WM x WN grid of wavefronts, or KS of them one behind the other) makes a BM x BN tile of sums.  What bounds these tiles are the
// loads of their steps, 60 KB per us and CU where the DMA alone reaches 100: 64 x 64 tiles, two to a CU, 0.5 us per step, 128 x 128 ones 1.05.
//
// Steps.  K is consumed 256 values (128 bytes of a row) at a time, copied global -> LDS by the 128-bit DMA load (gemm_tile.h).  Eight
// 16-byte chunks make a row of 128 bytes in LDS, one chunk being one block of 32 values; they are permuted by chunk ^ swz(row), so that
// the lanes which are served together touch different banks, and since the DMA cannot scatter inside a wave the permutation is applied to
// the global side.
// Scales.  A row's scales of two steps, a pair, are 16 bytes.  They travel by the same DMA into a ring of their own, 16 bytes per row.
// (Loaded into registers instead, the compiler's wait for them would be one for the DMA loads too, which it does not know of.)  As
// they lie in the tensor, each row's 16 bytes are a line for the L1 and the L2 to look up, and a pair of a 256 x 256 tile 512 lines next to
// 1024 of codes: up to 0.28 us per step, where power leaves that to be seen.  Large products have them arranged first, 64 rows to a KiB (MxScales).
// K's end.  Of a last step of fewer than eight blocks the missing chunks are filled with chunk 0, and their scales are 0, 2^-127, in arranged
// rows or by a mask: products of two such blocks are below 2^-243 and vanish in fp32.
// Products.  v_mfma_scale_f32_32x32x64_f8f6f4, W first: lane (i = l & 31, h = l >> 5) gives row i's chunk 4 h + j to product j of a
// step, and the four bytes of its scales of the step are those of chunks 4 h ... 4 h + 3: the instruction picks byte j.  Any order of
// K would do that both operands share; this one needs neither shifts nor shuffles of scales.  Out of registers and on quantized normal
// numbers these run at 6.8 PFLOP/s (on zeros 9.8: the limit on numbers is power).  16x16x128 draws less, 7.6 (9.7), but no tile here is built on it.
// Rows.  LDS row f 32 W + w 32 + i of an operand is row i of fragment f of wave row (column) w, W of them.  Of 32 rows of W a lane receives
// rows 8 q + 4 h + r (q, r = 0 ... 3); fragment 2 T + t takes columns 64 T + 16 q + 8 h + 4 t + r of the wave's, so that a pair of fragments
// gives a lane eight neighbouring columns: 16 bytes of a row of Y, stored as they are.
// GATED: a tile has BN / 2 columns; fragments with t = 0 are rows of the gate, those with t = 1 the rows N further, of columns
// 32 T + 16 h + 4 q + r, so a lane holds both factors of its columns.
// A single fragment (FN = 1) has columns 8 q + 4 h + r, gated: for q < 2 of the gate, for the others the rows N further of column - 16.
#pragma once
#include <type_traits>

#include "gemm_tile.h"
#include "mx.h"

namespace mslk_amd {

constexpr int kMxStep = 128;          // bytes of a row per step

// Two stages.  What a wave multiplies is in registers before its step's stage takes the step after the next: two steps are in flight, which the
// memory's latency asks for (with one in flight, 16 groups of 64 rows, gated 5120 x 4096, take 71 us instead of 62).
// WM x WN waves share a step's products (between barriers), or KS waves take the pairs of steps in turn, each with stages and the whole tile's
// sums of its own and without a barrier; at the end the sums meet in LDS.  The latter for small tiles, which would otherwise wait a memory round
// trip and a barrier for every step's few products.
template <int BM_, int BN_, int WM_, int WN_, int KS_>
struct MxShape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, KS = KS_;
  static constexpr int NW = WM * WN, NTHREADS = NW * KS * 64;       // waves that share a step
  static constexpr int FM = BM / WM / 32, FN = BN / WN / 32;        // fragments of 32 rows per wave
  static constexpr int X_BYTES = BM * kMxStep, W_BYTES = BN * kMxStep;
  static constexpr int LX = BM / 8 / NW, LW = BN / 8 / NW;          // DMA loads per wave and step
  // Scales of two steps: DMA loads per wave (the rows of X, then of W, S_ROWS a load; the last ones may have none).  KS > 1: four bytes a lane, for rows
  // that begin on four bytes; else 16, a fourth of the loads (with four, 16 groups of 64 rows, gated 5120 x 4096, take 2 % more).
  static constexpr int S_ROWS = KS > 1 ? 16 : 64, LS = ((BM + BN) / S_ROWS + NW - 1) / NW;
  static constexpr int S_BYTES = LS * NW * S_ROWS * 16;
  static constexpr int PART_BYTES = 2 * (X_BYTES + W_BYTES + S_BYTES);   // of the waves that share steps
  static constexpr int LDS_BYTES = KS * PART_BYTES;
  static_assert(KS == 1 || NW == 1, "steps are shared, or taken in turn");
  static_assert(BM % (32 * WM) == 0 && (BN % (64 * WN) == 0 || (KS > 1 && BN == 32)) && BM % (8 * NW) == 0 && BN % (8 * NW) == 0 && BM % S_ROWS == 0 && BN % S_ROWS == 0, "whole fragments and loads");
};

// Scales of a tile: row r of it is row `first` + r behind `base`, which is the first of 64.
struct MxTileScales {
  const uint8_t* base;
  uint32_t block, row, first;   // bytes of 64 rows, of one
  int pair_stride;
  MSLK_AMD_DEVINL MxTileScales() = default;
  MSLK_AMD_DEVINL MxTileScales(const MxScales& s, int64_t first_row)
      : base(s.data + (first_row >> 6) * s.block), block((uint32_t)s.block), row(s.row), first((uint32_t)first_row & 63), pair_stride(s.pair_stride) {}
  MSLK_AMD_DEVINL uint32_t offset(int r) const {   // of the 16 bytes for steps 0 and 1
    const uint32_t at = first + (uint32_t)r;
    return (at >> 6) * block + (at & 63) * row;
  }
};

// What a tile reads: first rows of its operands, valid rows (>= 1), steps [0, steps) of which the last has `last_chunks` blocks.
struct MxOperands {
  const uint8_t *x, *w;
  MxTileScales xs, ws;
  int rows_x, rows_w;       // rows_w: of the gate's rows, if gated
  uint32_t ld;              // bytes between rows of x and of w
  uint32_t up, up_rows;     // gated: bytes (rows) from a gate's row to its partner
  int steps, last_chunks;
};

MSLK_AMD_DEVINL int mx_swz(int row) { return (row >> 1) & 7; }

MSLK_AMD_DEVINL v8i mx_operand(v4i a) { return v8i{a[0], a[1], a[2], a[3], 0, 0, 0, 0}; }

template <typename TS, bool GATED>
struct MxTile {
  uint32_t x_off[TS::LX], w_off[TS::LW];   // of this lane's chunk of a load, step 0
  uint32_t s_off[TS::LS];                  // of this lane's scales, relative to xs or ws
  uint32_t s_last;                         // which bytes of a word of scales of the last step are those of its blocks
  MxOperands o;

  // Of a wave: its place among those that share a step, and which step of KS it takes.
  MSLK_AMD_DEVINL static int wave_id() { return TS::KS == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0; }
  MSLK_AMD_DEVINL static int turn_id() { return TS::KS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

  // Row of the tile that LDS row r of X holds.
  MSLK_AMD_DEVINL static int x_row(int r) { return ((r >> 5) % TS::WM) * (TS::BM / TS::WM) + r / (32 * TS::WM) * 32 + (r & 31); }
  // Row of W (of the tile's) that LDS row r of W holds, and whether it is one of the second half.
  MSLK_AMD_DEVINL static int w_row(int r, bool& up) {
    const int wn = (r >> 5) % TS::WN, tn = r / (32 * TS::WN), i = r & 31;
    if constexpr (TS::FN == 1) {
      up = GATED && i >= 16;
      return GATED ? i & 15 : i;
    }
    up = GATED && (tn & 1) != 0;
    if constexpr (GATED) return wn * (TS::BN / TS::WN / 2) + (tn >> 1) * 32 + ((i >> 2) & 1) * 16 + (i >> 3) * 4 + (i & 3);
    else return wn * (TS::BN / TS::WN) + (tn >> 1) * 64 + (tn & 1) * 4 + (i >> 2) * 8 + (i & 3);
  }
  // First of the 8 LDS rows that load q of this wave fills.
  MSLK_AMD_DEVINL static int x_load_row(int q) { return (wave_id() * TS::LX + q) * 8; }
  MSLK_AMD_DEVINL static int w_load_row(int q) { return (wave_id() * TS::LW + q) * 8; }

  MSLK_AMD_DEVINL void init(const MxOperands& operands) {
    o = operands;
    o.x = uniform_ptr(o.x);
    o.w = uniform_ptr(o.w);
    o.xs.base = uniform_ptr(o.xs.base);
    o.ws.base = uniform_ptr(o.ws.base);
    const int lane = threadIdx.x & 63, wave = wave_id();
    const int mine = o.last_chunks - 4 * (lane >> 5);
    s_last = mine >= 4 ? ~0u : mine <= 0 ? 0u : (1u << (8 * mine)) - 1;
#pragma unroll
    for (int q = 0; q < TS::LX; ++q) {   // rows beyond the valid ones read the last valid one again: their sums are not stored
      const int r = x_load_row(q) + (lane >> 3);
      x_off[q] = (uint32_t)min(x_row(r), o.rows_x - 1) * o.ld + (((lane & 7) ^ mx_swz(r)) << 4);
    }
#pragma unroll
    for (int q = 0; q < TS::LW; ++q) {
      const int r = w_load_row(q) + (lane >> 3);
      bool up;
      const int row = min(w_row(r, up), o.rows_w - 1);
      w_off[q] = (uint32_t)row * o.ld + (up ? o.up : 0u) + (((lane & 7) ^ mx_swz(r)) << 4);
    }
#pragma unroll
    for (int i = 0; i < TS::LS; ++i) {   // the list of LDS rows of X, then of W
      const int r = (wave * TS::LS + i) * TS::S_ROWS + lane * TS::S_ROWS / 64;
      bool up = false;
      if (r >= TS::BM) {
        const int row = min(w_row(min(r - TS::BM, TS::BN - 1), up), o.rows_w - 1);
        s_off[i] = o.ws.offset(row + (up ? (int)o.up_rows : 0));
      } else {
        s_off[i] = o.xs.offset(min(x_row(r), o.rows_x - 1));
      }
      if (TS::S_ROWS == 16) s_off[i] += (lane & 3) * 4;
    }
  }

  MSLK_AMD_DEVINL static char* x_stage(char* lds, int i) { return lds + i * TS::X_BYTES; }
  MSLK_AMD_DEVINL static char* w_stage(char* lds, int i) { return lds + 2 * TS::X_BYTES + i * TS::W_BYTES; }
  MSLK_AMD_DEVINL static char* s_stage(char* lds, int i) { return lds + 2 * (TS::X_BYTES + TS::W_BYTES) + i * TS::S_BYTES; }

  // What is added to the offsets of a step's loads: 0, but in a last step of fewer blocks lanes of missing chunks go back to chunk 0.
  // Loads of even and of odd number differ: swz() of their rows does, in bit 2.
  struct Adjust { uint32_t even, odd; };
  MSLK_AMD_DEVINL Adjust adjust(int kt) const {
    const int lane = threadIdx.x & 63, c = (lane & 7) ^ (lane >> 4);
    const int chunks = kt + 1 < o.steps ? 8 : o.last_chunks;
    return Adjust{c < chunks ? 0u : (uint32_t)(-16 * c), (c ^ 4) < chunks ? 0u : (uint32_t)(-16 * (c ^ 4))};
  }
  // Load i of the scales of steps 2 pair and 2 pair + 1 into `stage`; lanes of words behind the last block go back to the pair's first word.
  MSLK_AMD_DEVINL void copy_scales(char* stage, int pair, int i) {
    const int64_t from = (int64_t)pair * o.xs.pair_stride;   // (the same for both)
    const int load = wave_id() * TS::LS + i, word = threadIdx.x & 3, blocks = (o.steps - 1 - 2 * pair) * 8 + o.last_chunks;
    const uint8_t* base = uniform_ptr((load * TS::S_ROWS >= TS::BM ? o.ws.base : o.xs.base) + from);
    char* const dst = stage + load * TS::S_ROWS * 16;
    if constexpr (TS::S_ROWS == 16) dma4(base, s_off[i] + (word * 4 < blocks ? 0u : (uint32_t)(-4 * word)), dst);
    else dma16(base, s_off[i], dst);
  }
  // Global -> LDS copy of four bytes per lane, as dma16().
  MSLK_AMD_DEVINL static void dma4(const uint8_t* base, uint32_t off, char* lds_wave_base) {
    const uint32_t dst = (uint32_t)(uintptr_t)(lds_ptr_t)lds_wave_base;
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" : : "v"(off), "s"(base), "s"(dst) : "memory", "m0");
  }

  // At most `PENDING` of this wave's youngest loads are in flight and its LDS accesses are done; then the workgroup's barrier.
  template <int PENDING, bool BARRIER = true>
  MSLK_AMD_DEVINL static void wait_and_barrier() {
    static_assert(PENDING >= 0 && PENDING < 64, "vmcnt is a 6-bit counter");
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | (PENDING & 15) | ((PENDING >> 4) << 14));
    if constexpr (BARRIER) __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }

  // The same, with the barrier where waves share steps.
  template <int PENDING>
  MSLK_AMD_DEVINL static void wait() { wait_and_barrier<PENDING, TS::KS == 1>(); }

  // Chunk 4 h + j of this lane's row of a fragment of 32 W rows at `rows`; w: of the W waves that share it, this one.
  MSLK_AMD_DEVINL static v4i chunk(const char* rows, int w, int j) {
    const int lane = threadIdx.x & 63, i = lane & 31;
    return *reinterpret_cast<const v4i*>(rows + (w * 32 + i) * kMxStep + (((4 * (lane >> 5) + j) ^ mx_swz(i)) << 4));
  }
  MSLK_AMD_DEVINL static v4i x_chunk(const char* stage, int tm, int j) { return chunk(stage + tm * (32 * TS::WM * kMxStep), wave_id() / TS::WN, j); }
  MSLK_AMD_DEVINL static v4i w_chunk(const char* stage, int tn, int j) { return chunk(stage + tn * (32 * TS::WN * kMxStep), wave_id() % TS::WN, j); }
  MSLK_AMD_DEVINL static void load_scales(const char* stage, int kt, uint32_t (&sx)[TS::FM], uint32_t (&sw)[TS::FN]) {
    const int lane = threadIdx.x & 63, wave = wave_id();
    const char* at = stage + (kt & 1) * 8 + (lane >> 5) * 4 + (lane & 31) * 16;
#pragma unroll
    for (int tm = 0; tm < TS::FM; ++tm) sx[tm] = *reinterpret_cast<const uint32_t*>(at + (tm * TS::WM + wave / TS::WN) * 512);
#pragma unroll
    for (int tn = 0; tn < TS::FN; ++tn) sw[tn] = *reinterpret_cast<const uint32_t*>(at + TS::BM * 16 + (tn * TS::WN + wave % TS::WN) * 512);
  }
  template <int J>
  MSLK_AMD_DEVINL static void multiply(const v4i& wf, const v4i& xf, uint32_t sw, uint32_t sx, v16f& acc) {
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx_operand(wf), mx_operand(xf), acc, 4, 4, J, (int)sw, J, (int)sx);
  }

  // acc (KS > 1: of the first wave) = the tile's sums.
  MSLK_AMD_DEVINL void run(char* lds, v16f (&acc)[TS::FN][TS::FM]) {
#pragma unroll
    for (int tn = 0; tn < TS::FN; ++tn)
#pragma unroll
      for (int tm = 0; tm < TS::FM; ++tm)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[tn][tm][r] = 0.f;
    char* const mine = lds + turn_id() * TS::PART_BYTES;
    constexpr int CODES = TS::LX + TS::LW;   // loads of a step; a pair's scales go in front of its first step's
    int turns = o.steps;
    if constexpr (TS::KS > 1) {
      const int pairs = ((o.steps + 1) / 2 - turn_id() + TS::KS - 1) / TS::KS, last = turn_id() + (pairs - 1) * TS::KS;
      turns = 2 * pairs - (pairs > 0 && 2 * last + 1 == o.steps ? 1 : 0);
    }
    auto fetch = [&](int t) { issue(mine, 2 * (turn_id() + (t >> 1) * TS::KS) + (t & 1), t & 1, (t >> 1) & 1); };
    if (turns > 0) fetch(0);
    if (turns > 1) fetch(1);
    for (int t = 0; t < turns; ++t) {
      // in flight behind the loads of this turn: those of the next
      if (t + 1 == turns) wait<0>();
      else if ((t & 1) == 0) wait<CODES>();
      else wait<CODES + TS::LS>();
      const char *x = x_stage(mine, t & 1), *w = w_stage(mine, t & 1);
      v4i xf[TS::FM][4], wf[TS::FN][4];
      uint32_t sx[TS::FM], sw[TS::FN];
      load_scales(s_stage(mine, (t >> 1) & 1), t, sx, sw);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int tm = 0; tm < TS::FM; ++tm) xf[tm][j] = x_chunk(x, tm, j);
#pragma unroll
        for (int tn = 0; tn < TS::FN; ++tn) wf[tn][j] = w_chunk(w, tn, j);
      }
      if (t + 2 < turns) {
        wait<63>();   // for the reads: the stage is free
        fetch(t + 2);
      }
      if constexpr (TS::S_ROWS == 16) {
        const uint32_t there = 2 * (turn_id() + (t >> 1) * TS::KS) + (t & 1) + 1 == o.steps ? s_last : ~0u;
#pragma unroll
        for (int tm = 0; tm < TS::FM; ++tm) sx[tm] &= there;
#pragma unroll
        for (int tn = 0; tn < TS::FN; ++tn) sw[tn] &= there;
      }
      auto product = [&](auto j) {
        constexpr int J = decltype(j)::value;
#pragma unroll
        for (int tn = 0; tn < TS::FN; ++tn)
#pragma unroll
          for (int tm = 0; tm < TS::FM; ++tm) multiply<J>(wf[tn][J], xf[tm][J], sw[tn], sx[tm], acc[tn][tm]);
      };
      product(std::integral_constant<int, 0>{});
      product(std::integral_constant<int, 1>{});
      product(std::integral_constant<int, 2>{});
      product(std::integral_constant<int, 3>{});
    }
    if constexpr (TS::KS > 1) add_sums(lds, acc);
  }

  // The loads of step kt into stage `at`; with a pair's first step, in front of them those of its scales into `scales`.
  MSLK_AMD_DEVINL void issue(char* mine, int kt, int at, int scales) {
    if ((kt & 1) == 0) {
#pragma unroll
      for (int i = 0; i < TS::LS; ++i) copy_scales(s_stage(mine, scales), kt >> 1, i);
    }
    const Adjust a = adjust(kt);
    const uint8_t *x = o.x + (int64_t)kt * kMxStep, *w = o.w + (int64_t)kt * kMxStep;
#pragma unroll
    for (int q = 0; q < TS::LX; ++q) {
      const int r = x_load_row(q);
      dma16(x, x_off[q] + ((r >> 3) & 1 ? a.odd : a.even), x_stage(mine, at) + r * kMxStep);
    }
#pragma unroll
    for (int q = 0; q < TS::LW; ++q) {
      const int r = w_load_row(q);
      dma16(w, w_off[q] + ((r >> 3) & 1 ? a.odd : a.even), w_stage(mine, at) + r * kMxStep);
    }
  }

  // KS > 1: the first wave's sums become those of all, through LDS: [wave - 1][fragment][q][lane] of four.
  MSLK_AMD_DEVINL static void add_sums(char* lds, v16f (&acc)[TS::FN][TS::FM]) {
    constexpr int QUADS = TS::FN * TS::FM * 4;
    static_assert((TS::KS - 1) * QUADS * 1024 <= TS::LDS_BYTES, "room for the sums");
    v4f* const at = reinterpret_cast<v4f*>(lds) + (threadIdx.x & 63);
    const int wave = turn_id();
    wait_and_barrier<0>();   // nobody reads or fills stages any more
    if (wave > 0) {
#pragma unroll
      for (int i = 0; i < QUADS; ++i) {
        const v16f& a = acc[(i >> 2) / TS::FM][(i >> 2) % TS::FM];
        at[((wave - 1) * QUADS + i) * 64] = v4f{a[4 * (i & 3)], a[4 * (i & 3) + 1], a[4 * (i & 3) + 2], a[4 * (i & 3) + 3]};
      }
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int k = 0; k < TS::KS - 1; ++k)
#pragma unroll
        for (int i = 0; i < QUADS; ++i) {
          const v4f v = at[(k * QUADS + i) * 64];
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[(i >> 2) / TS::FM][(i >> 2) % TS::FM][4 * (i & 3) + r] += v[r];
        }
    }
  }
};

}  // namespace mslk_amd
