// The 256 x 256 tile of a product of two MXFP4 matrices: one workgroup of four waves per CU, each with 128 x 128 sums in all 256 of its
// accumulator registers, products pipelined by hand, tiles one after the other without a gap.  Chunks, scales, rows of fragments and K's
// end are as in mx_tile.h.
//
// A step (256 values) is four groups of products, one fragment of W each; all fragments of X and the first of W are in registers when it
// begins.  In front of the last group the wave waits for the loads of the next step and passes the barrier: nobody reads this step's rows
// any more, and those of the next one are complete.  Behind the barrier each chunk of X is replaced by the next step's as soon as the last
// product that uses it is issued, so neither the barrier nor LDS latency keeps the matrix cores waiting.
//
// Loads.  X has two stages of 32 KiB, W a ring of ten fragments of 8 KiB, of which a step takes four: that and the scales are the LDS of a
// CU.  Step k issues, with groups 1 and 2, fragments 0 and 1 of W of step k + 2 (places 8 and 9 behind this step's first); behind the
// barrier, fragments 2 and 3 (places that this step has left) and X (the stage that this step has left).  At the barrier the loads of
// groups 1 and 2 may be in flight.  The last two steps of a tile issue the first two of the next one, so the first barrier of that one need
// not wait for the stores of the one before, which are younger than what it waits for (loads and stores end in order).
//
// Rows.  LDS row r of X is row r of the tile: fragment t of a wave's four is 32 of rows 64 t ... 64 t + 63.  A tile of at most 64 or 128 rows
// (the last one of an operand or of a group; small operands are cut into such) takes a loop over one or two fragments.
//
// What bounds it is power: a step of a 256 x 256 tile takes 1.32 us on operands of zeros and 1.65 to 2.0, by card, on quantized normal numbers,
// whose products alone take 1.25 out of registers; 16384 x 16384 x 16384 runs at 4.8 PFLOP/s (6.6 on zeros), 4096 x 4096 x 4096 in 38.5 us (31).
//
// No branch is taken inside a step: the compiler moves products, which touch no memory, behind one, and away from the loads and reads
// that they are to be issued between.
#pragma once
#include "mx_tile.h"

namespace mslk_amd {

struct MxLarge {
  static constexpr int BM = 256, BN = 256, WM = 2, WN = 2, FM = 4, FN = 4, NTHREADS = 256;
  static constexpr int X_BYTES = BM * kMxStep, PLACES = 10, PLACE_BYTES = 64 * kMxStep;
  static constexpr int S_BYTES = (BM + BN) * 16;                   // scales of two steps
  static constexpr int LDS_BYTES = 2 * X_BYTES + PLACES * PLACE_BYTES + 2 * S_BYTES;
};

template <bool GATED>
struct MxLargeTile {
  using TS = MxLarge;
  using Rows = MxTile<MxShape<256, 256, 2, 2, 1>, GATED>;   // which row of the tile an LDS row holds
  // Of the tile whose loads are being issued; `steps` and the layout are the same for all.
  uint32_t x_off[8], w_off[8], s_off[2];
  const uint8_t *x, *w, *s_base;
  int pair_stride, steps, last_chunks;
  int quad;   // place of the scales of its first two steps
  int rows_x, rows_w;
  uint32_t first_x, first_w;   // what the offsets were formed for

  MSLK_AMD_DEVINL static int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

  // A load covers 8 LDS rows, or the 16 bytes of scales of 64 rows.  The loads of X are dealt to the waves in turn; wave v makes loads
  // 2 v and 2 v + 1 of each fragment of W, and 2 v and 2 v + 1 of the scales (of X, then of W).
  template <bool FIRST>
  MSLK_AMD_DEVINL void init(const MxOperands& o) {
    x = uniform_ptr(o.x);
    w = uniform_ptr(o.w);
    s_base = uniform_ptr(wave_id() < 2 ? o.xs.base : o.ws.base);
    // (most tiles have all their rows and columns, and the offsets of the one before)
    if (!FIRST && o.rows_x == rows_x && o.rows_w == rows_w && o.xs.first == first_x && o.ws.first == first_w) return;
    rows_x = o.rows_x;
    rows_w = o.rows_w;
    first_x = o.xs.first;
    first_w = o.ws.first;
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));   // formed again for each tile, not kept
    const int wave = wave_id();
    bool up;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int r = (q * 4 + wave) * 8 + (lane >> 3);
      x_off[q] = (uint32_t)min(r, o.rows_x - 1) * o.ld + (((lane & 7) ^ mx_swz(r)) << 4);
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int r = w_load_row(wave, q) + (lane >> 3);
      const int row = min(Rows::w_row(r, up), o.rows_w - 1);
      w_off[q] = (uint32_t)row * o.ld + (up ? o.up : 0u) + (((lane & 7) ^ mx_swz(r)) << 4);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = ((wave & 1) * 2 + i) * 64 + lane;
      const uint32_t sx = o.xs.offset(min(r, o.rows_x - 1));
      const int row = min(Rows::w_row(r, up), o.rows_w - 1);
      const uint32_t sw = o.ws.offset(row + (up ? o.up_rows : 0));
      s_off[i] = wave < 2 ? sx : sw;
    }
    // (one register each: formed by a 64-bit multiply-add they would keep both halves)
#pragma unroll
    for (int q = 0; q < 8; ++q) asm volatile("" : "+v"(x_off[q]), "+v"(w_off[q]));
    asm volatile("" : "+v"(s_off[0]), "+v"(s_off[1]));
  }
  MSLK_AMD_DEVINL static int w_load_row(int wave, int q) { return (q >> 1) * 64 + (wave * 2 + (q & 1)) * 8; }

  MSLK_AMD_DEVINL static char* x_stage(char* lds, int i) { return lds + i * TS::X_BYTES; }
  MSLK_AMD_DEVINL static char* w_place(char* lds, int i) { return lds + 2 * TS::X_BYTES + i * TS::PLACE_BYTES; }
  MSLK_AMD_DEVINL static char* s_stage(char* lds, int i) { return lds + 2 * TS::X_BYTES + TS::PLACES * TS::PLACE_BYTES + (i & 1) * TS::S_BYTES; }
  MSLK_AMD_DEVINL static int wrap(int place) { return place < TS::PLACES ? place : place - TS::PLACES; }

  // Where the loads of step kt come from.  MAY_END: it may be the last one, with fewer chunks; lanes of missing chunks go back to chunk 0.
  struct From { const uint8_t *x, *w; uint32_t even, odd; };   // rows of an even and an odd eight: swz() differs in bit 2
  template <bool MAY_END>
  MSLK_AMD_DEVINL From from(int kt) const {
    From f{x + (int64_t)kt * kMxStep, w + (int64_t)kt * kMxStep, 0, 0};
    if constexpr (MAY_END) {
      const int lane = threadIdx.x & 63, c = (lane & 7) ^ (lane >> 4), chunks = kt + 1 < steps ? 8 : last_chunks;
      f.even = c < chunks ? 0u : (uint32_t)(-16 * c);
      f.odd = (c ^ 4) < chunks ? 0u : (uint32_t)(-16 * (c ^ 4));
    }
    return f;
  }
  template <bool MAY_END>
  MSLK_AMD_DEVINL void copy_x(char* stage, const From& f, int q) {
    dma16(f.x, x_off[q] + (MAY_END ? wave_id() & 1 ? f.odd : f.even : 0u), stage + (q * 4 + wave_id()) * 1024);
  }
  template <bool MAY_END>
  MSLK_AMD_DEVINL void copy_w(char* place, const From& f, int q) {   // place: of fragment q / 2
    dma16(f.w, w_off[q] + (MAY_END ? q & 1 ? f.odd : f.even : 0u), place + (wave_id() * 2 + (q & 1)) * 1024);
  }
  MSLK_AMD_DEVINL void copy_scales(char* lds, int pair) {
#pragma unroll
    for (int i = 0; i < 2; ++i) dma16(s_base + (int64_t)pair * pair_stride, s_off[i], s_stage(lds, quad + pair) + (wave_id() * 2 + i) * 1024);
  }

  template <int PENDING>
  MSLK_AMD_DEVINL static void wait_and_barrier() { Rows::template wait_and_barrier<PENDING>(); }

  MSLK_AMD_DEVINL static v4i x_chunk(const char* stage, int tm, int j) { return Rows::chunk(stage + tm * 64 * kMxStep, wave_id() / 2, j); }
  MSLK_AMD_DEVINL static v4i w_chunk(const char* place, int j) { return Rows::chunk(place, wave_id() % 2, j); }

  struct Held {   // of the step at hand (of X, the fragments with valid rows)
    v4i x[4][4], w[2][4];
    uint32_t sx[4], sw[4];
    int stage, place, quad;   // of its X, of its first fragment of W, of its scales
    int odd;                  // which of the two steps of the scales
  };
  MSLK_AMD_DEVINL static void load_scales(char* lds, int quad, int odd, uint32_t (&sx)[4], uint32_t (&sw)[4]) {
    const int lane = threadIdx.x & 63, wave = wave_id();
    const char* at = s_stage(lds, quad) + odd * 8 + (lane >> 5) * 4 + (lane & 31) * 16;
#pragma unroll
    for (int tm = 0; tm < 4; ++tm) sx[tm] = *reinterpret_cast<const uint32_t*>(at + (tm * 2 + wave / 2) * 512);
#pragma unroll
    for (int tn = 0; tn < 4; ++tn) sw[tn] = *reinterpret_cast<const uint32_t*>(at + TS::BM * 16 + (tn * 2 + wave % 2) * 512);
  }

  // F: fragments of X with valid rows.  XL: loads of X that the step issues.  FIRST: of a tile, sums begin with it.  quad_next, odd_next: of the scales of the step that follows.
  template <int TN, int F, int XL, bool MAY_END, bool FIRST>
  MSLK_AMD_DEVINL void group(char* lds, const From& f, int quad_next, int odd_next, Held& held, v16f (&acc)[4][F]) {
    constexpr bool LAST = TN == 3;
    constexpr int SLOTS = 4 * F, ND = TN == 0 ? 0 : LAST ? 4 + XL : 2;
    uint32_t sx[4], sw[4];
    const char *w_next = w_place(lds, wrap(held.place + TN + 1)), *x_next = x_stage(lds, held.stage ^ 1);
    const int to = wrap(held.place + 8);
    if constexpr (LAST) {
      wait_and_barrier<FIRST ? 4 + stores(F) : 4>();
      load_scales(lds, quad_next, odd_next, sx, sw);
    }
    auto product = [&](auto jj) {
      constexpr int J = decltype(jj)::value;
      held.w[(TN + 1) & 1][J] = w_chunk(w_next, J);
#pragma unroll
      for (int tm = 0; tm < F; ++tm) {
        if constexpr (FIRST && J == 0)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[TN][tm][r] = 0.f;
        Rows::template multiply<J>(held.w[TN & 1][J], held.x[tm][J], held.sw[TN], held.sx[tm], acc[TN][tm]);
        const int slot = J * F + tm;
#pragma unroll
        for (int q = slot * ND / SLOTS; q < (slot + 1) * ND / SLOTS; ++q) {
          if constexpr (!LAST) copy_w<MAY_END>(w_place(lds, wrap(to + TN - 1)), f, (TN - 1) * 2 + q);
          else if (q < 4) copy_w<MAY_END>(w_place(lds, wrap(to + 2 + (q >> 1))), f, 4 + q);
          else copy_x<MAY_END>(x_stage(lds, held.stage), f, q - 4);
        }
        if constexpr (LAST) held.x[tm][J] = x_chunk(x_next, tm, J);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    product(std::integral_constant<int, 0>{});
    product(std::integral_constant<int, 1>{});
    product(std::integral_constant<int, 2>{});
    product(std::integral_constant<int, 3>{});
    if constexpr (LAST) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        held.sx[t] = sx[t];
        held.sw[t] = sw[t];
      }
      held.place = wrap(held.place + 4);
      held.stage ^= 1;
    }
  }
  // One step, with the loads of step `kt` of the tile that init() took last; ends_tile: the next step is the first of a tile.
  template <int F, int XL, bool MAY_END, bool FIRST>
  MSLK_AMD_DEVINL void step(char* lds, int kt, bool ends_tile, Held& held, v16f (&acc)[4][F]) {
    const From f = from<MAY_END>(kt);
    const int quad_next = held.quad + (held.odd | (int)ends_tile), odd_next = ends_tile ? 0 : held.odd ^ 1;
    group<0, F, XL, MAY_END, FIRST>(lds, f, quad_next, odd_next, held, acc);
    group<1, F, XL, MAY_END, FIRST>(lds, f, quad_next, odd_next, held, acc);
    group<2, F, XL, MAY_END, FIRST>(lds, f, quad_next, odd_next, held, acc);
    group<3, F, XL, MAY_END, FIRST>(lds, f, quad_next, odd_next, held, acc);
    held.quad = quad_next;
    held.odd = odd_next;
  }

  // First tile of a workgroup; at least two steps.
  MSLK_AMD_DEVINL void start(char* lds, const MxOperands& o, Held& held) {
    steps = o.steps;
    last_chunks = o.last_chunks;
    quad = 0;
    pair_stride = o.xs.pair_stride;
    init<true>(o);
    copy_scales(lds, 0);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const From f = from<true>(s);
#pragma unroll
      for (int q = 0; q < 8; ++q) copy_x<true>(x_stage(lds, s), f, q);
#pragma unroll
      for (int q = 0; q < 8; ++q) copy_w<true>(w_place(lds, s * 4 + (q >> 1)), f, q);
    }
    wait_and_barrier<0>();   // (no stores: see run())
    held.stage = held.place = held.quad = held.odd = 0;
  }
  // Stores of a whole tile, per wave.
  MSLK_AMD_DEVINL static constexpr int stores(int f) { return (GATED ? 4 : 8) * f; }
  // acc = the sums of the tile that was begun, of which the first 64 F rows are valid; begins with tile `next` (any valid one if there is none).
  // Since the loads of this tile's first two steps were issued there have been at least stores(F) stores, or a wait for everything.
  template <int F>
  MSLK_AMD_DEVINL void run(char* lds, const MxOperands& next, Held& held, v16f (&acc)[4][F]) {
    // (Read here and not in the last step before: they would be held over its sums' way out.)
    load_scales(lds, held.quad, 0, held.sx, held.sw);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      held.w[0][j] = w_chunk(w_place(lds, held.place), j);
#pragma unroll
      for (int tm = 0; tm < F; ++tm) held.x[tm][j] = x_chunk(x_stage(lds, held.stage), tm, j);
    }
    // What a step begins with: the scales of a pair; the next tile.
    auto begin = [&](int kt) {
      if ((kt & 1) == 0 && kt + 2 < steps) copy_scales(lds, (kt >> 1) + 1);   // of steps kt + 2 and kt + 3
      if (kt + 2 == steps) init<false>(next);
      if (kt + 1 == steps) {   // (with an odd number of steps the place is in use until now)
        quad += (steps + 1) >> 1;
        copy_scales(lds, 0);
      }
    };
    auto issued = [&](int kt) { return kt + 2 < steps ? kt + 2 : kt + 2 - steps; };
    begin(0);
    step<F, 8, true, true>(lds, issued(0), false, held, acc);
    int kt = 1;
    for (; kt + 3 < steps; ++kt) {
      if ((kt & 1) == 0) copy_scales(lds, (kt >> 1) + 1);
      step<F, 2 * F, false, false>(lds, kt + 2, false, held, acc);
    }
    for (; kt < steps; ++kt) {
      begin(kt);
      step<F, 8, true, false>(lds, issued(kt), kt + 1 == steps, held, acc);
    }
  }
};

}  // namespace mslk_amd
