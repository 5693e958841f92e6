// Products of MXFP4 matrices for gfx950: dense, with a gated activation, and for groups of rows (formats: mx.h, tile: mx_tile.h).
#include "kernels.h"
#include "mx_device.h"
#include "mx_tile_large.h"
#include "rows.h"

namespace mslk_amd {
namespace {

// Columns n + 8 h ... of the bias, which lie on 16 bytes, as fp32; n is the same for all lanes.  By scalar loads: a vector load's wait would be
// one for the stores and the DMA loads in front of it, too.
MSLK_AMD_DEVINL void load_bias(const MxProblem& p, int n, int h, float (&b)[8]) {
  typedef const __attribute__((address_space(4))) uint32_t* constant_ptr;
  const constant_ptr at = (constant_ptr)((uintptr_t)p.bias + (uintptr_t)n * (p.bias_dtype == 1 ? 4 : 2));
  uint32_t v[8];
  if (p.bias_dtype == 1) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = h ? at[8 + e] : at[e];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t two = h ? at[4 + e] : at[e];
      v[2 * e] = two << 16;
      v[2 * e + 1] = two & 0xFFFF0000u;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) b[e] = __uint_as_float(v[e]);
}

// Columns n ... n + 7 of the bias, which differ from lane to lane and may end; vectors: the bias and its columns in eights lie on 16 bytes.
MSLK_AMD_DEVINL void load_bias_columns(const MxProblem& p, int n, bool vectors, float (&b)[8]) {
  if (vectors && p.bias_dtype == 1) {
    const float4* at = reinterpret_cast<const float4*>(static_cast<const float*>(p.bias) + min(n, p.N - 8));
    const float4 lo = at[0], hi = at[1];
    b[0] = lo.x; b[1] = lo.y; b[2] = lo.z; b[3] = lo.w;
    b[4] = hi.x; b[5] = hi.y; b[6] = hi.z; b[7] = hi.w;
  } else if (vectors) {
    const uint4 two = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.bias) + min(n, p.N - 8));
    const uint32_t v[4] = {two.x, two.y, two.z, two.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = bf16_bits_to_f32((v[e >> 1] >> (16 * (e & 1))) & 0xFFFFu);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = bias_at(p, min(n + e, p.N - 1));
  }
}

// As store16_stream(), at a scalar base and a lane's offset.  (The data registers may be reused behind the statement: its wait states.)
MSLK_AMD_DEVINL void store16_at(char* base, uint32_t off, uint4 val) {
  const v4i v = {(int)val.x, (int)val.y, (int)val.z, (int)val.w};
  asm volatile("global_store_dwordx4 %0, %1, %2 nt\n\ts_nop 1" : : "v"(off), "v"(v), "s"(base) : "memory");
}

// Sums of a tile to Y: rows m0 ... m0 + rows - 1, columns from n0.  Fragment tm of wave row wm begins at row wm * WAVE_ROW + tm * FRAG_ROW.
// A lane's pieces of eight columns (16 bytes) are four of the eight of a row's line: by register bits r1, r0; the others have the other h.
// Exchanging r0 with bit 4 of the lane and r1 with bit 3 leaves a register eight rows' whole lines, which are then written past the L2:
// left in 32-byte pieces they reached the memory as such.
// FULL: every row and column of the tile is valid, its rows and the bias begin on 16 bytes; N < 2^25.
template <int FM, int FN, int WN, int WAVE_ROW, int FRAG_ROW, bool GATED, bool BIAS, bool F16, bool FULL>
MSLK_AMD_DEVINL void store_tile(const MxProblem& p, const v16f (&acc)[FN][FM], int m0, int rows, int n0) {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));   // formed again here, not kept over the products
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN, h = lane >> 5;
  const int first = n0 + wn * (FN * 32) / (GATED ? 2 : 1);
  const bool aligned = (p.N & 7) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
  constexpr int LINES = GATED ? (FN + 3) / 4 : FN / 2, PIECES = GATED && FN == 2 ? 2 : 4;   // of 64 columns; of a lane in a line
  // column of piece r of line t for the lanes of half h
  auto column = [&](int t, int r, int half) { return GATED ? t * 64 + (r >> 1) * 32 + half * 16 + (r & 1) * 8 : t * 64 + r * 16 + half * 8; };
  // after the exchange: this lane's piece and row of each register
  const int piece = ((lane >> 3) & 1) * 2 + ((lane >> 4) & 1), row8 = lane & 7;
  const uint32_t lane_off = 2u * ((uint32_t)row8 * (uint32_t)p.N + (uint32_t)column(0, piece, h));
#pragma unroll
  for (int t = 0; t < LINES; ++t) {
    // (Of the large tile's last rows and columns the bias is read where it is added: there are no registers to hold it.)
    constexpr bool HELD = BIAS && (FULL || FM * FN <= 4);
    float b[4][8];
    if constexpr (HELD) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (FULL) load_bias(p, first + column(t, r, 0), h, b[r]);
        else load_bias_columns(p, first + column(t, r, h), (p.N & 7) == 0 && (reinterpret_cast<uintptr_t>(p.bias) & 15) == 0, b[r]);
      }
    }
#pragma unroll
    for (int tm = 0; tm < FM; ++tm) {
      const int row0 = wm * WAVE_ROW + tm * FRAG_ROW;
      if (!FULL && row0 >= rows) break;
      uint32_t w[4][4], gates = 0;
      auto values = [&](auto far) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if constexpr (GATED) {
              const int T = t * 2 + (r >> 1), at = 8 * (r & 1) + e;
              v[e] = r < PIECES ? gated_value<decltype(far)::value>(acc[2 * T][tm][at], acc[2 * T + 1][tm][at]) : 0.f;
              if (r < PIECES) gates = farther(gates, acc[2 * T][tm][at]);
            } else {
              v[e] = acc[2 * t + (e >> 2)][tm][4 * r + (e & 3)];
              if constexpr (HELD) v[e] += b[r][e];
              else if constexpr (BIAS) v[e] += bias_at(p, min(first + column(t, r, h) + e, p.N - 1));
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) w[r][e] = pack_out_x2<F16>(v[2 * e], v[2 * e + 1]);
        }
      };
      values(std::false_type{});
      if (GATED && far_gates(gates)) values(std::true_type{});
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int r = 0; r < 4; r += 2) {   // r0 and bit 4: even 16 lanes of one, odd ones of the other
          const auto s = __builtin_amdgcn_permlane16_swap(w[r][e], w[r + 1][e], false, false);
          w[r][e] = s[0];
          w[r + 1][e] = s[1];
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {      // r1 and bit 3
          const uint32_t lo = w[r][e], hi = w[r + 2][e];
          w[r][e] = __builtin_amdgcn_update_dpp(lo, hi, 0x128, 0xF, 0xC, false);
          w[r + 2][e] = __builtin_amdgcn_update_dpp(hi, lo, 0x128, 0xF, 0x3, false);
        }
      }
      if constexpr (FULL) {
        // one address for all lanes, and the lane's place in the eight rows
        char* const base = reinterpret_cast<char*>(p.y + (int64_t)(m0 + row0) * p.N + first + t * 64);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          store16_at(base + (int64_t)((r & 1) * 16 + (r >> 1) * 8) * p.N * 2, lane_off, make_uint4(w[r][0], w[r][1], w[r][2], w[r][3]));
        continue;
      }
      const int n = first + column(t, piece, h), columns = p.N - n;
      const bool mine = columns > 0 && piece < PIECES;
      uint16_t* const base = p.y + (int64_t)(m0 + row0) * p.N + n;
#pragma unroll
      for (int r = 0; r < 4; ++r) {   // rows with bit 4 = r & 1, bit 3 = r >> 1
        const int m = (r & 1) * 16 + (r >> 1) * 8 + row8;
        uint16_t* dst = base + (int64_t)m * p.N;
        if (mine && row0 + m < rows) {
          if (aligned) {
            store16_stream(dst, make_uint4(w[r][0], w[r][1], w[r][2], w[r][3]));
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (e < columns) dst[e] = (uint16_t)(w[r][e >> 1] >> ((e & 1) * 16));
          }
        }
      }
    }
  }
}

// The same of a single fragment: pieces of four columns, 8 bytes.
template <bool GATED, bool BIAS, bool F16>
MSLK_AMD_DEVINL void store_fragment(const MxProblem& p, const v16f& acc, int m0, int rows, int n0) {
  const int lane = threadIdx.x & 63, h = lane >> 5, m = lane & 31;
  if (m >= rows) return;
  const bool aligned = (p.N & 3) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 7) == 0;
#pragma unroll
  for (int q = 0; q < (GATED ? 2 : 4); ++q) {
    const int n = n0 + 8 * q + 4 * h;
    if (n >= p.N) continue;
    float v[4];
    uint32_t gates = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      v[r] = acc[4 * q + r];
      if constexpr (GATED) {
        gates = farther(gates, acc[4 * q + r]);
        v[r] = gated_value<false>(acc[4 * q + r], acc[4 * q + 8 + r]);
      }
      if constexpr (BIAS) v[r] += bias_at(p, min(n + r, p.N - 1));
    }
    if (GATED && far_gates(gates)) {
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = gated_value<true>(acc[4 * q + r], acc[4 * q + 8 + r]);
    }
    const uint32_t w[2] = {pack_out_x2<F16>(v[0], v[1]), pack_out_x2<F16>(v[2], v[3])};
    uint16_t* dst = p.y + (int64_t)(m0 + m) * p.N + n;
    if (aligned) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n + r < p.N) dst[r] = (uint16_t)(w[r >> 1] >> ((r & 1) * 16));
    }
  }
}

// Operands of the tile of rows m0 ..., columns n0 ...; w_row: first row of W's group.
template <bool GATED>
MSLK_AMD_DEVINL MxOperands operands_of(const MxProblem& p, int m0, int rows, int64_t w_row, int n0, int columns) {
  const int64_t ld = p.K / 2;
  const int blocks = p.K / kMxBlock;
  MxOperands o;
  o.x = p.xq + m0 * ld;
  o.w = p.wq + (w_row + n0) * ld;
  o.xs = MxTileScales(p.xs, m0);
  o.ws = MxTileScales(p.ws, w_row + n0);
  o.rows_x = rows;
  o.rows_w = min(p.N - n0, columns);
  o.ld = (uint32_t)ld;
  o.up = GATED ? (uint32_t)(p.N * ld) : 0u;
  o.up_rows = GATED ? (uint32_t)p.N : 0u;
  o.steps = (blocks + 7) / 8;
  o.last_chunks = blocks - (o.steps - 1) * 8;
  return o;
}

// One tile per workgroup; the grid goes on along y (rows.h).
template <typename TS, bool GATED, bool GROUPS, bool BIAS, bool F16>
__global__ __launch_bounds__(TS::NTHREADS) void mx_kernel(MxProblem p, int tiles_m, int tiles_n) {
  static_assert(TS::LDS_BYTES <= 160 * 1024, "LDS of a CU");
  __shared__ __attribute__((aligned(1024))) char lds[TS::LDS_BYTES];
  constexpr int COLUMNS = GATED ? TS::BN / 2 : TS::BN;
  int m0, rows, tn;
  int64_t w_row = 0;
  if constexpr (GROUPS) {
    GroupTile t;
    if (!find_group_tile<TS::BM>(p, tiles_n, (int)row_block(), t)) return;
    m0 = t.row0;
    rows = t.rows;
    tn = t.tn;
    w_row = (int64_t)t.g * p.N * (GATED ? 2 : 1);
  } else {
    const int t = entry_of((int)row_block(), tiles_m * tiles_n);
    if (t < 0) return;
    int tm;
    tile_at(t, tiles_m, tiles_n, tm, tn);
    m0 = tm * TS::BM;
    rows = min(p.M - m0, TS::BM);
  }
  const int n0 = tn * COLUMNS;
  v16f acc[TS::FN][TS::FM];
  MxTile<TS, GATED> tile;
  tile.init(operands_of<GATED>(p, m0, rows, w_row, n0, COLUMNS));
  tile.run(lds, acc);
  if (MxTile<TS, GATED>::turn_id() != 0) return;
  if constexpr (TS::FN == 1) store_fragment<GATED, BIAS, F16>(p, acc[0][0], m0, rows, n0);
  else
    store_tile<TS::FM, TS::FN, TS::WN, TS::BM / TS::WM, 32, GATED, BIAS, F16, false>(p, acc, m0, rows, n0);
}

// Row tiles of at most 256 rows, as listed in device memory.
struct RowTile { int row0, rows, group, unused; };
static_assert(sizeof(RowTile) == 16, "read as four words");

// A workgroup per CU that walks the 256-column tiles, in rounds: of each round's entries, neighbours all, XCD x takes a run.  (A list has long
// tiles first, so those of a round are about as long; runs of the whole list leave the XCDs different amounts, 16 experts of 8192 rows 236 us
// instead of 225, and equal ones gain nothing: 8192 x 28672 x 4096 521 and 515.)
// One matrix: tiles of a last round that half of the workgroups would be enough for are cut into two of 128 rows (2048 x 10240 x 8192 114 us, 100).
// A list's last tiles are short already (cut, 16 experts of 8192 rows take 2 % more).
template <bool GATED, bool BIAS, bool F16>
__global__ __launch_bounds__(256) void mx_walk_kernel(MxProblem p, int tiles_m, int tiles_n) {
  using TS = MxLarge;
  using Tile = MxLargeTile<GATED>;
  __shared__ __attribute__((aligned(1024))) char lds[TS::LDS_BYTES];
  constexpr int COLUMNS = GATED ? TS::BN / 2 : TS::BN;
  // (read by scalar loads, which wait for no store)
  typedef const __attribute__((address_space(4))) int* constant_ptr;
  const constant_ptr list = (constant_ptr)(uintptr_t)p.row_tiles;
  if (list != nullptr) tiles_m = list[1];   // (the first entry holds their number as its rows)
  const int wgs = gridDim.x, xcd = blockIdx.x % kXcds, slot = blockIdx.x / kXcds;
  const int whole = tiles_m * tiles_n / wgs * wgs, rest = tiles_m * tiles_n - whole;
  const bool cut = list == nullptr && 2 * rest <= wgs;
  const int total = cut ? whole + 2 * rest : whole + rest;
  auto entry = [&](int round) {   // this workgroup's `round`th entry, -1: none
    const int first = round * wgs, here = min(total - first, wgs), run = (here + kXcds - 1) / kXcds, at = xcd * run + slot;
    return slot < run && at < here ? first + at : -1;
  };
  const bool aligned = (p.N & 7) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0 && (!BIAS || (reinterpret_cast<uintptr_t>(p.bias) & 15) == 0);
  struct Place { int m0, rows, n0; int64_t w_row; };
  auto place_of = [&](int t, Place& at) {   // false: none, or the empty half of a tile
    if (t < 0) return false;
    const bool part = cut && t >= whole;
    const int half = part ? (t - whole) & 1 : 0;
    if (part) t = whole + ((t - whole) >> 1);
    int tm, tn;
    tile_at(t, tiles_m, tiles_n, tm, tn);
    if (list != nullptr) {
      const constant_ptr r = list + 4 * (1 + tm);   // row0, rows, group
      at = Place{r[0], r[1], tn * COLUMNS, (int64_t)r[2] * p.N * (GATED ? 2 : 1)};
      return true;
    }
    const int m0 = tm * MxLarge::BM + half * 128;
    if (m0 >= p.M) return false;
    at = Place{m0, min(p.M - m0, part ? 128 : MxLarge::BM), tn * COLUMNS, 0};
    return true;
  };
  auto operands = [&](const Place& at) { return operands_of<GATED>(p, at.m0, at.rows, at.w_row, at.n0, COLUMNS); };
  int round = 0;
  Place at;
  if (!place_of(entry(0), at)) return;
  Tile tile;
  typename Tile::Held held;
  tile.start(lds, operands(at), held);
  for (bool more = true; more;) {
    const Place here = at;
    more = place_of(entry(++round), at);   // (behind the last tile: itself once more)
    auto make = [&](auto fragments) {
      constexpr int F = decltype(fragments)::value;
      v16f acc[4][F];
      tile.template run<F>(lds, operands(at), held, acc);
      const bool full = here.rows == 64 * F && here.n0 + COLUMNS <= p.N && aligned;
      if (full) store_tile<F, 4, 2, 32, 64, GATED, BIAS, F16, true>(p, acc, here.m0, here.rows, here.n0);
      else store_tile<F, 4, 2, 32, 64, GATED, BIAS, F16, false>(p, acc, here.m0, here.rows, here.n0);
      if (!full || at.rows > 64 * F) wait_vmcnt0();   // fewer stores than the next tile counts on
    };
    if (here.rows > 192) make(std::integral_constant<int, 4>{});
    else if (here.rows > 128) make(std::integral_constant<int, 3>{});
    else if (here.rows > 64) make(std::integral_constant<int, 2>{});
    else make(std::integral_constant<int, 1>{});
  }
  wait_vmcnt0();   // the loads of a tile that does not follow end before the LDS is given away
}

// Tensors of scales, rows of `from` bytes, to the arranged layout (MxScales), of both operands in one launch.  A workgroup takes up to 8 pairs
// of 64 rows through LDS, so that it reads and writes whole lines; the first one makes the list of row tiles.
constexpr int kArrangePairs = 8;
struct ArrangeJob {
  const uint8_t* src;
  uint8_t* dst;
  int64_t rows;
  int workgroups;
};
// Row tiles of the groups, at most 256 rows each, the longest first (by the fragments that they take): list[0].rows of them behind list[0].
struct ListJob {
  const int64_t* m_sizes;   // nullptr: none
  RowTile* list;
  int G, M;
};

// Sums over the lanes up to and with this one, at most `most` (< 2^31).
template <int CTRL, int ROWS>
MSLK_AMD_DEVINL uint32_t add_from(uint32_t v, uint32_t most) {
  return min(v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false), most);
}
MSLK_AMD_DEVINL uint32_t lanes_to(uint32_t v, uint32_t most) {
  v = add_from<0x111, 0xF>(v, most);   // from 1, 2, 4, 8 lanes below inside 16
  v = add_from<0x112, 0xF>(v, most);
  v = add_from<0x114, 0xF>(v, most);
  v = add_from<0x118, 0xF>(v, most);
  v = add_from<0x142, 0xA>(v, most);   // lane 15 of a row to the second and fourth row
  return add_from<0x143, 0xC>(v, most);   // lane 31 to the upper half
}

// By one wave; `held` of the sizes are in LDS.
MSLK_AMD_DEVINL uint32_t group_size(const ListJob& job, int g) { return (uint32_t)max((int64_t)0, min(job.m_sizes[g], (int64_t)job.M)); }
MSLK_AMD_DEVINL void list_row_tiles(const ListJob& job, const uint32_t* sizes, int held) {
  constexpr int ROWS = MxLarge::BM;
  const int lane = threadIdx.x & 63;
  int at[4] = {0, 0, 0, 0};   // where the next tile of 4, 3, 2, 1 fragments goes; first their numbers
  for (int pass = 0; pass < 2; ++pass) {
    uint32_t before = 0;      // rows of the groups before these 64
    for (int g0 = 0; g0 < job.G; g0 += 64) {
      const int g = g0 + lane;
      const uint32_t size = g >= job.G ? 0u : g < held ? sizes[g] : group_size(job, g);
      const uint32_t to = lanes_to(size, (uint32_t)job.M);
      const uint32_t start = min(before + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)to, 0x138, 0xF, 0xF, false), (uint32_t)job.M);   // of the lane below
      const int live = (int)min(size, (uint32_t)job.M - start), rest = live % ROWS;
      const int whole = live / ROWS + (rest > 192 ? 1 : 0);                                      // tiles of four fragments
      const int other = rest == 0 || rest > 192 ? 0 : rest > 128 ? 1 : rest > 64 ? 2 : 3;        // place in `at` of the last one
      const uint32_t whole_to = lanes_to((uint32_t)whole, 0xFFFFFFFFu);
      if (pass == 1) {
        RowTile* out = job.list + 1 + at[0] + (int)whole_to - whole;
        for (int t = 0; t < whole; ++t) out[t] = RowTile{(int)start + t * ROWS, min(live - t * ROWS, ROWS), g, 0};
      }
      at[0] += __builtin_amdgcn_readlane((int)whole_to, 63);
#pragma unroll
      for (int c = 1; c < 4; ++c) {
        const uint64_t mine = __ballot(other == c);
        if (pass == 1 && other == c)
          job.list[1 + at[c] + __popcll(mine & ((uint64_t(1) << lane) - 1))] = RowTile{(int)start + live - rest, rest, g, 0};
        at[c] += __popcll(mine);
      }
      before = min(before + (uint32_t)__builtin_amdgcn_readlane((int)to, 63), (uint32_t)job.M);
    }
    if (pass == 0) {   // numbers to places
      int sum = 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int n = at[c];
        at[c] = sum;
        sum += n;
      }
      if (lane == 0) job.list[0] = RowTile{0, sum, 0, 0};
    }
  }
}

__global__ __launch_bounds__(256) void arrange_scales_kernel(ArrangeJob a, ArrangeJob b, ListJob tiles, int from, int pairs) {
  extern __shared__ __attribute__((aligned(16))) uint4 piece[];   // [row][pair], an odd number of pieces per row
  int at = (int)row_block();
  if (tiles.m_sizes != nullptr && at-- == 0) {
    uint32_t* const sizes = reinterpret_cast<uint32_t*>(piece);
    const int held = min(tiles.G, 64 * 4);
    for (int g = threadIdx.x; g < held; g += 256) sizes[g] = group_size(tiles, g);
    __syncthreads();
    if (threadIdx.x < 64) list_row_tiles(tiles, sizes, held);
    return;
  }
  const bool second = at >= a.workgroups;
  const ArrangeJob job = second ? b : a;
  if (second) at -= a.workgroups;
  if (at >= job.workgroups) return;   // behind the last one, in the grid's last line
  const int slabs = (pairs + kArrangePairs - 1) / kArrangePairs, block = at / slabs, pair0 = (at - block * slabs) * kArrangePairs;
  const int n = min(pairs - pair0, kArrangePairs), rows = (int)min((int64_t)64, job.rows - (int64_t)block * 64);
  const int pitch = n | 1;
  const uint32_t inverse = (65536u + (uint32_t)n - 1) / (uint32_t)n;   // i / n = i * inverse >> 16 for i < 64 n, n <= 8
  const uint8_t* src = job.src + (int64_t)block * 64 * from + pair0 * 16;
  uint4 v[kArrangePairs / 4];
#pragma unroll
  for (int t = 0; t < kArrangePairs / 4; ++t) {   // (all loads before the first store)
    const int i = t * 256 + threadIdx.x, r = (int)(((uint32_t)i * inverse) >> 16), q = i - r * n, left = from - (pair0 + q) * 16;
    const uint8_t* in = src + (int64_t)r * from + q * 16;
    v[t] = make_uint4(0, 0, 0, 0);
    if (r < rows && left >= 16) {
      __builtin_memcpy(&v[t], in, 16);   // (rows begin anywhere)
    } else if (r < rows) {
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (e < left) w[e >> 2] |= (uint32_t)in[e] << (8 * (e & 3));
      v[t] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
#pragma unroll
  for (int t = 0; t < kArrangePairs / 4; ++t) {
    const int i = t * 256 + threadIdx.x, r = (int)(((uint32_t)i * inverse) >> 16), q = i - r * n;
    if (r < rows) piece[r * pitch + q] = v[t];
  }
  __syncthreads();
  uint4* dst = reinterpret_cast<uint4*>(job.dst) + ((int64_t)block * pairs + pair0) * 64;
  for (int i = threadIdx.x; i < 64 * n; i += 256) {
    const int r = i & 63, q = i >> 6;
    if (r < rows) dst[i] = piece[r * pitch + q];
  }
}

int64_t pairs_of(int64_t K) { return (K + 511) / 512; }
int64_t arranged_bytes(int64_t rows, int64_t K) { return (rows + 63) / 64 * pairs_of(K) * 1024; }

// As many row tiles as the rows of all groups can make.
int64_t most_row_tiles(int64_t M, int64_t G, int64_t tile_rows) { return M / tile_rows + (G < M ? G : M); }

template <typename TS, bool GATED, bool GROUPS, bool BIAS, bool F16>
hipError_t launch_tiles(const MxProblem& p, hipStream_t s) {
  constexpr int COLUMNS = GATED ? TS::BN / 2 : TS::BN;
  const int64_t tiles_n = ((int64_t)p.N + COLUMNS - 1) / COLUMNS;
  const int64_t tiles_m = GROUPS ? most_row_tiles(p.M, p.G, TS::BM) : ((int64_t)p.M + TS::BM - 1) / TS::BM;
  const int64_t grid = (tiles_m * tiles_n + kXcds - 1) / kXcds * kXcds;
  if (grid >= (int64_t(1) << 30)) return hipErrorInvalidValue;
  if (dispatch_probe_record("mx_tiles<%d,%d,waves=%dx%dx%d>%s workgroups=%lld", TS::BM, TS::BN, TS::WM, TS::WN, TS::KS, GROUPS ? " groups" : "", (long long)grid))
    return hipSuccess;
  mx_kernel<TS, GATED, GROUPS, BIAS, F16><<<row_grid(grid), TS::NTHREADS, 0, s>>>(p, (int)tiles_m, (int)tiles_n);
  return hipGetLastError();
}

template <typename TS>
hipError_t launch_dense(const MxProblem& p, hipStream_t s) {
  if (p.gated) return p.out_f16 ? launch_tiles<TS, true, false, false, true>(p, s) : launch_tiles<TS, true, false, false, false>(p, s);
  if (p.bias_dtype != 0) return p.out_f16 ? launch_tiles<TS, false, false, true, true>(p, s) : launch_tiles<TS, false, false, true, false>(p, s);
  return p.out_f16 ? launch_tiles<TS, false, false, false, true>(p, s) : launch_tiles<TS, false, false, false, false>(p, s);
}
template <typename TS>
hipError_t launch_groups(const MxProblem& p, hipStream_t s) {
  if (p.gated) return p.out_f16 ? launch_tiles<TS, true, true, false, true>(p, s) : launch_tiles<TS, true, true, false, false>(p, s);
  return p.out_f16 ? launch_tiles<TS, false, true, false, true>(p, s) : launch_tiles<TS, false, true, false, false>(p, s);
}

template <bool GATED, bool BIAS, bool F16>
hipError_t launch_walk(const MxProblem& p, hipStream_t s) {
  constexpr int COLUMNS = GATED ? MxLarge::BN / 2 : MxLarge::BN;
  if (p.K <= 256) return hipErrorInvalidValue;   // (the tiles load two steps ahead)
  const int64_t tiles_n = ((int64_t)p.N + COLUMNS - 1) / COLUMNS;
  const int64_t tiles_m = p.row_tiles != nullptr ? most_row_tiles(p.M, p.G, MxLarge::BM) : ((int64_t)p.M + MxLarge::BM - 1) / MxLarge::BM;
  if (tiles_m * tiles_n >= (int64_t(1) << 30)) return hipErrorInvalidValue;
  const int64_t grid = (2 * tiles_m * tiles_n + kXcds - 1) / kXcds * kXcds, cus = device_compute_units();
  const unsigned wgs = (unsigned)(grid < cus ? grid : cus);
  if (dispatch_probe_record("mx_walk%s tiles=%lld workgroups=%u", p.row_tiles != nullptr ? " groups" : "", (long long)(tiles_m * tiles_n), wgs)) return hipSuccess;
  mx_walk_kernel<GATED, BIAS, F16><<<wgs, MxLarge::NTHREADS, 0, s>>>(p, (int)tiles_m, (int)tiles_n);
  return hipGetLastError();
}

template <bool F16>
hipError_t launch_walk(const MxProblem& p, hipStream_t s) {
  if (p.gated) return launch_walk<true, false, F16>(p, s);
  return p.bias_dtype != 0 ? launch_walk<false, true, F16>(p, s) : launch_walk<false, false, F16>(p, s);
}

enum Way : int {
  kStream,     // few rows, scales that the DMA cannot take: mx_stream.hip
  k32x32, k32x64, k64x64Long, k64x64,   // the small ones
  k128x128,
  k64x128,     // groups only
  kWalk,       // 256-column tiles (at least two steps)
};
using Tile32x32 = MxShape<32, 32, 1, 1, 4>;         // two workgroups per CU
using Tile32x64 = MxShape<32, 64, 1, 1, 4>;         // one
using Tile64x64Long = MxShape<64, 64, 1, 1, 4>;     // one
using Tile64x64 = MxShape<64, 64, 1, 1, 2>;         // two
using Tile64x128 = MxShape<64, 128, 2, 2, 1>;       // two
using Tile128x128 = MxShape<128, 128, 2, 2, 1>;     // two
// Scales are fetched by 16 bytes of a row, by the small tiles by 4.
bool fetched_in_place(int64_t K, bool small, bool scales_aligned) { return K % (small ? 128 : 512) == 0 && scales_aligned; }

// The smallest tiles of which each CU gets no more than it holds at once, since their steps' loads, not their products, are waited for.  µs:
//   16 x 4096 x 14336   32x32 8.9, 32x64 11.7, 64x64 14.9
//   64 x 4096 x 14336   32x32 9.5, 32x64 13.0, 64x64 18.0
//   64 x 8192 x 8192    32x64 9.7, 32x32 10.5, 64x64 12.8 (two waves 14.7), 128x128 26.1
//   16 x 16384 x 4096   32x32 8.2, 32x64 8.7, 64x64 10.0 (up to 32 rows two of the smallest to a CU, as they read no weights twice)
//   128 x 8192 x 8192   64x64 13.3 (two waves 15.2), 32x64 16.1, 128x128 26.6
//   256 x 8192 x 8192   64x64 of two waves 19.3 (four 23.3), 128x128 27.1
//   500 x 8192 x 4096   128x128 17.0, walk 20.5, 64x64 21.6
//   1000 x 10240 x 8192 walk 51.8, 128x128 65.0
// Two 128x128 tiles to a CU only with a short K: 1000 x 8192 x 1024 9.5 (walk 11.7), 500 x 14336 x 2048 13.5 (15.3), 500 x 10240 x 4096 20.9 (21.1),
// 500 x 10240 x 8192 34.6 (34.7), 2000 x 4096 x 14336 73.7 (66.1); one to a CU 500 x 8192 x 8192 29.2 (32.9).
// Up to 32 rows whose scales would have to be arranged first take the kernel that needs no such launch, if there is a CU for every 32 columns
// (16 x 4096 x 4128 6.5, arranged 8.6; 32 x 8192 x 5152 7.9, 11.2).
// Groups of few rows on average wait for weights, too: 64x128 tiles (16 groups, 256 rows, 2 x 5120 x 4096 74.2, walk 79.5; 8 groups, 512 rows,
// 4096 x 14336 77.0 and 102.5; 32 groups, 256 rows, 2 x 1024 x 2048 14.0 and 19.1; a few crowded groups of more rows go the other way: 16 groups, 1024 rows,
// 2 x 5120 x 4096 93.4 and 86.2), but for many of a short K the walk, which has no gap between its tiles and no workgroups for tiles that groups might have
// had (128 groups, 512 rows, 2 x 768 x 2048 36.9, 64x128 38.6; of four rows each 49.1 and 46.7).
Way way_of(int64_t M, int64_t N, int64_t K, int gated, int64_t G, bool grouped, bool scales_aligned) {
  const int64_t cus = device_compute_units(), columns = N * (gated ? 2 : 1);
  auto tiles = [&](int64_t bm, int64_t bn) { return (grouped ? most_row_tiles(M, G, bm) : (M + bm - 1) / bm) * ((columns + bn - 1) / bn); };
  if (!grouped && M <= 32 && columns <= 32 * cus && !fetched_in_place(K, true, scales_aligned)) return kStream;
  if (!grouped && tiles(32, 32) <= (M <= 32 ? 2 : 1) * cus) return k32x32;
  if (!grouped && tiles(32, 64) <= cus) return k32x64;
  if (tiles(64, 64) <= 2 * cus) return tiles(64, 64) <= cus ? k64x64Long : k64x64;
  const bool short_k = K <= 256, wide = N >= (1 << 25);   // what the walk does not take
  if (grouped) return M <= 64 || (M <= 64 * G && (K >= 4096 || tiles(64, 128) <= 4 * cus)) || short_k || wide ? k64x128 : kWalk;
  return tiles(128, 128) <= (K < 4096 ? 2 : 1) * cus || short_k || wide ? k128x128 : kWalk;
}

// Whether the scales are arranged first.  If they can be fetched in place, the launch in front has to be worth it.
// The walk: from 128 steps of 256 x 256 sums per CU on (arranged / in place, us: 4096 x 4096 x 4096 41.4 / 39.0, 16 experts, 2048 rows, 8192 x 5120
// 122 / 116, 8192 x 8192 x 2048 86 / 83, 8192 x 8192 x 4096 139 / 136, 8192 x 8192 x 8192 246 / 243, 16384 x 8192 x 16384 923 / 945, 16 experts, 16384 rows
// 416 / 425, 32768 rows 793 / 809).
// Tiles of fewer rows wait for codes, or have few steps.
bool arranges(Way way, int64_t M, int64_t N, int64_t K, int gated, bool scales_aligned) {
  if (!fetched_in_place(K, way < k128x128, scales_aligned)) return true;
  const double products = (double)M * (double)(N * (gated ? 2 : 1)) * (double)K;
  return way == kWalk && products >= 128. * device_compute_units() * (256 * 256 * 256);
}

}  // namespace

size_t mx_workspace_bytes(int64_t M, int64_t N, int64_t K, int gated, int G, bool grouped, bool scales_aligned) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const Way way = way_of(M, N, K, gated, G, grouped, scales_aligned);
  if (way == kStream) return 0;
  const int64_t list = way == kWalk && grouped ? (1 + most_row_tiles(M, G, MxLarge::BM)) * (int64_t)sizeof(RowTile) : 0;
  if (!arranges(way, M, N, K, gated, scales_aligned)) return (size_t)list;
  return (size_t)(list + arranged_bytes(M, K) + arranged_bytes(N * (gated ? 2 : 1) * (grouped ? G : 1), K));
}

hipError_t launch_mx_mm(MxProblem p, void* workspace, bool scales_aligned, hipStream_t s) {
  const bool grouped = p.m_sizes != nullptr;
  const Way way = way_of(p.M, p.N, p.K, p.gated, p.G, grouped, scales_aligned);
  if (way == kStream) return launch_mx_stream(p, s);
  const int from = p.K / kMxBlock, pairs = (int)pairs_of(p.K);
  const bool listed = way == kWalk && grouped, arranged = p.K > 0 && arranges(way, p.M, p.N, p.K, p.gated, scales_aligned);
  ArrangeJob a{}, b{};
  ListJob tiles{};
  uint8_t* room = static_cast<uint8_t*>(workspace);
  if (listed) {
    tiles = ListJob{p.m_sizes, reinterpret_cast<RowTile*>(room), p.G, p.M};
    p.row_tiles = room;
    room += (1 + most_row_tiles(p.M, p.G, MxLarge::BM)) * (int64_t)sizeof(RowTile);
  }
  const MxScales in_tensor{nullptr, (int64_t)from * 64, from, 16}, in_order{nullptr, (int64_t)pairs * 1024, 16, 1024};
  auto scales = [&](MxScales& s, int64_t rows, ArrangeJob& job) {
    const uint8_t* tensor = s.data;
    s = arranged ? in_order : in_tensor;
    s.data = tensor;
    if (!arranged) return true;
    const int64_t wgs = (rows + 63) / 64 * ((pairs + kArrangePairs - 1) / kArrangePairs);
    if (wgs >= (int64_t(1) << 29)) return false;
    job = ArrangeJob{tensor, room, rows, (int)wgs};
    s.data = room;
    room += arranged_bytes(rows, p.K);
    return true;
  };
  if (!scales(p.xs, p.M, a) || !scales(p.ws, (int64_t)p.N * (p.gated ? 2 : 1) * (grouped ? p.G : 1), b)) return hipErrorInvalidValue;
  if ((listed || arranged) && !dispatch_probe_record(!arranged ? "list_row_tiles" : listed ? "arrange_scales with list_row_tiles" : "arrange_scales")) {
    const int most = pairs < kArrangePairs ? pairs : kArrangePairs;
    arrange_scales_kernel<<<row_grid((int64_t)a.workgroups + b.workgroups + (listed ? 1 : 0)), 256, 64 * (most | 1) * 16, s>>>(a, b, tiles, from, pairs);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  if (way == kWalk) return p.out_f16 ? launch_walk<true>(p, s) : launch_walk<false>(p, s);
  if (way == k64x64Long) return grouped ? launch_groups<Tile64x64Long>(p, s) : launch_dense<Tile64x64Long>(p, s);
  if (way == k64x64) return grouped ? launch_groups<Tile64x64>(p, s) : launch_dense<Tile64x64>(p, s);
  if (way == k64x128) return launch_groups<Tile64x128>(p, s);
  if (way == k32x32) return launch_dense<Tile32x32>(p, s);
  return way == k32x64 ? launch_dense<Tile32x64>(p, s) : launch_dense<Tile128x128>(p, s);
}

}  // namespace mslk_amd
