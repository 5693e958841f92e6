// Products of MXFP4 matrices for gfx950: dense, with a gated activation, and for groups of rows (formats: mx.h, tile: mx_tile.h).
#include "kernels.h"
#include "mx_device.h"
#include "mx_tile_large.h"

namespace mslk_amd {
namespace {

// Eight columns n ... n + 7 of the bias, as fp32; `whole`: they exist and lie on 16 bytes.
MSLK_AMD_DEVINL void load_bias(const MxProblem& p, int n, bool whole, float (&b)[8]) {
  if (!whole) {
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = bias_at(p, min(n + e, p.N - 1));
  } else if (p.bias_dtype == 1) {
    const float4 *f = reinterpret_cast<const float4*>(static_cast<const float*>(p.bias) + n), lo = f[0], hi = f[1];
    b[0] = lo.x; b[1] = lo.y; b[2] = lo.z; b[3] = lo.w;
    b[4] = hi.x; b[5] = hi.y; b[6] = hi.z; b[7] = hi.w;
  } else {
    const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.bias) + n);
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      b[2 * e] = bf16_bits_to_f32(v[e] & 0xFFFFu);
      b[2 * e + 1] = bf16_bits_to_f32(v[e] >> 16);
    }
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
// FULL: every row and column of the tile is valid and its rows begin on 16 bytes; N < 2^25.
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
    float b[4][8];
    if constexpr (BIAS) {
      const bool bias_aligned = (reinterpret_cast<uintptr_t>(p.bias) & 15) == 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = first + column(t, r, h);
        load_bias(p, n, bias_aligned && (FULL || n + 8 <= p.N), b[r]);
      }
    }
#pragma unroll
    for (int tm = 0; tm < FM; ++tm) {
      const int row0 = wm * WAVE_ROW + tm * FRAG_ROW;
      if (!FULL && row0 >= rows) break;
      uint32_t w[4][4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if constexpr (GATED) {
            const int T = t * 2 + (r >> 1), at = 8 * (r & 1) + e;
            v[e] = r < PIECES ? gated_value(acc[2 * T][tm][at], acc[2 * T + 1][tm][at]) : 0.f;
          } else {
            v[e] = acc[2 * t + (e >> 2)][tm][4 * r + (e & 3)];
            if constexpr (BIAS) v[e] += b[r][e];
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) w[r][e] = pack_out_x2<F16>(v[2 * e], v[2 * e + 1]);
      }
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

// One tile per workgroup.
template <typename TS, bool GATED, bool GROUPS, bool BIAS, bool F16>
__global__ __launch_bounds__(TS::NTHREADS) void mx_kernel(MxProblem p, int tiles_m, int tiles_n) {
  __shared__ __attribute__((aligned(1024))) char lds[TS::LDS_BYTES];
  constexpr int COLUMNS = GATED ? TS::BN / 2 : TS::BN;
  int m0, rows, tn;
  int64_t w_row = 0;
  if constexpr (GROUPS) {
    GroupTile t;
    if (!find_group_tile<TS::BM>(p, tiles_n, blockIdx.x, t)) return;
    m0 = t.row0;
    rows = t.rows;
    tn = t.tn;
    w_row = (int64_t)t.g * p.N * (GATED ? 2 : 1);
  } else {
    const int t = entry_of(blockIdx.x, tiles_m * tiles_n);
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
  store_tile<TS::FM, TS::FN, TS::WN, TS::BM / TS::WM, 32, GATED, BIAS, F16, false>(p, acc, m0, rows, n0);
}

// Row tiles: of p.tile_rows rows, or as listed in device memory.
struct RowTile { int row0, rows, group, unused; };

// A workgroup per CU that walks the 256-column tiles: XCD x keeps its run of neighbouring entries, its workgroups take them in turn.
template <bool GATED, bool BIAS, bool F16>
__global__ __launch_bounds__(256) void mx_walk_kernel(MxProblem p, int tiles_m, int tiles_n) {
  using TS = MxLarge;
  using Tile = MxLargeTile<GATED>;
  __shared__ __attribute__((aligned(1024))) char lds[TS::LDS_BYTES];
  constexpr int COLUMNS = GATED ? TS::BN / 2 : TS::BN;
  const RowTile* const list = static_cast<const RowTile*>(p.row_tiles);
  if (list != nullptr) tiles_m = list[0].rows;   // (the first entry holds their number)
  const int total = tiles_m * tiles_n, per_xcd = (total + kXcds - 1) / kXcds, first = (int)(blockIdx.x % kXcds) * per_xcd, stride = gridDim.x / kXcds;
  const int end = min(per_xcd, total - first);
  int j = blockIdx.x / kXcds;
  if (j >= end) return;
  const bool aligned = (p.N & 7) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
  struct Place { int m0, rows, n0; int64_t w_row; };
  auto place_of = [&](int t) {
    int tm, tn;
    tile_at(t, tiles_m, tiles_n, tm, tn);
    if (list != nullptr) {
      const RowTile r = list[1 + tm];
      return Place{r.row0, r.rows, tn * COLUMNS, (int64_t)r.group * p.N * (GATED ? 2 : 1)};
    }
    return Place{tm * p.tile_rows, min(p.M - tm * p.tile_rows, p.tile_rows), tn * COLUMNS, 0};
  };
  auto operands = [&](const Place& at) { return operands_of<GATED>(p, at.m0, at.rows, at.w_row, at.n0, COLUMNS); };
  Place at = place_of(first + j);
  Tile tile;
  typename Tile::Held held;
  tile.start(lds, operands(at), held);
  for (;;) {
    const Place here = at;
    j += stride;
    if (j < end) at = place_of(first + j);   // (behind the last tile: itself once more)
    auto make = [&](auto fragments) {
      constexpr int F = decltype(fragments)::value;
      v16f acc[4][F];
      tile.template run<F>(lds, operands(at), held, acc);
      if (here.rows == 64 * F && here.n0 + COLUMNS <= p.N && aligned) store_tile<F, 4, 2, 32, 64, GATED, BIAS, F16, true>(p, acc, here.m0, here.rows, here.n0);
      else store_tile<F, 4, 2, 32, 64, GATED, BIAS, F16, false>(p, acc, here.m0, here.rows, here.n0);
    };
    if (here.rows > 128) make(std::integral_constant<int, 4>{});
    else if (here.rows > 64) make(std::integral_constant<int, 2>{});
    else make(std::integral_constant<int, 1>{});
    if (j >= end) break;
  }
  wait_vmcnt0();   // the loads of a tile that does not follow end before the LDS is given away
}

// Tensors of scales, rows of `from` bytes, to the arranged layout (MxScales); both operands in one launch.  A lane moves 16 bytes, eight
// lanes a line of one row, eight rows to the lines of eight pairs.
struct ArrangeJob {
  const uint8_t* src;
  uint8_t* dst;
  int64_t rows, workgroups;
};
// Row tiles of the groups (at most 256 rows each), in the first workgroup: list[0].rows of them behind list[0].
struct ListJob {
  const int64_t* m_sizes;   // nullptr: none
  RowTile* list;
  int G, M;
};
MSLK_AMD_DEVINL void list_row_tiles(const ListJob& job) {
  __shared__ int64_t rows_to[512];   // rows of the groups up to and with this one, tiles likewise
  __shared__ int tiles_to[512];
  int64_t rows_before = 0;
  int tiles_before = 0;
  const int i = threadIdx.x;
  for (int g0 = 0; g0 < job.G; g0 += 512) {
    const int g = g0 + i;
    const int64_t size = g < job.G ? max((int64_t)0, min(job.m_sizes[g], (int64_t)job.M)) : 0;
    rows_to[i] = size;
    __syncthreads();
    for (int d = 1; d < 512; d *= 2) {
      const int64_t add = i >= d ? rows_to[i - d] : 0;
      __syncthreads();
      rows_to[i] += add;
      __syncthreads();
    }
    const int64_t start = rows_before + rows_to[i] - size;
    const int live = (int)max((int64_t)0, min(size, job.M - start)), tiles = (live + MxLarge::BM - 1) / MxLarge::BM;
    tiles_to[i] = tiles;
    __syncthreads();
    for (int d = 1; d < 512; d *= 2) {
      const int add = i >= d ? tiles_to[i - d] : 0;
      __syncthreads();
      tiles_to[i] += add;
      __syncthreads();
    }
    RowTile* out = job.list + 1 + tiles_before + tiles_to[i] - tiles;
    for (int t = 0; t < tiles; ++t) out[t] = RowTile{(int)start + t * MxLarge::BM, min(live - t * MxLarge::BM, MxLarge::BM), g, 0};
    rows_before += rows_to[511];
    tiles_before += tiles_to[511];
    __syncthreads();
  }
  if (i == 0) job.list[0] = RowTile{0, tiles_before, 0, 0};
}

__global__ __launch_bounds__(512) void arrange_scales_kernel(ArrangeJob a, ArrangeJob b, ListJob tiles, int from, int pairs) {
  if (tiles.m_sizes != nullptr && blockIdx.x == 0) list_row_tiles(tiles);
  const bool second = blockIdx.x >= a.workgroups;
  const ArrangeJob job = second ? b : a;
  const int64_t at = blockIdx.x - (second ? a.workgroups : 0);
  const int slabs = (pairs + 7) / 8;   // a workgroup: 64 rows, eight pairs
  const int64_t block = at / slabs;
  const int pair = (int)(at - block * slabs) * 8 + (threadIdx.x & 7), r = threadIdx.x >> 3;
  const int64_t row = block * 64 + r;
  if (pair >= pairs || row >= job.rows) return;
  const int col = pair * 16;
  const uint8_t* in = job.src + row * from + col;
  uint32_t w[4];
  if (col + 16 <= from) {
    __builtin_memcpy(w, in, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (col + 4 * i + b < from) w[i] |= (uint32_t)in[4 * i + b] << (8 * b);
    }
  }
  reinterpret_cast<uint4*>(job.dst)[(block * pairs + pair) * 64 + r] = make_uint4(w[0], w[1], w[2], w[3]);
}

int64_t pairs_of(int64_t K) { return (K + 511) / 512; }
int64_t arranged_bytes(int64_t rows, int64_t K) { return (rows + 63) / 64 * pairs_of(K) * 1024; }

// As many row tiles as the rows of all groups can make.
int64_t most_row_tiles(int64_t M, int64_t G, int64_t tile_rows) { return M / tile_rows + (G < M ? G : M); }

template <typename TS, bool GATED, bool GROUPS, bool BIAS, bool F16>
hipError_t launch_tiles(const MxProblem& p, hipStream_t s) {
  constexpr int COLUMNS = GATED ? TS::BN / 2 : TS::BN;
  const int64_t tiles_n = (p.N + COLUMNS - 1) / COLUMNS;
  const int64_t tiles_m = GROUPS ? most_row_tiles(p.M, p.G, TS::BM) : (p.M + TS::BM - 1) / TS::BM;
  const int64_t grid = (tiles_m * tiles_n + kXcds - 1) / kXcds * kXcds;
  if (grid * TS::NTHREADS >= (int64_t(1) << 32)) return hipErrorInvalidValue;
  mx_kernel<TS, GATED, GROUPS, BIAS, F16><<<(unsigned)grid, TS::NTHREADS, 0, s>>>(p, (int)tiles_m, (int)tiles_n);
  return hipGetLastError();
}

template <typename TS, bool F16>
hipError_t launch_tiles(const MxProblem& p, hipStream_t s) {
  if (p.m_sizes != nullptr) return p.gated ? launch_tiles<TS, true, true, false, F16>(p, s) : launch_tiles<TS, false, true, false, F16>(p, s);
  if (p.gated) return launch_tiles<TS, true, false, false, F16>(p, s);
  return p.bias_dtype != 0 ? launch_tiles<TS, false, false, true, F16>(p, s) : launch_tiles<TS, false, false, false, F16>(p, s);
}

template <bool GATED, bool BIAS, bool F16>
hipError_t launch_walk(const MxProblem& p, hipStream_t s) {
  constexpr int COLUMNS = GATED ? MxLarge::BN / 2 : MxLarge::BN;
  const int64_t tiles_n = (p.N + COLUMNS - 1) / COLUMNS;
  const int64_t tiles_m = p.row_tiles != nullptr ? most_row_tiles(p.M, p.G, p.tile_rows) : (p.M + p.tile_rows - 1) / p.tile_rows;
  if (tiles_m * tiles_n >= (int64_t(1) << 31)) return hipErrorInvalidValue;
  const int64_t grid = (tiles_m * tiles_n + kXcds - 1) / kXcds * kXcds, cus = device_compute_units();
  mx_walk_kernel<GATED, BIAS, F16><<<(unsigned)(grid < cus ? grid : cus), MxLarge::NTHREADS, 0, s>>>(p, (int)tiles_m, (int)tiles_n);
  return hipGetLastError();
}

template <bool F16>
hipError_t launch_walk(const MxProblem& p, hipStream_t s) {
  if (p.gated) return launch_walk<true, false, F16>(p, s);
  return p.bias_dtype != 0 ? launch_walk<false, true, F16>(p, s) : launch_walk<false, false, F16>(p, s);
}

enum Way : int {
  kStream,   // few rows: mx_stream.hip
  kTiles,    // 64 x 128 tiles
  kWalk,     // 256-column tiles (at least two steps)
};
Way way_of(int64_t M, int64_t N, int64_t K, int gated, bool grouped) {
  constexpr int kStreamTiles = 384;
  if (!grouped && M <= 64 && N * (gated ? 2 : 1) <= 32 * kStreamTiles) return kStream;
  return M <= 64 || K <= 256 || N >= (1 << 25) ? kTiles : kWalk;
}

// Rows of a row tile: as many as leave every CU a tile.
int rows_of_tile(int64_t M, int64_t N, int gated) {
  const int64_t tiles_n = (N * (gated ? 2 : 1) + 255) / 256, cus = device_compute_units();
  if ((M + 255) / 256 * tiles_n > cus / 2) return 256;
  return (M + 127) / 128 * tiles_n > cus / 2 ? 128 : 64;
}

}  // namespace

size_t mx_workspace_bytes(int64_t M, int64_t N, int64_t K, int gated, int G, bool grouped, bool scales_aligned) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const Way way = way_of(M, N, K, gated, grouped);
  if (way == kStream || (way == kTiles && K % 512 == 0 && scales_aligned)) return 0;
  const int64_t list = way == kWalk && grouped ? (1 + most_row_tiles(M, G, MxLarge::BM)) * (int64_t)sizeof(RowTile) : 0;
  return (size_t)(arranged_bytes(M, K) + arranged_bytes(N * (gated ? 2 : 1) * (grouped ? G : 1), K) + list);
}

hipError_t launch_mx_mm(MxProblem p, void* workspace, bool scales_aligned, hipStream_t s) {
  const bool grouped = p.m_sizes != nullptr;
  const Way way = way_of(p.M, p.N, p.K, p.gated, grouped);
  if (way == kStream) return launch_mx_stream(p, s);
  const int from = p.K / kMxBlock, pairs = (int)pairs_of(p.K);
  p.tile_rows = grouped ? MxLarge::BM : rows_of_tile(p.M, p.N, p.gated);
  if (p.K > 0 && (way == kWalk || p.K % 512 != 0 || !scales_aligned)) {
    const int64_t rows_w = (int64_t)p.N * (p.gated ? 2 : 1) * (grouped ? p.G : 1);
    uint8_t *xs = static_cast<uint8_t*>(workspace), *ws = xs + arranged_bytes(p.M, p.K), *list = ws + arranged_bytes(rows_w, p.K);
    const int64_t slabs = (pairs + 7) / 8;
    const ArrangeJob a{p.xs.data, xs, p.M, (p.M + 63) / 64 * slabs}, b{p.ws.data, ws, rows_w, (rows_w + 63) / 64 * slabs};
    ListJob tiles{};
    if (way == kWalk && grouped) {
      tiles = ListJob{p.m_sizes, reinterpret_cast<RowTile*>(list), p.G, p.M};
      p.row_tiles = list;
    }
    if ((a.workgroups + b.workgroups) * 512 >= (int64_t(1) << 32)) return hipErrorInvalidValue;
    arrange_scales_kernel<<<(unsigned)(a.workgroups + b.workgroups), 512, 0, s>>>(a, b, tiles, from, pairs);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    p.xs = MxScales{xs, (int64_t)pairs * 1024, 16, 1024};
    p.ws = MxScales{ws, (int64_t)pairs * 1024, 16, 1024};
  } else {
    p.xs = MxScales{p.xs.data, (int64_t)from * 64, from, 16};
    p.ws = MxScales{p.ws.data, (int64_t)from * 64, from, 16};
  }
  if (way == kWalk) return p.out_f16 ? launch_walk<true>(p, s) : launch_walk<false>(p, s);
  return p.out_f16 ? launch_tiles<MxShape<64, 128, 2, 2, 4>, true>(p, s) : launch_tiles<MxShape<64, 128, 2, 2, 4>, false>(p, s);
}

}  // namespace mslk_amd
