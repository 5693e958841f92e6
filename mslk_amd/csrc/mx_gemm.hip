// Products of MXFP4 matrices for gfx950: dense, with a gated activation, and for groups of rows (formats: mx.h, tile: mx_tile.h).
#include "kernels.h"
#include "mx_device.h"
#include "mx_tile_large.h"

namespace mslk_amd {
namespace {

// Eight columns n ... n + 7 of a row's bias, as fp32; `whole`: they exist and lie on 16 bytes.
template <int BIAS>
MSLK_AMD_DEVINL void load_bias(const MxProblem& p, int n, bool whole, float (&b)[8]) {
  if constexpr (BIAS == 0) {
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = 0.f;
  } else if (whole) {
    if constexpr (BIAS == 1) {
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
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = n + e < p.N ? n + e : p.N - 1;
      b[e] = BIAS == 1 ? static_cast<const float*>(p.bias)[at] : bf16_bits_to_f32(static_cast<const uint16_t*>(p.bias)[at]);
    }
  }
}

// Sums of a tile to Y: rows m0 ... m0 + rows - 1, columns from n0.
// A lane's pieces of eight columns (16 bytes) are two of a row's eight in a line: four of its own (register bits r1, r0), times its h.
// Exchanging r0 with bit 4 of the lane and r1 with bit 3 leaves a register eight rows' whole lines, which are then written past the L2:
// left in 32-byte pieces they reached the memory as such.
template <typename TS, bool GATED, int BIAS, bool F16>
MSLK_AMD_DEVINL void store_tile(const MxProblem& p, const v16f (&acc)[TS::FN][TS::FM], int m0, int rows, int n0) {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));   // formed again here, not kept over the products
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / TS::WN, wn = wave % TS::WN, h = lane >> 5;
  const int first = n0 + wn * (TS::BN / TS::WN) / (GATED ? 2 : 1);
  const bool aligned = (p.N & 7) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
  const bool bias_aligned = BIAS != 0 && (reinterpret_cast<uintptr_t>(p.bias) & 15) == 0;
  constexpr int LINES = GATED ? (TS::FN + 3) / 4 : TS::FN / 2;   // of 64 columns; the last one of a gated tile with FN = 2 is half empty
  float b[LINES][4][8];
  // column of piece r of line t for the lanes of half h
  auto column = [&](int t, int r, int half) { return GATED ? t * 64 + (r >> 1) * 32 + half * 16 + (r & 1) * 8 : t * 64 + r * 16 + half * 8; };
#pragma unroll
  for (int t = 0; t < LINES; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = first + column(t, r, h);
      load_bias<BIAS>(p, n, bias_aligned && n + 8 <= p.N, b[t][r]);
    }
  // after the exchange: this lane's piece and row of each register
  const int piece = ((lane >> 3) & 1) * 2 + ((lane >> 4) & 1), row8 = lane & 7;
#pragma unroll
  for (int tm = 0; tm < TS::FM; ++tm) {
    const int row0 = wm * (TS::BM / TS::WM) + tm * 32;
#pragma unroll
    for (int t = 0; t < LINES; ++t) {
      constexpr int PIECES = GATED && TS::FN == 2 ? 2 : 4;
      uint32_t w[4][4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if constexpr (GATED) {
            if (r >= PIECES) { v[e] = 0.f; continue; }
            const int T = t * 2 + (r >> 1), at = 8 * (r & 1) + e;
            v[e] = gated_value(acc[2 * T][tm][at], acc[2 * T + 1][tm][at]);
          } else {
            v[e] = acc[2 * t + (e >> 2)][tm][4 * r + (e & 3)];
            if constexpr (BIAS != 0) v[e] += b[t][r][e];
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
      const int n = first + column(t, piece, h), columns = p.N - n;
      const bool mine = columns > 0 && piece < PIECES;
#pragma unroll
      for (int r = 0; r < 4; ++r) {   // rows with bit 4 = r & 1, bit 3 = r >> 1
        const int m = row0 + (r & 1) * 16 + (r >> 1) * 8 + row8;
        uint16_t* dst = p.y + (int64_t)(m0 + m) * p.N + n;
        if (mine && m < rows) {
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

template <typename TS, bool GATED>
MSLK_AMD_DEVINL void store_tile(const MxProblem& p, const v16f (&acc)[TS::FN][TS::FM], int m0, int rows, int n0) {
  if constexpr (GATED) {
    if (p.out_f16) store_tile<TS, true, 0, true>(p, acc, m0, rows, n0);
    else store_tile<TS, true, 0, false>(p, acc, m0, rows, n0);
  } else {
    if (p.out_f16) {
      if (p.bias_dtype == 0) store_tile<TS, false, 0, true>(p, acc, m0, rows, n0);
      else if (p.bias_dtype == 1) store_tile<TS, false, 1, true>(p, acc, m0, rows, n0);
      else store_tile<TS, false, 2, true>(p, acc, m0, rows, n0);
    } else {
      if (p.bias_dtype == 0) store_tile<TS, false, 0, false>(p, acc, m0, rows, n0);
      else if (p.bias_dtype == 1) store_tile<TS, false, 1, false>(p, acc, m0, rows, n0);
      else store_tile<TS, false, 2, false>(p, acc, m0, rows, n0);
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
template <typename TS, bool GATED, bool GROUPS>
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
  const MxOperands o = operands_of<GATED>(p, m0, rows, w_row, n0, COLUMNS);
  v16f acc[TS::FN][TS::FM];
  if constexpr (std::is_same_v<TS, MxLarge>) {
    MxLargeTile<GATED> tile;
    typename MxLargeTile<GATED>::Held held;
    tile.start(lds, o, held);
    tile.run(lds, o, held, acc);
    wait_vmcnt0();   // (the loads of a tile that does not follow end before the LDS is given away)
  } else {
    MxTile<TS, GATED> tile;
    tile.init(o);
    tile.run(lds, acc);
  }
  store_tile<TS, GATED>(p, acc, m0, rows, n0);
}

// A workgroup per CU that walks the tiles: XCD x keeps its run of neighbouring entries, its workgroups take them in turn.
template <bool GATED>
__global__ __launch_bounds__(256) void mx_walk_kernel(MxProblem p, int tiles_m, int tiles_n) {
  using TS = MxLarge;
  __shared__ __attribute__((aligned(1024))) char lds[TS::LDS_BYTES];
  constexpr int COLUMNS = GATED ? TS::BN / 2 : TS::BN;
  const int total = tiles_m * tiles_n, per_xcd = (total + kXcds - 1) / kXcds, first = (int)(blockIdx.x % kXcds) * per_xcd, stride = gridDim.x / kXcds;
  const int end = min(per_xcd, total - first);
  int j = blockIdx.x / kXcds;
  if (j >= end) return;
  int tm, tn;
  tile_at(first + j, tiles_m, tiles_n, tm, tn);
  MxLargeTile<GATED> tile;
  typename MxLargeTile<GATED>::Held held;
  tile.start(lds, operands_of<GATED>(p, tm * TS::BM, min(p.M - tm * TS::BM, TS::BM), 0, tn * COLUMNS, COLUMNS), held);
  for (;;) {
    const int m0 = tm * TS::BM, n0 = tn * COLUMNS;
    j += stride;
    if (j < end) tile_at(first + j, tiles_m, tiles_n, tm, tn);   // (behind the last tile: itself once more)
    v16f acc[TS::FN][TS::FM];
    tile.run(lds, operands_of<GATED>(p, tm * TS::BM, min(p.M - tm * TS::BM, TS::BM), 0, tn * COLUMNS, COLUMNS), held, acc);
    store_tile<TS, GATED>(p, acc, m0, min(p.M - m0, TS::BM), n0);
    if (j >= end) break;
  }
  wait_vmcnt0();
}

// Tensors of scales, rows of `from` bytes, to the arranged layout (MxScales); both operands in one launch.  A lane moves 16 bytes, eight
// lanes a line of one row, eight rows to the lines of eight pairs.
struct ArrangeJob {
  const uint8_t* src;
  uint8_t* dst;
  int64_t rows, workgroups;
};
__global__ __launch_bounds__(512) void arrange_scales_kernel(ArrangeJob a, ArrangeJob b, int from, int pairs) {
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

template <typename TS, bool GATED, bool GROUPS>
hipError_t launch(const MxProblem& p, hipStream_t s) {
  constexpr int COLUMNS = GATED ? TS::BN / 2 : TS::BN;
  const int64_t tiles_n = (p.N + COLUMNS - 1) / COLUMNS;
  // (groups: as many row tiles as the sizes could make)
  const int64_t tiles_m = GROUPS ? (int64_t)p.M / TS::BM + (p.G < p.M ? p.G : p.M) : (p.M + TS::BM - 1) / TS::BM;
  const int64_t grid = (tiles_m * tiles_n + kXcds - 1) / kXcds * kXcds;
  if (grid * TS::NTHREADS >= (int64_t(1) << 32)) return hipErrorInvalidValue;
  if constexpr (std::is_same_v<TS, MxLarge> && !GROUPS) {
    const int cus = device_compute_units();
    mx_walk_kernel<GATED><<<(unsigned)(grid < cus ? grid : cus), TS::NTHREADS, 0, s>>>(p, (int)tiles_m, (int)tiles_n);
  } else {
    mx_kernel<TS, GATED, GROUPS><<<(unsigned)grid, TS::NTHREADS, 0, s>>>(p, (int)tiles_m, (int)tiles_n);
  }
  return hipGetLastError();
}

template <typename TS>
hipError_t launch(const MxProblem& p, hipStream_t s) {
  if (p.m_sizes != nullptr) return p.gated ? launch<TS, true, true>(p, s) : launch<TS, false, true>(p, s);
  return p.gated ? launch<TS, true, false>(p, s) : launch<TS, false, false>(p, s);
}

// Few rows: the weights are streamed (mx_stream.hip).
constexpr int kStreamTiles = 384;
bool takes_stream(int64_t M, int64_t N, int gated, bool grouped) { return !grouped && M <= 64 && N * (gated ? 2 : 1) <= 32 * kStreamTiles; }
// Whether the 256 x 256 tiles take the others (at least two steps).
bool takes_large(int64_t K) { return K > 256; }

}  // namespace

size_t mx_workspace_bytes(int64_t M, int64_t N, int64_t K, int gated, int G, bool grouped, bool scales_aligned) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  if (takes_stream(M, N, gated, grouped) || (K % 512 == 0 && scales_aligned && !(takes_large(K) && M > 64))) return 0;
  return (size_t)(arranged_bytes(M, K) + arranged_bytes(N * (gated ? 2 : 1) * (grouped ? G : 1), K));
}

hipError_t launch_mx_mm(MxProblem p, void* workspace, bool scales_aligned, hipStream_t s) {
  if (takes_stream(p.M, p.N, p.gated, p.m_sizes != nullptr)) return launch_mx_stream(p, s);
  const bool large = takes_large(p.K) && p.M > 64;
  const int from = p.K / kMxBlock, pairs = (int)pairs_of(p.K);
  if (p.K > 0 && (large || p.K % 512 != 0 || !scales_aligned)) {
    const int64_t rows_w = (int64_t)p.N * (p.gated ? 2 : 1) * (p.m_sizes != nullptr ? p.G : 1);
    uint8_t *xs = static_cast<uint8_t*>(workspace), *ws = xs + arranged_bytes(p.M, p.K);
    const int64_t slabs = (pairs + 7) / 8;
    const ArrangeJob a{p.xs.data, xs, p.M, (p.M + 63) / 64 * slabs}, b{p.ws.data, ws, rows_w, (rows_w + 63) / 64 * slabs};
    if ((a.workgroups + b.workgroups) * 512 >= (int64_t(1) << 32)) return hipErrorInvalidValue;
    arrange_scales_kernel<<<(unsigned)(a.workgroups + b.workgroups), 512, 0, s>>>(a, b, from, pairs);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    p.xs = MxScales{xs, (int64_t)pairs * 1024, 16, 1024};
    p.ws = MxScales{ws, (int64_t)pairs * 1024, 16, 1024};
  } else {
    p.xs = MxScales{p.xs.data, (int64_t)from * 64, from, 16};
    p.ws = MxScales{p.ws.data, (int64_t)from * 64, from, 16};
  }
  if (large) return launch<MxLarge>(p, s);
  return launch<MxShape<64, 128, 2, 2, 4>>(p, s);
}

}  // namespace mslk_amd
