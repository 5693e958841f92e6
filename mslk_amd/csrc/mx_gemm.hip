// Products of MXFP4 matrices for gfx950: dense, with a gated activation, and for groups of rows (formats: mx.h, tile: mx_tile.h).
#include "kernels.h"
#include "mx_tile.h"

namespace mslk_amd {
namespace {

constexpr int kXcds = 8;
constexpr int kPanel = 4;   // row tiles that share the weights of a panel in an XCD's L2

// y = silu(gate) * up in fp32.  For gates below -88 exp(-gate) is infinite and the result -0, as it should be; the exponential and the
// reciprocal are good to about 2 units of fp32, far below the rounding to 16 bits that follows.
MSLK_AMD_DEVINL float gated_value(float gate, float up) { return gate * __builtin_amdgcn_rcpf(1.f + __expf(-gate)) * up; }

MSLK_AMD_DEVINL float bias_at(const MxProblem& p, int n) {
  if (p.bias_dtype == 1) return static_cast<const float*>(p.bias)[n];
  if (p.bias_dtype == 2) return bf16_bits_to_f32(static_cast<const uint16_t*>(p.bias)[n]);
  return 0.f;
}

MSLK_AMD_DEVINL uint32_t pack_x2(float a, float b, int out_f16) { return out_f16 ? pack_f16x2(a, b) : pack_bf16x2(a, b); }

// Eight columns n ... n + 7 of one row of Y; `whole`: all of them exist and their 16 bytes are aligned.
MSLK_AMD_DEVINL void store8(uint16_t* dst, const float (&v)[8], int columns, bool whole, int out_f16) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = pack_x2(v[2 * e], v[2 * e + 1], out_f16);
  if (whole) {
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < columns) dst[e] = (uint16_t)(w[e >> 1] >> ((e & 1) * 16));
  }
}

// Sums of a tile to Y (or, as they are, to p.part): rows m0 ... m0 + rows - 1, columns from n0.
template <typename TS, bool GATED>
MSLK_AMD_DEVINL void store_tile(const MxProblem& p, const v16f (&acc)[TS::FN][TS::FM], int m0, int rows, int n0, int slice) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / TS::WN, wn = wave % TS::WN, i = lane & 31, h = lane >> 5;
  const bool aligned = (p.N & 7) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
#pragma unroll
  for (int T = 0; T < TS::FN / 2; ++T) {
#pragma unroll
    for (int c = 0; c < (GATED ? 2 : 4); ++c) {   // pieces of eight columns
      const int n = GATED ? n0 + (wn * (TS::BN / TS::WN) + T * 64) / 2 + 16 * h + 8 * c : n0 + wn * (TS::BN / TS::WN) + T * 64 + 16 * c + 8 * h;
      const bool whole = aligned && n + 8 <= p.N;
      float b[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = !GATED && p.bias_dtype != 0 && n + e < p.N ? bias_at(p, n + e) : 0.f;
#pragma unroll
      for (int tm = 0; tm < TS::FM; ++tm) {
        const int m = wm * (TS::BM / TS::WM) + tm * 32 + i;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if constexpr (GATED) v[e] = gated_value(acc[2 * T][tm][8 * c + e], acc[2 * T + 1][tm][8 * c + e]);
          else v[e] = acc[2 * T + (e >> 2)][tm][4 * c + (e & 3)] + b[e];
        }
        if (m < rows && n < p.N) store8(p.y + (int64_t)(m0 + m) * p.N + n, v, p.N - n, whole, p.out_f16);
      }
    }
  }
}

// Entry t of the tiles of `tiles_m` x `tiles_n`: panels of up to kPanel row tiles, column by column.
MSLK_AMD_DEVINL void tile_at(int t, int tiles_m, int tiles_n, int& tm, int& tn) {
  const int panel = kPanel * tiles_n, first = (t / panel) * kPanel;
  const int rows = min(tiles_m - first, kPanel);
  tm = __builtin_amdgcn_readfirstlane(first + (t % panel) % rows);
  tn = __builtin_amdgcn_readfirstlane((t % panel) / rows);
}

// Workgroup ids are dealt to the XCDs in turn: XCD x takes a run of neighbouring entries of the list.
MSLK_AMD_DEVINL int entry_of(int wg, int total) {
  const int per_xcd = (total + kXcds - 1) / kXcds, t = (wg % kXcds) * per_xcd + wg / kXcds;
  return wg / kXcds < per_xcd && t < total ? t : -1;
}

// Group and tile of entry t among the row tiles of all groups (R_g = ceil(size / BM) each) times tiles_n.  Returns false behind the
// last one.  Every lane takes part.
struct GroupTile { int g, row0, rows, tm, tn; };
template <int BM>
MSLK_AMD_DEVINL bool find_group_tile(const MxProblem& p, int tiles_n, int wg, GroupTile& out) {
  const int lane = threadIdx.x & 63;
  auto size_at = [&](int g) { return g < p.G ? (int)max((int64_t)0, min(p.m_sizes[g], (int64_t)p.M)) : 0; };
  // all row tiles (rows beyond M do not exist, whatever the sizes say)
  int tiles = 0;
  int64_t rows_before = 0;
  for (int g0 = 0; g0 < p.G; g0 += 64) {
    int64_t end = size_at(g0 + lane);
    const int mine = (int)end;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int64_t up = __shfl_up(end, d, 64);
      if (lane >= d) end += up;
    }
    const int64_t start = rows_before + end - mine;
    int r = (int)max((int64_t)0, min((int64_t)mine, p.M - start));
    r = (r + BM - 1) / BM;
#pragma unroll
    for (int d = 32; d > 0; d /= 2) r += __shfl_xor(r, d, 64);
    tiles += r;
    rows_before += __shfl(end, 63, 64);
  }
  const int t = entry_of(wg, tiles * tiles_n);
  if (t < 0) return false;
  int before = 0;
  rows_before = 0;
  for (int g0 = 0; g0 < p.G; g0 += 64) {
    int64_t end = size_at(g0 + lane);
    const int mine = (int)end;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int64_t up = __shfl_up(end, d, 64);
      if (lane >= d) end += up;
    }
    const int64_t start = rows_before + end - mine;
    const int live = (int)max((int64_t)0, min((int64_t)mine, p.M - start));
    int last = (live + BM - 1) / BM * tiles_n;   // entries up to and with this group's
    const int own = last;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int up = __shfl_up(last, d, 64);
      if (lane >= d) last += up;
    }
    const uint64_t holds = __ballot(t >= before + last - own && t < before + last);
    if (holds != 0) {
      const int src = __ffsll((unsigned long long)holds) - 1;
      out.g = __builtin_amdgcn_readfirstlane(g0 + src);
      const int row0 = __shfl((int)start, src, 64), size = __shfl(live, src, 64), at = t - (before + __shfl(last - own, src, 64));
      tile_at(at, (size + BM - 1) / BM, tiles_n, out.tm, out.tn);
      out.row0 = __builtin_amdgcn_readfirstlane(row0) + out.tm * BM;
      out.rows = min(__builtin_amdgcn_readfirstlane(size) - out.tm * BM, BM);
      return true;
    }
    before += __shfl(last, 63, 64);
    rows_before += __shfl(end, 63, 64);
  }
  return false;
}

template <typename TS, bool GATED, bool GROUPS>
__global__ __launch_bounds__(TS::NTHREADS) void mx_kernel(MxProblem p, int tiles_m, int tiles_n) {
  __shared__ __attribute__((aligned(1024))) char lds[TS::LDS_BYTES];
  constexpr int COLUMNS = GATED ? TS::BN / 2 : TS::BN;
  const int64_t ld = p.K / 2;
  int m0, rows, tn;
  const uint8_t *w = p.wq, *ws = p.ws;
  if constexpr (GROUPS) {
    GroupTile t;
    if (!find_group_tile<TS::BM>(p, tiles_n, blockIdx.x, t)) return;
    m0 = t.row0;
    rows = t.rows;
    tn = t.tn;
    const int64_t rows_w = (int64_t)t.g * p.N * (GATED ? 2 : 1);
    w += rows_w * ld;
    ws += rows_w * p.w_pitch;
  } else {
    const int t = entry_of(blockIdx.x, tiles_m * tiles_n);
    if (t < 0) return;
    int tm;
    tile_at(t, tiles_m, tiles_n, tm, tn);
    m0 = tm * TS::BM;
    rows = min(p.M - m0, TS::BM);
  }
  const int n0 = tn * COLUMNS;
  MxOperands o;
  o.x = p.xq + m0 * ld;
  o.w = w + n0 * ld;
  o.xs = p.xs + (int64_t)m0 * p.x_pitch;
  o.ws = ws + (int64_t)n0 * p.w_pitch;
  o.rows_x = rows;
  o.rows_w = min(p.N - n0, COLUMNS);
  o.ld = (uint32_t)ld;
  o.x_pitch = p.x_pitch;
  o.w_pitch = p.w_pitch;
  o.up = (uint32_t)(p.N * ld);
  o.up_scale = (uint32_t)((int64_t)p.N * p.w_pitch);
  const int blocks = p.K / kMxBlock;
  o.steps = (blocks + 7) / 8;
  o.last_chunks = blocks - (o.steps - 1) * 8;
  MxTile<TS, GATED> tile;
  tile.init(o);
  v16f acc[TS::FN][TS::FM];
  tile.run(lds, acc);
  store_tile<TS, GATED>(p, acc, m0, rows, n0, 0);
}

// Rows of scales of `from` bytes -> rows of `to` bytes (a multiple of 16), filled up with 127 (1.0).
__global__ __launch_bounds__(256) void pad_scales_kernel(const uint8_t* __restrict__ src, uint8_t* __restrict__ dst, int64_t pieces, int from, int to) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;   // 16 bytes of dst
  if (at >= pieces) return;
  const int per_row = to / 16;
  const int64_t row = at / per_row;
  const int col = (int)(at - row * per_row) * 16;
  const uint8_t* in = src + row * from + col;
  uint32_t w[4];
  if (col + 16 <= from) {
    __builtin_memcpy(w, in, 16);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = 0x7F7F7F7Fu;
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (col + 4 * i + b < from) w[i] = (w[i] & ~(0xFFu << (8 * b))) | ((uint32_t)in[4 * i + b] << (8 * b));
    }
  }
  reinterpret_cast<uint4*>(dst)[at] = make_uint4(w[0], w[1], w[2], w[3]);
}

hipError_t pad_scales(const uint8_t* src, uint8_t* dst, int64_t rows, int from, int to, hipStream_t s) {
  const int64_t pieces = rows * (to / 16);
  pad_scales_kernel<<<(unsigned)((pieces + 255) / 256), 256, 0, s>>>(src, dst, pieces, from, to);
  return hipGetLastError();
}

template <typename TS, bool GATED, bool GROUPS>
hipError_t launch(const MxProblem& p, hipStream_t s) {
  const int64_t tiles_n = (p.N + (GATED ? TS::BN / 2 : TS::BN) - 1) / (GATED ? TS::BN / 2 : TS::BN);
  // (groups: as many row tiles as the sizes could make)
  const int64_t tiles_m = GROUPS ? (int64_t)p.M / TS::BM + (p.G < p.M ? p.G : p.M) : (p.M + TS::BM - 1) / TS::BM;
  const int64_t grid = (tiles_m * tiles_n + kXcds - 1) / kXcds * kXcds;
  if (grid * TS::NTHREADS >= (int64_t(1) << 32)) return hipErrorInvalidValue;
  mx_kernel<TS, GATED, GROUPS><<<(unsigned)grid, TS::NTHREADS, 0, s>>>(p, (int)tiles_m, (int)tiles_n);
  return hipGetLastError();
}

template <typename TS>
hipError_t launch(const MxProblem& p, hipStream_t s) {
  if (p.m_sizes != nullptr) return p.gated ? launch<TS, true, true>(p, s) : launch<TS, false, true>(p, s);
  return p.gated ? launch<TS, true, false>(p, s) : launch<TS, false, false>(p, s);
}

int64_t padded_pitch(int64_t K) { return (K + 511) / 512 * 16; }

}  // namespace

size_t mx_workspace_bytes(int64_t M, int64_t N, int64_t K, int gated, int G, bool grouped, bool scales_aligned) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  if (K % 512 == 0 && scales_aligned) return 0;
  return (size_t)((M + N * (gated ? 2 : 1) * (grouped ? G : 1)) * padded_pitch(K));
}

hipError_t launch_mx_mm(MxProblem p, void* workspace, bool scales_aligned, hipStream_t s) {
  const int from = p.K / kMxBlock;
  p.x_pitch = p.w_pitch = from;
  if (p.K % 512 != 0 || !scales_aligned) {   // rows of scales that the 16-byte loads of two steps cannot fetch
    const int to = (int)padded_pitch(p.K);
    const int64_t rows_w = (int64_t)p.N * (p.gated ? 2 : 1) * (p.m_sizes != nullptr ? p.G : 1);
    uint8_t *xs = static_cast<uint8_t*>(workspace), *ws = xs + (int64_t)p.M * to;
    if (const hipError_t e = pad_scales(p.xs, xs, p.M, from, to, s); e != hipSuccess) return e;
    if (const hipError_t e = pad_scales(p.ws, ws, rows_w, from, to, s); e != hipSuccess) return e;
    p.xs = xs;
    p.ws = ws;
    p.x_pitch = p.w_pitch = to;
  }
  if (p.M <= 64) return launch<MxShape<64, 128, 2, 2, 4>>(p, s);
  return launch<MxShape<256, 256, 2, 2, 2>>(p, s);
}

}  // namespace mslk_amd
