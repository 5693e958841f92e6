// Device code that the MXFP4 products share: the gated activation, bias, and which tile a workgroup makes.
#pragma once
#include "common.h"
#include "mx.h"

namespace mslk_amd {
namespace {

constexpr int kXcds = 8;
constexpr int kPanel = 4;   // row tiles that share the weights of a panel in an XCD's L2

// y = silu(gate) * up in fp32, silu(gate) = gate / (1 + exp(-gate)).  exp(-gate) is off by |gate| 2^-24 of itself (its argument times log2(e), rounded) and
// about two units, the reciprocal by one: far below the rounding to 16 bits that follows, as |gate| is below 2^7 here.
// Below -87 the reciprocal is no normal number any more, and from -88.7 on exp(-gate) is infinite, but up may bring the product back into range (gate -90,
// up 1e30: -7e-8).  There silu(gate) = gate exp(gate) to the last bit; exp(gate) = 2^n 2^f, |f| <= 1/2, and 2^n is multiplied to up first.
// FAR: some gate may be that far.  Callers look at all gates of a lane (far_gates()) and make their values again if one of the wave's is.  That look is what
// it costs otherwise: 2047 x (2 x 10000) x 4128 takes 100.5 us in the kernel instead of 99.2, 128 experts of 2 x 768 x 2048 93 instead of 92.
template <bool FAR>
MSLK_AMD_DEVINL float gated_value(float gate, float up) {
  const float near = gate * __builtin_amdgcn_rcpf(1.f + __expf(-gate)) * up;
  if constexpr (!FAR) return near;
  constexpr float kLog2e = 1.44269504088896340736f;
  const float x = fmaxf(gate, -1000.f), n = rintf(x * kLog2e);   // (what is below -1000 ends at 0 all the same; -infinity times that is NaN)
  return gate < -87.f ? gate * __builtin_amdgcn_exp2f(fmaf(x, kLog2e, -n)) * ldexpf(up, (int)n) : near;
}
// The largest bits of gates seen: those of -87 are below those of every smaller number.
MSLK_AMD_DEVINL uint32_t farther(uint32_t most, float gate) { return max(most, __float_as_uint(gate)); }
MSLK_AMD_DEVINL bool far_gates(uint32_t most) { return __builtin_expect(__any(most > 0xC2AE0000u), 0); }

MSLK_AMD_DEVINL float bias_at(const MxProblem& p, int n) {
  return p.bias_dtype == 1 ? static_cast<const float*>(p.bias)[n] : bf16_bits_to_f32(static_cast<const uint16_t*>(p.bias)[n]);
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
template <int BM>
MSLK_AMD_DEVINL int row_tiles_of(int rows) { return (int)(((uint32_t)rows + (BM - 1)) / BM); }   // (rows may be 2^31 - 1)
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
    r = row_tiles_of<BM>(r);
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
    int last = row_tiles_of<BM>(live) * tiles_n;   // entries up to and with this group's
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
      tile_at(at, row_tiles_of<BM>(size), tiles_n, out.tm, out.tn);
      out.row0 = __builtin_amdgcn_readfirstlane(row0) + out.tm * BM;
      out.rows = min(__builtin_amdgcn_readfirstlane(size) - out.tm * BM, BM);
      return true;
    }
    before += __shfl(last, 63, 64);
    rows_before += __shfl(end, 63, 64);
  }
  return false;
}

}  // namespace
}  // namespace mslk_amd
