// Products of few rows of X with MXFP4 weights for gfx950 (formats: mx.h), for rows of scales that do not begin on 4 bytes: they go to
// registers from wherever they lie, and no launch arranges them first.  The weights are read once, and they are what counts: 16 x 4096 x 4128 takes
// 6.3 us a call.
//
// A workgroup makes 32 columns (gated: 16, from 16 rows of the gate and their 16 partners) of up to 32 rows of X.  Its waves take K's
// pairs of steps, 512 values, in turn, each with a part of the LDS for itself: no barrier until their sums meet in LDS, and no sums
// go through memory.  A wave asks for the rows of U pairs at once, 256 bytes of four rows per load (the 128-bit DMA load, mx_tile.h),
// waits for them and multiplies.  (Loaded into registers as the instructions want them, 64 bytes of 16 rows at a time, a load takes the
// texture path four times as long: 1 row x 8192 x 8192 10.8 us, 16 rows x 28672 x 4096 19.6.)
// Lane (i = l & 31, h = l >> 5) gives row i's chunk (block) 8 h + j to product j of eight (v_mfma_scale_f32_32x32x64_f8f6f4, W first); its
// scales are eight neighbouring bytes, loaded into registers from wherever they begin.
#include "gemm_tile.h"
#include "kernels.h"
#include "mx_device.h"
#include "rows.h"

namespace mslk_amd {
namespace {

constexpr int kPairBytes = 256;   // of a row

// Chunk c of row r of a fragment lies at c ^ swz(r): the rows that are served together (mx_tile.h) then touch all banks.
MSLK_AMD_DEVINL int pair_swz(int r) { return (r & 3) | ((((r >> 2) ^ (r >> 3)) & 3) << 2); }

// XR rows of X; WAVES waves, U pairs at a time.
template <int XR_, int WAVES_, int U_>
struct StreamShape {
  static constexpr int XR = XR_, WAVES = WAVES_, U = U_;
  static constexpr int W_BYTES = 32 * kPairBytes, X_BYTES = XR * kPairBytes;
  static constexpr int WAVE_BYTES = U * (W_BYTES + X_BYTES);
  static constexpr int SUM_BYTES = WAVES * 4096;                  // behind the products, in the same place
  static constexpr int LDS_BYTES = WAVES * WAVE_BYTES > SUM_BYTES ? WAVES * WAVE_BYTES : SUM_BYTES;
  static_assert(XR % 4 == 0 && XR <= 32 && LDS_BYTES <= 160 * 1024, "whole loads, the LDS of a CU");
};

// Scales of this lane's eight chunks, 8 h ... 8 h + 7 of `blocks` (missing ones 0: products of two such blocks vanish).
MSLK_AMD_DEVINL uint2 load_scales8(const uint8_t* s, int blocks) {
  const int h = (threadIdx.x & 63) >> 5;
  uint2 v = make_uint2(0, 0);
  if (blocks >= 16) {
    __builtin_memcpy(&v, s + 8 * h, 8);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (8 * h + j < blocks) (j < 4 ? v.x : v.y) |= (uint32_t)s[8 * h + j] << (8 * (j & 3));
  }
  return v;
}

// Rows m0 ... m0 + rows - 1 (at most XR), columns from n0; w_row: first row of W's group.
template <typename S, bool GATED>
MSLK_AMD_DEVINL void stream_tile(const MxProblem& p, char* lds, int m0, int rows, int64_t w_row, int n0) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 31, h = lane >> 5;
  const int64_t ld = p.K / 2, pitch = p.K / kMxBlock;
  const int blocks = p.K / kMxBlock, pairs = (blocks + 15) >> 4;
  // rows beyond the last one read it again: their sums are not stored
  auto row_of_w = [&](int r) { return w_row + (GATED ? min(n0 + (r & 15), p.N - 1) + (int64_t)(r >> 4) * p.N : min(n0 + r, p.N - 1)); };
  auto row_of_x = [&](int r) { return (int64_t)m0 + min(r, rows - 1); };
  char* const mine = lds + wave * S::WAVE_BYTES;
  const uint8_t *w_at[8], *x_at[S::XR / 4], *w_scale = p.ws.data + row_of_w(i) * pitch, *x_scale = p.xs.data + row_of_x(min(i, S::XR - 1)) * pitch;
#pragma unroll
  for (int q = 0; q < 8; ++q) w_at[q] = p.wq + row_of_w(q * 4 + (lane >> 4)) * ld;
#pragma unroll
  for (int q = 0; q < S::XR / 4; ++q) x_at[q] = p.xq + row_of_x(q * 4 + (lane >> 4)) * ld;
  v16f acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.f;
  for (int first = wave; first < pairs; first += S::U * S::WAVES) {
    uint2 sw[S::U], sx[S::U];
#pragma unroll
    for (int u = 0; u < S::U; ++u) {
      const int pair = min(first + u * S::WAVES, pairs - 1), there = blocks - pair * 16;   // (behind the last pair: it once more, not multiplied)
      const int64_t at = (int64_t)pair * kPairBytes;
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const int c = (lane & 15) ^ pair_swz(q * 4 + (lane >> 4));
        __builtin_amdgcn_global_load_lds((gbl_ptr_t)(w_at[q] + at + (c < there ? c * 16 : 0)), (lds_ptr_t)(mine + u * S::W_BYTES + q * 1024), 16, 0, 2);
      }
      sw[u] = load_scales8(w_scale + pair * 16, there);
    }
#pragma unroll
    for (int u = 0; u < S::U; ++u) {
      const int pair = min(first + u * S::WAVES, pairs - 1), there = blocks - pair * 16;
      const int64_t at = (int64_t)pair * kPairBytes;
#pragma unroll
      for (int q = 0; q < S::XR / 4; ++q) {
        const int c = (lane & 15) ^ pair_swz(q * 4 + (lane >> 4));
        __builtin_amdgcn_global_load_lds((gbl_ptr_t)(x_at[q] + at + (c < there ? c * 16 : 0)), (lds_ptr_t)(mine + S::U * S::W_BYTES + u * S::X_BYTES + q * 1024), 16, 0, 0);
      }
      sx[u] = load_scales8(x_scale + pair * 16, there);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): this wave's rows are in its part of the LDS
#pragma unroll
    for (int u = 0; u < S::U; ++u) {
      if (first + u * S::WAVES < pairs) {
        const char *wb = mine + u * S::W_BYTES, *xb = mine + S::U * S::W_BYTES + u * S::X_BYTES;
        auto product = [&](auto jj) {
          constexpr int J = decltype(jj)::value;
          auto chunk = [&](const char* b, int r) { return *reinterpret_cast<const v4i*>(b + r * kPairBytes + (((8 * h + J) ^ pair_swz(r)) << 4)); };
          auto operand = [](v4i a) { return v8i{a[0], a[1], a[2], a[3], 0, 0, 0, 0}; };
          const v4i wf = chunk(wb, i), xf = chunk(xb, min(i, S::XR - 1));
          acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(wf), operand(xf), acc, 4, 4, J & 3, (int)(J < 4 ? sw[u].x : sw[u].y), J & 3,
                                                                (int)(J < 4 ? sx[u].x : sx[u].y));
        };
        product(Int<0>{}); product(Int<1>{}); product(Int<2>{}); product(Int<3>{});
        product(Int<4>{}); product(Int<5>{}); product(Int<6>{}); product(Int<7>{});
      }
    }
  }
  // Row m = i of a wave's sums: 32 columns, in pieces of four (q, h) at piece ^ (i & 7).
  __syncthreads();
  char* const sums = lds + wave * 4096;
#pragma unroll
  for (int q = 0; q < 4; ++q)
    *reinterpret_cast<float4*>(sums + i * 128 + (((2 * q + h) ^ (i & 7)) << 4)) = make_float4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
  __syncthreads();
  auto total = [&](int m, int piece) {   // columns 4 piece ... of row m
    const char* at = lds + m * 128 + ((piece ^ (m & 7)) << 4);
    v4f s = *reinterpret_cast<const v4f*>(at);
#pragma unroll
    for (int k = 1; k < S::WAVES; ++k) s += *reinterpret_cast<const v4f*>(at + k * 4096);
    return s;
  };
  constexpr int PIECES = GATED ? 4 : 8;
  for (int t = threadIdx.x; t < rows * PIECES; t += S::WAVES * 64) {
    const int m = t / PIECES, piece = t % PIECES, n = n0 + 4 * piece;
    if (n >= p.N) continue;
    v4f v = total(m, piece);
    if constexpr (GATED) {
      const v4f gate = v, up = total(m, piece + 4);
      uint32_t gates = 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        gates = farther(gates, gate[r]);
        v[r] = gated_value<false>(gate[r], up[r]);
      }
      if (far_gates(gates)) {
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = gated_value<true>(gate[r], up[r]);
      }
    } else if (p.bias_dtype != 0) {
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] += bias_at(p, min(n + r, p.N - 1));
    }
    uint16_t* dst = p.y + (int64_t)(m0 + m) * p.N + n;
    uint32_t o[2];
    if (p.out_f16) {
      o[0] = pack_f16x2(v[0], v[1]);
      o[1] = pack_f16x2(v[2], v[3]);
    } else {
      o[0] = pack_bf16x2(v[0], v[1]);
      o[1] = pack_bf16x2(v[2], v[3]);
    }
    if ((p.N & 3) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 7) == 0) {
      *reinterpret_cast<uint2*>(dst) = make_uint2(o[0], o[1]);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n + r < p.N) dst[r] = (uint16_t)(o[r >> 1] >> ((r & 1) * 16));
    }
  }
}

template <typename S, bool GATED>
__global__ __launch_bounds__(S::WAVES * 64) void mx_stream_kernel(MxProblem p) {
  __shared__ __attribute__((aligned(1024))) char lds[S::LDS_BYTES];
  stream_tile<S, GATED>(p, lds, 0, p.M, 0, blockIdx.x * (GATED ? 16 : 32));
}

template <typename S>
hipError_t launch(const MxProblem& p, unsigned grid, hipStream_t s) {
  if (dispatch_probe_record("mx_stream<%d,waves=%d> workgroups=%u", S::XR, S::WAVES, grid)) return hipSuccess;
  if (p.gated) mx_stream_kernel<S, true><<<grid, S::WAVES * 64, 0, s>>>(p);
  else mx_stream_kernel<S, false><<<grid, S::WAVES * 64, 0, s>>>(p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_mx_stream(const MxProblem& p, hipStream_t s) {
  const int columns = p.gated ? 16 : 32;
  const int64_t grid = ((int64_t)p.N + columns - 1) / columns;
  if (grid * 512 >= (int64_t(1) << 32)) return hipErrorInvalidValue;
  if (p.M <= 8) return launch<StreamShape<8, 8, 2>>(p, (unsigned)grid, s);
  if (p.M <= 16) return launch<StreamShape<16, 8, 1>>(p, (unsigned)grid, s);
  return launch<StreamShape<32, 8, 1>>(p, (unsigned)grid, s);
}

}  // namespace mslk_amd
