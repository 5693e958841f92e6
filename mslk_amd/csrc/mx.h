// Microscaled 4-bit floating point (MXFP4): what its translation units share.
//
// A row of K values is K / 32 blocks.  A block is 32 e2m1 codes (sign, 2 exponent bits, 1 mantissa bit: magnitudes 0, 0.5, 1, 1.5, 2,
// 3, 4, 6), two to a byte, the earlier value in the low half, and one scale byte s that stands for 2^(s - 127); 255 is NaN.  Codes
// [rows, K / 2] and scales [rows, K / 32], both row-major: the layouts of the OCP microscaling specification.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace mslk_amd {

constexpr int kMxBlock = 32;

// a [rows, K] of dtype 0 bf16, 1 fp16, 2 fp32, row stride in elements; K % 32 == 0.
hipError_t launch_quantize_mxfp4(const void* a, int dtype, int64_t rows, int64_t K, int64_t row_stride, void* codes, void* scales,
                                 hipStream_t s);
// out [rows, K] of the same dtype codes, everything contiguous.
hipError_t launch_dequantize_mxfp4(const void* codes, const void* scales, int64_t rows, int64_t K, void* out, int dtype, hipStream_t s);

// Where scales lie: those of row r, blocks 16 p ... 16 p + 15 are the 16 bytes at data + (r / 64) * block + (r % 64) * row + p * pair_stride,
// all multiples of 16 (for the small tiles, of 4).  A tensor's own: row = K / 32, block = 64 row, pair_stride = 16.  Arranged: [rows / 64][pairs][64][16],
// blocks beyond K 0.
struct MxScales {
  const uint8_t* data;
  int64_t block;
  int row, pair_stride;
};

// Y[m, n] = sum_k X[m, k] W[n, k] + bias[n]; gated: W has 2 N rows, gate rows first, and Y = silu(X Wg^T) * (X Wu^T).
// Groups (m_sizes != nullptr): W [G, rows of W, K]; the rows of X are those of group 0, of group 1, ...
struct MxProblem {
  const uint8_t *xq, *wq;          // codes, rows of K / 2 bytes
  MxScales xs, ws;
  const void* bias;
  uint16_t* y;
  const int64_t* m_sizes;
  const void* row_tiles;           // list of the groups' row tiles in device memory, nullptr without
  int M, N, K;                     // N: columns of Y
  int G;
  int bias_dtype;                  // 0 none, 1 fp32, 2 bf16
  int out_f16;
  int gated;
};
// Bytes of workspace that launch_mx_mm() wants for this problem (scales_aligned: both tensors of scales begin on 16 bytes).
size_t mx_workspace_bytes(int64_t M, int64_t N, int64_t K, int gated, int G, bool grouped, bool scales_aligned);
// p.xs.data and p.ws.data: the tensors; the rest of p.xs and p.ws is filled in.
hipError_t launch_mx_stream(const MxProblem& p, hipStream_t s);   // of it, few rows of X (mx_stream.hip): tensors of scales as they are
hipError_t launch_mx_mm(MxProblem p, void* workspace, bool scales_aligned, hipStream_t s);

}  // namespace mslk_amd
