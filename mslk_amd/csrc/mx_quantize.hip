// Rows of values to blocks of 32 e2m1 codes with a shared power of two, and back (formats: mx.h).
//
// Of a block with the largest magnitude a: scale 2^E, E = max(floor(log2 a) - 2, -127), so that a lands in [4, 8), and
// code = e2m1(v 2^-E), to nearest, of two as near the one with mantissa bit 0, magnitudes above 6 to 6.  Multiplying by a power of
// two is exact, so the conversion is the only rounding.  A block with a NaN or an infinity gets scale 255 and codes 0: NaN.
//
// Both are bound by memory.  A lane holds 8 values (16 bytes of 16-bit ones), so that a wave reads and writes whole lines; four
// neighbouring lanes are a block and find its maximum by data-parallel moves, on the bits, where NaN > infinity > numbers.
// Values of half of the Infinity Cache and more go past the caches (STREAM), there and back: 8192 x 28672 bf16 values take 177 us in all instead of 224
// (5.3 TB/s of values: the codes stay in the cache between the two), 8192 x 8192 55 instead of 60.  Fewer are left where a reader may find them.
#include <type_traits>

#include "mx.h"
#include "quant_math.h"

namespace mslk_amd {
namespace {

constexpr int kThreads = 256;

// Words: 16 bytes of elements, which begin on any element.
template <int DTYPE> struct Elements {
  typedef uint16_t type;
  typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));
};
template <> struct Elements<2> {
  typedef float type;
  typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(4)));
};

constexpr int64_t kStreamBytes = int64_t(1) << 27;

// 8 consecutive values as fp32.
template <int DTYPE, bool STREAM>
MSLK_AMD_DEVINL void load8(const typename Elements<DTYPE>::type* p, float (&v)[8]) {
  typedef typename Elements<DTYPE>::Words Words;
  auto load4 = [&](int at) {
    const Words* from = reinterpret_cast<const Words*>(p) + at;
    if constexpr (STREAM) return __builtin_nontemporal_load(from);
    else return *from;
  };
  if constexpr (DTYPE == 2) {
    const Words lo = load4(0), hi = load4(1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = __uint_as_float(lo[i]);
      v[4 + i] = __uint_as_float(hi[i]);
    }
  } else {
    const Words w = load4(0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = Traits<DTYPE>::to_f32(w[i] & 0xFFFFu);
      v[2 * i + 1] = Traits<DTYPE>::to_f32(w[i] >> 16);
    }
  }
}

MSLK_AMD_DEVINL uint32_t max_of_4_lanes(uint32_t m) {
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, true));   // lanes 1 0 3 2
  return max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, true));   // lanes 2 3 0 1
}

// U vectors of 8 values per lane, kThreads vectors apart, all loads in front of the arithmetic.  Vector v of the launch is vector
// v % per_row of row v / per_row; FLAT: rows follow one another without a gap.
template <int DTYPE, int U, bool FLAT, bool STREAM>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const typename Elements<DTYPE>::type* __restrict__ a, int64_t row_stride, uint32_t per_row,
                                                            int64_t vectors, uint32_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const int64_t first = (int64_t)blockIdx.x * (kThreads * U) + threadIdx.x;
  float v[U][8];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = first + u * kThreads;
    if (i < vectors) {
      int64_t at = i * 8;
      if constexpr (!FLAT) {
        const uint32_t row = (uint32_t)i / per_row;   // (launches of rows with gaps are cut below 2^32 vectors)
        at = row * row_stride + (int64_t)((uint32_t)i - row * per_row) * 8;
      }
      load8<DTYPE, STREAM>(a + at, v[u]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[u][e] = 0.f;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = first + u * kThreads;
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(v[u][e]) & 0x7FFFFFFFu);
    m = max_of_4_lanes(m);
    const uint32_t field = m >> 23;   // floor(log2 a) + 127, 0 for denormal numbers and 0
    const uint32_t s = field == 255 ? 255u : field > 2 ? field - 2 : 0u;
    const float to_code = __uint_as_float((254u - s) << 23);   // 2^(127 - s)
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[u][0] * to_code, v[u][1] * to_code, 1.f, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[u][2] * to_code, v[u][3] * to_code, 1.f, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[u][4] * to_code, v[u][5] * to_code, 1.f, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[u][6] * to_code, v[u][7] * to_code, 1.f, 3);
    if (s == 255) c = 0;
    if (i < vectors) {
      codes[i] = c;
      if ((threadIdx.x & 3) == 0) scales[i >> 2] = (uint8_t)s;
    }
  }
}

template <int DTYPE, int U, bool STREAM>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t vectors,
                                                              void* __restrict__ out) {
  const int64_t first = (int64_t)blockIdx.x * (kThreads * U) + threadIdx.x;
  uint32_t c[U], s[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = first + u * kThreads;
    c[u] = i < vectors ? codes[i] : 0u;
    s[u] = i < vectors ? scales[i >> 2] : 0u;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = first + u * kThreads;
    if (i >= vectors) break;
    const float scale = __uint_as_float(s[u] == 255 ? 0x7FC00000u : s[u] == 0 ? 0x00400000u : s[u] << 23);   // 2^(s - 127); 2^-127 is denormal
    float v[8];
    auto two = [&](int at, auto pair) {
      v[at] = pair[0] * scale;
      v[at + 1] = pair[1] * scale;
    };
    two(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], 1.f, 0));
    two(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], 1.f, 1));
    two(4, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], 1.f, 2));
    two(6, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], 1.f, 3));
    typedef uint32_t Words __attribute__((ext_vector_type(4)));
    auto store4 = [&](int64_t at, Words w) {
      Words* to = static_cast<Words*>(out) + at;
      if constexpr (STREAM) __builtin_nontemporal_store(w, to);
      else *to = w;
    };
    if constexpr (DTYPE == 2) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        store4(2 * i + h, Words{__float_as_uint(v[4 * h]), __float_as_uint(v[4 * h + 1]), __float_as_uint(v[4 * h + 2]), __float_as_uint(v[4 * h + 3])});
    } else {
      store4(i, Words{pack_out_x2<DTYPE == 1>(v[0], v[1]), pack_out_x2<DTYPE == 1>(v[2], v[3]), pack_out_x2<DTYPE == 1>(v[4], v[5]),
                      pack_out_x2<DTYPE == 1>(v[6], v[7])});
    }
  }
}

// Calls f(first vector, vectors, vectors per lane, whether they are streamed) for launches that HIP takes (fewer than 2^32 work-items): four vectors
// per lane keep enough loads in flight, where that still makes a workgroup for every CU.  bytes: of all values.
template <typename F>
hipError_t in_launches(int64_t vectors, int64_t bytes, F f) {
  constexpr int64_t kMost = int64_t(1) << 31;   // a multiple of all that a launch is divided into
  for (int64_t at = 0; at < vectors; at += kMost) {
    const int64_t n = vectors - at < kMost ? vectors - at : kMost;
    const std::integral_constant<int, 1> one{};
    const std::integral_constant<int, 4> four{};
    if (n <= 4 * 256 * kThreads) f(at, n, one, std::false_type{});
    else if (bytes < kStreamBytes) f(at, n, four, std::false_type{});
    else f(at, n, four, std::true_type{});
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
  }
  return hipSuccess;
}
unsigned blocks(int64_t vectors, int u) { return (unsigned)((vectors + kThreads * u - 1) / (kThreads * u)); }

template <int DTYPE>
hipError_t quantize(const void* a, int64_t rows, int64_t K, int64_t row_stride, uint32_t* codes, uint8_t* scales, hipStream_t s) {
  typedef typename Elements<DTYPE>::type T;
  const T* x = static_cast<const T*>(a);
  const int64_t per_row = K / 8, bytes = rows * K * (int64_t)sizeof(T);
  if (row_stride == K || rows == 1)
    return in_launches(rows * per_row, bytes, [&](int64_t at, int64_t n, auto u, auto stream) {
      quantize_kernel<DTYPE, u, true, stream><<<blocks(n, u), kThreads, 0, s>>>(x + at * 8, 0, 1, n, codes + at, scales + at / 4);
    });
  const int64_t most = (int64_t(1) << 31) / per_row;   // rows of a launch; K < 2^31
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t first = r * per_row;
    const hipError_t e = in_launches((rows - r < most ? rows - r : most) * per_row, bytes, [&](int64_t, int64_t n, auto u, auto stream) {
      quantize_kernel<DTYPE, u, false, stream><<<blocks(n, u), kThreads, 0, s>>>(x + r * row_stride, row_stride, (uint32_t)per_row, n, codes + first, scales + first / 4);
    });
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <int DTYPE>
hipError_t dequantize(const uint32_t* codes, const uint8_t* scales, int64_t vectors, void* out, hipStream_t s) {
  const int64_t each = DTYPE == 2 ? 32 : 16;
  return in_launches(vectors, vectors * each, [&](int64_t at, int64_t n, auto u, auto stream) {
    dequantize_kernel<DTYPE, u, stream><<<blocks(n, u), kThreads, 0, s>>>(codes + at, scales + at / 4, n, static_cast<char*>(out) + at * each);
  });
}

}  // namespace

hipError_t launch_quantize_mxfp4(const void* a, int dtype, int64_t rows, int64_t K, int64_t row_stride, void* codes, void* scales, hipStream_t s) {
  uint32_t* c = static_cast<uint32_t*>(codes);
  uint8_t* o = static_cast<uint8_t*>(scales);
  if (dtype == 0) return quantize<0>(a, rows, K, row_stride, c, o, s);
  if (dtype == 1) return quantize<1>(a, rows, K, row_stride, c, o, s);
  return quantize<2>(a, rows, K, row_stride, c, o, s);
}

hipError_t launch_dequantize_mxfp4(const void* codes, const void* scales, int64_t rows, int64_t K, void* out, int dtype, hipStream_t s) {
  const uint32_t* c = static_cast<const uint32_t*>(codes);
  const uint8_t* o = static_cast<const uint8_t*>(scales);
  const int64_t vectors = rows * (K / 8);
  if (dtype == 0) return dequantize<0>(c, o, vectors, out, s);
  if (dtype == 1) return dequantize<1>(c, o, vectors, out, s);
  return dequantize<2>(c, o, vectors, out, s);
}

}  // namespace mslk_amd
