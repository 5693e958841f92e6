// New keys and values of packed tokens -> paged cache, queries and keys rotated by their positions on the way.
//
// Row (token, head) of the fused projection is read once and written once: queries to q_out, keys and values to the slot
// that the page table gives their position.  Channel pairs (a, b) of the rotated part become (a cos - b sin, b cos + a sin) in
// 32 bits, rounded once; with e4m3 caches a row's codes are x * (448 / amax) and its scale amax / 448, both from the unrounded
// row.
//
// A team of eight lanes holds a row in registers, two vectors of VEC channels per lane and unit: the two partners of VEC
// rotations (half of the rotated part apart, or neighbours with `interleaved`), or the next 2 VEC unrotated channels.
#include "attention.h"
#include "rows.h"

namespace mslk_amd {
namespace {

constexpr int kTeam = 8, kThreads = 256, kRowsPerBlock = kThreads / kTeam;

// VEC consecutive 16-bit channels.
template <bool F16, int VEC>
MSLK_AMD_DEVINL void load_vec(const uint16_t* src, float* x) {
  using E = Elem<F16>;
  if constexpr (VEC == 1) {
    x[0] = E::lo(*src);
  } else {
    typedef uint32_t words __attribute__((ext_vector_type(VEC / 2)));
    uint32_t w[VEC / 2];
    if constexpr (VEC == 2) w[0] = *reinterpret_cast<const uint32_t*>(src);
    else {
      const words v = *reinterpret_cast<const words*>(src);
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) w[i] = v[i];
    }
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      x[2 * i] = E::lo(w[i]);
      x[2 * i + 1] = E::hi(w[i]);
    }
  }
}
template <bool F16, int VEC>
MSLK_AMD_DEVINL void store_vec(uint16_t* dst, const float* x) {
  using E = Elem<F16>;
  if constexpr (VEC == 1) {
    *dst = (uint16_t)E::pack(x[0], 0.f);
  } else {
    uint32_t w[VEC / 2];
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) w[i] = E::pack(x[2 * i], x[2 * i + 1]);
    if constexpr (VEC == 2) *reinterpret_cast<uint32_t*>(dst) = w[0];
    else if constexpr (VEC == 4) *reinterpret_cast<v2u*>(dst) = v2u{w[0], w[1]};
    else *reinterpret_cast<v4u*>(dst) = v4u{w[0], w[1], w[2], w[3]};
  }
}
template <int VEC>
MSLK_AMD_DEVINL void store_codes(uint8_t* dst, const float* x, float inv) {
  if constexpr (VEC == 1) {
    *dst = (uint8_t)cvt_pk_e4m3fn(__fmul_rn(x[0], inv), 0.f);
  } else {
    uint32_t h[VEC / 2];
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) h[i] = cvt_pk_e4m3fn(__fmul_rn(x[2 * i], inv), __fmul_rn(x[2 * i + 1], inv));
    if constexpr (VEC == 2) *reinterpret_cast<uint16_t*>(dst) = (uint16_t)h[0];
    else if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(dst) = h[0] | (h[1] << 16);
    else *reinterpret_cast<v2u*>(dst) = v2u{h[0] | (h[1] << 16), h[2] | (h[3] << 16)};
  }
}

// Sequence of a token: the last one that starts at or in front of it and is not empty; -1 for tokens of no sequence.
MSLK_AMD_DEVINL int sequence_of(const int32_t* cu, int sequences, int64_t token) {
  int lo = 0, hi = sequences;   // first sequence that ends behind the token
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (cu[mid + 1] > token) hi = mid;
    else lo = mid + 1;
  }
  return lo < sequences && cu[lo] <= token ? lo : -1;
}

template <bool F16, bool FP8, bool INTERLEAVED, int VEC>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs p, Divider heads, int64_t rows) {
  constexpr int kUnits = kMaxHeadDim / (2 * VEC * kTeam);   // per lane
  const int64_t row = row_block() * kRowsPerBlock + threadIdx.x / kTeam;
  if (row >= rows) return;
  const int lane = threadIdx.x % kTeam;
  const int64_t token = heads.magic == 0 ? row : row < (int64_t(1) << 31) ? (int64_t)divide((uint32_t)row, heads) : row / heads.d;
  const int h = (int)(row - token * heads.d);
  const bool is_q = h < p.Hq, is_v = h >= p.Hq + p.Hkv;
  const int kv_head = is_q ? 0 : is_v ? h - p.Hq - p.Hkv : h - p.Hq;
  const uint16_t* src = is_q   ? p.q.data + token * p.q.token_stride + h * p.q.head_stride
                        : is_v ? p.v.data + token * p.v.token_stride + kv_head * p.v.head_stride
                               : p.k.data + token * p.k.token_stride + kv_head * p.k.head_stride;

  // the token's place
  int64_t position = -1;
  const int seq = p.cu_seqlens == nullptr ? (token < p.sequences ? (int)token : -1) : sequence_of(p.cu_seqlens, p.sequences, token);
  if (seq >= 0) position = (int64_t)p.cache.lens[seq] - (p.cu_seqlens == nullptr ? 1 : p.cu_seqlens[seq + 1] - token);
  const bool padding = position < 0;
  bool placed = !padding && (p.rotary == nullptr || position < p.rotary_positions);
  int64_t page = 0;
  int slot = 0;
  if (placed) {
    const int index = (int)divide((uint32_t)position, p.cache.page_size);
    slot = (int)position - index * (int)p.cache.page_size.d;
    placed = index < p.cache.table_width;
    if (placed) {
      page = p.cache.table[seq * p.cache.table_stride + index];
      placed = page >= 0 && page < p.cache.pages;
    }
  }
  if (!placed && !is_q) return;

  const int turned = is_v || p.rotary == nullptr ? 0 : p.rotary_dim;   // rotated channels
  const int half = turned / 2;
  const int turning = half / VEC;                                        // units that are rotated
  const int units = turning + (p.D - turned + 2 * VEC - 1) / (2 * VEC);
  float x[kUnits][2][VEC];
  int at[kUnits][2];   // first channels of a unit's vectors, D where there is none
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int u = lane + i * kTeam;
    at[i][0] = at[i][1] = p.D;
    if (u < units) {
      if (u >= turning) {
        at[i][0] = turned + (u - turning) * 2 * VEC;
        at[i][1] = at[i][0] + VEC;
      } else if (INTERLEAVED) {
        at[i][0] = u * 2 * VEC;
        at[i][1] = at[i][0] + VEC;
      } else {
        at[i][0] = u * VEC;
        at[i][1] = at[i][0] + half;
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (at[i][j] < p.D) load_vec<F16, VEC>(src + at[i][j], x[i][j]);
  }
  if (placed && turned != 0) {
    const float* cosines = p.rotary + position * p.rotary_dim;
    const float* sines = cosines + half;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      const int u = lane + i * kTeam;
      if (u >= turning) continue;
      if constexpr (!INTERLEAVED) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float cs = cosines[u * VEC + e], sn = sines[u * VEC + e], a = x[i][0][e], b = x[i][1][e];
          x[i][0][e] = __fsub_rn(__fmul_rn(a, cs), __fmul_rn(b, sn));
          x[i][1][e] = __fadd_rn(__fmul_rn(b, cs), __fmul_rn(a, sn));
        }
      } else {
        float flat[2 * VEC];
#pragma unroll
        for (int e = 0; e < 2 * VEC; ++e) flat[e] = x[i][e / VEC][e % VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float cs = cosines[u * VEC + e], sn = sines[u * VEC + e], a = flat[2 * e], b = flat[2 * e + 1];
          flat[2 * e] = __fsub_rn(__fmul_rn(a, cs), __fmul_rn(b, sn));
          flat[2 * e + 1] = __fadd_rn(__fmul_rn(b, cs), __fmul_rn(a, sn));
        }
#pragma unroll
        for (int e = 0; e < 2 * VEC; ++e) x[i][e / VEC][e % VEC] = flat[e];
      }
    }
  }

  if (is_q) {
    uint16_t* dst = p.q_out + (token * p.Hq + h) * p.D;
    const float other = padding ? 0.f : __builtin_nanf("");
#pragma unroll
    for (int i = 0; i < kUnits; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (at[i][j] >= p.D) continue;
        if (!placed)
#pragma unroll
          for (int e = 0; e < VEC; ++e) x[i][j][e] = other;
        store_vec<F16, VEC>(dst + at[i][j], x[i][j]);
      }
    return;
  }
  const int64_t* stride = is_v ? p.cache.v_stride : p.cache.k_stride;
  const int64_t to = page * stride[0] + slot * stride[1] + kv_head * stride[2];
  if constexpr (!FP8) {
    uint16_t* dst = (uint16_t*)(is_v ? p.cache.v : p.cache.k) + to;
#pragma unroll
    for (int i = 0; i < kUnits; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (at[i][j] < p.D) store_vec<F16, VEC>(dst + at[i][j], x[i][j]);
  } else {
    uint32_t top = 0;   // magnitudes compare as integers, NaN above infinity
#pragma unroll
    for (int i = 0; i < kUnits; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (at[i][j] < p.D)
#pragma unroll
          for (int e = 0; e < VEC; ++e) top = max(top, __float_as_uint(x[i][j][e]) & 0x7FFFFFFFu);
    const float seen = __uint_as_float(team_max<kTeam>(top, nullptr)), amax = seen < 1e-12f ? 1e-12f : seen;
    const float inv = 448.0f / amax;
    uint8_t* dst = (uint8_t*)(is_v ? p.cache.v : p.cache.k) + to;
#pragma unroll
    for (int i = 0; i < kUnits; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (at[i][j] < p.D) store_codes<VEC>(dst + at[i][j], x[i][j], inv);
    if (lane == 0) {
      const int64_t* ss = is_v ? p.cache.v_scale_stride : p.cache.k_scale_stride;
      (is_v ? p.cache.v_scale : p.cache.k_scale)[page * ss[0] + slot * ss[1] + kv_head * ss[2]] = amax / 448.0f;
    }
  }
}

template <bool F16, bool FP8, bool INTERLEAVED>
hipError_t pick(const AppendArgs& p, hipStream_t s) {
  const int64_t rows = p.tokens * (p.Hq + 2 * p.Hkv);
  const int64_t blocks = (rows + kRowsPerBlock - 1) / kRowsPerBlock;
  const Divider heads = divider((uint32_t)(p.Hq + 2 * p.Hkv));
  // the widest vectors that fit between the partners of a rotation
  const int fit = p.rotary == nullptr ? 8 : p.rotary_dim / 2;
#define MSLK_AMD_APPEND(VEC) hipLaunchKernelGGL((append_kernel<F16, FP8, INTERLEAVED, VEC>), row_grid(blocks), dim3(kThreads), 0, s, p, heads, rows)
  if (fit % 8 == 0) MSLK_AMD_APPEND(8);
  else if (fit % 4 == 0) MSLK_AMD_APPEND(4);
  else if (fit % 2 == 0) MSLK_AMD_APPEND(2);
  else MSLK_AMD_APPEND(1);
#undef MSLK_AMD_APPEND
  return hipGetLastError();
}

}  // namespace

hipError_t launch_append_kv(const AppendArgs& p, hipStream_t s) {
  if (p.dtype == 1) {
    if (p.fp8) return p.interleaved ? pick<true, true, true>(p, s) : pick<true, true, false>(p, s);
    return p.interleaved ? pick<true, false, true>(p, s) : pick<true, false, false>(p, s);
  }
  if (p.fp8) return p.interleaved ? pick<false, true, true>(p, s) : pick<false, true, false>(p, s);
  return p.interleaved ? pick<false, false, true>(p, s) : pick<false, false, false>(p, s);
}

}  // namespace mslk_amd
