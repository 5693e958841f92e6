// New keys and values of packed tokens -> paged cache, queries and keys rotated by their positions on the way.
//
// Row (token, head) of the fused projection is read once and written once: queries to q_out, keys and values to the slot
// that the page table gives their position.  Channel pairs (a, b) of the rotated part become (a cos - b sin, b cos + a sin) in
// 32 bits, rounded once; with e4m3 caches a row's codes are x * (448 / amax) and its scale amax / 448, both from the unrounded
// row.
//
// A team of eight lanes holds a row in registers, two vectors of VEC channels per lane and unit: the two partners of VEC
// rotations (half of the rotated part apart, or neighbours with `interleaved`), or the next 2 VEC unrotated channels.  A workgroup
// takes 32 consecutive rows: it asks for them and looks up the places of their tokens meanwhile, one lane a token (the sequence,
// its length, the page: loads that wait for one another).
//
// Bound: the memory where there are many tokens: 8191 tokens, 64 heads of 128 and 8 of keys and values, 340 MB in 70.5 us, 4.8 TB/s (a
// copy of that size moves 5.1).  Asked for behind its place, a row waited for that whole chain: 97 us.  Few tokens are bound by the
// chain and the launch: 3.2 us for one, 4.4 us for 64 in e4m3.  Four rows to a team, instead of one, left 73.0 us in 16 bits and took 71.1
// instead of 76.6 in e4m3, but 6.9 instead of 3.8 us at 64 tokens.
#include "attention.h"
#include "rows.h"

namespace mslk_amd {
namespace {

constexpr int kTeam = 8, kThreads = 256, kBlockRows = kThreads / kTeam;
constexpr int kBlockTokens = kBlockRows / 3 + 2;   // a token has at least three rows

// VEC consecutive 16-bit channels.
template <int VEC> struct Raw {
  static constexpr int kWords = VEC == 1 ? 1 : VEC / 2;
  uint32_t w[kWords];
};
template <int VEC>
MSLK_AMD_DEVINL Raw<VEC> load_raw(const uint16_t* src) {
  Raw<VEC> r;
  if constexpr (VEC == 1) r.w[0] = *src;
  else if constexpr (VEC == 2) r.w[0] = *reinterpret_cast<const uint32_t*>(src);
  else {
    typedef uint32_t words __attribute__((ext_vector_type(VEC / 2)));
    const words v = __builtin_nontemporal_load(reinterpret_cast<const words*>(src));
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) r.w[i] = v[i];
  }
  return r;
}
template <bool F16, int VEC>
MSLK_AMD_DEVINL void to_floats(const Raw<VEC>& r, float* x) {
  using E = Elem<F16>;
#pragma unroll
  for (int i = 0; i < Raw<VEC>::kWords; ++i) {
    x[2 * i] = E::lo(r.w[i]);
    if constexpr (VEC > 1) x[2 * i + 1] = E::hi(r.w[i]);
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

// Where a token goes.
struct Place {
  int position, page, slot;
  int state;   // 0: stored, 1: padding, 2: has no place
};
MSLK_AMD_DEVINL Place place_of(const AppendArgs& p, int64_t token) {
  Place r{0, 0, 0, 1};
  const int seq = p.cu_seqlens == nullptr ? (token < p.sequences ? (int)token : -1) : sequence_of(p.cu_seqlens, p.sequences, token);
  if (seq < 0) return r;
  const int64_t position = (int64_t)p.cache.lens[seq] - (p.cu_seqlens == nullptr ? 1 : p.cu_seqlens[seq + 1] - token);
  if (position < 0) return r;
  r.state = 2;
  if (p.rotary != nullptr && position >= p.rotary_positions) return r;
  r.position = (int)position;
  const int index = (int)divide((uint32_t)position, p.cache.page_size);
  r.slot = r.position - index * (int)p.cache.page_size.d;
  if (index >= p.cache.table_width) return r;
  r.page = p.cache.table[seq * p.cache.table_stride + index];
  if (r.page >= 0 && r.page < p.cache.pages) r.state = 0;
  return r;
}

template <bool F16, bool FP8, bool INTERLEAVED, int VEC>
__global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs p, Divider heads, int64_t rows) {
  constexpr int kUnits = kMaxHeadDim / (2 * VEC * kTeam);   // per lane
  __shared__ Place places[kBlockTokens];
  const int64_t row0 = row_block() * kBlockRows;
  if (row0 >= rows) return;
  const int64_t token0 = row0 < (int64_t(1) << 31) ? (int64_t)divide((uint32_t)row0, heads) : row0 / heads.d;
  const int lane = threadIdx.x % kTeam, team = threadIdx.x / kTeam;
  const int lead = (int)(row0 - token0 * heads.d);   // rows of the first token that are in front of the block
  const int count = (int)min(rows - row0, (int64_t)kBlockRows);

  const int r = lead + min(team, count - 1);   // (teams behind the last row repeat it and store nothing)
  const int in_block = (int)divide((uint32_t)r, heads), h = r - in_block * (int)heads.d;
  const int64_t token = token0 + in_block;
  const bool is_q = h < p.Hq, is_v = h >= p.Hq + p.Hkv;
  const int kv_head = is_q ? 0 : is_v ? h - p.Hq - p.Hkv : h - p.Hq;
  const uint16_t* src = is_q   ? p.q.data + token * p.q.token_stride + h * p.q.head_stride
                        : is_v ? p.v.data + token * p.v.token_stride + kv_head * p.v.head_stride
                               : p.k.data + token * p.k.token_stride + kv_head * p.k.head_stride;
  const int turned = is_v || p.rotary == nullptr ? 0 : p.rotary_dim, half = turned / 2, turning = half / VEC;   // rotated channels, units
  const int units = turning + (p.D - turned + 2 * VEC - 1) / (2 * VEC);
  int at[kUnits][2];   // first channels of a unit's two vectors, D where there is none
  Raw<VEC> raw[kUnits][2];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int u = lane + i * kTeam;
    at[i][0] = at[i][1] = p.D;
    if (u < units) {
      at[i][0] = u >= turning ? turned + (u - turning) * 2 * VEC : INTERLEAVED ? u * 2 * VEC : u * VEC;
      at[i][1] = u >= turning || INTERLEAVED ? at[i][0] + VEC : at[i][0] + half;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (at[i][j] < p.D) raw[i][j] = load_raw<VEC>(src + at[i][j]);
  }
  if ((int)threadIdx.x <= (int)divide((uint32_t)(lead + count - 1), heads)) places[threadIdx.x] = place_of(p, token0 + threadIdx.x);
  __syncthreads();

  if (team >= count) return;
  const Place place = places[in_block];
  const bool placed = place.state == 0;
  if (!placed && !is_q) return;
  float x[kUnits][2][VEC];
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const int u = lane + i * kTeam;
#pragma unroll
    for (int j = 0; j < 2; ++j) to_floats<F16, VEC>(raw[i][j], x[i][j]);
    if (!placed || u >= turning) continue;
    const float* cosines = p.rotary + (int64_t)place.position * p.rotary_dim + u * VEC;
    const float* sines = cosines + half;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      // partners: element e of the two vectors, or neighbours in the 2 VEC channels that they make up
      float& a = INTERLEAVED ? x[i][2 * e / VEC][2 * e % VEC] : x[i][0][e];
      float& b = INTERLEAVED ? x[i][(2 * e + 1) / VEC][(2 * e + 1) % VEC] : x[i][1][e];
      const float cs = cosines[e], sn = sines[e], a0 = a, b0 = b;
      a = __fsub_rn(__fmul_rn(a0, cs), __fmul_rn(b0, sn));
      b = __fadd_rn(__fmul_rn(b0, cs), __fmul_rn(a0, sn));
    }
  }

  if (is_q) {
    uint16_t* dst = p.q_out + (token * p.Hq + h) * p.D;
    const float other = place.state == 1 ? 0.f : __builtin_nanf("");
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
  const int64_t to = place.page * stride[0] + place.slot * stride[1] + kv_head * stride[2];
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
      (is_v ? p.cache.v_scale : p.cache.k_scale)[place.page * ss[0] + place.slot * ss[1] + kv_head * ss[2]] = amax / 448.0f;
    }
  }
}

template <bool F16, bool FP8, bool INTERLEAVED>
hipError_t pick(const AppendArgs& p, hipStream_t s) {
  const int64_t rows = p.tokens * (p.Hq + 2 * p.Hkv), blocks = (rows + kBlockRows - 1) / kBlockRows;
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
