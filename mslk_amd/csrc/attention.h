// Arguments of the attention kernels and device helpers they share.
#pragma once
#include "common.h"

namespace mslk_amd {

constexpr int kMaxHeadDim = 256;

// Rows of heads: element (token, head, channel) at data[token * token_stride + head * head_stride + channel].
struct HeadRows {
  const uint16_t* data;
  int64_t token_stride, head_stride;
};

// n / d = umulhi(n, magic) >> shift for n < 2^31, d > 1; magic 0: d = 1.
struct Divider {
  uint32_t d, magic, shift;
};
inline Divider divider(uint32_t d) {
  Divider v{d, 0, 0};
  if (d > 1) {   // 2^shift < d <= 2^(shift + 1): magic = ceil(2^(32 + shift) / d) < 2^32, exact for n < 2^31
    while ((uint64_t(2) << v.shift) < d) ++v.shift;
    v.magic = (uint32_t)(((uint64_t(1) << (32 + v.shift)) + d - 1) / d);
  }
  return v;
}
MSLK_AMD_DEVINL uint32_t divide(uint32_t n, const Divider& v) { return v.magic == 0 ? n : __umulhi(n, v.magic) >> v.shift; }

// A paged cache: row (page, slot, head) of the keys at k + page * k_stride[0] + slot * k_stride[1] + head * k_stride[2], and so
// on.  Strides in elements (bytes for e4m3 codes).
struct PagedCache {
  void *k, *v;
  float *k_scale, *v_scale;              // e4m3 only: one scale per row
  int64_t k_stride[3], v_stride[3], k_scale_stride[3], v_scale_stride[3];
  int pages;
  Divider page_size;
  const int32_t* table;                  // [sequences, table_width] page numbers
  int table_width;
  int64_t table_stride;
  const int32_t* lens;                   // [sequences] keys per sequence
};

struct AppendArgs {
  HeadRows q, k, v;
  uint16_t* q_out;                       // [tokens, Hq, D]
  PagedCache cache;
  const int32_t* cu_seqlens;             // nullptr: token i is the one new token of sequence i
  const float* rotary;                   // [positions, rotary_dim]: cosines, then sines; nullptr: no rotation
  int64_t rotary_positions;
  int rotary_dim, interleaved;
  int64_t tokens;
  int sequences, Hq, Hkv, D, dtype, fp8;
};
hipError_t launch_append_kv(const AppendArgs& p, hipStream_t s);

struct DecodeArgs {
  HeadRows q;                            // a token per sequence
  PagedCache cache;
  uint16_t* out;                         // [sequences, Hq, D]
  float* lse;                            // [sequences, Hq]
  float* partial;                        // workspace: the pieces of divided head blocks, ...
  int* ends;                             // ... and the first and last of each
  int sequences, Hq, Hkv, D, dtype, fp8;
  float scale;
};
size_t decode_workspace_bytes(int64_t sequences, int64_t Hq, int64_t Hkv, int64_t D, int64_t longest);
hipError_t launch_attention_decode(const DecodeArgs& p, hipStream_t s);

struct PromptArgs {
  HeadRows q, k, v;
  uint16_t* out;                         // [tokens, Hq, D]
  float* lse;                            // [tokens, Hq]
  const int32_t *cu_q, *cu_k;            // [sequences + 1]
  int64_t tokens, keys;
  int sequences, Hq, Hkv, D, dtype, causal;
  Divider group;                         // heads of queries per head of keys
  float scale;
};
hipError_t launch_attention_prompt(const PromptArgs& p, hipStream_t s);

// ---------------------------------------------------------------------------------------------------------------------
// 16-bit element types: operands of the matrix instructions and the rounding of two sums
// ---------------------------------------------------------------------------------------------------------------------
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

template <bool F16> struct Elem;
template <> struct Elem<false> {
  MSLK_AMD_DEVINL static v4f mfma16(v4i a, v4i b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
  MSLK_AMD_DEVINL static uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
  MSLK_AMD_DEVINL static float lo(uint32_t w) { return __uint_as_float(w << 16); }
  MSLK_AMD_DEVINL static float hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
};
template <> struct Elem<true> {
  MSLK_AMD_DEVINL static v4f mfma16(v4i a, v4i b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
  MSLK_AMD_DEVINL static uint32_t pack(float a, float b) {
    const f32x2_t v = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2_t));
  }
  MSLK_AMD_DEVINL static float lo(uint32_t w) { return (float)__builtin_bit_cast(f16x2_t, w)[0]; }
  MSLK_AMD_DEVINL static float hi(uint32_t w) { return (float)__builtin_bit_cast(f16x2_t, w)[1]; }
};

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
MSLK_AMD_DEVINL float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
MSLK_AMD_DEVINL float log2_fast(float x) { return __builtin_amdgcn_logf(x); }

// Over the lanes of a wave.
MSLK_AMD_DEVINL int wave_sum(int v) {   // in every lane
  v += __builtin_amdgcn_update_dpp(0, v, 0x128, 0xF, 0xF, false);   // rotated by 8 inside 16 lanes, ...
  v += __builtin_amdgcn_update_dpp(0, v, 0x124, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x122, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x121, 0xF, 0xF, false);
  return __builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16) + __builtin_amdgcn_readlane(v, 32) + __builtin_amdgcn_readlane(v, 48);
}
MSLK_AMD_DEVINL int wave_scan(int v, int lane) {   // inclusive sum
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);   // from 1, 2, 4, 8 lanes below, inside 16 lanes
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
  const int a = __builtin_amdgcn_readlane(v, 15), b = a + __builtin_amdgcn_readlane(v, 31), c = b + __builtin_amdgcn_readlane(v, 47);
  return v + (lane < 16 ? 0 : lane < 32 ? a : lane < 48 ? b : c);
}

// Over the two halves of the wave.
MSLK_AMD_DEVINL float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
MSLK_AMD_DEVINL float sum_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
MSLK_AMD_DEVINL float max_rows16(float x) {   // over the four groups of 16 lanes
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return max_halves(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
MSLK_AMD_DEVINL float sum_rows16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return sum_halves(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

}  // namespace mslk_amd
