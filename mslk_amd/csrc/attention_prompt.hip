// Attention of packed prompts:  O = softmax(scale Q K^T + mask) V  per sequence and head, heads of queries sharing keys.
//
// One pass over the keys per block of queries with the running maximum m and sum l of a softmax: for a tile of keys
// s = q k, m' = max(m, s), l' = l 2^(c(m - m')) + sum 2^(c(s - m')), O' = O 2^(c(m - m')) + 2^(c(s - m')) V with
// c = scale log2(e), and O / l at the end.
//
// A workgroup of four waves takes 128 queries of one head, a wave 32 of them.  Both products are v_mfma_f32_32x32x16 with the
// keys first: S^T = K Q^T leaves a lane one query and half of the tile's keys, so a row's maximum and sum are sums inside a lane
// and one exchange between the wave's halves, and exp2 of S^T is, without moving between lanes, the second operand of
// O^T = V^T P^T: the k slots of that product are dealt to the keys in the order in which the lane holds them, and V is read out
// of LDS with the transposing loads in the same order.
#include "attention.h"
#include "gemm_tile.h"
#include "rows.h"

namespace mslk_amd {
namespace {

constexpr int kWaves = 4, kBlockQ = 32 * kWaves, kTileK = 64;

typedef __attribute__((address_space(3))) v2i lds_v2i;
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

// What a workgroup works on: `rows` queries from q_row on, the first of them query q0 of its sequence, over `keys` keys from
// k_row on; query i of the sequence sees keys up to i + shift.
struct Work {
  int64_t q_row, k_row;
  int q0, rows, keys, shift;
};

MSLK_AMD_DEVINL int clamp_offset(int v, int64_t limit) { return (int)min((int64_t)max(v, 0), limit); }

// Block `index` of the packed queries: the blocks of sequence 0 (last queries first: they see the most keys), of sequence 1, ...,
// then those of the tokens in front of and behind all sequences, which see nothing.
MSLK_AMD_DEVINL bool find_work(const PromptArgs& p, int index, Work& w) {
  const int lane = threadIdx.x & 63;
  int before = 0;   // blocks of the sequences looked at so far
  for (int base = 0; base < p.sequences; base += 64) {
    const int b = base + lane;
    int start = 0, len = 0;
    if (b < p.sequences) {
      start = clamp_offset(p.cu_q[b], p.tokens);
      len = max(clamp_offset(p.cu_q[b + 1], p.tokens) - start, 0);
    }
    const int blocks = (len + kBlockQ - 1) / kBlockQ;
    int upto = blocks;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int v = __shfl_up(upto, d, 64);
      if (lane >= d) upto += v;
    }
    const uint64_t hit = __ballot(index < before + upto);
    if (hit != 0) {
      const int src = __builtin_ctzll(hit);
      const int first = before + __shfl(upto - blocks, src, 64), n = __shfl(blocks, src, 64);
      start = __shfl(start, src, 64);
      len = __shfl(len, src, 64);
      const int b_hit = base + src;
      w.q0 = (n - 1 - (index - first)) * kBlockQ;
      w.rows = min(len - w.q0, kBlockQ);
      w.q_row = start + w.q0;
      int k_start = start, k_len = len;
      if (p.cu_k != p.cu_q) {
        k_start = clamp_offset(p.cu_k[b_hit], p.keys);
        k_len = max(clamp_offset(p.cu_k[b_hit + 1], p.keys) - k_start, 0);
      }
      w.k_row = k_start;
      w.keys = k_len;
      w.shift = p.causal ? k_len - len : k_len;   // not causal: every query sees everything
      return true;
    }
    before += __shfl(upto, 63, 64);
  }
  // tokens of no sequence
  const int head = clamp_offset(p.cu_q[0], p.tokens), tail = clamp_offset(p.cu_q[p.sequences], p.tokens);
  const int head_blocks = (head + kBlockQ - 1) / kBlockQ;
  index -= before;
  const bool front = index < head_blocks;
  if (!front) index -= head_blocks;
  const int64_t from = (front ? 0 : tail) + (int64_t)index * kBlockQ, to = front ? head : p.tokens;
  if (from >= to) return false;
  w = Work{from, 0, 0, (int)min(to - from, (int64_t)kBlockQ), 0, -1};
  return true;
}

// 16 bits of a value, 0 if it is an infinity or a NaN.
template <bool F16> MSLK_AMD_DEVINL uint32_t without_wild(uint32_t bits) { return (bits & 0x7FFFu) >= (F16 ? 0x7C00u : 0x7F80u) ? 0u : bits; }

// Whether rows first ... first + 31 of a tile in LDS hold such a value: two lanes per row.
template <bool F16, int ROW_BYTES, typename Swizzle>
MSLK_AMD_DEVINL bool any_wild(const char* tile, int first, int chunks, Swizzle swizzle) {
  typedef unsigned short us2 __attribute__((ext_vector_type(2)));
  const int lane = threadIdx.x & 63, r = first + lane / 2;
  us2 top = {0, 0};
  for (int c = lane & 1; c < chunks; c += 2) {
    const v4i x = *reinterpret_cast<const v4i*>(tile + r * ROW_BYTES + ((c ^ swizzle(r)) << 4));
#pragma unroll
    for (int i = 0; i < 4; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(us2, x[i] & 0x7FFF7FFF));
  }
  return __ballot(max(top[0], top[1]) >= (F16 ? 0x7C00 : 0x7F80)) != 0;
}

// DP: head dimension rounded up to what the operands are padded to.
template <bool F16, int DP>
__global__ __launch_bounds__(64 * kWaves, DP <= 128 ? 2 : 1) void prompt_kernel(PromptArgs p, int blocks) {
  using E = Elem<F16>;
  constexpr int kSlots = DP <= 64 ? 8 : DP <= 128 ? 16 : 32;   // 16-byte chunks of a row in LDS, a power of two
  constexpr int kRowBytes = kSlots * 16, kTileBytes = kTileK * kRowBytes;
  constexpr int kSteps = DP / 16, kBlocksD = DP / 32;
  constexpr int kLoads = kTileBytes / 1024 / kWaves;           // wave-level copies of a tile per wave
  __shared__ __attribute__((aligned(1024))) char lds[4 * kTileBytes];   // keys, keys, values, values

  const int64_t id = row_block();
  if (id >= (int64_t)blocks * p.Hq) return;
  int head, index;
  if (p.Hkv % 8 == 0) {   // workgroup i runs on XCD i % 8: heads that share keys on one XCD
    const int per = p.Hq / 8, i = (int)(id / 8);
    head = (int)(id % 8) * per + i % per;
    index = i / per;
  } else {
    head = (int)(id % p.Hq);
    index = (int)(id / p.Hq);
  }
  Work w;
  if (!find_work(p, index, w)) return;
  w.q_row = ((int64_t)__builtin_amdgcn_readfirstlane((int)(w.q_row >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)w.q_row);
  w.k_row = ((int64_t)__builtin_amdgcn_readfirstlane((int)(w.k_row >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)w.k_row);
  w.q0 = __builtin_amdgcn_readfirstlane(w.q0);
  w.rows = __builtin_amdgcn_readfirstlane(w.rows);
  w.keys = __builtin_amdgcn_readfirstlane(w.keys);
  w.shift = __builtin_amdgcn_readfirstlane(w.shift);

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int chunks = p.D / 8;   // 16-byte chunks of a row

  // queries: lane (col, half) holds channels 16 step + 8 half ... + 7 of query 32 wave + col; zeros beyond D
  const int row = 32 * wave + col;
  v4i q[kSteps];
  {
    const uint16_t* src = p.q.data + (w.q_row + min(row, w.rows - 1)) * p.q.token_stride + (int64_t)head * p.q.head_stride;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int c = 2 * s + half;
      q[s] = c < chunks ? *reinterpret_cast<const v4i*>(src + c * 8) : v4i{0, 0, 0, 0};
    }
  }

  const int kv_head = head / (p.Hq / p.Hkv);
  const uint8_t* k_base = reinterpret_cast<const uint8_t*>(p.k.data + w.k_row * p.k.token_stride + (int64_t)kv_head * p.k.head_stride);
  const uint8_t* v_base = reinterpret_cast<const uint8_t*>(p.v.data + w.k_row * p.v.token_stride + (int64_t)kv_head * p.v.head_stride);
  const uint32_t k_pitch = (uint32_t)p.k.token_stride * 2, v_pitch = (uint32_t)p.v.token_stride * 2;

  // Copies of tile t: slot (row r, chunk c) of LDS holds chunk c ^ swizzle(r) of row r.  Rows beyond the last key repeat it, so
  // that nothing of another sequence is ever multiplied; chunks beyond D repeat the last one (their queries are zero, and the
  // columns of the output are dropped).
  constexpr int kRowsPerCopy = 64 / kSlots;
  auto issue = [&](const uint8_t* base, uint32_t pitch, int t, char* buf, auto swizzle) {
    const int valid = w.keys - t * kTileK;
    const uint8_t* tile = uniform_ptr(base + (int64_t)t * kTileK * pitch);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int r = (wave * kLoads + i) * kRowsPerCopy + lane / kSlots;
      const int c = (lane % kSlots) ^ swizzle(r);
      const uint32_t off = (uint32_t)min(r, valid - 1) * pitch + (uint32_t)min(c, chunks - 1) * 16;
      dma16(tile, off, buf + (wave * kLoads + i) * 1024);
    }
  };
  auto k_swizzle = [](int r) { return kSlots == 8 ? (r >> 1) & 7 : r & 15; };
  auto v_swizzle = [](int r) { return kSlots == 8 ? (2 * r) & 6 : (4 * r) & 12; };

  // keys that the block's last query sees
  const int seen = min(w.keys, w.q0 + w.rows + w.shift);
  const int tiles = seen <= 0 ? 0 : (seen + kTileK - 1) / kTileK;
  const int limit = w.q0 + row + w.shift;                                  // last key that this lane's query sees
  const int wave_first = w.q0 + 32 * wave + w.shift, wave_last = wave_first + 31;
  const float c = p.scale * kLog2e;

  v16f o[kBlocksD];
#pragma unroll
  for (int d = 0; d < kBlocksD; ++d) o[d] = v16f{};
  float m = -__builtin_inff(), l = 0.f;

  if (tiles > 0) {
    issue(k_base, k_pitch, 0, lds, k_swizzle);
    issue(v_base, v_pitch, 0, lds + 2 * kTileBytes, v_swizzle);
  }
  // lane-constant parts of the LDS addresses
  const int v_key = 4 * half + (lane & 15) / 4, v_byte = 32 * ((lane >> 4) & 1) + 8 * (lane & 3);

  for (int t = 0; t < tiles; ++t) {
    const char* kb = lds + (t & 1) * kTileBytes;
    const char* vb = lds + (2 + (t & 1)) * kTileBytes;
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0): this wave's copies of tile t are in LDS, its reads of t - 1 done
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if (t + 1 < tiles) {
      issue(k_base, k_pitch, t + 1, lds + ((t + 1) & 1) * kTileBytes, k_swizzle);
      issue(v_base, v_pitch, t + 1, lds + (2 + ((t + 1) & 1)) * kTileBytes, v_swizzle);
    }
    const int key0 = t * kTileK;
    if (key0 > wave_last || 32 * wave >= w.rows) continue;   // nothing to see for this wave

    v16f s[2] = {v16f{}, v16f{}};
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int r = 32 * g + col;
        const v4i a = *reinterpret_cast<const v4i*>(kb + r * kRowBytes + (((2 * i + half) ^ k_swizzle(r)) << 4));
        s[g] = E::mfma32(a, q[i], s[g]);
      }
    }
    // lane (col, half) holds keys key0 + 32 g + 4 half + r % 4 + 8 (r / 4)
    bool wild = false;   // the tile holds a value that is not finite, of a key that not all of the wave's queries see
    if (key0 + kTileK > w.keys || key0 + kTileK - 1 > wave_first) {
      const int first = min(max(wave_first + 1 - key0, 0), kTileK - 32);   // rows of the tile from here on are hidden from some
      if (key0 + kTileK - 1 > wave_first) wild = any_wild<F16, kRowBytes>(vb, first, chunks, v_swizzle);
      if (first < kTileK - 32) wild |= any_wild<F16, kRowBytes>(vb, kTileK - 32, chunks, v_swizzle);
      const int last = min(limit, w.keys - 1) - key0 - 4 * half;
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[g][r] = 32 * g + r % 4 + 8 * (r / 4) <= last ? s[g][r] : -__builtin_inff();
    }
    float top = s[0][0];
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[g][r]);
    top = max_halves(top);
    const float m_new = fmaxf(m, top);
    const float base = m_new == -__builtin_inff() ? 0.f : m_new * c;
    const float shrink = exp2_fast(m * c - base);
    m = m_new;
    float sum = 0.f;
    v4i pk[4];
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float a = exp2_fast(__builtin_fmaf(s[g][r], c, -base)), b = exp2_fast(__builtin_fmaf(s[g][r + 1], c, -base));
        sum += a + b;
        pk[2 * g + r / 8][(r % 8) / 2] = (int)E::pack(a, b);
      }
    l = l * shrink + sum;
#pragma unroll
    for (int d = 0; d < kBlocksD; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] *= shrink;
    // k slot 8 half + j of step u: key 16 u + 4 half + j (j < 4), 16 u + 8 + 4 half + j - 4 (j >= 4)
    auto product = [&](auto tame) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int d = 0; d < kBlocksD; ++d) {
          v4i a;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int r = 16 * u + 8 * x + v_key;
            const char* at = vb + r * kRowBytes + ((((64 * d + v_byte) >> 4) ^ v_swizzle(r)) << 4) + (v_byte & 15);
            const v2i two = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at)));
            a[2 * x] = tame(two[0]);
            a[2 * x + 1] = tame(two[1]);
          }
          o[d] = E::mfma32(a, pk[u], o[d]);
        }
    };
    if (!wild) {
      product([](int x) { return x; });
    } else {
      // Queries that do not see a key have the weight 0 for it, which does not silence an infinity or a NaN: such values are left
      // out of the product and added where they are seen.
      product([](int x) { return (int)(without_wild<F16>((uint32_t)x & 0xFFFFu) | without_wild<F16>((uint32_t)x >> 16) << 16); });
      for (int r = 0; r < kTileK; ++r) {
        if (key0 + r > limit || key0 + r >= w.keys) continue;
#pragma unroll
        for (int d = 0; d < kBlocksD; ++d)
#pragma unroll
          for (int y = 0; y < 16; ++y) {
            const int ch = 32 * d + y % 4 + 8 * (y / 4) + 4 * half;
            const uint32_t x = *reinterpret_cast<const uint16_t*>(vb + r * kRowBytes + (((ch >> 3) ^ v_swizzle(r)) << 4) + (ch & 7) * 2);
            if (without_wild<F16>(x) != x) o[d][y] += E::lo(x);
          }
      }
    }
  }

  if (row >= w.rows) return;
  l = sum_halves(l);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* dst = p.out + ((w.q_row + row) * p.Hq + head) * p.D;
#pragma unroll
  for (int d = 0; d < kBlocksD; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int ch = 32 * d + 8 * g + 4 * half;
      if (ch < p.D) {
        const v2i v = {(int)E::pack(o[d][4 * g] * inv, o[d][4 * g + 1] * inv), (int)E::pack(o[d][4 * g + 2] * inv, o[d][4 * g + 3] * inv)};
        *reinterpret_cast<v2i*>(dst + ch) = v;
      }
    }
  if (half == 0) p.lse[(w.q_row + row) * p.Hq + head] = l == 0.f ? -__builtin_inff() : m * p.scale + log2_fast(l) * kLn2;
}

template <bool F16, int DP>
hipError_t launch(const PromptArgs& p, hipStream_t s) {
  const int64_t blocks = p.tokens / kBlockQ + (p.sequences < p.tokens ? p.sequences : p.tokens) + 2;
  hipLaunchKernelGGL((prompt_kernel<F16, DP>), row_grid(blocks * p.Hq), dim3(64 * kWaves), 0, s, p, (int)blocks);
  return hipGetLastError();
}

template <bool F16>
hipError_t pick(const PromptArgs& p, hipStream_t s) {
  if (p.D <= 64) return launch<F16, 64>(p, s);
  if (p.D <= 96) return launch<F16, 96>(p, s);
  if (p.D <= 128) return launch<F16, 128>(p, s);
  if (p.D <= 192) return launch<F16, 192>(p, s);
  return launch<F16, 256>(p, s);
}

}  // namespace

hipError_t launch_attention_prompt(const PromptArgs& p, hipStream_t s) { return p.dtype == 1 ? pick<true>(p, s) : pick<false>(p, s); }

}  // namespace mslk_amd
