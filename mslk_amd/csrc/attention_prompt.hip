// Attention of packed prompts:  O = softmax(scale Q K^T + mask) V  per sequence and head, heads of queries sharing keys.
//
// One pass over the keys per block of queries with a reference m near the running maximum and the running sum l of a softmax in base
// 2: for a tile of keys s = q k, l' = l 2^(m - m') + sum 2^(c s - m'), O' = O 2^(m - m') + 2^(c s - m') V with c = scale log2(e), and
// O / l at the end.  m is the rounded product of c and a score, and everything is taken from that one number: where it stays, the
// sums are scaled by exactly 1, however large the scores are.
//
// A workgroup takes 128 or 64 queries of one head, a wave 32 or 16 of them; tiles of 64 keys and values are copied into LDS, two of
// each.  Both products are v_mfma_f32_16x16x32 with the keys first: S^T = K Q^T leaves a lane one query and a quarter of the tile's
// keys, so a row's maximum and sum are sums inside a lane and two exchanges between lanes, and exp2 of S^T is, without moving
// between lanes, the second operand of O^T = V^T P^T: the k slots of that product are dealt to the keys in the order in which the
// lane holds them, and V is read out of LDS with the transposing loads in the same order.
//
// The reference m follows the maximum when it is left behind by more than 8 powers of two, so that the sums are seldom scaled; weights
// are below 2^8 and rounded once to 16 bits, l sums them unrounded.
//
// The weights' rounding is the one thing here that a computation in 32 bits does not have: it adds 2^-9 in bf16 (2^-12 in fp16) to an
// output that is rounded by as much itself, 0.0019 to 0.0023 from 64 bits instead of 0.0016.  Two numbers per weight, as in
// attention_decode.hip, would be half as many matrix instructions again in a kernel that these bind.
//
// Bound (profiles/attention_rules.txt): long prompts by the power of the matrix cores: 16384 tokens, 32 heads of 128 on 8, causal, 1780 to
// 1960 us by the card, 1120 to 1240 TFLOP/s of what the mask leaves; busy 0.63 of the time at 1.72 GHz, and with operands of zeros just as
// busy at 2.23 GHz and 26 % faster; without any softmax it would gain 18 %.  (The 32x32x16 form of both products was 8 % slower.)  Ragged
// batches (8192 tokens in nine sequences, 64 heads: 427 to 459 us) lose the rest to products behind the mask, 13 % of all, and to the
// tiles that the mask cuts, 17 %, whose copies, products and softmax do not overlap; so do heads of 96 without a mask (46 us, matrix
// cores busy 0.31 at full clock: two workgroups per CU are too few to hide one another's softmax).  Few and short prompts are bound by a
// tile's chain of copies, products and softmax, 0.7 us for a workgroup of 64 queries alone: 100 tokens 6.0 us, 1000 tokens 21.
#include <algorithm>

#include "attention.h"
#include "gemm_tile.h"

namespace mslk_amd {
namespace {

constexpr int kTileK = 64, kHalfK = 32;
constexpr int kGridY = 32768;   // blocks of queries per grid row

// DP: head dimension rounded up to what the operands are padded to.  Q: queries of a workgroup.
template <int DP, int Q> struct Shape {
  // Blocks of 16 queries per wave.  Two halve the reads of LDS per matrix instruction (16384 tokens, D = 128: 1955 us, with eight waves of
  // one block 2375; 8192 tokens, D = 64: 323 / 342).  Beyond D = 128 two do not fit 256 registers, and one wave per SIMD has nothing to run
  // beside its softmax: 8192 tokens, 16 heads of 256, 579 us with eight waves of one block; four waves of two had taken 940 where that
  // form took 550.
  static constexpr int kB = DP <= 128 && Q == 128 ? 2 : 1;
  static constexpr int kWaveQ = 16 * kB, kWaves = Q / kWaveQ;
};

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

// What a workgroup works on: `rows` queries from q_row on, the first of them query q0 of its sequence, over `keys` keys from
// k_row on; query i of the sequence sees keys up to i + shift.
struct Work {
  int64_t q_row, k_row;
  int q0, rows, keys, shift;
};

// A sequence of the packed queries and its keys; blocks of Q queries.
template <int Q> struct Sequence {
  int start, len, k_start, k_len;
  MSLK_AMD_DEVINL int blocks() const { return (len + Q - 1) / Q; }
  // Blocks that visit at least `tiles` tiles of keys: the last ones.
  MSLK_AMD_DEVINL int blocks_of(int tiles, bool causal) const {
    const int n = blocks();
    if (tiles <= 0) return n;
    const uint32_t keys = (uint32_t)(tiles - 1) * kTileK + 1;   // the last query has to see this many
    if (keys > (uint32_t)k_len) return 0;
    const int queries = (int)keys - (k_len - len);
    return !causal || queries <= 0 ? n : n - (queries - 1) / Q;
  }
};

MSLK_AMD_DEVINL int clamp_offset(int v, int64_t limit) { return (int)min((int64_t)max(v, 0), limit); }
MSLK_AMD_DEVINL int64_t uniform64(int64_t v) {
  return ((int64_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}
template <int Q>
MSLK_AMD_DEVINL Sequence<Q> sequence(const PromptArgs& p, int b) {
  Sequence<Q> s{0, 0, 0, 0};
  if (b >= p.sequences) return s;
  s.start = clamp_offset(p.cu_q[b], p.tokens);
  s.len = max(clamp_offset(p.cu_q[b + 1], p.tokens) - s.start, 0);
  s.k_start = s.start;
  s.k_len = s.len;
  if (p.cu_k != p.cu_q) {
    s.k_start = clamp_offset(p.cu_k[b], p.keys);
    s.k_len = max(clamp_offset(p.cu_k[b + 1], p.keys) - s.k_start, 0);
  }
  return s;
}
// Block `index` of the packed queries: sequence by sequence, its last queries, which see the most keys, first; or, `sorted` (up to 64
// sequences), in the order of how many tiles of keys they visit, most first.  Behind them the tokens in front of and behind all
// sequences, which see nothing.
//
// Few workgroups are sorted, so that the last ones to start are short; of many, those that run together rather share keys in the
// L2.  Sorted against not, us: 8192 tokens in 9 sequences, causal, D = 128, 600 workgroups 51.3 / 51.8, 1200 69.4 / 71.1, 2400 163.5 /
// 162.3, 4800 258 / 253; 6000 tokens in 13 sequences, not causal, D = 96, 976 workgroups 47.5 / 48.6, 1952 84.3 / 85.9, 3904 152.6 /
// 152.2; 4873 tokens in 8 sequences, causal, 1536 workgroups 59.4 / 64.0.
constexpr int kSortedBlocks = 2048;
template <int Q>
MSLK_AMD_DEVINL bool find_work(const PromptArgs& p, int index, bool sorted, Work& w) {
  const int lane = threadIdx.x & 63;
  int before = 0;   // blocks of the sequences looked at so far
  for (int base = 0; base < p.sequences; base += 64) {
    const Sequence<Q> s = sequence<Q>(p, base + lane);
    const int n = s.blocks();
    int src = -1, block = 0;
    if (sorted) {
      const int all = wave_sum(n);
      if (index < all) {
        // the largest number of tiles that more than `index` blocks visit
        int low = 0, high = (int)(min(p.keys, (int64_t)INT32_MAX) / kTileK) + 1;
        while (low < high) {
          const int mid = low + (high - low + 1) / 2;
          if (wave_sum(s.blocks_of(mid, p.causal)) > index) low = mid;
          else high = mid - 1;
        }
        const int here = s.blocks_of(low, p.causal), more = s.blocks_of(low + 1, p.causal), rank = index - wave_sum(more);
        const int upto = wave_scan(here - more, lane);   // blocks with just as many tiles
        src = __builtin_ctzll(__ballot(rank < upto));
        block = __builtin_amdgcn_readlane(n - here, src) + rank - __builtin_amdgcn_readlane(upto - (here - more), src);
      } else {
        before = all;
      }
    } else {
      const int upto = wave_scan(n, lane);
      const uint64_t hit = __ballot(index < before + upto);
      if (hit != 0) {
        src = __builtin_ctzll(hit);
        block = __builtin_amdgcn_readlane(n, src) - 1 - (index - before - __builtin_amdgcn_readlane(upto - n, src));
      } else {
        before += __builtin_amdgcn_readlane(upto, 63);
      }
    }
    if (src >= 0) {
      const int len = __builtin_amdgcn_readlane(s.len, src);
      w.keys = __builtin_amdgcn_readlane(s.k_len, src);
      w.k_row = __builtin_amdgcn_readlane(s.k_start, src);
      w.q0 = block * Q;
      w.rows = min(len - w.q0, Q);
      w.q_row = __builtin_amdgcn_readlane(s.start, src) + w.q0;
      w.shift = p.causal ? w.keys - len : w.keys;   // not causal: every query sees everything
      return true;
    }
  }
  // tokens of no sequence
  const int head = clamp_offset(p.cu_q[0], p.tokens), tail = clamp_offset(p.cu_q[p.sequences], p.tokens);
  const int head_blocks = (head + Q - 1) / Q;
  index -= before;
  const bool front = index < head_blocks;
  if (!front) index -= head_blocks;
  const int64_t from = (front ? 0 : tail) + (int64_t)index * Q, to = front ? head : p.tokens;
  if (from >= to) return false;
  w = Work{from, 0, 0, (int)min(to - from, (int64_t)Q), 0, -1};
  return true;
}

// 16 bits of a value, 0 if it is an infinity or a NaN.
template <bool F16> MSLK_AMD_DEVINL uint32_t without_wild(uint32_t bits) { return (bits & 0x7FFFu) >= (F16 ? 0x7C00u : 0x7F80u) ? 0u : bits; }

// Whether one of 32 rows in LDS holds such a value; two lanes a row.  (Rare: the lane number is hidden from the compiler, which
// would compute the addresses in front of the loop and keep them.)
template <bool F16, int ROW_BYTES, int CHUNKS, typename Swizzle>
MSLK_AMD_DEVINL bool any_wild(const char* rows, Swizzle swizzle) {
  typedef unsigned short us2 __attribute__((ext_vector_type(2)));
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  const int r = lane / 2;
  us2 top = {0, 0};
#pragma unroll
  for (int c = 0; c < CHUNKS / 2; ++c) {
    const v4i x = *reinterpret_cast<const v4i*>(rows + r * ROW_BYTES + (((2 * c + (lane & 1)) ^ swizzle(r)) << 4));
#pragma unroll
    for (int i = 0; i < 4; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(us2, x[i] & 0x7FFF7FFF));
  }
  return __ballot(max(top[0], top[1]) >= (F16 ? 0x7C00 : 0x7F80)) != 0;
}

// Rows of a head's keys or values from a tile's first one on, as a buffer: what lies beyond the last row is read as zeros (a row's pitch
// is at least its length).
struct Rows {
  uint64_t base;
  uint32_t pitch, row_bytes;
  int left;   // rows
  v4i buffer;
  MSLK_AMD_DEVINL Rows(const HeadRows& r, int64_t row, int head, int D, int rows)
      : base(reinterpret_cast<uint64_t>(r.data + row * r.token_stride + (int64_t)head * r.head_stride)), pitch((uint32_t)r.token_stride * 2),
        row_bytes((uint32_t)D * 2), left(rows) {
    describe();
  }
  MSLK_AMD_DEVINL void describe() {
    buffer = v4i{(int)(uint32_t)base, (int)(uint32_t)(base >> 32), left <= 0 ? 0 : (int)((uint32_t)(min(left, kTileK) - 1) * pitch + row_bytes), 0x00020000};
  }
  MSLK_AMD_DEVINL void next() {
    base += (uint64_t)kTileK * pitch;
    left -= kTileK;
    describe();
  }
};

constexpr uint32_t kOutside = 0xFFFFFF00u;   // of any buffer of 64 rows that are less than 2^26 bytes apart

// 64 pieces of 16 bytes into LDS at `to`, `from` bytes into the buffer, lane after lane.  To the compiler it is a value made from
// `token`, so that it can lie between matrix instructions and LDS reads can be moved past it; the fences in front of it and behind
// it hold the token.
MSLK_AMD_DEVINL void copy_piece(v4i buffer, uint32_t from, uint32_t to, int& token) {
  asm("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : "+s"(token) : "v"(from), "s"(buffer), "s"(to) : "m0");
}

template <bool F16, int DP, int Q>
__global__ __launch_bounds__((64 * Shape<DP, Q>::kWaves), 2) void prompt_kernel(PromptArgs p, int blocks) {
  using E = Elem<F16>;
  using S = Shape<DP, Q>;
  constexpr int kB = S::kB, kWaveQ = S::kWaveQ, kWaves = S::kWaves;
  constexpr int kSlots = DP / 8;   // 16-byte chunks of a row in LDS
  constexpr int kRowBytes = kSlots * 16, kTileBytes = kTileK * kRowBytes;
  constexpr int kSteps = DP / 32, kBlocksD = DP / 16;
  constexpr int kLoads = kTileBytes / 1024 / kWaves;           // wave-level copies of a tile per wave
  __shared__ __attribute__((aligned(1024))) char lds[4 * kTileBytes];   // keys, keys, values, values

  int head = blockIdx.x;
  const int index = blockIdx.y + blockIdx.z * kGridY;
  if (index >= blocks) return;
  // Workgroup i runs on XCD i % 8: heads that share keys on one XCD, where the KV heads can be dealt out evenly.  With against without, us: 64
  // heads on 8, 8192 tokens in nine sequences 457 / 480, 4096 tokens 281 / 286; 16 heads of 96 on 16 46.8 / 48.4; 32 heads on 8, 16384 tokens
  // 1963 / 1964.
  if (p.Hkv % 8 == 0) head = head % 8 * (p.Hq / 8) + head / 8;
  Work w;
  if (!find_work<Q>(p, index, p.sequences > 1 && p.sequences <= 64 && (int64_t)blocks * p.Hq <= kSortedBlocks, w)) return;
  w.q_row = uniform64(w.q_row);
  w.k_row = uniform64(w.k_row);
  w.q0 = __builtin_amdgcn_readfirstlane(w.q0);
  w.rows = __builtin_amdgcn_readfirstlane(w.rows);
  w.keys = __builtin_amdgcn_readfirstlane(w.keys);
  w.shift = __builtin_amdgcn_readfirstlane(w.shift);

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, group = lane >> 4;
  const int chunks = p.D / 8;   // 16-byte chunks of a row

  const int kv_head = (int)divide((uint32_t)head, p.group);
  const uint32_t k_pitch = (uint32_t)p.k.token_stride * 2, v_pitch = (uint32_t)p.v.token_stride * 2;
  // Which 16-byte chunk of its row a slot of LDS holds: chosen so that the 16 (8-byte loads: 32) lanes that are served together find
  // their rows in different banks (64 of 4 bytes: rows of 16 or 32 chunks begin in the same one, of 8 or 24 in two in turn, of 12 in four).
  // Of a 16-byte load these are rows 0 to 3 and 12 to 15 of one `group` and 4 to 11 of its neighbour.
  auto k_swizzle = [](int r) { return kSlots % 16 == 8 ? (r >> 1) & 7 : kSlots == 12 ? ((r >> 1) & 2) ^ 3 * ((r >> 3) & 1) : r & 15; };
  auto v_swizzle = [](int r) { return kSlots % 16 == 8 ? r & 6 : kSlots == 12 ? (r >> 1) & 2 : (2 * r) & 14; };

  // Copies of a tile: slot (row r, chunk c) of LDS holds chunk c ^ swizzle(r) of row r.  Rows beyond the last key and chunks beyond D
  // lie outside the buffer and come as zeros.
  uint32_t k_off[kLoads], v_off[kLoads];   // of this lane's pieces from a tile's first row
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int slot = (wave * kLoads + i) * 64 + lane, r = slot / kSlots;
    const int k_chunk = (slot % kSlots) ^ k_swizzle(r), v_chunk = (slot % kSlots) ^ v_swizzle(r);
    k_off[i] = k_chunk < chunks ? (uint32_t)r * k_pitch + (uint32_t)k_chunk * 16 : kOutside;
    v_off[i] = v_chunk < chunks ? (uint32_t)r * v_pitch + (uint32_t)v_chunk * 16 : kOutside;
  }
  const uint32_t lds_wave = __builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(lds_ptr_t)lds + wave * kLoads * 1024);

  const int wave_row = kWaveQ * wave;
  const int seen = min(w.keys, w.q0 + w.rows + w.shift);                   // keys that the block's last query sees
  const int tiles = seen <= 0 ? 0 : (seen + kTileK - 1) / kTileK;
  const int limit = w.q0 + wave_row + col + w.shift;                       // last key that this lane's first query sees
  const int wave_first = w.q0 + wave_row + w.shift;
  const int wave_seen = wave_row >= w.rows ? 0 : max(min(w.keys, wave_first + kWaveQ), 0);
  const int wave_tiles = (wave_seen + kTileK - 1) / kTileK;
  const int whole = min(min(w.keys, w.q0 + w.shift + 1) / kTileK, tiles);  // tiles that every query of the block sees whole
  const float c = p.scale * kLog2e;

  Rows k_rows(p.k, w.k_row, kv_head, p.D, min(w.keys, tiles * kTileK)), v_rows(p.v, w.k_row, kv_head, p.D, min(w.keys, tiles * kTileK));
  int token = 0;
  auto piece = [&](int i, int parity) {   // copies 0 to kLoads - 1: values of the next tile; from kLoads on: keys of the one after it
    if (i < kLoads) copy_piece(v_rows.buffer, v_off[i], lds_wave + (2 + (parity ^ 1)) * kTileBytes + i * 1024, token);
    else copy_piece(k_rows.buffer, k_off[i - kLoads], lds_wave + parity * kTileBytes + (i - kLoads) * 1024, token);
  };
  if (tiles > 0) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) piece(kLoads + i, 0);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) piece(i, 1);
  }
  // queries: lane (col, group) holds channels 32 step + 8 group ... + 7 of query wave_row + 16 b + col; zeros beyond D
  v4i q[kB][kSteps];
#pragma unroll
  for (int b = 0; b < kB; ++b) {
    const uint16_t* src = p.q.data + (w.q_row + min(wave_row + 16 * b + col, w.rows - 1)) * p.q.token_stride + (int64_t)head * p.q.head_stride;
#pragma unroll
    for (int x = 0; x < kSteps; ++x) {
      const int ch = 4 * x + group;
      q[b][x] = ch < chunks ? *reinterpret_cast<const v4i*>(src + ch * 8) : v4i{0, 0, 0, 0};
    }
  }

  v4f o[kB][kBlocksD], s[kB][4];
  v4i pk[kB][2];
  float m[kB], l[kB];
#pragma unroll
  for (int b = 0; b < kB; ++b) {
#pragma unroll
    for (int d = 0; d < kBlocksD; ++d) o[b][d] = v4f{};
    m[b] = -__builtin_inff();
    l[b] = 0.f;
  }

  auto next = [&] {
    v_rows.next();
    k_rows.next();
  };
  auto fence = [&] {   // this wave's copies are in LDS and its reads are done; so are the other waves'
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" : "+s"(token) : : "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" : "+s"(token) : : "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  // where a lane reads keys and values in LDS: a row's 16 bytes of a step's channels; four keys by 16 channels per 16 lanes
  int k_at[kSteps], v_at[kBlocksD];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) k_at[i] = col * kRowBytes + (((4 * i + group) ^ k_swizzle(col)) << 4);
  const int v_key = 4 * group + col / 4;
#pragma unroll
  for (int d = 0; d < kBlocksD; ++d) v_at[d] = v_key * kRowBytes + (((2 * d + ((lane >> 1) & 1)) ^ v_swizzle(v_key)) << 4) + 8 * (lane & 1);

  // S^T of a half tile: lane (col, group) holds keys 16 g + 4 group + r in s[g][r], g = 0, 1 of the first half and 2, 3 of the second
  auto scores = [&](int parity, int h) {
    const char* kb = lds + parity * kTileBytes;
#pragma unroll
    for (int g = 2 * h; g < 2 * h + 2; ++g) {
#pragma unroll
      for (int b = 0; b < kB; ++b) s[b][g] = v4f{};
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const v4i a = *reinterpret_cast<const v4i*>(kb + k_at[i] + g * 16 * kRowBytes);
#pragma unroll
        for (int b = 0; b < kB; ++b) s[b][g] = E::mfma16(a, q[b][i], s[b][g]);
      }
    }
  };
  // O^T += V^T P^T of half tile u; k slot 8 group + j: key 32 u + 4 group + j (j < 4), 32 u + 16 + 4 group + j - 4 (j >= 4)
  auto product = [&](int parity, int u, auto tame) {
    const char* vb = lds + (2 + parity) * kTileBytes;
#pragma unroll
    for (int d = 0; d < kBlocksD; ++d) {
      v4i a;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const v2i two = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(vb + v_at[d] + (32 * u + 16 * x) * kRowBytes)));
        a[2 * x] = tame(two[0]);
        a[2 * x + 1] = tame(two[1]);
      }
#pragma unroll
      for (int b = 0; b < kB; ++b) o[b][d] = E::mfma16(a, pk[b][u], o[b][d]);
    }
  };
  auto same = [](int x) { return x; };
  auto softmax = [&] {
    float shrink[kB], base[kB], largest = 0.f;
#pragma unroll
    for (int b = 0; b < kB; ++b) {
      float top = s[b][0][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) top = fmaxf(top, s[b][r / 4][r % 4]);
      top = max_rows16(top);
      top *= c;
      // the reference follows the maximum when it is left behind by more than 8 powers of two: the weights stay below 2^8
      const float m_new = top > m[b] + 8.f ? top : m[b];
      base[b] = m_new == -__builtin_inff() ? 0.f : m_new;
      shrink[b] = exp2_fast(m[b] - base[b]);
      m[b] = m_new;
      largest = fmaxf(largest, __builtin_fabsf(base[b]));
    }
    float by = c;
    if (__ballot(largest > 0x1p24f) != 0) {
      // The product in a weight's fused multiply-add is not rounded, that in the reference is: here by more than a power of two, and
      // at the same score too, which may leave the range of 16 bits.  Both rounded instead.
      by = 1.f;
#pragma unroll
      for (int b = 0; b < kB; ++b) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float x = s[b][r / 4][r % 4] * c;
          s[b][r / 4][r % 4] = x - base[b];
        }
        base[b] = 0.f;
      }
    }
#pragma unroll
    for (int b = 0; b < kB; ++b) {
      float sum = 0.f;
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          const float x = exp2_fast(__builtin_fmaf(s[b][g][r], by, -base[b])), y = exp2_fast(__builtin_fmaf(s[b][g][r + 1], by, -base[b]));
          sum += x + y;
          pk[b][g / 2][2 * (g % 2) + r / 2] = (int)E::pack(x, y);   // the weights' one rounding; l sums them unrounded
        }
      l[b] = __builtin_fmaf(l[b], shrink[b], sum);
      asm volatile("" : "+v"(l[b]));   // summed here: put off, it keeps the weights in registers
    }
    bool moved = false;
#pragma unroll
    for (int b = 0; b < kB; ++b) moved |= shrink[b] != 1.f;
    if (__ballot(moved) != 0)
#pragma unroll
      for (int b = 0; b < kB; ++b)
#pragma unroll
        for (int d = 0; d < kBlocksD; ++d) o[b][d] *= shrink[b];
  };
  auto interleave = [&] {   // LDS reads ahead of the matrix instructions that need them
    __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
    for (int i = 0; i < 2 * kBlocksD - 4; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, kB, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
#pragma unroll
    for (int i = 0; i < 4 * kSteps; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, kB, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 4 * kB, 0);
  };

  if (tiles > 0) {
    fence();
    k_rows.next();
#pragma unroll
    for (int i = 0; i < kLoads; ++i) piece(kLoads + i, 1);
    scores(0, 0);
    scores(0, 1);
    const int pairs = max((whole - 1) / 2, 0);   // of tiles that are whole, and so is the next
    for (int i = 0; i < pairs; ++i) {
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        softmax();
        fence();
        next();
#pragma unroll
        for (int j = 0; j < 2 * kLoads; ++j) piece(j, y);
        product(y, 0, same);
        product(y, 1, same);
        scores(y ^ 1, 0);
        scores(y ^ 1, 1);
        interleave();
      }
    }
#pragma unroll 1
    for (int t = 2 * pairs; t < tiles; ++t) {
      const int key0 = t * kTileK;
      const bool both = key0 + kHalfK < wave_seen;   // the wave sees keys of the second half
      if (t < wave_tiles) {
        if (key0 + kTileK > w.keys || key0 + kTileK - 1 > wave_first) {
#pragma unroll
          for (int b = 0; b < kB; ++b) {
            const int last = min(limit + 16 * b, w.keys - 1) - key0 - 4 * group;
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
              for (int r = 0; r < 4; ++r) s[b][g][r] = 16 * g + r <= last ? s[b][g][r] : -__builtin_inff();
          }
        }
        softmax();
      }
      fence();
      next();
      if (t + 1 < tiles) {
#pragma unroll
        for (int i = 0; i < 2 * kLoads; ++i) piece(i, t & 1);
      }
      if (t < wave_tiles) {
        const char* vb = lds + (2 + (t & 1)) * kTileBytes;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          if (u == 1 && !both) break;
          // Queries that do not see a key have the weight 0 for it, which does not silence an infinity or a NaN: where a half tile
          // holds such a value and a key that not all of the wave's queries see, these values are left out of the product and
          // added where they are seen.
          const char* rows = vb + u * kHalfK * kRowBytes;
          if (key0 + kHalfK * u + kHalfK - 1 <= wave_first || !any_wild<F16, kRowBytes, kBlocksD * 2>(rows, v_swizzle)) {
            product(t & 1, u, same);
          } else {
            product(t & 1, u, [](int x) { return (int)(without_wild<F16>((uint32_t)x & 0xFFFFu) | without_wild<F16>((uint32_t)x >> 16) << 16); });
#pragma unroll 1
            for (int r = 0; r < kHalfK; ++r) {
              const int key = key0 + kHalfK * u + r;
              if (key >= w.keys) break;
              int side = 8 * (group & 1);
              asm volatile("" : "+v"(side));
#pragma unroll
              for (int d = 0; d < kBlocksD; ++d)
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                  const uint32_t x = *reinterpret_cast<const uint16_t*>(rows + r * kRowBytes + side + (((2 * d + group / 2) ^ v_swizzle(r)) << 4) + y * 2);
                  const bool bad = without_wild<F16>(x) != x;
#pragma unroll
                  for (int b = 0; b < kB; ++b)
                    if (bad && key <= limit + 16 * b) o[b][d][y] += E::lo(x);
                }
            }
          }
        }
        if (t + 1 < wave_tiles) {
          scores((t + 1) & 1, 0);
          if (key0 + kTileK + kHalfK < wave_seen) scores((t + 1) & 1, 1);   // (else masked: what is left in there does not matter)
        }
      }
    }
  }

#pragma unroll
  for (int b = 0; b < kB; ++b) {
    const int row = wave_row + 16 * b + col;
    const float total = sum_rows16(l[b]);
    const float inv = total == 0.f ? 0.f : 1.f / total;
    uint16_t* dst = p.out + ((w.q_row + row) * p.Hq + head) * p.D;
#pragma unroll
    for (int d = 0; d < kBlocksD; d += 2) {   // neighbours in `group` exchange halves of two blocks of 16 channels: 16 bytes per lane
      v4i x;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const auto two = __builtin_amdgcn_permlane16_swap(E::pack(o[b][d][2 * y] * inv, o[b][d][2 * y + 1] * inv),
                                                          E::pack(o[b][d + 1][2 * y] * inv, o[b][d + 1][2 * y + 1] * inv), false, false);
        x[y] = (int)two[0];
        x[2 + y] = (int)two[1];
      }
      const int ch = 16 * (d + (group & 1)) + 8 * (group / 2);
      if (row < w.rows && ch < p.D) *reinterpret_cast<v4i*>(dst + ch) = x;
    }
    if (group == 0 && row < w.rows) p.lse[(w.q_row + row) * p.Hq + head] = total == 0.f ? -__builtin_inff() : (m[b] + log2_fast(total)) * kLn2;
  }
}

template <bool F16, int DP, int Q>
hipError_t launch(const PromptArgs& p, int64_t blocks, hipStream_t s) {
  hipLaunchKernelGGL((prompt_kernel<F16, DP, Q>), dim3((unsigned)p.Hq, (unsigned)std::min<int64_t>(blocks, kGridY), (unsigned)((blocks + kGridY - 1) / kGridY)),
                     dim3(64 * Shape<DP, Q>::kWaves), 0, s, p, (int)blocks);
  return hipGetLastError();
}
// Few workgroups of 128 queries (up to two per CU, or one where LDS holds no second) leave the matrix cores waiting for one another's
// softmax and the last workgroup long: blocks of 64 queries then, in waves of 16, though LDS is read twice as often.  128 against 64, us:
// D = 128 on 32 heads, causal: 100 tokens (96 workgroups) 8.0 / 6.0, 256 (160) 11.5 / 8.0, 500 (192) 16.4 / 11.2, 1000 (320) 26.8 / 20.5,
// 1400 (448) 35.3 / 29.0, 2048 (608) 52.4 / 53.0; 20 sequences of 100 tokens on 16 heads (592) 14.9 / 14.8; 6000 tokens in 13 sequences on
// 16 heads of 96 (976) 50.4 / 55.0.  D = 64 on 32 heads: 1000 tokens 18.3 / 12.8, 2048 33.3 / 31.6.  D = 256, 1000 tokens: 16 heads (160)
// 36.6 / 29.6, 32 heads (320) 39.4 / 39.3.
template <int DP> constexpr int kFewBlocks = DP <= 128 ? 512 : 256;
template <bool F16, int DP>
hipError_t launch(const PromptArgs& p, hipStream_t s) {
  const int64_t parts = std::min<int64_t>(p.sequences, p.tokens) + 2;
  const int64_t blocks = p.tokens / 128 + parts;
  if (blocks * p.Hq <= kFewBlocks<DP>) return launch<F16, DP, 64>(p, p.tokens / 64 + parts, s);
  return launch<F16, DP, 128>(p, blocks, s);
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
