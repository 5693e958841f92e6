// Attention of one new token per sequence over a paged cache, keys and values in 16 bits or as e4m3 codes with a scale per row.
//
// The work is the stream of keys and values: a block of up to 16 query heads that share a KV head reads it once.  A wave takes
// 32 keys at a time straight from memory into the operands of v_mfma_f32_16x16x32: S^T = K Q^T has the keys as rows (lane (i, g)
// loads channels 8 g ... of keys i and 16 + i), which leaves a lane eight scores of one head in the order in which exp2 of them is the
// second operand of O^T = V^T P^T; a lane of group g loads 8 channels of each of its eight keys of V and pairs them up in registers.
//
// The softmax runs in base 2 with reference m: P = 2^(c s - m), c = scale log2(e).  With e4m3 caches the weight of a key's codes
// is P times the value row's scale, so m is the maximum of c s + log2(scale): the weights stay at most 1 (fp16: 2^15) whatever the scales
// are.  The second product takes each weight as the sum of two 16-bit numbers: rounded to one, weights added 2^-9 in bf16 to an output
// that is rounded by as much itself (against 64 bits 0.0023 instead of 0.0016).  Twice the matrix instructions are free where the memory
// binds; 8 sequences with heads of 64 take 22.8 instead of 22.0 us.
//
// Keys are divided evenly whatever the lengths: every (sequence, head block) has its tiles of 32 keys, all tiles stand in one line,
// and wave i of W, each a workgroup of its own, takes the i-th of W equal parts of the line.  Where a part begins or ends inside a
// (sequence, head block), what was summed there is written out in 32 bits, together with where the pieces of the block begin and
// end, and a second launch joins them in their order.  (Short caches are not cut: a wave each for their head blocks.)
//
// Bound: the memory.  64 heads of 128 on 8: one sequence of 131071 keys (537 MB) 92.5 us, 5.8 TB/s; 32 sequences of up to 8192 keys
// (515 MB) 94.3 us, 5.5 TB/s; 128 sequences in e4m3 (1269 MB) 234 us, 5.4 TB/s, and 6 % less where a pool keeps its scales by head (one
// row of 4 bytes per key and head lies among those of the other heads, whose waves fetch the same lines).  A copy moves 5.1 TB/s
// on the same card, a plain read 6.2.  Short caches are bound by what waits for one another: the lengths, the page numbers, the rows,
// the second launch: 700 keys on 8 KV heads take 5.1 + 3.0 us in the two kernels, 8.1 to 8.5 us a call in a graph.  With heads of 64 half of
// a load of values, of the second product and of a piece is padding, and a tile holds half the bytes: 8 sequences of up to 3001 keys
// (60 MB) 23 us, 2.6 TB/s.
#include "attention.h"
#include "rows.h"

#include <utility>

namespace mslk_amd {
namespace {

constexpr int kTile = 32, kHeads = 16;
// A line of at most kMostParts tiles is cut into parts of one tile, a longer one into kLongParts parts.  Two waves fit a SIMD up to D = 128
// (kMostParts of them the GPU), but in a long line one keeps the memory busy and there is half as much to join: 1024 against 2048 parts,
// us, heads of 128: one sequence of 131071 keys 94.3 / 99.4, 4 of 4096 19.4 / 20.8, 128 in e4m3 243 / 252; heads of 256, 16 on 4, 32 sequences of
// up to 4096 keys 62.6 / 67.5, in e4m3 38.1 / 44.7; heads of 64 in e4m3 50.8 / 52.4.  Heads of 64 in 16 bits, whose tiles hold half the
// bytes, are better off the other way: 8 sequences of up to 3001 keys 24.1 / 21.2, 32 of up to 8192 63.9 / 61.8.  Short lines have no
// tile to load while another is computed: 256 sequences of 4 keys (2048 tiles) took 11.5 in parts of one, 14.0 in 1024 parts.
constexpr int kMostParts = 2048, kLongParts = 1024;

// Where the page tables hold few keys, or not many more than there are head blocks, a wave takes a whole head block instead, and there
// is nothing to join.  In parts against whole, us, 32 heads on 8: 100 keys, 1 sequence 7.4 / 6.8, 64 sequences 14.9 / 9.3; 250 keys, 1
// sequence 7.5 / 10.2, 16 10.9 / 10.8, 64 18.3 / 14.9; 500 keys, 16 sequences 16.7 / 18.9, 32 18.6 / 19.1, 128 52.2 / 49.2; 1000 keys, 16
// sequences 19.1 / 32.4, 64 53.0 / 48.9, 128 94.5 / 92.1, and of 1 to 1000 keys 77.7 / 60.7 (a part there holds pieces of several
// blocks, each with its own start).  Longer ones, 64 of 1 to 4000 keys: 95.4 / 132.9, the longest block long after the others.
constexpr int kWholeKeys = 128, kMostWholeKeys = 1024;

struct Line {          // how the work is divided
  int head_blocks;     // per sequence: KV heads x blocks of kHeads query heads
  Divider by_head_blocks;
  int per_kv;          // blocks of query heads per KV head
  int group;           // query heads per KV head
  int parts;
  int joined;          // whether a head block may be cut
};

// A length that the page table cannot hold counts as one key more than it holds: that key has no page.  (Room for at most 2^30 keys.)
MSLK_AMD_DEVINL int length_of(const DecodeArgs& p, int b) {
  return min(max(p.cache.lens[b], 0), p.cache.table_width * (int)p.cache.page_size.d + 1);
}
MSLK_AMD_DEVINL int tiles_of(int len) { return max(1, (len + kTile - 1) / kTile); }

// Part `w` of the line: tiles [begin, end), the sequence that holds the first of them and the tiles in front of that sequence.  (A line
// has fewer than 2^31 tiles; 64-bit divisions would take longer than a tile.)
struct Part {
  int index, begin, end, before, seq, len;
};
MSLK_AMD_DEVINL bool find_part(const DecodeArgs& p, const Line& ln, int w, Part& r) {
  if (!ln.joined) {   // a head block each
    if (w >= ln.parts) return false;
    r.seq = (int)divide((uint32_t)w, ln.by_head_blocks);
    r.len = __builtin_amdgcn_readfirstlane(length_of(p, r.seq));
    r.index = 0;
    r.before = 0;
    r.begin = (w - r.seq * ln.head_blocks) * tiles_of(r.len);
    r.end = r.begin + tiles_of(r.len);
    return true;
  }
  const int lane = threadIdx.x;
  int len = lane < p.sequences ? length_of(p, lane) : 0;
  int n = lane < p.sequences ? tiles_of(len) : 0, upto = wave_scan(n, lane);
  uint32_t total = __builtin_amdgcn_readlane(upto, 63);
  for (int base = 64; base < p.sequences; base += 64) {
    total += wave_sum(base + lane < p.sequences ? tiles_of(length_of(p, base + lane)) : 0);
  }
  total *= ln.head_blocks;
  const uint32_t parts = total <= kMostParts ? total : kLongParts;   // none of them empty
  if ((uint32_t)w >= parts) return false;
  // Workgroup i runs on XCD i % 8.  Neighbours in the line go to one XCD where they share lines: the scales of the heads of a key
  // (128 sequences in e4m3, 64 heads on 8: 245.5 -> 242.8 us), the pieces that one join reads and the page table (700 keys: 8.7 -> 8.1).
  // Long lines of 16-bit rows, which share nothing, are better spread: 64 sequences of 1024 keys 54.4, by neighbours 55.4; 32 of up to
  // 4096 keys, 16 heads of 256 on 4, 62.5 / 63.1; though 8 of up to 3001 keys, 16 heads of 64, 24.1 / 23.8.
  if (p.fp8 || parts == total) w = (w % 8) * (parts / 8) + min((uint32_t)w % 8, parts % 8) + w / 8;
  r.index = w;
  const uint32_t each = parts == total ? 1 : total / parts, more = total - each * parts;   // the first `more` parts hold one tile more
  r.begin = w * each + min((uint32_t)w, more);
  r.end = r.begin + each + ((uint32_t)w < more ? 1 : 0);
  r.before = 0;
  for (int base = 0; base < p.sequences; base += 64) {
    if (base > 0) {
      len = base + lane < p.sequences ? length_of(p, base + lane) : 0;
      n = base + lane < p.sequences ? tiles_of(len) : 0;
      upto = wave_scan(n, lane);
    }
    const uint64_t hit = __ballot(r.begin < r.before + upto * ln.head_blocks);
    if (hit != 0) {
      const int src = __builtin_ctzll(hit);
      r.before += __builtin_amdgcn_readlane(upto - n, src) * ln.head_blocks;
      r.len = __builtin_amdgcn_readlane(len, src);
      r.seq = base + src;
      return true;
    }
    r.before += __builtin_amdgcn_readlane(upto, 63) * ln.head_blocks;
  }
  return false;
}

// The value that lane N of the lane's group of 16 holds.
template <int N>
MSLK_AMD_DEVINL int from16(int x) { return __builtin_amdgcn_update_dpp(0, x, 0x150 + N, 0xF, 0xF, false); }
template <int N>
MSLK_AMD_DEVINL float from16(float x) { return __uint_as_float((uint32_t)from16<N>((int)__float_as_uint(x))); }
template <int N>
MSLK_AMD_DEVINL int64_t from16(int64_t x) { return ((int64_t)from16<N>((int)(x >> 32)) << 32) | (uint32_t)from16<N>((int)x); }

template <typename F, int... I>
MSLK_AMD_DEVINL void each8(F f, std::integer_sequence<int, I...>) { (f(Int<I>{}), ...); }
template <typename F>
MSLK_AMD_DEVINL void each8(F f) { each8(f, std::make_integer_sequence<int, 8>{}); }   // f(Int<0>{}), ... f(Int<7>{})

// Eight e4m3 codes -> eight 16-bit values (exact).
template <bool F16>
MSLK_AMD_DEVINL v4i widen(v2i codes) {
  v4i r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (F16) {
      r[2 * i] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[i], 1.f, false));
      r[2 * i + 1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[i], 1.f, true));
    } else {
      r[2 * i] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[i], 1.f, false));
      r[2 * i + 1] = __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes[i], 1.f, true));
    }
  }
  return r;
}

// A pair of weights, each as the sum of two 16-bit numbers: 16 bits of it in bf16 and 20 in fp16, where rounding to one would leave 8 and
// 11.  The first is truncated from a number below the weight, so that both are positive: with one zero or negative, a key's
// infinite value would give NaN.  (fp16: the second is zero for weights of less than 2^-28 of the largest.)
constexpr float kAbove16 = 15.f;   // fp16: weights below 2^15 instead of 1, so that small ones keep their bits too
template <bool F16>
MSLK_AMD_DEVINL void split(float x, float y, int& first, int& second) {
  using E = Elem<F16>;
  constexpr int kStep = F16 ? 1 << 12 : 1;
  const uint32_t below_x = max((int)__float_as_uint(x) - kStep, 0), below_y = max((int)__float_as_uint(y) - kStep, 0);
  if constexpr (F16) {
    first = __builtin_bit_cast(int, __builtin_amdgcn_cvt_pkrtz(__uint_as_float(below_x), __uint_as_float(below_y)));
    second = (int)E::pack(x - E::lo((uint32_t)first), y - E::hi((uint32_t)first));
  } else {
    first = (int)__builtin_amdgcn_perm(below_y, below_x, 0x07060302u);
    second = (int)E::pack(x - __uint_as_float(below_x & 0xFFFF0000u), y - __uint_as_float(below_y & 0xFFFF0000u));
  }
}

// How a cache holds its rows, and what of a key row a lane fetches at once: 8 channels of 16 bits, 16 e4m3 codes, or 8 where the
// rows do not begin on 16-byte boundaries.
enum Rows : int { kRows16Bit, kRowsE4m3, kRowsE4m3By8 };
template <Rows R> struct RowTraits {
  typedef v4i key_t;
  typedef v2i value_t;
};
template <> struct RowTraits<kRows16Bit> {
  typedef v4i key_t, value_t;
};
template <> struct RowTraits<kRowsE4m3By8> {
  typedef v2i key_t, value_t;
};
// A load of values covers whole rows, whose lines no other load asks for: non-temporal.  A load of keys takes 64 bytes of each of its
// rows and the next one the rest of the line, which has to be there still (in e4m3 247 us with plain loads of keys, 346 with
// non-temporal ones of half the width).
template <typename T>
MSLK_AMD_DEVINL T stream(const char* at) { return __builtin_nontemporal_load(reinterpret_cast<const T*>(at)); }

// Key j (0 ... 7) of group g in a tile: the order in which lane (i, g) holds its scores.
MSLK_AMD_DEVINL int key_of(int j, int g) { return (j & 3) + 4 * g + 16 * (j >> 2); }

// STEPS: channels of a key in steps of 32; SETS: channels of a value in sets of 128.
template <bool F16, Rows ROWS, int STEPS, int SETS>
__global__ __launch_bounds__(64, STEPS <= 4 ? 2 : 1) void decode_kernel(DecodeArgs p, Line ln) {
  using E = Elem<F16>;
  using key_t = typename RowTraits<ROWS>::key_t;
  using value_t = typename RowTraits<ROWS>::value_t;
  constexpr bool FP8 = ROWS != kRows16Bit;
  constexpr int kDP = 128 * SETS, kElem = FP8 ? 1 : 2;
  constexpr int kLeast = STEPS == 2 ? 1 : STEPS == 3 ? 65 : STEPS == 4 ? (FP8 ? 65 : 97) : STEPS == 6 ? 129 : 193;   // smallest D
  constexpr int kPer = ROWS == kRowsE4m3 ? 2 : 1;            // steps of a piece of a key: channels 32 kPer x + 8 kPer g + 8 y ... + 7 in step
  static_assert(STEPS % kPer == 0, "pieces cover whole steps");   // kPer x + y of lane (i, g)
  const int key_pieces = p.D / (8 * kPer);
  // strides in pieces of eight channels: 32 bits reach for them
  const uint32_t k_page = (uint32_t)(p.cache.k_stride[0] >> 3), k_slot = (uint32_t)(p.cache.k_stride[1] >> 3);
  const uint32_t v_page = (uint32_t)(p.cache.v_stride[0] >> 3), v_slot = (uint32_t)(p.cache.v_stride[1] >> 3);
  const int lane = threadIdx.x, i = lane & 15, g = lane >> 4;
  const int chunks = p.D / 8;
  const float c = p.scale * kLog2e;

  Part part;
  if (!find_part(p, ln, (int)row_block(), part)) return;
  int at = part.begin;
  int seq = part.seq, len = part.len;

  while (true) {
    const int tiles = tiles_of(len);
    const int hb = (uint32_t)(at - part.before) / (uint32_t)tiles, tile0 = at - part.before - hb * tiles;
    const int n = min(tiles - tile0, part.end - at);
    const int kv_head = ln.per_kv == 1 ? hb : hb / ln.per_kv, first = (hb - kv_head * ln.per_kv) * kHeads, heads = min(ln.group - first, kHeads);
    const int head0 = kv_head * ln.group + first;
    const int key_begin = tile0 * kTile, key_end = min(len, (tile0 + n) * kTile);

    const int32_t* table = p.cache.table + seq * p.cache.table_stride;
    const char* k_base = (const char*)p.cache.k + kv_head * p.cache.k_stride[2] * kElem;
    const char* v_base = (const char*)p.cache.v + kv_head * p.cache.v_stride[2] * kElem;
    const float* ks_base = p.cache.k_scale + kv_head * p.cache.k_scale_stride[2];
    const float* vs_base = p.cache.v_scale + kv_head * p.cache.v_scale_stride[2];

    // Pages of the keys whose rows or scales a lane fetches: keys i and 16 + i, and key (i % 8, g).  Keys beyond the end repeat the
    // last one; a sequence without keys, whose first look-up stands in front of the test for that, asks for the place of key 0.
    const int last_key = max(key_end - 1, 0);
    struct Place { int page[3], slot[3]; };
    auto places = [&](int key0) {
      Place r;
#pragma unroll
      for (int x = 0; x < 3; ++x) {
        const int key = min(key0 + (x == 0 ? i : x == 1 ? 16 + i : key_of(i & 7, g)), last_key);
        const int index = (int)divide((uint32_t)key, p.cache.page_size);
        r.slot[x] = key - index * (int)p.cache.page_size.d;
        r.page[x] = (uint32_t)index < (uint32_t)p.cache.table_width ? table[index] : -1;
      }
      return r;
    };
    struct Tile {
      key_t k[2][STEPS / kPer];
      value_t v[SETS][8];
      float scale;     // e4m3: of key (i % 8, g), of its key row where i < 8, of its value row otherwise
      uint64_t bad;    // lanes whose key (i % 8, g) has no page
    };
    auto load = [&](Tile& t, int key0, const Place& where) {
      uint32_t page[3], slot[3];
#pragma unroll
      for (int x = 0; x < 3; ++x) {
        const bool lost = (uint32_t)where.page[x] >= (uint32_t)p.cache.pages;
        if (x == 2) t.bad = __ballot(lost);
        slot[x] = lost ? 0 : where.slot[x];
        page[x] = lost ? 0 : where.page[x];
      }
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int64_t row = (int64_t)(((uint64_t)page[b] * k_page + (uint64_t)slot[b] * k_slot) * (8 * kElem));
#pragma unroll
        for (int x = 0; x < STEPS / kPer; ++x) t.k[b][x] = *reinterpret_cast<const key_t*>(k_base + row + min(4 * x + g, key_pieces - 1) * (int)sizeof(key_t));
        __builtin_amdgcn_sched_barrier(0);   // a row's address is done with before the next one's
      }
      const int64_t mine = (int64_t)(((uint64_t)page[2] * v_page + (uint64_t)slot[2] * v_slot) * (8 * kElem));
      each8([&](auto j) {
        const int64_t row = from16<decltype(j)::value>(mine);
#pragma unroll
        for (int x = 0; x < SETS; ++x) t.v[x][decltype(j)::value] = stream<value_t>(v_base + row + min(16 * x + i, chunks - 1) * 8 * kElem);
        __builtin_amdgcn_sched_barrier(0);
      });
      if constexpr (FP8) {
        const bool is_v = i >= 8;
        const uint32_t by_page = (uint32_t)(is_v ? p.cache.v_scale_stride[0] : p.cache.k_scale_stride[0]);
        const uint32_t by_slot = (uint32_t)(is_v ? p.cache.v_scale_stride[1] : p.cache.k_scale_stride[1]);
        t.scale = (is_v ? vs_base : ks_base)[(uint64_t)page[2] * by_page + (uint64_t)slot[2] * by_slot];
      }
    };

    v4i q[STEPS];
    v4f o[SETS][8];
    float m = -__builtin_inff(), l = 0.f;
    auto compute = [&](const Tile& t, int key0) {
      v4f s[2] = {v4f{}, v4f{}};
      // A piece of a key.  Channels beyond D: zeros of q would not silence an infinity that was read in their place.
      auto key_piece = [&](int b, int x) {
        if (32 * kPer * (x + 1) <= kLeast || 4 * x + g < key_pieces) return t.k[b][x];
        return key_t{};
      };
#pragma unroll
      for (int x = 0; x < STEPS; ++x)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if constexpr (ROWS == kRows16Bit) s[b] = E::mfma16(key_piece(b, x), q[x], s[b]);
          else if constexpr (ROWS == kRowsE4m3By8) s[b] = E::mfma16(widen<F16>(key_piece(b, x)), q[x], s[b]);
          else s[b] = E::mfma16(widen<F16>(v2i{key_piece(b, x / 2)[2 * (x % 2)], key_piece(b, x / 2)[2 * (x % 2) + 1]}), q[x], s[b]);
        }
      float e[8], vs[8], lg = 0.f;
      if constexpr (FP8) lg = fminf(fmaxf(log2_fast(t.scale), -60.f), 60.f);
      each8([&](auto jj) {
        constexpr int j = decltype(jj)::value;
        e[j] = s[j >> 2][j & 3] * c;
        vs[j] = 1.f;
        if constexpr (FP8) {
          e[j] *= from16<j>(t.scale);
          vs[j] = from16<8 + j>(t.scale);
        }
      });
      if (t.bad != 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (t.bad >> (16 * g + j) & 1) e[j] = __builtin_nanf("");
      }
      if (key0 + kTile > key_end) {   // n copies of the last key: 1 / n of its weight each (none, and an infinite value would give NaN)
        const float share = log2_fast((float)(key0 + kTile - key_end + 1));
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (key0 + key_of(j, g) >= key_end - 1) e[j] -= share;
      }
      float top = m;
      each8([&](auto jj) {
        constexpr int j = decltype(jj)::value;
        if constexpr (FP8) top = fmaxf(top, e[j] + from16<8 + j>(lg));
        else top = fmaxf(top, e[j]);
      });
      top = max_rows16(top);
      const float peak = top == -__builtin_inff() ? 0.f : top, base = peak - (F16 ? kAbove16 : 0.f);
      if (__ballot(top != m) != 0) {   // some head's maximum has moved
        const float shrink = exp2_fast(m - peak);
        l *= shrink;
#pragma unroll
        for (int x = 0; x < SETS; ++x)
#pragma unroll
          for (int j = 0; j < 8; ++j) o[x][j] *= shrink;
        m = top;
      }
      float w[8], sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[j] = exp2_fast(e[j] - base);
        sum += w[j];
        if constexpr (FP8) w[j] *= vs[j];
      }
      l += sum;
      int first[4], second[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) split<F16>(w[2 * j], w[2 * j + 1], first[j], second[j]);
      const v4i pk = {first[0], first[1], first[2], first[3]}, rest = {second[0], second[1], second[2], second[3]};
#pragma unroll
      for (int x = 0; x < SETS; ++x) {
        v4i val[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (FP8) val[j] = widen<F16>(t.v[x][j]);
          else val[j] = t.v[x][j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          v4i a;   // channel 8 i + j of the lane's eight keys
#pragma unroll
          for (int y = 0; y < 4; ++y)
            a[y] = (int)__builtin_amdgcn_perm((uint32_t)val[2 * y + 1][j / 2], (uint32_t)val[2 * y][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
          o[x][j] = E::mfma16(a, rest, E::mfma16(a, pk, o[x][j]));
        }
      }
    };

    Tile ta, tb;
    Place next = places(key_begin);
    {
      const uint16_t* src = p.q.data + seq * p.q.token_stride + (int64_t)(head0 + min(i, heads - 1)) * p.q.head_stride;
#pragma unroll
      for (int x = 0; x < STEPS; ++x) {
        const int ch = 4 * kPer * (x / kPer) + kPer * g + x % kPer;
        q[x] = ch < chunks && i < heads ? *reinterpret_cast<const v4i*>(src + ch * 8) : v4i{0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int x = 0; x < SETS; ++x)
#pragma unroll
      for (int j = 0; j < 8; ++j) o[x][j] = v4f{};
    // Two tiles in registers and the pages of a third.  Loads come back in order: pages are asked for in front of the rows of the
    // tile before theirs, so that waiting for them waits for nothing younger.
    int key0 = key_begin;
    if (key0 < key_end) {
      Place after = places(key0 + kTile);
      load(ta, key0, next);
      while (true) {
        next = places(key0 + 2 * kTile);
        load(tb, key0 + kTile, after);
        compute(ta, key0);
        key0 += kTile;
        if (key0 >= key_end) break;
        after = places(key0 + 2 * kTile);
        load(ta, key0 + kTile, next);
        compute(tb, key0);
        key0 += kTile;
        if (key0 >= key_end) break;
      }
    }

    l = sum_rows16(l);
    const bool whole = n == tiles;
    const int slot = 2 * part.index + (at == part.begin ? 0 : 1);
    if (ln.joined && lane == 0) {
      int* ends = p.ends + 2 * (seq * (int64_t)ln.head_blocks + hb);
      if (tile0 == 0) ends[0] = slot;
      if (tile0 + n == tiles) ends[1] = slot;
    }
    if (i < heads) {   // lane (i, g) holds channels 128 x + 32 g + 8 r + j of head i in o[x][j][r]
      const int64_t row = (int64_t)seq * p.Hq + head0 + i;
      float* piece = p.partial + (int64_t)slot * (kHeads * (kDP + 2));
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int x = 0; x < SETS; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int ch = 128 * x + 32 * g + 8 * r;
          if (whole) {
            if (ch < p.D) {
              v4i v;
#pragma unroll
              for (int y = 0; y < 4; ++y) v[y] = (int)E::pack(o[x][2 * y][r] * inv, o[x][2 * y + 1][r] * inv);
              *reinterpret_cast<v4i*>(p.out + row * p.D + ch) = v;
            }
          } else {
            *reinterpret_cast<v4f*>(piece + i * kDP + ch) = v4f{o[x][0][r], o[x][1][r], o[x][2][r], o[x][3][r]};
            *reinterpret_cast<v4f*>(piece + i * kDP + ch + 4) = v4f{o[x][4][r], o[x][5][r], o[x][6][r], o[x][7][r]};
          }
        }
      if (g == 0) {
        if (whole) {
          p.lse[row] = l == 0.f ? -__builtin_inff() : (m + log2_fast(l) - (F16 ? kAbove16 : 0.f)) * kLn2;
        } else {
          piece[kHeads * kDP + i] = m;
          piece[kHeads * kDP + kHeads + i] = l;
        }
      }
    }

    at += n;
    if (at >= part.end) break;
    if (at - part.before == tiles * ln.head_blocks) {
      part.before = at;
      if (++seq >= p.sequences) break;
      len = length_of(p, seq);
    }
  }
}

// Joins the pieces of a head block where there is more than one: 3 to 6 us, most of it the launch and the two loads that wait for one
// another.  (A workgroup of eight waves per head block, joined in LDS in one launch, took 12.3 us for 700 keys and 55 for 4 sequences
// of 4096, against 9.2 and 19.6: too few waves load.)  Workgroup (x, y, z): `per` heads of head block z kRowGridX + x, from y * per on.  A team
// of kDP / 4 lanes, four channels each, sums the pieces of a head, or every n-th of them where there are fewer heads than teams.
typedef float v2f __attribute__((ext_vector_type(2)));
constexpr int kJoinThreads = 256;
template <bool F16, int SETS>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(DecodeArgs p, Line ln, int per) {
  using E = Elem<F16>;
  constexpr int kDP = 128 * SETS, kLanes = kDP / 4, kTeams = kJoinThreads / kLanes, kPiece = kHeads * (kDP + 2);
  __shared__ __attribute__((aligned(16))) float sums[kTeams][kDP];
  __shared__ v2f weights[kTeams];
  const int lane = threadIdx.x % kLanes, team = threadIdx.x / kLanes;
  const uint32_t block = blockIdx.z * (uint32_t)kRowGridX + blockIdx.x;
  const int seq = (int)divide(block, ln.by_head_blocks), hb = block - seq * ln.head_blocks;
  if (seq >= p.sequences) return;
  const int first = p.ends[2 * (int64_t)block], last = p.ends[2 * (int64_t)block + 1];
  if (first == last) return;   // one piece: its wave has written the result
  const int pieces = last / 2 - first / 2 + 1;
  const int kv_head = ln.per_kv == 1 ? hb : hb / ln.per_kv, from = (hb - kv_head * ln.per_kv) * kHeads, heads = min(ln.group - from, kHeads);
  const int h0 = blockIdx.y * per, hn = min(per, heads - h0);
  if (hn <= 0) return;
  // piece 0 lies in slot `first`, piece i in the first slot of its wave
  const auto piece = [&](int i) { return p.partial + (int64_t)(i == 0 ? first : (first & ~1) + 2 * i) * kPiece; };
  const int groups = hn == 1 ? kTeams : max(kTeams / hn, 1), share = min(hn, kTeams);
  const int group = share == 1 ? team : team / share, mine = team - group * share;   // (teams left over repeat the last group's work and store nothing)
  for (int h = h0 + mine; h < h0 + hn; h += share) {
    // One pass, a reference that follows the maximum: nothing that is loaded waits for anything but `ends`.
    float top = -__builtin_inff(), total = 0.f;
    v4f acc = {0.f, 0.f, 0.f, 0.f};
    const auto add = [&](float m, float l, v4f o) {
      const float next = fmaxf(top, m), base = next == -__builtin_inff() ? 0.f : next;
      const float a = exp2_fast(top - base), b = exp2_fast(m - base);
      total = total * a + l * b;
      acc = acc * a + o * b;
      top = next;
    };
#pragma unroll 4
    for (int i = group; i < pieces; i += groups)
      add(piece(i)[kHeads * kDP + h], piece(i)[kHeads * kDP + kHeads + h], *reinterpret_cast<const v4f*>(piece(i) + h * kDP + 4 * lane));
    if (groups > 1) {   // (then every head has its teams at once)
      *reinterpret_cast<v4f*>(&sums[team][4 * lane]) = acc;
      if (lane == 0) weights[team] = v2f{top, total};
      __syncthreads();
      if (group == 0)
        for (int i = 1; i < groups; ++i) add(weights[i * share + mine][0], weights[i * share + mine][1], *reinterpret_cast<const v4f*>(&sums[i * share + mine][4 * lane]));
    }
    if (group == 0) {
      const int64_t row = (int64_t)seq * p.Hq + kv_head * ln.group + from + h;
      const float inv = total == 0.f ? 0.f : 1.f / total;
      if (4 * lane < p.D)
        *reinterpret_cast<v2i*>(p.out + row * p.D + 4 * lane) = v2i{(int)E::pack(acc[0] * inv, acc[1] * inv), (int)E::pack(acc[2] * inv, acc[3] * inv)};
      if (lane == 0) p.lse[row] = total == 0.f ? -__builtin_inff() : (top + log2_fast(total) - (F16 ? kAbove16 : 0.f)) * kLn2;
    }
  }
}

Line line_of(int64_t sequences, int64_t Hq, int64_t Hkv, int64_t longest) {
  Line r;
  r.group = (int)(Hq / Hkv);
  r.per_kv = (r.group + kHeads - 1) / kHeads;
  r.head_blocks = (int)Hkv * r.per_kv;
  r.by_head_blocks = divider((uint32_t)r.head_blocks);
  const int64_t tiles = longest / kTile + 1;   // (longest + 1 keys, see length_of())
  const int64_t blocks = sequences * r.head_blocks, all = blocks * tiles;
  r.joined = longest > kWholeKeys && (longest > kMostWholeKeys || blocks < longest / 2);
  r.parts = (int)(!r.joined ? blocks : all < kMostParts ? all : kMostParts);   // at most; what there is of them the lengths decide
  return r;
}
int padded(int64_t D) { return D <= 128 ? 128 : 256; }

template <bool F16, Rows ROWS, int STEPS, int SETS>
hipError_t launch(const DecodeArgs& p, const Line& ln, hipStream_t s) {
  hipLaunchKernelGGL((decode_kernel<F16, ROWS, STEPS, SETS>), row_grid(ln.parts), dim3(64), 0, s, p, ln);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || !ln.joined) return e;
  // heads of a workgroup: as many as leave two workgroups per CU
  const int64_t blocks = (int64_t)p.sequences * ln.head_blocks;
  const int most = ln.group < kHeads ? ln.group : kHeads;
  int per = most;
  while (per > 1 && blocks * ((most + per - 1) / per) < 512) per = (per + 1) / 2;
  const dim3 lines = row_grid(blocks);
  hipLaunchKernelGGL((join_kernel<F16, SETS>), dim3(lines.x, (most + per - 1) / per, lines.y), dim3(kJoinThreads), 0, s, p, ln, per);
  return hipGetLastError();
}

template <bool F16, Rows ROWS>
hipError_t pick(const DecodeArgs& p, const Line& ln, hipStream_t s) {
  if (p.D <= 64) return launch<F16, ROWS, 2, 1>(p, ln, s);
  if constexpr (ROWS == kRows16Bit)
    if (p.D <= 96) return launch<F16, ROWS, 3, 1>(p, ln, s);
  if (p.D <= 128) return launch<F16, ROWS, 4, 1>(p, ln, s);
  if (p.D <= 192) return launch<F16, ROWS, 6, 2>(p, ln, s);
  return launch<F16, ROWS, 8, 2>(p, ln, s);
}
template <bool F16>
hipError_t pick_rows(const DecodeArgs& p, const Line& ln, hipStream_t s) {
  if (!p.fp8) return pick<F16, kRows16Bit>(p, ln, s);
  const int64_t* st = p.cache.k_stride;
  const bool by16 = p.D % 16 == 0 && (reinterpret_cast<uintptr_t>(p.cache.k) | st[0] | st[1] | st[2]) % 16 == 0;
  return by16 ? pick<F16, kRowsE4m3>(p, ln, s) : pick<F16, kRowsE4m3By8>(p, ln, s);
}

size_t partial_bytes(const Line& ln, int64_t D) { return (size_t)2 * ln.parts * kHeads * (padded(D) + 2) * sizeof(float); }

}  // namespace

size_t decode_workspace_bytes(int64_t sequences, int64_t Hq, int64_t Hkv, int64_t D, int64_t longest) {
  const Line ln = line_of(sequences, Hq, Hkv, longest);
  return ln.joined ? partial_bytes(ln, D) + (size_t)2 * sequences * ln.head_blocks * sizeof(int) : 0;
}

hipError_t launch_attention_decode(const DecodeArgs& args, hipStream_t s) {
  DecodeArgs p = args;
  const Line ln = line_of(p.sequences, p.Hq, p.Hkv, (int64_t)p.cache.table_width * p.cache.page_size.d);
  p.ends = (int*)((char*)p.partial + partial_bytes(ln, p.D));
  return p.dtype == 1 ? pick_rows<true>(p, ln, s) : pick_rows<false>(p, ln, s);
}

}  // namespace mslk_amd
