// Attention of one new token per sequence over a paged cache, keys and values in 16 bits or as e4m3 codes with a scale per row.
//
// The work is the stream of keys and values: a block of up to 16 query heads that share a KV head reads it once.  A wave takes
// 32 keys at a time straight from memory into the operands of v_mfma_f32_16x16x32: S^T = K Q^T has the keys as rows (lane (i, g)
// loads channels 8 g ... of key i), which leaves a lane eight scores of one head in the order in which exp2 of them is the second
// operand of O^T = V^T P^T; a lane of group g loads 8 channels of each of its eight keys of V and pairs them up in registers.
//
// The softmax runs in base 2 with reference m: P = 2^(c s - m), c = scale log2(e).  With e4m3 caches the weight of a key's codes
// is P times the value row's scale, so m is the maximum of c s + log2(scale): the weights stay at most 1 and keep their precision
// in 16 bits whatever the scales are.
//
// Keys are divided evenly whatever the lengths: every (sequence, head block) counts its keys in units, all units stand in one
// line, and workgroup i of W takes the i-th of W equal parts of the line.  Where a part begins or ends inside a (sequence, head
// block), what was summed there is written out in 32 bits, and a second launch joins the pieces in their order.
#include "attention.h"
#include "rows.h"

namespace mslk_amd {
namespace {

constexpr int kWaves = 4, kThreads = 64 * kWaves, kTile = 32, kUnit = kTile * kWaves, kHeads = 16;

struct Line {          // how the work is divided
  int head_blocks;     // per sequence: KV heads x blocks of kHeads query heads
  int per_kv;          // blocks of query heads per KV head
  int group;           // query heads per KV head
  int workgroups;
};

MSLK_AMD_DEVINL int64_t part_begin(int64_t total, int w, int workgroups) { return total * w / workgroups; }

// A length that the page table cannot hold counts as one key more than it holds: that key has no page.
MSLK_AMD_DEVINL int length_of(const DecodeArgs& p, int b) {
  const int64_t most = (int64_t)p.cache.table_width * p.cache.page_size.d + 1;
  return (int)min((int64_t)max(p.cache.lens[b], 0), min(most, (int64_t)1 << 30));
}
MSLK_AMD_DEVINL int units_of(int len) { return max(1, (len + kUnit - 1) / kUnit); }

MSLK_AMD_DEVINL int wave_scan(int v, int lane) {   // inclusive sum over the lanes
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int u = __shfl_up(v, d, 64);
    if (lane >= d) v += u;
  }
  return v;
}
MSLK_AMD_DEVINL int64_t total_units(const DecodeArgs& p) {   // of one head block, over the sequences
  const int lane = threadIdx.x & 63;
  int64_t sum = 0;
  for (int b = lane; b < p.sequences; b += 64) sum += units_of(length_of(p, b));
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) sum += __shfl_xor(sum, d, 64);
  return sum;
}
// Sequence that holds unit `unit` of the line (head_blocks times its units each), and the units in front of it.
MSLK_AMD_DEVINL int sequence_at(const DecodeArgs& p, const Line& ln, int64_t unit, int64_t& before) {
  const int lane = threadIdx.x & 63;
  before = 0;
  for (int base = 0; base < p.sequences; base += 64) {
    const int b = base + lane;
    const int n = b < p.sequences ? units_of(length_of(p, b)) : 0;
    const int upto = wave_scan(n, lane);
    const uint64_t hit = __ballot(unit < before + (int64_t)upto * ln.head_blocks);
    if (hit != 0) {
      const int src = __builtin_ctzll(hit);
      before += (int64_t)__shfl(upto - n, src, 64) * ln.head_blocks;
      return base + src;
    }
    before += (int64_t)__shfl(upto, 63, 64) * ln.head_blocks;
  }
  return p.sequences;   // beyond the line
}

// Two e4m3 codes -> two 16-bit values (exact).
template <bool F16>
MSLK_AMD_DEVINL v4i widen(v2i codes) {
  v4i r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(codes[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(codes[i], true);
    r[2 * i] = (int)Elem<F16>::pack(lo[0], lo[1]);
    r[2 * i + 1] = (int)Elem<F16>::pack(hi[0], hi[1]);
  }
  return r;
}

template <bool FP8> struct RowPiece;   // 8 channels of a row
template <> struct RowPiece<false> { typedef v4i type; };
template <> struct RowPiece<true> { typedef v2i type; };

// STEPS: channels of a key in steps of 32; SETS: channels of a value in sets of 128.
template <bool F16, bool FP8, int STEPS, int SETS>
struct Tile {
  using piece_t = typename RowPiece<FP8>::type;
  piece_t k[2][STEPS], v[SETS][8];
  float k_scale, v_scale;   // of key `lane` (FP8; lanes 0 ... 31)
  uint64_t bad;             // keys without a page
};

template <bool F16, bool FP8, int STEPS, int SETS>
__global__ __launch_bounds__(kThreads, STEPS <= 4 ? 2 : 1) void decode_kernel(DecodeArgs p, Line ln) {
  using E = Elem<F16>;
  using T = Tile<F16, FP8, STEPS, SETS>;
  using piece_t = typename T::piece_t;
  constexpr int kDP = 128 * SETS, kPitch = kDP + 4, kElem = FP8 ? 1 : 2;
  __shared__ __attribute__((aligned(16))) float sums[kWaves][kHeads][kPitch];
  __shared__ float tops[kWaves][kHeads], totals[kWaves][kHeads];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i = lane & 15, g = lane >> 4;
  const int chunks = p.D / 8;
  const float c = p.scale * kLog2e;

  const int64_t all = total_units(p) * ln.head_blocks;
  int64_t at = part_begin(all, blockIdx.x, ln.workgroups);
  const int64_t begin = at, end = part_begin(all, blockIdx.x + 1, ln.workgroups);
  if (at >= end) return;
  int64_t before;
  int seq = sequence_at(p, ln, at, before);
  if (seq >= p.sequences) return;

  while (at < end) {
    const int len = length_of(p, seq), units = units_of(len);
    const int hb = (int)((at - before) / units), unit0 = (int)((at - before) - (int64_t)hb * units);
    const int n_units = (int)min((int64_t)(units - unit0), end - at);
    const int kv_head = hb / ln.per_kv, first = (hb - kv_head * ln.per_kv) * kHeads, heads = min(ln.group - first, kHeads);
    const int head0 = kv_head * ln.group + first;
    const int key_begin = unit0 * kUnit, key_end = min(len, (unit0 + n_units) * kUnit);

    v4i q[STEPS];
    {
      const uint16_t* src = p.q.data + seq * p.q.token_stride + (int64_t)(head0 + min(i, heads - 1)) * p.q.head_stride;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const int ch = 4 * s + g;
        q[s] = ch < chunks && i < heads ? *reinterpret_cast<const v4i*>(src + ch * 8) : v4i{0, 0, 0, 0};
      }
    }
    const int32_t* table = p.cache.table + seq * p.cache.table_stride;
    const char* k_base = (const char*)p.cache.k + kv_head * p.cache.k_stride[2] * kElem;
    const char* v_base = (const char*)p.cache.v + kv_head * p.cache.v_stride[2] * kElem;

    v4f o[SETS][8];
#pragma unroll
    for (int x = 0; x < SETS; ++x)
#pragma unroll
      for (int j = 0; j < 8; ++j) o[x][j] = v4f{};
    float m = -__builtin_inff(), l = 0.f;

    // Place of key key0 + (lane & 31): keys beyond the end repeat the last one.
    struct Place { int page, slot; };
    auto place_of = [&](int key0) {
      const int key = min(key0 + (lane & 31), key_end - 1);
      const int index = (int)divide((uint32_t)key, p.cache.page_size);
      Place r;
      r.slot = key - index * (int)p.cache.page_size.d;
      r.page = index < p.cache.table_width ? table[index] : -1;
      return r;
    };
    auto load = [&](T& t, Place at_lane) {
      const bool lost = at_lane.page < 0 || at_lane.page >= p.cache.pages;
      t.bad = __ballot(lost) & 0xFFFFFFFFu;
      const int page = lost ? 0 : at_lane.page, slot = lost ? 0 : at_lane.slot;
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int pg = __shfl(page, 16 * b + i, 64), sl = __shfl(slot, 16 * b + i, 64);
        const char* row = k_base + ((int64_t)pg * p.cache.k_stride[0] + (int64_t)sl * p.cache.k_stride[1]) * kElem;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) t.k[b][s] = *reinterpret_cast<const piece_t*>(row + min(4 * s + g, chunks - 1) * 8 * kElem);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = (j & 3) + 4 * g + 16 * (j >> 2);
        const int pg = __shfl(page, key, 64), sl = __shfl(slot, key, 64);
        const char* row = v_base + ((int64_t)pg * p.cache.v_stride[0] + (int64_t)sl * p.cache.v_stride[1]) * kElem;
#pragma unroll
        for (int x = 0; x < SETS; ++x) t.v[x][j] = *reinterpret_cast<const piece_t*>(row + min(16 * x + i, chunks - 1) * 8 * kElem);
      }
      if constexpr (FP8) {
        const bool is_v = lane >= 32;
        const int64_t* st = is_v ? p.cache.v_scale_stride : p.cache.k_scale_stride;
        const float sc = (is_v ? p.cache.v_scale : p.cache.k_scale)[page * st[0] + slot * st[1] + kv_head * st[2]];
        t.k_scale = sc;   // lanes 0 ... 31: of the key, 32 ... 63: of the value
      }
    };
    auto compute = [&](const T& t, int key0) {
      v4f s[2] = {v4f{}, v4f{}};
#pragma unroll
      for (int x = 0; x < STEPS; ++x)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          if constexpr (FP8) s[b] = E::mfma16(widen<F16>(t.k[b][x]), q[x], s[b]);
          else s[b] = E::mfma16(t.k[b][x], q[x], s[b]);
        }
      float e[8], vs[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = (j & 3) + 4 * g + 16 * (j >> 2);
        e[j] = s[j >> 2][j & 3] * c;
        vs[j] = 1.f;
        if constexpr (FP8) {
          e[j] *= __shfl(t.k_scale, key, 64);
          vs[j] = __shfl(t.k_scale, key + 32, 64);
        }
        if (t.bad != 0 && (t.bad >> key & 1)) e[j] = __builtin_nanf("");
        if (key0 + key >= key_end) e[j] = -__builtin_inff();
      }
      float top = m;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (FP8) top = fmaxf(top, e[j] + fminf(fmaxf(log2_fast(vs[j]), -60.f), 60.f));
        else top = fmaxf(top, e[j]);
      }
      top = max_rows16(top);
      const float base = top == -__builtin_inff() ? 0.f : top;
      const float shrink = exp2_fast(m - base);
      m = top;
      float w[8], sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[j] = exp2_fast(e[j] - base);
        sum += w[j];
        if constexpr (FP8) w[j] = key0 + (j & 3) + 4 * g + 16 * (j >> 2) < key_end ? w[j] * vs[j] : 0.f;
      }
      l = l * shrink + sum;
      v4i pk;
#pragma unroll
      for (int j = 0; j < 4; ++j) pk[j] = (int)E::pack(w[2 * j], w[2 * j + 1]);
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
          o[x][j] *= shrink;
          o[x][j] = E::mfma16(a, pk, o[x][j]);
        }
      }
    };

    // two tiles in registers, the places of a third
    const int step = kTile * kWaves;
    int key0 = key_begin + wave * kTile;
    if (key0 < key_end) {
      T ta, tb;
      load(ta, place_of(key0));
      Place next = place_of(key0 + step);
      while (true) {
        load(tb, next);
        next = place_of(key0 + 2 * step);
        compute(ta, key0);
        key0 += step;
        if (key0 >= key_end) break;
        load(ta, next);
        next = place_of(key0 + 2 * step);
        compute(tb, key0);
        key0 += step;
        if (key0 >= key_end) break;
      }
    }

    // join the waves
    l = sum_rows16(l);
    if (g == 0) {
      tops[wave][i] = m;
      totals[wave][i] = l;
    }
    __syncthreads();
    float top = tops[0][i];
#pragma unroll
    for (int x = 1; x < kWaves; ++x) top = fmaxf(top, tops[x][i]);
    const float mine = m == -__builtin_inff() ? 0.f : exp2_fast(m - top);
#pragma unroll
    for (int x = 0; x < SETS; ++x)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const v4f v = {o[x][4 * y][r] * mine, o[x][4 * y + 1][r] * mine, o[x][4 * y + 2][r] * mine, o[x][4 * y + 3][r] * mine};
          *reinterpret_cast<v4f*>(&sums[wave][i][128 * x + (4 * g + r) * 8 + 4 * y]) = v;
        }
    __syncthreads();
    {
      const int h = threadIdx.x / 16, cl = threadIdx.x % 16;
      float t2 = tops[0][h];
#pragma unroll
      for (int x = 1; x < kWaves; ++x) t2 = fmaxf(t2, tops[x][h]);
      float total = 0.f;
#pragma unroll
      for (int x = 0; x < kWaves; ++x) total += tops[x][h] == -__builtin_inff() ? totals[x][h] : totals[x][h] * exp2_fast(tops[x][h] - t2);
      const bool whole = n_units == units;
      const int64_t slot = 2 * (int64_t)blockIdx.x + (at == begin ? 0 : 1);
      float* part = p.partial + slot * (kHeads * (kDP + 2));
      if (h < heads) {
        const int64_t out_row = (int64_t)seq * p.Hq + head0 + h;
        const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
        for (int x = 0; x < SETS; ++x) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[e] = 0.f;
#pragma unroll
            for (int y = 0; y < kWaves; ++y) v[e] += sums[y][h][128 * x + cl * 8 + e];
          }
          const int ch = 128 * x + cl * 8;
          if (whole) {
            if (ch < p.D)
              *reinterpret_cast<v4i*>(p.out + out_row * p.D + ch) = v4i{(int)E::pack(v[0] * inv, v[1] * inv), (int)E::pack(v[2] * inv, v[3] * inv),
                                                                        (int)E::pack(v[4] * inv, v[5] * inv), (int)E::pack(v[6] * inv, v[7] * inv)};
          } else {
            *reinterpret_cast<v4f*>(part + h * kDP + ch) = v4f{v[0], v[1], v[2], v[3]};
            *reinterpret_cast<v4f*>(part + h * kDP + ch + 4) = v4f{v[4], v[5], v[6], v[7]};
          }
        }
        if (cl == 0) {
          if (whole) {
            p.lse[out_row] = total == 0.f ? -__builtin_inff() : (t2 + log2_fast(total)) * kLn2;
          } else {
            part[kHeads * kDP + h] = t2;
            part[kHeads * kDP + kHeads + h] = total;
          }
        }
      }
    }
    __syncthreads();   // the LDS is written again

    at += n_units;
    if (at - before == (int64_t)units * ln.head_blocks) {
      before = at;
      ++seq;
      if (seq >= p.sequences) break;
    }
  }
}

// Sequence blockIdx.y, query head blockIdx.x: joins the pieces of its line where there is more than one.
template <bool F16, int SETS>
__global__ __launch_bounds__(64) void join_kernel(DecodeArgs p, Line ln) {
  using E = Elem<F16>;
  constexpr int kDP = 128 * SETS;
  const int lane = threadIdx.x, head = blockIdx.x, seq = blockIdx.y;
  int64_t before = 0, total = 0;
  for (int b = lane; b < p.sequences; b += 64) {
    const int n = units_of(length_of(p, b));
    total += n;
    if (b < seq) before += n;
  }
#pragma unroll
  for (int d = 32; d >= 1; d /= 2) {
    total += __shfl_xor(total, d, 64);
    before += __shfl_xor(before, d, 64);
  }
  total *= ln.head_blocks;
  const int units = units_of(length_of(p, seq));
  const int kv_head = head / ln.group, in_group = head - kv_head * ln.group, hb = kv_head * ln.per_kv + in_group / kHeads, h = in_group % kHeads;
  const int64_t from = before * ln.head_blocks + (int64_t)hb * units, to = from + units;
  // first workgroup whose part holds unit `from`: the largest w with total * w / W <= from
  const int W = ln.workgroups;
  int w = (int)(((from + 1) * W - 1) / total);
  if (part_begin(total, w + 1, W) >= to) return;   // one piece: written by its workgroup
  float m = -__builtin_inff(), l = 0.f;
  v2f acc[SETS];
#pragma unroll
  for (int x = 0; x < SETS; ++x) acc[x] = v2f{0.f, 0.f};
  for (; w < W; ++w) {
    const int64_t b = part_begin(total, w, W);
    if (b >= to) break;
    if (part_begin(total, w + 1, W) == b) continue;   // an empty part
    const float* part = p.partial + (2 * (int64_t)w + (b >= from ? 0 : 1)) * (kHeads * (kDP + 2));
    const float pm = part[kHeads * kDP + h], pl = part[kHeads * kDP + kHeads + h];
    const float top = fmaxf(m, pm), base = top == -__builtin_inff() ? 0.f : top;
    const float f = exp2_fast(m - base), pf = exp2_fast(pm - base);
    l = l * f + pl * pf;
    m = top;
#pragma unroll
    for (int x = 0; x < SETS; ++x) {
      const v2f v = *reinterpret_cast<const v2f*>(part + h * kDP + 128 * x + 2 * lane);
      acc[x] = acc[x] * f + v * pf;
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t row = (int64_t)seq * p.Hq + head;
#pragma unroll
  for (int x = 0; x < SETS; ++x) {
    const int ch = 128 * x + 2 * lane;
    if (ch < p.D) *reinterpret_cast<uint32_t*>(p.out + row * p.D + ch) = E::pack(acc[x][0] * inv, acc[x][1] * inv);
  }
  if (lane == 0) p.lse[row] = l == 0.f ? -__builtin_inff() : (m + log2_fast(l)) * kLn2;
}

struct Plan {
  Line line;
  bool joined;   // whether a line may be cut
};
Plan plan_of(int64_t sequences, int64_t Hq, int64_t Hkv, int64_t longest) {
  Plan r;
  r.line.group = (int)(Hq / Hkv);
  r.line.per_kv = (r.line.group + kHeads - 1) / kHeads;
  r.line.head_blocks = (int)Hkv * r.line.per_kv;
  const int64_t units = longest / kUnit + 1;   // (longest + 1 keys, see length_of())
  const int64_t all = sequences * r.line.head_blocks * units, most = 512;
  r.line.workgroups = (int)(all < most ? all : most);
  r.joined = units > 1;
  return r;
}
int padded(int64_t D) { return D <= 128 ? 128 : 256; }

template <bool F16, bool FP8, int STEPS, int SETS>
hipError_t launch(const DecodeArgs& p, const Plan& plan, hipStream_t s) {
  hipLaunchKernelGGL((decode_kernel<F16, FP8, STEPS, SETS>), dim3(plan.line.workgroups), dim3(kThreads), 0, s, p, plan.line);
  if (hipError_t e = hipGetLastError(); e != hipSuccess || !plan.joined) return e;
  hipLaunchKernelGGL((join_kernel<F16, SETS>), dim3(p.Hq, p.sequences), dim3(64), 0, s, p, plan.line);
  return hipGetLastError();
}

template <bool F16, bool FP8>
hipError_t pick(const DecodeArgs& p, const Plan& plan, hipStream_t s) {
  if (p.D <= 64) return launch<F16, FP8, 2, 1>(p, plan, s);
  if (p.D <= 96) return launch<F16, FP8, 3, 1>(p, plan, s);
  if (p.D <= 128) return launch<F16, FP8, 4, 1>(p, plan, s);
  if (p.D <= 192) return launch<F16, FP8, 6, 2>(p, plan, s);
  return launch<F16, FP8, 8, 2>(p, plan, s);
}

int64_t longest_of(int64_t table_width, int64_t page_size) {
  const int64_t n = table_width * page_size;
  return n < (int64_t(1) << 30) ? n : int64_t(1) << 30;
}

}  // namespace

size_t decode_workspace_bytes(int64_t sequences, int64_t Hq, int64_t Hkv, int64_t D, int64_t longest) {
  const Plan plan = plan_of(sequences, Hq, Hkv, longest_of(longest, 1));
  return plan.joined ? (size_t)2 * plan.line.workgroups * kHeads * (padded(D) + 2) * sizeof(float) : 0;
}

hipError_t launch_attention_decode(const DecodeArgs& p, hipStream_t s) {
  const Plan plan = plan_of(p.sequences, p.Hq, p.Hkv, longest_of(p.cache.table_width, p.cache.page_size.d));
  if (p.dtype == 1) return p.fp8 ? pick<true, true>(p, plan, s) : pick<true, false>(p, plan, s);
  return p.fp8 ? pick<false, true>(p, plan, s) : pick<false, false>(p, plan, s);
}

}  // namespace mslk_amd
