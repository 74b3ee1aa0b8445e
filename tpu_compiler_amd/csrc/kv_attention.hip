// Attention to a key/value cache of 4 or 8 bits: single tokens, a few tokens and prompts, over all tokens or a window and the first ones.
#include "kv_cache.hpp"

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

namespace tpuhip {

struct AttentionArgs {
  const uint8_t *data;
  const int32_t *q_starts, *kv_lens, *table;
  const uint16_t *q;
  uint16_t *out;
  float *part, *part_ml;        // of each split and row: DP sums; the maximum and the sum of the weights
  int *counters;                // of each tile: splits that have ended; NULL: another kernel joins them
  int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;
  FastDiv group, units_per_page, kv_heads;
  int heads, dim, pages, table_stride;
  int total_q, max_q, max_kv, window, sinks, bf16;
  FastDiv split_count;
  FastDiv class_heads;          // cache heads of a class of XCDs
  int classes, works, n_seq, one_tile;   // works: workgroups of a class
  int splits, chunk;            // a split takes `chunk` units of those that a wave's rows see (where all waves of a workgroup have the same)
  float scale;
};

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint2u __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t uint4u __attribute__((ext_vector_type(4), aligned(2)));   // memory takes any address

__device__ __forceinline__ float load16(uint32_t b, int bf16) {
  return bf16 ? bf16_to_f32(b & 0xFFFF) : (float)__builtin_bit_cast(_Float16, (uint16_t)b);
}
__device__ __forceinline__ uint32_t store16(float v, int bf16) {
  return bf16 ? __builtin_bit_cast(uint16_t, (__bf16)v) : __builtin_bit_cast(uint16_t, (_Float16)v);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2v){a, b}, half2v));
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2v){a, b}, bf16x2));
}
// two floats past the caches that a device's XCDs have of their own
__device__ __forceinline__ void store2(float *p, float x, float y) {
  __hip_atomic_store((uint64_t *)p, __builtin_bit_cast(uint64_t, (float2v){x, y}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2v load2(const float *p) {
  return __builtin_bit_cast(float2v, __hip_atomic_load((const uint64_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}
__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }

// inclusive sums over the lanes of a wave
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int sums_upto(int v) {
  v = dpp_add<0x111, 0xf>(v);                                  // from 1, 2, 4 and 8 lanes below in each 16,
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);                                  // from lane 15 to 16..31 and 47 to 48..63,
  return dpp_add<0x143, 0xc>(v);                               // from lane 31 to 32..63
}

// the largest of a wave's numbers, in a scalar register
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = dpp_max<0xB1>(v);                                        // of lanes 1 and 2 apart, of halves of 16 and of 16 turned round,
  v = dpp_max<0x4E>(v);
  v = dpp_max<0x141>(v);
  v = dpp_max<0x140>(v);
  const auto of = [&](int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
  return max(max(of(0), of(16)), max(of(32), of(48)));
}

// f over the four lanes of a column, 16 apart
template <typename F>
__device__ __forceinline__ float over_column(float v, F f) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float column_max(float v) {
  return over_column(v, [](float x, float y) { return fmaxf(x, y); });
}
__device__ __forceinline__ float column_sum(float v) {
  return over_column(v, [](float x, float y) { return x + y; });
}

// A tile of R rows of a sequence, the `slot`th of those of all sequences: which sequence, its first query, how many it has, the position
// of the first.  A lane counts the tiles of a sequence; the host knows a bound of their number only, and tile is -1 where there are
// fewer.  With one tile a sequence at most, the slot is the sequence.
struct Tile {
  int seq, tile, begin, n, first;
  template <int R>
  __device__ __forceinline__ static Tile find(const AttentionArgs &a, int slot) {
    Tile t;
    if (a.one_tile) {
      t.seq = slot;
      t.look_up(a);
      t.tile = t.n > 0 ? 0 : -1;
      return t;
    }
    for (int first = 0; first < a.n_seq; first += 64) {
      t.seq = min(first + ((int)threadIdx.x & 63), a.n_seq - 1);
      t.look_up(a);
      const int tiles = first + ((int)threadIdx.x & 63) < a.n_seq ? (t.n * (int)a.group.d + R - 1) / R : 0, upto = sums_upto(tiles);
      if (const uint64_t there = __ballot(upto > slot)) {
        const int at = __builtin_ctzll(there);
        return {first + at, __builtin_amdgcn_readlane(upto, at) - 1 - slot,   // the last tiles, which see the most, begin first
                __builtin_amdgcn_readlane(t.begin, at), __builtin_amdgcn_readlane(t.n, at), __builtin_amdgcn_readlane(t.first, at)};
      }
      slot -= __builtin_amdgcn_readlane(upto, 63);
    }
    return {0, -1, 0, 0, 0};
  }
  // the same in all lanes, for the compiler
  __device__ __forceinline__ Tile uniform() const {
    return {__builtin_amdgcn_readfirstlane(seq), __builtin_amdgcn_readfirstlane(tile), __builtin_amdgcn_readfirstlane(begin),
            __builtin_amdgcn_readfirstlane(n), __builtin_amdgcn_readfirstlane(first)};
  }
  __device__ __forceinline__ void look_up(const AttentionArgs &a) {
    begin = min(max(a.q_starts[seq], 0), a.total_q);
    n = min(min(max(a.q_starts[seq + 1], begin), a.total_q) - begin, a.max_q);
    first = min(max(a.kv_lens[seq], 0), a.max_kv) - n;
  }
};

// The units that rows at positions lo..hi see some token of: those of the first tokens, then those of the window up to hi.
struct UnitList {
  int sinks, low, count;
  __device__ __forceinline__ UnitList(const AttentionArgs &a, int lo, int hi) {
    low = a.window ? max(0, lo - a.window + 1) / kUnitTokens : 0;
    sinks = a.window ? min((a.sinks + kUnitTokens - 1) / kUnitTokens, low) : 0;
    count = hi < 0 ? 0 : sinks + hi / kUnitTokens - low + 1;
  }
  __device__ __forceinline__ int block(int i) const { return i < sinks ? i : low + i - sinks; }
};

constexpr int kAttentionWaves = 4, kXcds = 8;
constexpr int kMostTokens = 1 << 30;  // of a sequence: sums and differences of two positions are ints
constexpr float kNothing = -__FLT_MAX__;   // the maximum of no scores: below that of any
constexpr int kJoinAtOnce = 8;       // splits whose sums are loaded together
constexpr int kJoinWaves = 16;

// A wave takes 16 NC rows (a row: a query and one of the heads that share a cache head) and units of 32 tokens:
//   S^T = K Q^T   tokens x rows:    a lane has one row (of each 16) and the tokens 4g..4g+3, 16+4g..16+4g+3 of a unit, g = lane / 16
//   O^T = V^T P^T channels x rows:  which are just the lane's elements of the right operand here, so nothing is exchanged
// The left operands are the codes themselves: masked out of a dword, two of them are a pair of subnormal float16 numbers
// c 2^-24 (of a byte's upper half c 2^-20), which the matrix unit takes as they are and multiplies exactly.  Steps and offsets are applied to
// what is small: x = s_t (q.c_t) + m_t sum(q) to the scores, and P'_t = p_t s_t to the weights, with sum(p_t m_t) added to all channels.
// Scores, maxima and sums are 32 bits.  Weights times steps are rounded to float16, as the matrix unit takes no wider ones at this rate: against 64 bits
// a result's RMS error is 1.005 times that of its own rounding in bfloat16 and 1.06 times in float16 (a token to 513; to 8192 1.002 and 1.02).
// Of a workgroup's four waves, WR have rows of their own; the 4 / WR with the same rows take every so manieth unit and join their sums in LDS.
//
// Bounds.  Few rows: memory.  A unit of 128 channels in 4 bits is 4352 bytes, read once, straight into the lanes that multiply it (no
// barrier in the loop): one token for each of 64 sequences of 61 to 8192, 288 MB, takes 68 us, 4.3 TB/s (a copy moves 4.8, reading alone reaches
// 6.0); for one of 131072, 143 MB, 28 us and 4.5 for the join.  Many rows: the vector ALU.  A unit costs a wave 80 instructions to unpack and
// 7 a score (two fused products, half a maximum, an exponential, a sum, a step, an offset, half a conversion), 238 for 32 rows against 32
// matrix instructions of 16 cycles; 8192 tokens of 32 heads, causal, 0.55 TFLOP, take 588 us, 935 TFLOP/s, 77 % of a large float16 product,
// with the vector ALU busy for 83 % of the time and the matrix unit for 37 %.  More rows a wave would amortise unpacking, but 48 of 128 channels need the queries in LDS,
// all registers, and gained 2 %; fewer, 16, have three waves a SIMD and take 709 us.
// In between, latency: a SIMD with one wave issues a vector instruction every eight clocks instead of four to five, and a unit of 32 rows takes it
// 0.95 us, where two waves take 1.13 for one each.  Multiplying the next unit's keys before this one's scores, and handing on its params, took nothing
// off that and 5 % more where memory bounds.  A wave's way in and out is four units' worth of instructions.
template <typename U, int NC, int WR>
__global__ __launch_bounds__(64 * kAttentionWaves, 2) void kv_attention_kernel(AttentionArgs a) {
  constexpr int DP = U::kDim, KD = U::kRow / 16, STEPS = DP / 32, OB = DP / 16, WK = kAttentionWaves / WR;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const int group = (int)a.group.d;
  // Workgroups go to the XCDs in turn.  An XCD, or the 2, 4 or 8 of a class where there are fewer heads, takes every so manieth cache head
  // of all sequences: an L2 holds the keys and values that the workgroups on it read at a time, and sequences of any lengths
  // are shared out evenly.
  const uint32_t xcd = blockIdx.x % kXcds, of_head = xcd & (a.classes - 1);
  uint32_t work = blockIdx.x / kXcds * (kXcds / a.classes) + xcd / a.classes;
  if (work >= (uint32_t)a.works) return;
  uint32_t slot = a.class_heads.split(work);                   // the first tile of all heads, then the second one, ...
  const int kvh = (int)(work * a.classes + of_head);
  constexpr bool SPLIT = WR == 1;                              // the others are for rows enough: a tile's units are one workgroup's
  int split = 0;
  if constexpr (SPLIT) {
    split = (int)slot;
    slot = a.split_count.div(slot);
    split -= (int)(slot * a.split_count.d);
  }
  const Tile seq = Tile::find<16 * NC * WR>(a, (int)slot).uniform();
  const int tile = seq.tile, rows = seq.n * group;
  if (tile < 0) return;
  const int row0 = (tile * WR + wave / WK) * 16 * NC;
  if (WK == 1 && row0 >= rows) return;                         // the waves share nothing
  const int p_lo = seq.first + (int)a.group.div(row0), p_hi = seq.first + (int)a.group.div(max(min(row0 + 16 * NC, rows), 1) - 1);
  const UnitList list(a, p_lo, row0 < rows ? p_hi : -1);
  int i = 0, end = list.count, splits = 1;
  if constexpr (SPLIT) {
    i = split * a.chunk;
    end = min(end, i + a.chunk);
    if (split > 0 && i >= end) return;                         // no such split: what joins them counts them the same way
    splits = max(1, (list.count + a.chunk - 1) / a.chunk);     // that there are
  }
  i += wave % WK;

  // ---- queries
  int pos[NC];
  uint4v q[NC][STEPS];
#pragma unroll
  for (int nc = 0; nc < NC; ++nc) {
    uint32_t h = min(row0 + nc * 16 + col, rows - 1);           // past the last row: that one again, to be thrown away
    const int token = (int)a.group.split(h);
    pos[nc] = seq.first + token;
    const uint16_t *src = a.q + (int64_t)(seq.begin + token) * a.q_token_stride + (int64_t)(kvh * group + (int)h) * a.q_head_stride;
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      const int c0 = g * (DP / 4) + st * 8;
      uint4v raw = {0, 0, 0, 0};
      if (a.dim >= 8) {                                         // the last eight channels in place of eight that are not all there
        const int at = min(c0, a.dim - 8);
        raw = *(const uint4u *)(src + at);
        if (a.dim % 8 && at < c0) {
          const int by = min(c0 - at, 7) * 16;
          const uint64_t low = raw[0] | (uint64_t)raw[1] << 32, high = raw[2] | (uint64_t)raw[3] << 32;
          const uint64_t down = by < 64 ? low >> by | high << 1 << (63 - by) : high >> (by - 64), up = by < 64 ? high >> by : 0;
          raw = (uint4v){(uint32_t)down, (uint32_t)(down >> 32), (uint32_t)up, (uint32_t)(up >> 32)};
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) raw[e / 2] |= (e < a.dim ? src[min(e, a.dim - 1)] : 0u) << 16 * (e & 1);
      }
      q[nc][st] = raw;
    }
  }
  // ---- units: each lane looks up one of the wave's next 64
  int held = 0, held_at = -64 * WK;
  const auto unit_at = [&](int at) -> int {                    // -1: none
    if (at >= end) return -1;
    if (at >= held_at + 64 * WK) {
      held_at = at;
      const int mine = at + lane * WK;
      held = -1;
      if (mine < end) {
        uint32_t in_page = list.block(mine);
        const int page = a.table[(int64_t)seq.seq * a.table_stride + a.units_per_page.split(in_page)];
        if ((unsigned)page < (unsigned)a.pages) held = page * (int)a.units_per_page.d + (int)in_page;
      }
    }
    return __builtin_amdgcn_readlane(held, (at - held_at) / WK);
  };
  const auto address = [&](int unit) { return a.data + ((int64_t)max(unit, 0) * a.kv_heads.d + kvh) * U::kBytes; };
  uint32_t k_raw[2][KD], v_raw[U::kBlocks][2], param;         // of the unit that comes next
  const auto load_k = [&](const uint8_t *u) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t *at = (const uint32_t *)(u + (h * 16 + col) * U::kRow + g * (U::kRow / 4));
#pragma unroll
      for (int d = 0; d < KD; ++d) k_raw[h][d] = at[d];
    }
  };
  const auto load_params = [&](const uint8_t *u) { param = ((const uint32_t *)(u + U::kParams))[lane]; };
  const auto load_v = [&](const uint8_t *u) {
    u += U::kCodes;
    if constexpr (U::kPaired) {
#pragma unroll
      for (int b = 0; b < U::kBlocks; b += 2) {
        const uint4v w = *(const uint4v *)(u + b / 2 * 1024 + lane * 16);
        v_raw[b][0] = w[0], v_raw[b][1] = w[1], v_raw[b + 1][0] = w[2], v_raw[b + 1][1] = w[3];
      }
    } else {
#pragma unroll
      for (int b = 0; b < U::kBlocks; ++b) {
        const uint2 w = *(const uint2 *)(u + b * 512 + lane * 8);
        v_raw[b][0] = w.x, v_raw[b][1] = w.y;
      }
    }
  };

  // Loads are waited for in the order of their issue: params for the next unit go out when this one's have been handed on, keys when they have
  // been multiplied, then values, each a good part of a unit's work before they are used.  The compiler has to keep the order (it would
  // issue the params last, and wait for the values with the keys).
  const auto in_order = [] { asm volatile("" ::: "memory"); };
  int unit = unit_at(i);
  {
    const uint8_t *u = address(unit);
    load_params(u);
    in_order();
    load_k(u);
    in_order();
    load_v(u);
    in_order();
  }

  // ---- queries as the matrix unit takes them, while the first unit is on its way: the wave's times one power of two, the largest number
  // just below 2^15.  float16 holds all bits of those within 2^24 of it, and of smaller ones a multiple of 2^-38 of it.  A number past the
  // bounds of the exponent becomes an infinity, in its own row.
  ushort2v most2 = {0, 0};                                      // magnitudes are in order as integers
#pragma unroll
  for (int nc = 0; nc < NC; ++nc)
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      if (g * (DP / 4) + st * 8 >= a.dim) q[nc][st] = (uint4v){0, 0, 0, 0};
#pragma unroll
      for (int d = 0; d < 4; ++d) most2 = __builtin_elementwise_max(most2, __builtin_bit_cast(ushort2v, q[nc][st][d] & 0x7FFF7FFF));
    }
  const uint32_t infinite = a.bf16 ? 0x7F80 : 0x7C00;
  uint32_t most = max((uint32_t)most2[0], (uint32_t)most2[1]);
  if (__any(most >= infinite)) {                                // those are not to count
    most = 0;
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
      for (int st = 0; st < STEPS; ++st)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t v = q[nc][st][e / 2] >> 16 * (e & 1) & 0x7FFF;
          most = max(most, v < infinite ? v : 0u);
        }
  }
  most = wave_max(most);
  const int e2 = min(max((int)(__float_as_uint(load16(most, a.bf16)) >> 23) - 127 - 14, -100), 88);
  const float down = __uint_as_float((uint32_t)(127 - e2) << 23);
  const auto queries = [&](auto is_bf16) {
    constexpr int bf16 = decltype(is_bf16)::value;
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)   // odd channels lie in the upper halves of 4-bit bytes, 16 times their size
          v[e] = load16(q[nc][st][e / 2] >> 16 * (e & 1), bf16) * (U::kBits == 4 && e & 1 ? down / 16 : down);
        // in the order of the codes' pairs
        q[nc][st] = U::kBits == 4 ? (uint4v){pack_f16(v[0], v[4]), pack_f16(v[1], v[5]), pack_f16(v[2], v[6]), pack_f16(v[3], v[7])}
                                  : (uint4v){pack_f16(v[0], v[2]), pack_f16(v[1], v[3]), pack_f16(v[4], v[6]), pack_f16(v[5], v[7])};
      }
  };
  if (a.bf16)
    queries(std::true_type{});
  else
    queries(std::false_type{});
  // their sums, of the same rounded numbers: a token whose codes are all one
  float q_sum[NC];
  constexpr uint32_t one = 0x3C003C00, odd = U::kBits == 4 ? 0x4C004C00 : one;
#pragma unroll
  for (int nc = 0; nc < NC; ++nc) {
    float4v sum = {0, 0, 0, 0};
#pragma unroll
    for (int st = 0; st < STEPS; ++st)
      sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, (uint4v){one, odd, one, odd}), __builtin_bit_cast(half8, q[nc][st]), sum, 0, 0, 0);
    q_sum[nc] = ldexpf(sum[0], e2);
  }
  const float log2e = 1.44269504088896341f;
  const float offset_scale = a.scale * log2e, step_scale = ldexpf(offset_scale, e2 + 24);


  // ---- the sums
  float top[NC], limit[NC], total[NC], offsets[NC];   // limit: a score above it, relative to the maximum, raises that
  float4v o[OB][NC];
  // The rounding of weights times steps counts as much as the codes do, also where codes and offsets cancel.  For a float16 result it counts by the codes'
  // distance from their middle: sums of the rounded weights make o that of codes less the middle, which goes to the offsets, whose weights are not
  // rounded.  Of the RMS error of a token to 513, beside that of the result's own rounding, that leaves 0.35 of 1.03.  For bfloat16, whose own is eight
  // times as large, it is a tenth of it as it is, and four instructions for eight scores would be for nothing.
  const float middle = a.bf16 ? 0.0f : U::kLevels / 2.0f;
  float rounded[NC];
#pragma unroll
  for (int nc = 0; nc < NC; ++nc) {
    rounded[nc] = 0;
    top[nc] = 0;
    limit[nc] = -INFINITY;                                      // the row has seen nothing
    total[nc] = offsets[nc] = 0;
#pragma unroll
    for (int b = 0; b < OB; ++b) o[b][nc] = (float4v){0, 0, 0, 0};
  }
  // Steps of the values are taken times a power of two, the same for a wave: 2^8 to 2^10 for the largest that any row has seen.  Weights up
  // to 2^5 (of a maximum that lags) times these are below float16's 65504.  A row that has seen only far smaller ones, as the large ones
  // are hidden from it, has a maximum that is lower by its `lift`, so that its weights are larger by a power of two (limit: kLag and that):
  // a row's own largest step is 2^5 or more, with what float16 loses of subnormal weights 2^-30 of it.
  // An offset counts as a step of 2^-14 of it: what is rounded beside it is far below its own rounding, and its sum stays in bounds.
  const auto power = [](int e) { return __uint_as_float((uint32_t)min(max(e + 127, 0), 254) << 23); };
  const auto exponent = [](uint32_t bits) { return (int)(bits >> 23) - 127; };
  const auto size_of = [](float step, float offset) { return fmaxf(step, fabsf(offset) * 0x1p-14f); };   // of an offset that is a NaN, 0
  int v_exp = 0;
  float v_scale = 1, size_limit = 0;                            // size_limit: a token above it may not fit; 0: none so far
  uint32_t most_seen = 0;                                       // by any row; numbers that are not negative are in order as integers
  bool uneven = false;                                          // whether rows have seen different ones: the largest of each is in row_size
  constexpr int kMostSteps = 10, kLeastLift = 4, kMostLift = 100;
  constexpr float kLag = 5;

  __shared__ __attribute__((aligned(16))) float params[kAttentionWaves][128];
  __shared__ float row_size[kAttentionWaves][NC * 16];
  const int window = a.window ? a.window : kMostTokens;
  // A maximum or a step has gone up, which it seldom does after the first units: what has been summed, and this unit's scores, relative to
  // the new ones.  step, size: of the lane's token.
  const auto rescale = [&](int t0, bool all, float step, float size, float (&high)[NC], float4v (&s)[2][NC], float (&vs)[8], const float (&vm)[8]) {
    const auto steps = [&](float scale) {                       // from the steps themselves: with the scale so far they may be infinite
      if (lane >= 32) params[wave][lane] = step * scale;
#pragma unroll
      for (int h = 0; h < 2; ++h) *(float4v *)(vs + h * 4) = *(const float4v *)&params[wave][32 + h * 16 + g * 4];
    };
    const bool scaled = size_limit > 0;
    float lift[NC], v_change = 1;
    bool sizes = !scaled || ((size > size_limit) & (lane >= 32));
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      high[nc] = column_max(high[nc]);
      lift[nc] = fmaxf(limit[nc] - kLag, 0);
      sizes |= limit[nc] < 0 && high[nc] > -INFINITY;           // a row that begins to see
    }
    if (__any(sizes)) {
      float seen_size[NC];
#pragma unroll
      for (int nc = 0; nc < NC; ++nc) seen_size[nc] = uneven ? row_size[wave][nc * 16 + col] : __uint_as_float(most_seen);
      const int t = t0 + lane - 32;                             // the lane's token, and whether any row sees it
      const bool there = lane >= 32 && t <= p_hi && (t > p_lo - window || t < a.sinks);
      const uint32_t largest = wave_max(there ? __float_as_uint(size) : 0);
      const auto least = [&] { return ~wave_max(there ? ~__float_as_uint(size) : 0); };
      if (all || p_lo == p_hi) {                                // all rows see the same of the unit
        most_seen = max(most_seen, largest);
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) seen_size[nc] = fmaxf(seen_size[nc], __uint_as_float(largest));
      } else if (const uint32_t low = least(); exponent(max(most_seen, largest)) - exponent(low) < kLeastLift) {
        uneven = true;                                          // or about the same, if any, and so near the largest that no row which does is lifted
        most_seen = max(most_seen, largest);
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) seen_size[nc] = high[nc] > -INFINITY ? fmaxf(seen_size[nc], __uint_as_float(low)) : seen_size[nc];
      } else {
        uneven = true;
        if (scaled) steps(1);
        uint32_t most = 0;
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
          float sees = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) sees = s[j / 4][nc][j & 3] > -INFINITY ? fmaxf(sees, size_of(vs[j], vm[j])) : sees;
          seen_size[nc] = fmaxf(seen_size[nc], column_max(sees));
          most = max(most, __float_as_uint(seen_size[nc]));
        }
        most_seen = max(most_seen, wave_max(most));
      }
      if (most_seen && (!scaled || exponent(most_seen) + v_exp >= kMostSteps)) {
        const int now = min(8 - exponent(most_seen), 99);
        v_change = power(now - v_exp);
        v_exp = now;
        v_scale = power(now);
      }
      if (scaled) {
        steps(v_scale);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) vs[j] *= v_scale;
      }
      if (!all) {
#pragma unroll
        for (int j = 0; j < 8; ++j) vs[j] = fminf(vs[j], 0x1p15f);   // of a hidden one, whose weight is 0
      }
      int most_lift = 0;
      if (uneven) {
#pragma unroll
        for (int nc = 0; nc < NC; ++nc) {
          row_size[wave][nc * 16 + col] = seen_size[nc];
          const int by = seen_size[nc] > 0 ? 8 - exponent(__float_as_uint(seen_size[nc])) - v_exp : 0;
          lift[nc] = by < kLeastLift ? 0.0f : (float)min(by, kMostLift);
          most_lift = max(most_lift, (int)lift[nc]);
        }
        if (__any(most_lift)) most_lift = (int)wave_max(most_lift);
      }
      if (most_seen) size_limit = power(kMostSteps - v_exp - __builtin_amdgcn_readfirstlane(most_lift));
    }
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      const bool first = limit[nc] < 0, some = high[nc] > -INFINITY;
      const float up = (first ? some ? high[nc] : 0.0f : fmaxf(high[nc], limit[nc] - kLag)) - lift[nc], change = first ? 1.0f : exp2_fast(-up);
      limit[nc] = some || !first ? kLag + lift[nc] : limit[nc];
      top[nc] += up;
      total[nc] *= change;
      offsets[nc] *= change;
      rounded[nc] *= change * v_change;
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j / 4][nc][j & 3] -= up;
#pragma unroll
      for (int b = 0; b < OB; ++b) o[b][nc] *= change * v_change;
    }
  };
  const auto softmax = [&](int t0, float step, float size, float (&ks)[8], float (&km)[8], float (&vs)[8], float (&vm)[8], float4v (&s)[2][NC], uint4v (&p)[NC]) {
    const bool all = t0 + kUnitTokens - 1 <= p_lo && (t0 > p_hi - window || t0 + kUnitTokens - 1 < a.sinks);
    bool rise = (size > size_limit) & (lane >= 32);
    const auto scores = [&](const float (&top)[NC]) {           // s: x - top
#pragma unroll
      for (int nc = 0; nc < NC; ++nc)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          s[j / 4][nc][j & 3] = __builtin_fmaf(s[j / 4][nc][j & 3], ks[j], __builtin_fmaf(km[j], q_sum[nc], -top[nc]));
    };
    scores(top);
    if (!all) {
#pragma unroll
      for (int nc = 0; nc < NC; ++nc) {
        const int back = pos[nc] - t0 - g * 4, first = a.sinks - t0 - g * 4;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int t = j / 4 * 16 + (j & 3);
          const bool seen = ((uint32_t)(back - t) < (uint32_t)window) | ((t < first) & (t <= back));
          s[j / 4][nc][j & 3] = seen ? s[j / 4][nc][j & 3] : -INFINITY;
        }
      }
    }
    float high[NC];
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      high[nc] = s[0][nc][0];
#pragma unroll
      for (int j = 1; j < 8; ++j) high[nc] = fmaxf(high[nc], s[j / 4][nc][j & 3]);
      rise |= high[nc] > limit[nc];
    }
    if (__builtin_expect(__any(rise), 0)) rescale(t0, all, step, size, high, s, vs, vm);
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      float w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        w[j] = exp2_fast(s[j / 4][nc][j & 3]);
        total[nc] += w[j];
      }
      if (all) {
#pragma unroll
        for (int j = 0; j < 8; ++j) offsets[nc] = __builtin_fmaf(w[j], vm[j], offsets[nc]);
      } else {                                                  // what is masked may be a NaN, which is to show where it is not, however small its weight
#pragma unroll
        for (int j = 0; j < 8; ++j)
          offsets[nc] = s[j / 4][nc][j & 3] != -INFINITY ? __builtin_fmaf(w[j], vm[j], offsets[nc]) : offsets[nc];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] *= vs[j];
      p[nc] = (uint4v){pack_f16(w[0], w[1]), pack_f16(w[2], w[3]), pack_f16(w[4], w[5]), pack_f16(w[6], w[7])};
    }
    if (!a.bf16)
#pragma unroll
      for (int nc = 0; nc < NC; ++nc)
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          const uint32_t pair = p[nc][d];
          rounded[nc] = __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, pair), (half2v){1, 1}, rounded[nc], false);   // takes subnormal ones as they are
        }
  };

  for (; i < end; i += WK) {
    const int next = unit_at(i + WK);
    const uint8_t *u = address(next);
    const int t0 = unit < 0 ? kMostTokens : list.block(i) * kUnitTokens;   // a page outside the cache: nothing is seen
    // a lane has the keys' (lanes 0..31) or the values' step and offset of one token; through LDS each gets those of its eight
    if (lane >= 32 && t0 + lane - 32 > p_hi) param = 0;         // of no token yet
    float step = bf16_to_f32(param), offset = __uint_as_float(param & 0xFFFF0000);
    const float size = size_of(step, offset);                   // of the values' lanes
    if (lane < 32) {
      step *= step_scale;
      offset *= offset_scale;
    } else {
      offset = __builtin_fmaf(step, middle, offset);
    }
    params[wave][lane] = lane < 32 ? step : step * v_scale;
    params[wave][64 + lane] = offset;
    float ks[8], km[8], vs[8], vm[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      *(float4v *)(ks + h * 4) = *(const float4v *)&params[wave][h * 16 + g * 4];
      *(float4v *)(vs + h * 4) = *(const float4v *)&params[wave][32 + h * 16 + g * 4];
      *(float4v *)(km + h * 4) = *(const float4v *)&params[wave][64 + h * 16 + g * 4];
      *(float4v *)(vm + h * 4) = *(const float4v *)&params[wave][96 + h * 16 + g * 4];
    }
    load_params(u);
    in_order();
    float4v s[2][NC];
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) s[0][nc] = s[1][nc] = (float4v){0, 0, 0, 0};
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      uint4v w[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (U::kBits == 4) {
          const uint32_t d = k_raw[h][st];
          w[h] = (uint4v){d & 0x000F000F, d & 0x00F000F0, d >> 8 & 0x000F000F, d >> 8 & 0x00F000F0};
        } else {
          const uint32_t d = k_raw[h][2 * st], f = k_raw[h][2 * st + 1];
          w[h] = (uint4v){d & 0x00FF00FF, d >> 8 & 0x00FF00FF, f & 0x00FF00FF, f >> 8 & 0x00FF00FF};
        }
      }
#pragma unroll
      for (int nc = 0; nc < NC; ++nc) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          s[h][nc] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, w[h]), __builtin_bit_cast(half8, q[nc][st]), s[h][nc], 0, 0, 0);
      }
    }
    load_k(u);
    in_order();
    // bound by the vector ALU: a wave with scores to work on goes before one that feeds the matrix unit, and products of values, which
    // end its unit, before those of keys (a prompt of 8192 tokens: 598 us without, 585 with; parts of prompts 34.4 and 32.9)
    __builtin_amdgcn_s_setprio(2);
    uint4v p[NC];
    softmax(t0, step, size, ks, km, vs, vm, s, p);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int b = 0; b < U::kBlocks; ++b) {
      const uint32_t d = v_raw[b][0], f = v_raw[b][1];
      constexpr uint32_t low = U::kBits == 4 ? 0x000F000F : 0x00FF00FF;
      const uint4v w = {d & low, d >> 8 & low, f & low, f >> 8 & low};
#pragma unroll
      for (int nc = 0; nc < NC; ++nc)
        o[b][nc] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, w), __builtin_bit_cast(half8, p[nc]), o[b][nc], 0, 0, 0);
      if constexpr (U::kBits == 4) {
        const uint4v x = {d & 0x00F000F0, d >> 8 & 0x00F000F0, f & 0x00F000F0, f >> 8 & 0x00F000F0};
#pragma unroll
        for (int nc = 0; nc < NC; ++nc)
          o[OB / 2 + b][nc] =
              __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, x), __builtin_bit_cast(half8, p[nc]), o[OB / 2 + b][nc], 0, 0, 0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    load_v(u);
    in_order();
    unit = next;
  }

  // ---- results: channels 16 b + 4 g + 0..3 of a row in each lane
#pragma unroll
  for (int nc = 0; nc < NC; ++nc) {
    const int lift = limit[nc] > 0 ? (int)(limit[nc] - kLag) : 0;
    const float down = power(-lift), back = ldexpf(1.0f, 24 - v_exp - lift);
    total[nc] = column_sum(total[nc]) * down;
    offsets[nc] = __builtin_fmaf(column_sum(rounded[nc]), -middle * 0x1p-24f * back, column_sum(offsets[nc]) * down);
    top[nc] = limit[nc] < 0 ? kNothing : top[nc] + (float)lift;
#pragma unroll
    for (int b = 0; b < OB; ++b) {
      const float f = U::kBits == 4 && b >= OB / 2 ? back / 16 : back;
#pragma unroll
      for (int r = 0; r < 4; ++r) o[b][nc][r] = __builtin_fmaf(o[b][nc][r], f, offsets[nc]);
    }
  }
  const auto result = [&](int row) {
    uint32_t h = row;
    const int token = (int)a.group.split(h);
    return a.out + (int64_t)(seq.begin + token) * a.out_token_stride + (int64_t)(kvh * group + (int)h) * a.out_head_stride;
  };
  const auto write = [&](uint16_t *dst, int c0, float4v v) {   // four channels of a row's result
    const uint2u b = a.bf16 ? (uint2u){pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])} : (uint2u){pack_f16(v[0], v[1]), pack_f16(v[2], v[3])};
    if (c0 + 4 <= a.dim) {
      *(uint2u *)(dst + c0) = b;
    } else {
#pragma unroll
      for (int r = 0; r < 3; ++r)
        if (c0 + r < a.dim) dst[c0 + r] = (uint16_t)(b[r / 2] >> 16 * (r & 1));
    }
  };
  if constexpr (WK == 1) {
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      const int row = row0 + nc * 16 + col;
      if (row >= rows) continue;
      uint16_t *dst = result(row);
      const float inv = total[nc] != 0 ? 1.0f / total[nc] : 0.0f;
#pragma unroll
      for (int b = 0; b < OB; ++b) write(dst, b * 16 + g * 4, o[b][nc] * inv);
    }
  } else {
    __shared__ float sums[kAttentionWaves][16][DP + 4];
    __shared__ float tops[kAttentionWaves][16], totals[kAttentionWaves][16];
    const int64_t between = (int64_t)a.total_q * a.heads, first_row = ((int64_t)kvh * a.total_q + seq.begin) * group;
    constexpr int PARTS = 16 / WR;                               // threads a row
    const int r = threadIdx.x / PARTS % 16, first_wave = threadIdx.x / (PARTS * 16) * WK, part = threadIdx.x % PARTS;
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      if (nc) __syncthreads();
#pragma unroll
      for (int b = 0; b < OB; ++b) *(float4v *)&sums[wave][col][b * 16 + g * 4] = o[b][nc];
      if (g == 0) {
        tops[wave][col] = top[nc];
        totals[wave][col] = total[nc];
      }
      __syncthreads();
      const int row = (tile * WR + first_wave / WK) * 16 * NC + nc * 16 + r;
      if (row >= rows) continue;
      float high = tops[first_wave][r], w[WK], sum = 0;
#pragma unroll
      for (int k = 1; k < WK; ++k) high = fmaxf(high, tops[first_wave + k][r]);
#pragma unroll
      for (int k = 0; k < WK; ++k) {
        w[k] = exp2_fast(tops[first_wave + k][r] - high);
        sum = __builtin_fmaf(totals[first_wave + k][r], w[k], sum);
      }
      uint16_t *dst = result(row);
      const float inv = sum != 0 ? 1.0f / sum : 0.0f;
#pragma unroll
      for (int c = part * 4; c < DP; c += PARTS * 4) {
        float4v v = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < WK; ++k) v += *(const float4v *)&sums[first_wave + k][r][c] * w[k];
        if (SPLIT && splits > 1) {
          float *to = a.part + (split * between + first_row + row) * DP + c;
          store2(to, v[0], v[1]);
          store2(to + 2, v[2], v[3]);
          if (c == 0) store2(a.part_ml + (split * between + first_row + row) * 2, high, sum);
        } else {
          write(dst, c, v * inv);
        }
      }
    }
    if (!SPLIT || splits == 1 || !a.counters) return;
    // The last of a tile's splits to end joins them.  Their sums went past the caches of their XCDs (store2), so that they are where every
    // XCD sees them when their wave's vmcnt is 0, and the counter goes up after that; they are read past the caches too.  A release and
    // an acquire of the whole device would write back and drop an L2 for each workgroup: 28 us more for 1024 of them.
    __shared__ int last;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int *counter = a.counters + slot * a.kv_heads.d + kvh;
    if (threadIdx.x == 0) {
      const int before = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      last = before == splits - 1;
      if (last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next call
    }
    __syncthreads();
    if (!last) return;
    constexpr int FOURS = DP / 4;
    for (int at = threadIdx.x; at < min(16 * NC, rows - row0) * FOURS; at += 64 * kAttentionWaves) {
      const int row = row0 + at / FOURS, c = at % FOURS * 4;
      float high = kNothing, sum = 0;
      float4v v = {0, 0, 0, 0};
      for (int k0 = 0; k0 < splits; k0 += kJoinAtOnce) {
        float2v ml[kJoinAtOnce], x[kJoinAtOnce], y[kJoinAtOnce];
#pragma unroll
        for (int k = 0; k < kJoinAtOnce; ++k) {
          const int64_t from = first_row + min(k0 + k, splits - 1) * between + row;
          ml[k] = load2(a.part_ml + from * 2);
          x[k] = load2(a.part + from * DP + c);
          y[k] = load2(a.part + from * DP + c + 2);
        }
        float now = high;
#pragma unroll
        for (int k = 0; k < kJoinAtOnce; ++k) now = fmaxf(now, ml[k][0]);
        const float change = exp2_fast(high - now);
        high = now;
        sum *= change;
        v *= change;
#pragma unroll
        for (int k = 0; k < kJoinAtOnce; ++k) {
          const float w = k0 + k < splits ? exp2_fast(ml[k][0] - high) : 0.0f;
          sum = __builtin_fmaf(ml[k][1], w, sum);
          v[0] = __builtin_fmaf(x[k][0], w, v[0]);
          v[1] = __builtin_fmaf(x[k][1], w, v[1]);
          v[2] = __builtin_fmaf(y[k][0], w, v[2]);
          v[3] = __builtin_fmaf(y[k][1], w, v[3]);
        }
      }
      write(result(row), c, v * (sum != 0 ? 1.0f / sum : 0.0f));
    }
  }
}

// The splits of a row, joined: a workgroup a row, whose waves take every sixteenth split, a lane a channel of each 64.  Bound by latency: 64
// splits of 64 rows, 2 MB, take 4.5 us with the gap before it (34 us with the attention, and 40 where the last workgroups join so many).  Few splits of
// many rows are better joined there: 2 of 2048 rows take 68 us with the attention, and 97 with this kernel.
template <typename U, int NC>
__global__ __launch_bounds__(64 * kJoinWaves) void kv_join_kernel(AttentionArgs a) {
  constexpr int DP = U::kDim, C = (DP + 63) / 64, WAVES = kJoinWaves;
  __shared__ float sums[WAVES][C * 64], totals[WAVES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), kvh = blockIdx.y, group = (int)a.group.d;
  constexpr int R = 16 * NC;
  const Tile seq = Tile::find<R>(a, blockIdx.x / R).uniform();
  const int tile = seq.tile;
  if (tile < 0) return;
  const int rows = seq.n * group, row = tile * R + (int)blockIdx.x % R;
  if (row >= rows) return;
  const int row0 = tile * R;
  const UnitList list(a, seq.first + (int)a.group.div(row0), seq.first + (int)a.group.div(min(row0 + R, rows) - 1));
  const int splits = max(1, (list.count + a.chunk - 1) / a.chunk);
  if (splits == 1) return;                                     // written already
  const int64_t between = (int64_t)a.total_q * a.heads, at = ((int64_t)kvh * a.total_q + seq.begin) * group + row;
  float high = kNothing;
  for (int s = lane; s < splits; s += 64) high = fmaxf(high, a.part_ml[(at + s * between) * 2]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) high = fmaxf(high, __shfl_xor(high, d));
  float sum = 0, v[C] = {};
#pragma unroll 4
  for (int s = wave; s < splits; s += WAVES) {
    const float2v ml = *(const float2v *)(a.part_ml + (at + s * between) * 2);
    const float w = exp2_fast(ml[0] - high);
    sum = __builtin_fmaf(ml[1], w, sum);
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (DP % 64 == 0 || c * 64 + lane < DP) v[c] = __builtin_fmaf(a.part[(at + s * between) * DP + c * 64 + lane], w, v[c]);
  }
#pragma unroll
  for (int c = 0; c < C; ++c) sums[wave][c * 64 + lane] = v[c];
  if (lane == 0) totals[wave] = sum;
  __syncthreads();
  const int c = threadIdx.x;
  if (c >= a.dim) return;
  sum = 0;
  float x = 0;
#pragma unroll
  for (int k = 0; k < WAVES; ++k) {
    sum += totals[k];
    x += sums[k][c];
  }
  uint32_t h = row;
  const int token = (int)a.group.split(h);
  uint16_t *dst = a.out + (int64_t)(seq.begin + token) * a.out_token_stride + (int64_t)(kvh * group + (int)h) * a.out_head_stride;
  dst[c] = (uint16_t)store16(sum != 0 ? x / sum : 0.0f, a.bf16);
}

// Splits' sums: a split of 16 rows of 128 channels takes 8 KiB, three of them on each of 256 CUs 6 MiB.
constexpr size_t kJoinBytes = 32 << 20;
constexpr int kCounters = 16384, kJoinInKernel = 16;   // tiles with a counter; splits up to which the last workgroup joins them

int attention_workspace(tpuhip_ctx *ctx) {
  if (ctx->join) return TPUHIP_OK;
  hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
  TPUHIP_CHECK_HIP(hipStreamIsCapturing(ctx->stream, &capture));
  if (capture != hipStreamCaptureStatusNone || hipMalloc(&ctx->join, kCounters * 4 + kJoinBytes) != hipSuccess) {   // does without: one split
    (void)hipGetLastError();
    ctx->join = nullptr;
    return TPUHIP_OK;
  }
  const hipError_t e = hipMemsetAsync(ctx->join, 0, kCounters * 4, ctx->stream);
  if (e != hipSuccess) {
    (void)hipFree(ctx->join);
    ctx->join = nullptr;
    TPUHIP_CHECK_HIP(e);
  }
  return TPUHIP_OK;
}

}  // namespace tpuhip

using namespace tpuhip;

extern "C" {

int tpuhip_kv_attention(tpuhip_ctx *ctx, const tpuhip_kv_cache *cache, const tpuhip_kv_attention_desc *d, const void *q, void *out,
                        const int32_t *q_starts, const int32_t *kv_lens, const int32_t *page_table) {
  const char *what = "tpuhip_kv_attention";
  TPUHIP_REQUIRE(ctx && cache && d, "%s: NULL argument", what);
  TPUHIP_REQUIRE(cache->device == ctx->device, "%s: the cache lies on device %d, the context works on %d", what, cache->device,
                 ctx->device);
  TPUHIP_REQUIRE(d->dtype == TPUHIP_BF16 || d->dtype == TPUHIP_F16, "%s: queries in bfloat16 or float16, not type %d", what, d->dtype);
  const int kv_heads = cache->desc.kv_heads, dim = cache->desc.head_dim;
  TPUHIP_REQUIRE(d->heads >= 1 && d->heads % kv_heads == 0 && d->heads <= 65535, "%s: %d heads over the cache's %d", what, d->heads,
                 kv_heads);
  TPUHIP_REQUIRE(d->n_seq >= 0 && d->n_seq <= 65535, "%s: %d sequences", what, d->n_seq);
  TPUHIP_REQUIRE(d->total_q >= 0 && d->max_q >= 0 && d->max_kv >= 0, "%s: %d queries, at most %d a sequence, of %d tokens", what,
                 d->total_q, d->max_q, d->max_kv);
  TPUHIP_REQUIRE((int64_t)d->max_q * d->heads <= kMostTokens / 2 && d->max_kv <= kMostTokens, "%s: %d queries of %d heads, %d tokens",
                 what, d->max_q, d->heads, d->max_kv);
  TPUHIP_REQUIRE(d->window >= 0 && d->sinks >= 0, "%s: a window of %d, %d first tokens", what, d->window, d->sinks);
  TPUHIP_REQUIRE(std::isfinite(d->scale), "%s: the scale is not finite", what);
  if (d->n_seq == 0 || d->total_q == 0 || d->max_q == 0) return TPUHIP_OK;
  TPUHIP_REQUIRE(q && out && q_starts && kv_lens && (page_table || d->max_kv == 0), "%s: NULL argument", what);
  TPUHIP_REQUIRE(d->table_stride >= (d->max_kv + (int64_t)cache->desc.page_tokens - 1) / cache->desc.page_tokens,
                 "%s: %d pages a sequence for %d tokens", what, d->table_stride, d->max_kv);
  const int64_t strides[2][2] = {{d->q_token_stride, d->q_head_stride}, {d->out_token_stride, d->out_head_stride}};
  for (const auto &s : strides)
    TPUHIP_REQUIRE(s[0] >= 0 && s[1] >= 0 && s[0] <= INT64_MAX / 8 / d->total_q && s[1] <= INT64_MAX / 8 / d->heads, "%s: strides", what);
  const int64_t ts = d->out_token_stride, hs = d->out_head_stride;
  TPUHIP_REQUIRE(((d->heads == 1 || hs >= dim) && (d->total_q == 1 || ts >= (d->heads - 1) * hs + dim)) ||
                     ((d->total_q == 1 || ts >= dim) && (d->heads == 1 || hs >= (d->total_q - 1) * ts + dim)),
                 "%s: rows of the result overlap", what);
  TPUHIP_REQUIRE(q != out, "%s: the result takes the queries' place", what);
  TPUHIP_REQUIRE((uintptr_t)q % 2 == 0 && (uintptr_t)out % 2 == 0, "%s: q or out does not begin at an element", what);
  TPUHIP_CHECK_HIP(hipSetDevice(ctx->device));   // of the workspace, and of launches on its default stream
  AttentionArgs a{};
  a.data = cache->data;
  a.q_starts = q_starts;
  a.kv_lens = kv_lens;
  a.table = page_table;
  a.q = (const uint16_t *)q;
  a.out = (uint16_t *)out;
  a.q_token_stride = d->q_token_stride;
  a.q_head_stride = d->q_head_stride;
  a.out_token_stride = ts;
  a.out_head_stride = hs;
  a.heads = d->heads;
  a.group = FastDiv(d->heads / kv_heads);
  a.kv_heads = FastDiv(kv_heads);
  a.dim = dim;
  a.pages = cache->desc.pages;
  a.units_per_page = FastDiv(cache->units_per_page);
  a.table_stride = d->table_stride;
  a.total_q = d->total_q;
  a.max_q = d->max_q < d->total_q ? d->max_q : d->total_q;
  a.max_kv = d->max_kv;
  a.window = std::min(d->window, kMostTokens);
  a.sinks = std::min(d->sinks, d->max_kv);
  a.bf16 = d->dtype == TPUHIP_BF16;
  a.scale = d->scale;
  a.n_seq = d->n_seq;
  const int group = (int)a.group.d, num_cu = ctx->num_cu;
  const int64_t rows_max = (int64_t)a.max_q * group;             // of a sequence and cache head
  const int64_t rows_all = std::min<int64_t>(rows_max * d->n_seq, (int64_t)a.total_q * group) * kv_heads;
  return kv_dispatch(cache, [&](auto u) -> int {
    using U = decltype(u);
    const auto units_of = [&](int r) -> int64_t {               // that a tile of r rows sees at most
      const int64_t units = ceil_div64(a.max_kv, kUnitTokens);
      return a.window ? std::min<int64_t>(units, ceil_div64(a.sinks, kUnitTokens) + (a.window + r / group + 2) / kUnitTokens + 2) : units;
    };
    const auto run = [&](auto nc, auto wr) -> int {
      constexpr int NC = decltype(nc)::value, WR = decltype(wr)::value, R = 16 * NC * WR;
      a.one_tile = rows_max <= R;
      const int64_t slots = a.one_tile ? d->n_seq : std::min(ceil_div64(rows_max, R) * d->n_seq, (int64_t)a.total_q * group / R + d->n_seq);
      const int64_t base = slots * kv_heads, most = (UINT32_MAX / (64 * kAttentionWaves) - kXcds) / base;   // a launch has fewer than 2^32 threads
      TPUHIP_REQUIRE(most >= 1, "%s: %d queries of %d sequences over %d heads in one call", what, a.total_q, d->n_seq, kv_heads);
      a.splits = 1;
      if constexpr (WR == 1) {
        // Two workgroups a CU, without more than are there at a time (three, two with twice the rows or wider ones; heads of 64 have registers for
        // one more, but with 2, 3 or 4 a batch of 24 single tokens takes 26.5, 23.5 or 23.6 us there, 34.3, 32.7 or 32.5 with heads of 128, and a draft
        // 20.3, 21.1 or 21.3), and none of more than 128 units, as lengths may differ; but two units a wave at least, four with twice the rows, for a join takes as long (a wave takes
        // 1 us a unit, the join of two splits 1.6), and so few splits that the last one can join them rather than another kernel, where
        // these have six units a wave at most.
        const int64_t units = units_of(R), there = (NC == 1 && U::kDim <= 128 ? 3 : 2) * num_cu;
        int64_t splits = std::max<int64_t>(1, std::min(ceil_div64(2 * num_cu, base), there / base));
        splits = std::min(std::max(splits, ceil_div64(units, 128)), ceil_div64(units, 8 * NC));
        if (units <= kJoinInKernel * 24) splits = std::min<int64_t>(splits, kJoinInKernel / NC);
        splits = std::min({splits, most, (int64_t)kJoinBytes / ((int64_t)a.total_q * a.heads * (U::kDim + 2) * 4)});
        if (splits > 1) {
          if (int rc = attention_workspace(ctx)) return rc;
          if (!ctx->join) splits = 1;
        }
        splits = std::max<int64_t>(1, splits);                  // also where there are no tokens at all
        a.chunk = std::max(round_up((int)ceil_div64(units, splits), kAttentionWaves), 1);
        a.splits = (int)std::max<int64_t>(1, ceil_div64(units, a.chunk));
        a.part_ml = (float *)((char *)ctx->join + kCounters * 4);
        a.part = a.part_ml + (int64_t)a.splits * a.total_q * a.heads * 2;
      }
      const bool in_kernel = a.splits <= kJoinInKernel && base <= kCounters;
      a.counters = in_kernel ? (int *)ctx->join : nullptr;
      a.classes = kv_heads % 8 == 0 ? 8 : kv_heads % 4 == 0 ? 4 : kv_heads % 2 == 0 ? 2 : 1;
      a.class_heads = FastDiv(kv_heads / a.classes);
      a.split_count = FastDiv(a.splits);
      a.works = (int)(slots * a.splits * (kv_heads / a.classes));
      launch(ctx, kv_attention_kernel<U, NC, WR>, dim3((unsigned)(ceil_div64(a.works, kXcds / a.classes) * kXcds)), dim3(64 * kAttentionWaves), a);
      TPUHIP_CHECK_HIP(hipGetLastError());
      if constexpr (WR == 1)
        if (a.splits > 1 && !in_kernel) {   // a workgroup a row: no more than kJoinBytes have room for, and R - 1 past the end of each sequence
          launch(ctx, kv_join_kernel<U, NC>, dim3((unsigned)(slots * R), (unsigned)kv_heads), dim3(64 * kJoinWaves), a);
          TPUHIP_CHECK_HIP(hipGetLastError());
        }
      return TPUHIP_OK;
    };
    // The form of the kernel: 16 NC rows a wave, WR of the four waves with rows of their own.  Wide waves unpack codes less often, waves
    // with the same rows end a long list sooner, and there have to be workgroups for the CUs, more than two at a time where tiles differ.
    // Microseconds of 4 sequences of n tokens, causal, heads of 128 in 4 bits by fours (NC, WR; the chosen one in brackets; those of WR 1 with
    // their splits, the others have none):
    //    n  heads  rows a CU    2, 4     2, 2     2, 1     1, 4     1, 1
    //    64    4        16       9.2      8.8      8.4      6.8     [6.3]
    //   512    4        32      21.2     15.4     11.8     16.4    [10.4]
    //  1088    4        68      37.5     25.0    [20.6]    29.2     23.4
    //    64  128       128      11.2     12.7     20.1     [9.9]    20.6
    //   512   16       128      24.1    [21.4]    24.8     21.2     25.4
    //   256   64       256     [22.8]    26.5     38.2     23.3     37.3
    //  1088   64      1088    [129.4]   156.0    208.1    142.9    213.3
    // and of 64 queries of each behind 4096 tokens of 8 heads 116.5, 63.6, 23.5, 88.1 and [18.9]; of one prompt of 2176 of 32 heads (272 rows a
    // CU) 77.4, [70.3], 77.8, 71.0 and 80.4; of a draft, 24 sequences of 12 to 28 rows of 80 channels in 8 bits, 132.6, 74.3, [24.6], 107.4 and 27.1.
    // Rows of more than 128 channels have one block of 16 a wave, as two do not fit into registers.  Of 4 sequences with q queries each at the end of
    // n tokens, heads of 192 in 4 bits by fours (those of 256 take 1.1 to 1.3 times as long in all forms):
    //     q     n  heads  rows a CU    1, 4     1, 2     1, 1
    //    64    64    4        16        7.9      7.5     [7.3]
    //   512   512    4        32       19.6     13.7    [12.6]
    //    64  4096   32        32      109.9     61.0    [46.4]
    //    64  1000   64        64       34.3    [25.6]    31.3
    //   128  4096   32        64      111.0    [74.1]    80.8
    //  1088  1088    4        68       36.8    [27.0]    29.1
    //    64    64  128       128      [13.3]    18.7     29.8
    //   128  4096   64       128      137.2   [140.4]   150.6
    //   600  2000   16       150      104.1    [92.7]
    //   300   300   32       150      [22.5]    26.6     38.4
    //  1088  1088   16       272      [68.9]    68.0     91.6
    //  1088  1088   64      1088     [212.8]   252.3    344.0
    using std::integral_constant;
    const integral_constant<int, 1> one;
    const integral_constant<int, 2> two;
    const integral_constant<int, 4> four;
    const auto enough = [&](int rows_a_cu) { return rows_all > (int64_t)rows_a_cu * num_cu; };
    if constexpr (U::kDim <= 128) {
      const int64_t seen = units_of(32);
      if (rows_max <= 16 || (rows_max > 32 && !enough(32))) return run(one, one);
      if (rows_max <= 32) return run(two, one);
      if (seen <= 8) return run(one, four);
      if (!enough(80)) return run(two, one);
      if (!enough(seen <= 40 ? 255 : 511)) return run(two, two);
      return run(two, four);
    } else {
      if (rows_max <= 16 || !enough(48)) return run(one, one);
      if (!enough(units_of(16) <= 20 ? 100 : 255)) return run(one, two);
      return run(one, four);
    }
  });
}

}  // extern "C"
