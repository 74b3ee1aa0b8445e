// Attention to a key/value cache of 4 or 8 bits.
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
  int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;
  FastDiv group, units_per_page, kv_heads;
  int heads, dim, pages, table_stride, rows;   // rows: of a sequence and cache head at most
  int total_q, max_q, max_kv, window, sinks, bf16;
  int splits, chunk;            // a split takes `chunk` units of those that a wave's rows see
  int q_wide, out_wide;         // rows begin at dwords / at every fourth element
  float scale;
};

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4u __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ float load16(uint32_t b, int bf16) {
  return bf16 ? bf16_to_f32(b & 0xFFFF) : (float)__builtin_bit_cast(_Float16, (uint16_t)b);
}
__device__ __forceinline__ uint32_t store16(float v, int bf16) {
  return bf16 ? __builtin_bit_cast(uint16_t, (__bf16)v) : __builtin_bit_cast(uint16_t, (_Float16)v);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2v){a, b}, half2v));
}
__device__ __forceinline__ float exp2_fast(float v) { return __builtin_amdgcn_exp2f(v); }

// What a sequence's row of the call sees.
struct Sequence {
  int begin, n, first;          // its first query, how many, the position of the first
  __device__ __forceinline__ Sequence(const AttentionArgs &a, int seq) {
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

constexpr int kAttentionWaves = 4;
constexpr float kNothing = -1e30f;   // the maximum of no scores

// A wave takes 16 NC rows (a row: a query and one of the heads that share a cache head) and units of 32 tokens:
//   S^T = K Q^T   tokens x rows:    a lane has one row (of each 16) and the tokens 4g..4g+3, 16+4g..16+4g+3 of a unit, g = lane / 16
//   O^T = V^T P^T channels x rows:  which are just the lane's elements of the right operand here, so nothing is exchanged
// The left operands are the codes themselves: masked out of a dword, two of them are a pair of subnormal float16 numbers
// c 2^-24 (of a byte's upper half c 2^-20), which the matrix unit takes as they are and multiplies exactly.  Steps and offsets are applied to
// what is small: x = s_t (q.c_t) + m_t sum(q) to the scores, and P'_t = p_t s_t to the weights, with sum(p_t m_t) added to all channels.
// Four waves share a workgroup's rows (WR = 1: they take every fourth unit and join their sums in LDS) or have rows of their own (WR = 4).
template <typename U, int NC, int WR>
__global__ __launch_bounds__(64 * kAttentionWaves, 2) void kv_attention_kernel(AttentionArgs a) {
  constexpr int DP = U::kDim, KD = U::kRow / 16, STEPS = DP / 32, OB = DP / 16, WK = kAttentionWaves / WR;
  constexpr bool IN_LDS = NC > 1;                              // the queries: read once a unit, they need no registers
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const int kvh = blockIdx.y, group = (int)a.group.d;
  const Sequence seq(a, blockIdx.z);
  const int rows = seq.n * group, tiles = (rows + 16 * NC * WR - 1) / (16 * NC * WR);
  // the last tiles, which see the most, begin first
  const int tile = tiles - 1 - (int)blockIdx.x / a.splits, split = blockIdx.x % a.splits;
  if (tile < 0) return;
  const int row0 = (tile * WR + (WR > 1 ? wave : 0)) * 16 * NC;
  if (row0 >= rows) return;                                    // WR > 1 only: the workgroup shares nothing
  const int p_lo = seq.first + (int)a.group.div(row0), p_hi = seq.first + (int)a.group.div(min(row0 + 16 * NC, rows) - 1);
  const UnitList list(a, p_lo, p_hi);
  int i = split * a.chunk;
  const int end = min(list.count, i + a.chunk);
  if (split > 0 && i >= end) return;                           // no such split: the joining kernel counts them the same way
  i += WR > 1 ? 0 : wave;

  // ---- queries
  int pos[NC];
  float q_sum[NC];
  uint4v q[NC][STEPS];
  __shared__ uint4v q_shared[IN_LDS ? WR : 1][IN_LDS ? NC * STEPS * 64 : 1];   // WR = 1: the same from each wave
  uint32_t most = 0;
  int e2 = 0;
#pragma unroll
  for (int nc = 0; nc < NC; ++nc) {
    uint32_t h = row0 + nc * 16 + col;
    const bool valid = (int)h < rows;
    const int token = (int)a.group.split(h);
    pos[nc] = seq.first + token;
    const uint16_t *src = a.q + (int64_t)(seq.begin + token) * a.q_token_stride + (int64_t)(kvh * group + (int)h) * a.q_head_stride;
    q_sum[nc] = 0;
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      const int c0 = g * (DP / 4) + st * 8;
      uint4v raw = {0, 0, 0, 0};
      if (valid && c0 < a.dim) {
        if (a.q_wide && c0 + 8 <= a.dim) {
          raw = *(const uint4u *)(src + c0);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t b = src[min(c0 + e, a.dim - 1)];
            raw[e / 2] |= (c0 + e < a.dim ? b : 0) << 16 * (e & 1);
          }
        }
      }
      q[nc][st] = raw;
    }
  }
  const auto queries = [&](auto is_bf16) {
    constexpr int bf16 = decltype(is_bf16)::value;
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
      for (int st = 0; st < STEPS; ++st)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float v = load16(q[nc][st][e / 2] >> 16 * (e & 1), bf16);
          q_sum[nc] += v;
          const uint32_t size = __float_as_uint(v) & 0x7FFFFFFF;
          most = size < 0x7F800000 ? max(most, size) : most;
        }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, d));
    // the wave's queries times one power of two, the largest number just below 2^15: float16 holds bfloat16's 8 bits of all that are
    // within 2^29 of it.  A number past the bounds of the exponent becomes an infinity, in its own row.
    e2 = min(max((int)(most >> 23) - 127 - 14, -100), 88);
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)   // odd channels lie in the upper halves of 4-bit bytes, 16 times their size
          v[e] = ldexpf(load16(q[nc][st][e / 2] >> 16 * (e & 1), bf16), U::kBits == 4 && e & 1 ? -e2 - 4 : -e2);
        // in the order of the codes' pairs
        q[nc][st] = U::kBits == 4 ? (uint4v){pack_f16(v[0], v[4]), pack_f16(v[1], v[5]), pack_f16(v[2], v[6]), pack_f16(v[3], v[7])}
                                  : (uint4v){pack_f16(v[0], v[2]), pack_f16(v[1], v[3]), pack_f16(v[4], v[6]), pack_f16(v[5], v[7])};
      }
  };
  if (a.bf16)
    queries(std::true_type{});
  else
    queries(std::false_type{});
#pragma unroll
  for (int nc = 0; nc < NC; ++nc) {
    q_sum[nc] += __shfl_xor(q_sum[nc], 16);
    q_sum[nc] += __shfl_xor(q_sum[nc], 32);
  }
  if constexpr (IN_LDS) {
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
      for (int st = 0; st < STEPS; ++st) q_shared[WR > 1 ? wave : 0][(nc * STEPS + st) * 64 + lane] = q[nc][st];
  }
  const float log2e = 1.44269504088896341f;
  const float offset_scale = a.scale * log2e, step_scale = ldexpf(offset_scale, e2 + 24);

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
        const int page = a.table[(int64_t)blockIdx.z * a.table_stride + a.units_per_page.split(in_page)];
        if ((unsigned)page < (unsigned)a.pages) held = page * (int)a.units_per_page.d + (int)in_page;
      }
    }
    return __builtin_amdgcn_readlane(held, (at - held_at) / WK);
  };
  const auto address = [&](int unit) { return a.data + ((int64_t)max(unit, 0) * a.kv_heads.d + kvh) * U::kBytes; };
  uint32_t k_raw[2][KD], v_raw[U::kBlocks][2];
  uint32_t param;
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

  // ---- the sums
  float top[NC], limit[NC], total[NC], offsets[NC];   // limit: a score above it, relative to the maximum, raises that
  float4v o[OB][NC];
#pragma unroll
  for (int nc = 0; nc < NC; ++nc) {
    top[nc] = 0;
    limit[nc] = -INFINITY;                                      // the row has seen nothing
    total[nc] = offsets[nc] = 0;
#pragma unroll
    for (int b = 0; b < OB; ++b) o[b][nc] = (float4v){0, 0, 0, 0};
  }
  float v_scale = 1;            // steps of the values are taken times this power of two: 2^8 to 2^10 for the largest so far
  bool scaled = false;
  constexpr float kStepLimit = 1024, kLag = 5;   // weights up to 2^5 (of a maximum that lags), times steps up to 2^10: below float16's 65504

  __shared__ __attribute__((aligned(16))) float params[kAttentionWaves][128];
  const int window = a.window ? a.window : INT_MAX / 2;
  // A maximum or a step has gone up, which it seldom does after the first units: what has been summed, and this unit's scores, relative to
  // the new ones.
  const auto rescale = [&](float v_step, float (&high)[NC], float4v (&s)[2][NC], float (&vs)[8]) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v_step = fmaxf(v_step, __shfl_xor(v_step, d));
    float v_change = 1;
    if (v_step * v_scale > kStepLimit || !scaled) {
      scaled = true;
      const float now = ldexpf(1.0f, min(8 - ((int)(__float_as_uint(v_step) >> 23) - 127), 99));
      v_change = now / v_scale;
      v_scale = now;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) vs[j] *= v_change;
#pragma unroll
    for (int nc = 0; nc < NC; ++nc) {
      high[nc] = fmaxf(high[nc], __shfl_xor(high[nc], 16));
      high[nc] = fmaxf(high[nc], __shfl_xor(high[nc], 32));
      const bool first = limit[nc] < 0, some = high[nc] > -INFINITY;
      const float up = first ? some ? high[nc] : 0.0f : fmaxf(high[nc], 0.0f), change = first ? 1.0f : exp2_fast(-up);
      limit[nc] = some ? kLag : limit[nc];
      top[nc] += up;
      total[nc] *= change;
      offsets[nc] *= change;
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j / 4][nc][j & 3] -= up;
#pragma unroll
      for (int b = 0; b < OB; ++b) o[b][nc] *= change * v_change;
    }
  };
  const auto softmax = [&](int t0, float4v (&s)[2][NC], uint4v (&p)[NC]) {
    const bool all = t0 + kUnitTokens - 1 <= p_lo && (t0 > p_hi - window || t0 + kUnitTokens - 1 < a.sinks);
    // a lane has the keys' (lanes 0..31) or the values' step and offset of one token; through LDS each gets those of its eight
    float step = bf16_to_f32(param), offset = __uint_as_float(param & 0xFFFF0000);
    if (lane < 32) {
      step *= step_scale;
      offset *= offset_scale;
    } else if (t0 + lane - 32 > p_hi) {
      step = 0;                                                 // of no token yet
    }
    const float v_step = lane < 32 ? 0.0f : step;
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
    bool rise = v_step * v_scale > kStepLimit;
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
      for (int nc = 0; nc < NC; ++nc)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int t = t0 + j / 4 * 16 + g * 4 + (j & 3);
          const bool seen = (t <= pos[nc]) & ((t > pos[nc] - window) | (t < a.sinks));
          s[j / 4][nc][j & 3] = seen ? s[j / 4][nc][j & 3] : -INFINITY;
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
    if (__builtin_expect(__any(rise), 0)) rescale(v_step, high, s, vs);
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
      } else {                                                  // what is masked may be a NaN
#pragma unroll
        for (int j = 0; j < 8; ++j) offsets[nc] = w[j] != 0 ? __builtin_fmaf(w[j], vm[j], offsets[nc]) : offsets[nc];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] *= vs[j];
      p[nc] = (uint4v){pack_f16(w[0], w[1]), pack_f16(w[2], w[3]), pack_f16(w[4], w[5]), pack_f16(w[6], w[7])};
    }
  };

  int unit = unit_at(i);
  {
    const uint8_t *u = address(unit);
    load_k(u);
    load_params(u);
    load_v(u);
  }
  for (; i < end; i += WK) {
    const int next = unit_at(i + WK);
    const uint8_t *u = address(next);
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
        const uint4v rows = IN_LDS ? q_shared[WR > 1 ? wave : 0][(nc * STEPS + st) * 64 + lane] : q[nc][st];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          s[h][nc] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, w[h]), __builtin_bit_cast(half8, rows), s[h][nc], 0, 0, 0);
      }
    }
    load_k(u);
    uint4v p[NC];
    const int t0 = unit < 0 ? INT_MAX - kUnitTokens : list.block(i) * kUnitTokens;   // a page outside the cache: nothing is seen
    softmax(t0, s, p);
    load_params(u);
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
    load_v(u);
    unit = next;
  }

  // ---- results: channels 16 b + 4 g + 0..3 of a row in each lane
  const float back = 0x1p24f / v_scale;
#pragma unroll
  for (int nc = 0; nc < NC; ++nc) {
    total[nc] += __shfl_xor(total[nc], 16);
    total[nc] += __shfl_xor(total[nc], 32);
    offsets[nc] += __shfl_xor(offsets[nc], 16);
    offsets[nc] += __shfl_xor(offsets[nc], 32);
    if (limit[nc] < 0) top[nc] = kNothing;
#pragma unroll
    for (int b = 0; b < OB; ++b) {
      const float f = U::kBits == 4 && b >= OB / 2 ? back / 16 : back;
#pragma unroll
      for (int r = 0; r < 4; ++r) o[b][nc][r] = __builtin_fmaf(o[b][nc][r], f, offsets[nc]);
    }
  }
  // v[0..3]: four channels of a row's result or, of several splits, of its sums
  const auto write = [&](int row, int c0, float4v v, float high, float sum) {
    if (row >= rows) return;
    if (a.splits > 1) {
      const int64_t at = ((int64_t)split * gridDim.z + blockIdx.z) * gridDim.y + kvh;
      *(float4v *)(a.part + (at * a.rows + row) * DP + c0) = v;
      if (c0 == 0) *(float2v *)(a.part_ml + (at * a.rows + row) * 2) = (float2v){high, sum};
      return;
    }
    if (c0 >= a.dim) return;
    uint32_t h = row;
    const int token = (int)a.group.split(h);
    uint16_t *dst = a.out + (int64_t)(seq.begin + token) * a.out_token_stride + (int64_t)(kvh * group + (int)h) * a.out_head_stride + c0;
    const float inv = sum != 0 ? 1.0f / sum : 0.0f;
    v *= inv;
    if (a.out_wide && c0 + 4 <= a.dim) {
      *(uint2 *)dst = make_uint2(store16(v[0], a.bf16) | store16(v[1], a.bf16) << 16, store16(v[2], a.bf16) | store16(v[3], a.bf16) << 16);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (c0 + r < a.dim) dst[r] = (uint16_t)store16(v[r], a.bf16);
    }
  };
  if constexpr (WR > 1) {
#pragma unroll
    for (int nc = 0; nc < NC; ++nc)
#pragma unroll
      for (int b = 0; b < OB; ++b) write(row0 + nc * 16 + col, b * 16 + g * 4, o[b][nc], top[nc], total[nc]);
  } else {
    __shared__ float sums[WK][16][DP + 4];
    __shared__ float tops[WK][16], totals[WK][16];
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
      const int r = threadIdx.x >> 4, part = threadIdx.x & 15;
      float high = tops[0][r], w[WK], sum = 0;
#pragma unroll
      for (int k = 1; k < WK; ++k) high = fmaxf(high, tops[k][r]);
#pragma unroll
      for (int k = 0; k < WK; ++k) {
        w[k] = exp2_fast(tops[k][r] - high);
        sum = __builtin_fmaf(totals[k][r], w[k], sum);
      }
#pragma unroll
      for (int c = 0; c < DP; c += 64) {
        if (c + part * 4 >= DP) break;
        float4v v = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < WK; ++k) v += *(const float4v *)&sums[k][r][c + part * 4] * w[k];
        write(row0 + nc * 16 + r, c + part * 4, v, high, sum);
      }
    }
  }
}

// The splits of a row, joined: a wave a row, a lane a channel of each 64.
template <typename U, int ROWS>
__global__ __launch_bounds__(256) void kv_join_kernel(AttentionArgs a) {
  constexpr int DP = U::kDim, C = (DP + 63) / 64;
  const int lane = threadIdx.x & 63, kvh = blockIdx.y, group = (int)a.group.d;
  const int row = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Sequence seq(a, blockIdx.z);
  const int rows = seq.n * group;
  if (row >= rows) return;
  const int row0 = row / ROWS * ROWS;
  const UnitList list(a, seq.first + (int)a.group.div(row0), seq.first + (int)a.group.div(min(row0 + ROWS, rows) - 1));
  const int splits = max(1, (list.count + a.chunk - 1) / a.chunk);
  const int64_t at = ((int64_t)blockIdx.z * gridDim.y + kvh) * a.rows + row, between = (int64_t)gridDim.z * gridDim.y * a.rows;
  float high = kNothing;
  for (int s = lane; s < splits; s += 64) high = fmaxf(high, a.part_ml[(at + s * between) * 2]);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) high = fmaxf(high, __shfl_xor(high, d));
  float sum = 0, v[C] = {};
  for (int s = 0; s < splits; ++s) {
    const float2v ml = *(const float2v *)(a.part_ml + (at + s * between) * 2);
    const float w = exp2_fast(ml[0] - high);
    sum = __builtin_fmaf(ml[1], w, sum);
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (DP % 64 == 0 || c * 64 + lane < DP) v[c] = __builtin_fmaf(a.part[(at + s * between) * DP + c * 64 + lane], w, v[c]);
  }
  uint32_t h = row;
  const int token = (int)a.group.split(h);
  uint16_t *dst = a.out + (int64_t)(seq.begin + token) * a.out_token_stride + (int64_t)(kvh * group + (int)h) * a.out_head_stride;
  const float inv = sum != 0 ? 1.0f / sum : 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (c * 64 + lane < a.dim) dst[c * 64 + lane] = (uint16_t)store16(v[c] * inv, a.bf16);
}

// Splits' sums: a split of 16 rows of 128 channels takes 8 KiB, four of them on each of 256 CUs 8 MiB.
constexpr size_t kJoinBytes = 32 << 20;

int attention_workspace(tpuhip_ctx *ctx) {
  if (ctx->join) return TPUHIP_OK;
  hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
  TPUHIP_CHECK_HIP(hipStreamIsCapturing(ctx->stream, &capture));
  if (capture != hipStreamCaptureStatusNone || hipMalloc(&ctx->join, kJoinBytes) != hipSuccess) {   // does without: one split
    (void)hipGetLastError();
    ctx->join = nullptr;
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
  TPUHIP_REQUIRE((int64_t)d->max_q * d->heads <= INT_MAX / 2 && d->max_kv <= INT_MAX - 4096, "%s: %d queries of %d heads, %d tokens",
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
  TPUHIP_REQUIRE((uintptr_t)q % 2 == 0 && (uintptr_t)out % 2 == 0, "%s: q or out does not begin at an element", what);
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
  a.window = d->window;
  a.sinks = d->sinks;
  a.bf16 = d->dtype == TPUHIP_BF16;
  a.scale = d->scale;
  a.q_wide = (uintptr_t)q % 4 == 0 && d->q_token_stride % 2 == 0 && d->q_head_stride % 2 == 0;
  a.out_wide = (uintptr_t)out % 8 == 0 && ts % 4 == 0 && hs % 4 == 0;
  a.rows = a.max_q * (int)a.group.d;
  return kv_dispatch(cache, [&](auto u) -> int {
    using U = decltype(u);
    constexpr int WIDE = U::kDim <= 64 ? 4 : U::kDim <= 128 ? 3 : 2;   // 16s of rows a wave: their sums take DP / 4 registers each
    const auto run = [&](auto nc, auto wr) -> int {
      constexpr int NC = decltype(nc)::value, WR = decltype(wr)::value, R = 16 * NC * WR;
      const int tiles = (int)ceil_div64(a.rows, R);
      // units that a tile sees at most, and how many workgroups there would be
      int64_t units = ceil_div64(a.max_kv, kUnitTokens);
      if (a.window) units = std::min<int64_t>(units, ceil_div64(a.sinks, kUnitTokens) + (a.window + R / (int)a.group.d + 2) / kUnitTokens + 2);
      const int64_t base = (int64_t)tiles * kv_heads * d->n_seq, row_bytes = (int64_t)a.rows * kv_heads * d->n_seq * (U::kDim + 2) * 4;
      int64_t splits = std::max<int64_t>(1, std::min(ceil_div64(4 * ctx->num_cu, base), units / 16));
      splits = std::min(splits, std::max<int64_t>(1, (int64_t)kJoinBytes / row_bytes));
      if (splits > 1) {
        if (int rc = attention_workspace(ctx)) return rc;
        if (!ctx->join) splits = 1;
      }
      a.chunk = (int)std::max<int64_t>(round_up((int)ceil_div64(units, splits), 4 / WR), 1);
      a.splits = (int)std::max<int64_t>(1, ceil_div64(units, a.chunk));
      a.part_ml = (float *)ctx->join;
      a.part = a.part_ml + (int64_t)a.splits * a.rows * kv_heads * d->n_seq * 2;
      TPUHIP_REQUIRE((int64_t)tiles * a.splits <= INT_MAX, "%s: %d queries", what, a.max_q);
      launch(ctx, kv_attention_kernel<U, NC, WR>, dim3((unsigned)(tiles * a.splits), (unsigned)kv_heads, (unsigned)d->n_seq),
             dim3(64 * kAttentionWaves), a);
      TPUHIP_CHECK_HIP(hipGetLastError());
      if (a.splits > 1) {
        launch(ctx, kv_join_kernel<U, 16 * NC>, dim3((unsigned)ceil_div64(a.rows, 4), (unsigned)kv_heads, (unsigned)d->n_seq), dim3(256), a);
        TPUHIP_CHECK_HIP(hipGetLastError());
      }
      return TPUHIP_OK;
    };
    using std::integral_constant;
    if (a.rows <= 16) return run(integral_constant<int, 1>{}, integral_constant<int, 1>{});
    if (a.rows <= 16 * WIDE) return run(integral_constant<int, WIDE>{}, integral_constant<int, 1>{});
    return run(integral_constant<int, WIDE>{}, integral_constant<int, 4>{});
  });
}

}  // extern "C"
