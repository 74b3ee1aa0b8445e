// The key/value cache in 4 or 8 bits: its memory, rows on their way into it and out of it.
#include "kv_cache.hpp"

#include <algorithm>
#include <climits>
#include <new>
#include <type_traits>

namespace tpuhip {

// ---- elements ----------------------------------------------------------------------------------------------------------------------
struct Bf16 {
  uint16_t b;
};
__device__ __forceinline__ float to_f32(Bf16 v) { return bf16_to_f32(v.b); }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  return (T)v;
}
// to nearest, ties to even; a NaN stays one
template <>
__device__ __forceinline__ Bf16 from_f32<Bf16>(float v) {
  return {__builtin_bit_cast(uint16_t, (__bf16)v)};
}

// Bytes between registers and LDS or memory, by sixteen as far as that goes: at dwords, or (rows of any stride) at any element
typedef uint32_t dwords4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t row_dwords4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t row_dword __attribute__((aligned(2)));
template <int BYTES, typename V = dwords4, typename D = uint32_t>
__device__ __forceinline__ void copy_dwords(void *dst, const void *src) {
  static_assert(BYTES % 4 == 0);
  constexpr int full = BYTES / 16;
#pragma unroll
  for (int i = 0; i < full; ++i) ((V *)dst)[i] = ((const V *)src)[i];
#pragma unroll
  for (int i = full * 4; i < BYTES / 4; ++i) ((D *)dst)[i] = ((const D *)src)[i];
}
template <int BYTES>
__device__ __forceinline__ void copy_row(void *dst, const void *src) {
  copy_dwords<BYTES, row_dwords4, row_dword>(dst, src);
}

struct RowsArgs {
  uint8_t *data;
  const int32_t *slots;
  void *x[2];                   // keys, values
  int64_t token_stride[2], head_stride[2];
  FastDiv head_count;
  int tokens, heads, dim, most; // slots below `most` exist
  int half;                     // few workgroups: so many take whole units and as many what is left; 0: each takes both
  int wide;                     // all DP elements are there
};

// A workgroup takes 32 rows of one head, keys and values: eight threads a row, each with DP/16 channels of its lower half and as many
// of the upper one, which share the bytes of the values.
constexpr int kRowThreads = 8, kRowsThreads = kUnitTokens * kRowThreads;

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
// over the eight lanes of a row: neighbours, pairs, halves
template <typename F>
__device__ __forceinline__ float over8(float v, F f) {
  v = f(v, dpp<0xB1>(v));
  v = f(v, dpp<0x4E>(v));
  return f(v, dpp<0x141>(v));
}

// the upper 16 bits of the largest bfloat16 not above v: away from zero where v is negative
__device__ __forceinline__ uint32_t bf16_down(float v) {
  const uint32_t b = __float_as_uint(v);
  return (b + ((uint32_t)((int32_t)b >> 31) & 0xFFFF)) >> 16;
}

// Four dwords of four bytes as four dwords of the first, second, ... bytes
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400), b = __builtin_amdgcn_perm(w[3], w[2], 0x05010400);
  const uint32_t c = __builtin_amdgcn_perm(w[1], w[0], 0x07030602), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602);
  w[0] = __builtin_amdgcn_perm(b, a, 0x05040100);
  w[1] = __builtin_amdgcn_perm(b, a, 0x07060302);
  w[2] = __builtin_amdgcn_perm(d, c, 0x05040100);
  w[3] = __builtin_amdgcn_perm(d, c, 0x07060302);
}

// A unit's values on their way between rows in LDS, one token's bytes after the other's, and the columns they have in memory (v_at):
// a thread takes four columns, or eight of two neighbouring blocks, of the eight tokens that a lane of the attention kernel has, 32 or
// 64 bytes of memory next to each other, and turns bytes in registers.  Rows are a dword longer than their bytes: the threads of a
// wave then read and write different banks.
template <typename U>
struct ValueColumns {
  static constexpr int kStride = U::kRow + 4, kPair = U::kPaired ? 2 : 1, kThreads = U::kRow / (4 * kPair) * 4;
  static_assert(kThreads <= kRowsThreads);
  int g, c0;                    // tokens 4g.. and 16 + 4g.., columns c0..c0+3 (and c0+16..)
  __device__ __forceinline__ explicit ValueColumns(int at) {
    const int q = at & 3;
    g = at >> 2 & 3;
    c0 = (at >> 4) * 16 * kPair + q * 4;
  }
  __device__ __forceinline__ uint32_t *memory(uint8_t *values) const {
    return (uint32_t *)(values + (c0 / (16 * kPair)) * (512 * kPair) + (g * 16 + (c0 & 15)) * (8 * kPair));
  }
  // LDS: the dword of tokens' byte order in memory: the middle two of four change places
  __device__ __forceinline__ int row(int half, int k) const { return half * 16 + g * 4 + ((k >> 1) | (k & 1) << 1); }
  __device__ __forceinline__ void to_memory(const uint8_t *rows, uint8_t *values) const {
    uint32_t out[4][2 * kPair];
#pragma unroll
    for (int p = 0; p < kPair; ++p)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = *(const uint32_t *)(rows + row(half, k) * kStride + c0 + p * 16);
        transpose4(w);
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i][p * 2 + half] = w[i];
      }
    uint32_t *to = memory(values);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (U::kPaired)
        *(uint4 *)(to + i * 4) = make_uint4(out[i][0], out[i][1], out[i][2], out[i][3]);
      else
        *(uint2 *)(to + i * 2) = make_uint2(out[i][0], out[i][1]);
    }
  }
  __device__ __forceinline__ void to_rows(const uint8_t *values, uint8_t *rows) const {
    const uint32_t *from = memory(const_cast<uint8_t *>(values));
    uint32_t in[4][2 * kPair];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (U::kPaired) {
        const uint4 v = *(const uint4 *)(from + i * 4);
        in[i][0] = v.x, in[i][1] = v.y, in[i][2] = v.z, in[i][3] = v.w;
      } else {
        const uint2 v = *(const uint2 *)(from + i * 2);
        in[i][0] = v.x, in[i][1] = v.y;
      }
    }
#pragma unroll
    for (int p = 0; p < kPair; ++p)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = in[i][p * 2 + half];
        transpose4(w);
#pragma unroll
        for (int k = 0; k < 4; ++k) *(uint32_t *)(rows + row(half, k) * kStride + c0 + p * 16) = w[k];
      }
  }
};

// N bytes from registers to memory and back, in the largest pieces that their number allows
template <int N>
__device__ __forceinline__ void copy_bytes(void *dst, const void *src) {
  if constexpr (N % 4 == 0) {
    copy_dwords<N>(dst, src);
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) ((uint16_t *)dst)[i] = ((const uint16_t *)src)[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) ((uint8_t *)dst)[i] = ((const uint8_t *)src)[i];
  }
}

// x / L as a division rounds it: the same, with the inverse rounded to nearest
template <int L>
__device__ __forceinline__ float over_levels(float x) {
  constexpr float inv = 1.0f / L;
  const bool small = x < 0x1p-60f;
  x *= small ? 0x1p64f : 1.0f;
  const float q = x * inv;
  return __builtin_fmaf(__builtin_fmaf(-q, (float)L, x), inv, q) * (small ? 0x1p-64f : 1.0f);
}

// a number that the compiler takes for another one each time: what follows from it is worked out where it is used, and only then
__device__ __forceinline__ int here(int v) {
  asm("" : "+v"(v));
  return v;
}

// the low bytes of N dwords, or zeros
template <int N>
__device__ __forceinline__ void store_bytes(uint8_t *at, const uint32_t (&b)[N], bool none) {
  if constexpr (N % 4 == 0) {
    uint32_t w[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      w[i] = __builtin_amdgcn_perm(b[4 * i + 1], b[4 * i], 0x0C0C0400) | __builtin_amdgcn_perm(b[4 * i + 3], b[4 * i + 2], 0x04000C0C);
      w[i] = none ? 0 : w[i];
    }
    copy_dwords<N>(at, w);
  } else {
    uint8_t w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = none ? 0 : b[i];
    copy_bytes<N>(at, w);
  }
}

// What a workgroup does with the slots around its 32 tokens: where a whole unit's tokens stand in order, wherever that begins, they are one
// workgroup's, the one among whose tokens is the first; what is left of its own 32 it takes one by one.  Each wave finds out for itself.
struct Runs {
  int start, slot;              // the first token of the unit and its slot; start -1: none
  uint32_t left;                // which of the 32
  int slots;                    // of tokens first - 32 + lane, -1: none or not in the cache
  __device__ __forceinline__ Runs(const RowsArgs &a, int first) {
    const int lane = threadIdx.x & 63;
    const auto at = [&](int i) {
      const int s = a.slots[min(max(i, 0), a.tokens - 1)];
      return (unsigned)i < (unsigned)a.tokens && (unsigned)s < (unsigned)a.most ? s : -1;
    };
    slots = at(first - 32 + lane);
    const int further = at(first + 32 + lane);
    // tokens of which the next one stands in the next slot (wave_shl:1 brings the next lane's)
    const int next0 = __builtin_amdgcn_update_dpp(__builtin_amdgcn_readlane(further, 0), slots, 0x130, 0xf, 0xf, false);
    const int next1 = __builtin_amdgcn_update_dpp(-1, further, 0x130, 0xf, 0xf, false);
    const uint64_t link0 = __ballot(slots >= 0 && next0 == slots + 1), link1 = __ballot(further >= 0 && next1 == further + 1);
    const uint32_t links = (uint32_t)(lane ? link0 >> lane | link1 << (64 - lane) : link0);
    const uint64_t starts = __ballot(slots >= 0 && (slots & 31) == 0 && (links & 0x7FFFFFFF) == 0x7FFFFFFF);
    const uint32_t own = (uint32_t)(starts >> 32);
    const int k = own ? __builtin_ctz(own) : 0;
    start = own ? first + k : -1;
    slot = __builtin_amdgcn_readlane(slots, 32 + k);
    const bool taken = lane >= 32 && (uint32_t)(starts >> (lane - 31)) != 0;
    left = (uint32_t)(__ballot(first - 32 + lane < a.tokens && !taken) >> 32);
  }
  // where row `row` of the unit, or of the 32, belongs
  __device__ __forceinline__ int slot_of(bool whole, int row) const { return whole ? slot + row : __shfl(slots, 32 + row); }
};

// A row's m, s and c, in one pass: it is read once, into registers, its minimum and maximum found among its eight threads (which keep a NaN),
// and codes are made with eight instructions an element.  Whole units (prompts, wherever they begin) are written as they lie in memory,
// 16 bytes a thread; other tokens as rows of keys, and values by bytes, or by dwords where the four tokens of one are there.
// Bound by memory: 65536 tokens of 8 heads of 128 bfloat16 channels in 4 bits, 340 MB, take 53.6 us, 4.8 TB/s where that begins at a unit and
// 3.9 where it does not (with twice the instructions an element it was the vector ALU, and 62 us).
template <typename U, typename T, bool WIDE>
__global__ __launch_bounds__(kRowsThreads) void kv_write_kernel(RowsArgs a) {
  constexpr int E = U::kDim / 16, HALF = U::kDim / 2, B = E * U::kBits / 8, STRIDE = ValueColumns<U>::kStride;
  __shared__ __attribute__((aligned(16))) uint8_t keys[U::kCodes], values[kUnitTokens * STRIDE];
  __shared__ __attribute__((aligned(16))) uint32_t params[2 * kUnitTokens];
  __shared__ int slots[kUnitTokens];
  const bool second = a.half && blockIdx.x >= (unsigned)a.half;
  uint32_t at_head = second ? blockIdx.x - a.half : blockIdx.x;   // the heads of a token next to each other, as in memory
  const int first = (int)a.head_count.split(at_head) * kUnitTokens, head = (int)at_head;
  const int t = threadIdx.x & (kRowThreads - 1), row = threadIdx.x / kRowThreads;
  T raw[2][2 * E];
  const auto load = [&](int begin) {
    const int at = min(begin + row, a.tokens - 1);             // a row to read in any case
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const T *src = (const T *)a.x[kv] + (int64_t)at * a.token_stride[kv] + (int64_t)head * a.head_stride[kv];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c0 = h * HALF + t * E;
        if (WIDE || c0 + E <= a.dim) {
          copy_row<E * sizeof(T)>(raw[kv] + h * E, src + c0);
        } else {
          const int c = here(c0);
#pragma unroll
          for (int e = 0; e < E; ++e) raw[kv][h * E + e] = src[min(c + e, a.dim - 1)];   // past the end, the last one again
        }
      }
    }
  };
  const Runs runs(a, first);
  for (int whole = runs.start >= 0 && !second; whole >= 0; --whole) {
    if (!whole && (!runs.left || (a.half && !second))) return;
    load(whole ? runs.start : first);
    int slot = runs.slot_of(whole, row);
    if (!whole && !(runs.left >> row & 1)) slot = -1;
    if (!whole && runs.start >= 0) __syncthreads();            // LDS holds the unit
    if (t == 0) slots[row] = slot;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      float x[2 * E];
#pragma unroll
      for (int e = 0; e < 2 * E; ++e) x[e] = to_f32(raw[kv][e]);
      float lo = x[0], hi = x[0];                              // a NaN stays
#pragma unroll
      for (int e = 1; e < 2 * E; ++e) {
        lo = __builtin_elementwise_minimum(lo, x[e]);
        hi = __builtin_elementwise_maximum(hi, x[e]);
      }
      lo = over8(lo, [](float p, float q) { return __builtin_elementwise_minimum(p, q); });
      hi = over8(hi, [](float p, float q) { return __builtin_elementwise_maximum(p, q); });
      uint32_t mb = bf16_down(lo);
      const float m = bf16_to_f32(mb);
      const float step = over_levels<U::kLevels>(hi - m);
      uint32_t sb = 0x8000u ^ bf16_down(-step);
      float s = bf16_to_f32(sb);
      if (!(lo >= -__FLT_MAX__ && hi <= __FLT_MAX__ && s <= __FLT_MAX__)) {
        mb = 0x7FC0;
        sb = 0;
        s = 0;
      } else if (s < 0x1p-126f) {
        sb = 0;
        s = 0;
      }
      // c = rint((x - m) / s), where ties are common among bfloat16 numbers: a product with an inverse that is good to a unit, and the
      // remainder of that, which is exact, times the inverse again.  So a quotient that a float holds, as all ties are, comes out as it
      // is; at a scale where neither the inverse nor the remainder leaves the normal numbers.  m is not above the minimum and L s not
      // below the rest, so c lies in 0..L; it comes in the low bits of a float that has no room for fractions.
      const float scale = s > 0x1p100f ? 0x1p-64f : s < 0x1p-90f ? 0x1p64f : 1.0f;
      const float ss = s * scale, inv = __builtin_amdgcn_rcpf(ss), ms = -m * scale;
      uint32_t c[2 * E];
#pragma unroll
      for (int e = 0; e < 2 * E; ++e) {
        const float d = __builtin_fmaf(x[e], scale, ms), q0 = d * inv;
        c[e] = __float_as_uint(__builtin_fmaf(__builtin_fmaf(-q0, ss, d), inv, q0) + 0x1.8p23f);
      }
      if constexpr (!WIDE) {                                   // what is added holds zeros
#pragma unroll
        for (int e = 0; e < 2 * E; ++e) c[e] = e / E * HALF + t * E + e % E < a.dim ? c[e] : 0;
      }
      const bool none = !(s > 0);
      if (U::kBits == 4 && kv == 1) {
        uint32_t b[E];
#pragma unroll
        for (int e = 0; e < E; ++e) b[e] = c[e] | c[E + e] << 4;
        store_bytes<E>(values + row * STRIDE + t * E, b, none);
      } else {
        uint8_t *at = kv ? values + row * STRIDE : keys + row * U::kRow;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t b[B];
#pragma unroll
          for (int i = 0; i < B; ++i) b[i] = U::kBits == 4 ? c[h * E + 2 * i % E] | c[h * E + (2 * i + 1) % E] << 4 : c[h * E + i % E];
          store_bytes<B>(at + h * (U::kRow / 2) + t * B, b, none);
        }
      }
      if (t == 0) params[kv * kUnitTokens + row] = mb << 16 | sb;
    }
    __syncthreads();
    uint8_t *dst = a.data + ((int64_t)(slot >> 5) * a.heads + head) * U::kBytes;
    if (whole) {
      for (int i = threadIdx.x; i < ValueColumns<U>::kThreads; i += kRowsThreads) ValueColumns<U>(i).to_memory(values, dst + U::kCodes);
      // the other threads first
      for (int i = kRowsThreads - 1 - threadIdx.x; i < U::kCodes / 16; i += kRowsThreads) ((uint4 *)dst)[i] = ((const uint4 *)keys)[i];
      if (threadIdx.x < 16) ((uint4 *)(dst + U::kParams))[threadIdx.x] = ((const uint4 *)params)[threadIdx.x];
      continue;
    }
    if (slot < 0) return;
    const int place = slot & 31;
    constexpr int KB = U::kRow / kRowThreads;
    copy_bytes<KB>(dst + place * U::kRow + t * KB, keys + row * U::kRow + t * KB);
    if (t < 2) ((uint32_t *)(dst + U::kParams))[t * kUnitTokens + place] = params[t * kUnitTokens + row];
    dst += U::kCodes;
    const int in4 = place & 3, lead = row - in4;
    bool four = lead >= 0 && lead + 3 < kUnitTokens;
    if (four)
      for (int i = 0; i < 4; ++i) four &= slots[lead + i] == slot - in4 + i;
    if (four) {                                                // each of the four writes a quarter of the columns
      for (int j = (in4 * kRowThreads + t) * 4; j < U::kRow; j += 16 * kRowThreads) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = *(const uint32_t *)(values + (lead + ((k >> 1) | (k & 1) << 1)) * STRIDE + j);
        transpose4(w);
#pragma unroll
        for (int i = 0; i < 4; ++i) *(uint32_t *)(dst + U::v_at(j + i, place & ~3)) = w[i];
      }
    } else {
      for (int j = t; j < U::kRow; j += kRowThreads) dst[U::v_at(j, place)] = values[row * STRIDE + j];
    }
  }
}

// m + s c.  Bound by memory: whole units are read as they lie, other tokens row by row with the values' bytes gathered; rows are written
// once: 65536 tokens of 8 heads of 128 channels, 4 bits to bfloat16, 340 MB, take 56 us, 4.5 TB/s with the launch.
template <typename U, typename T, bool WIDE>
__global__ __launch_bounds__(kRowsThreads) void kv_read_kernel(RowsArgs a) {
  constexpr int E = U::kDim / 16, HALF = U::kDim / 2, B = E * U::kBits / 8, STRIDE = ValueColumns<U>::kStride;
  __shared__ __attribute__((aligned(16))) uint8_t values[kUnitTokens * STRIDE];
  const bool second = a.half && blockIdx.x >= (unsigned)a.half;
  uint32_t at_head = second ? blockIdx.x - a.half : blockIdx.x;   // the heads of a token next to each other, as in memory
  const int first = (int)a.head_count.split(at_head) * kUnitTokens, head = (int)at_head;
  const int t = threadIdx.x & (kRowThreads - 1), row = threadIdx.x / kRowThreads;
  const Runs runs(a, first);
  for (int whole = runs.start >= 0 && !second; whole >= 0; --whole) {
    if (!whole && (!runs.left || (a.half && !second))) return;
    const int at = (whole ? runs.start : first) + row;
    const bool there = whole || (runs.left >> row & 1);
    const int slot = runs.slot_of(whole, row);
    const int place = slot & 31;
    const uint8_t *unit = a.data + ((int64_t)max(slot >> 5, 0) * a.heads + head) * U::kBytes;   // none: any, and zeros below
    uint8_t bytes[2][2 * B];
    uint32_t param[2];
    if (whole && threadIdx.x < ValueColumns<U>::kThreads) ValueColumns<U>(threadIdx.x).to_rows(unit + U::kCodes, values);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) param[kv] = ((const uint32_t *)(unit + U::kParams))[kv * kUnitTokens + place];
#pragma unroll
    for (int h = 0; h < 2; ++h) copy_bytes<B>(bytes[0] + h * B, unit + place * U::kRow + h * (U::kRow / 2) + t * B);
    if (whole) {
      __syncthreads();
      if constexpr (U::kBits == 4) {
        copy_bytes<E>(bytes[1], values + row * STRIDE + t * E);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) copy_bytes<E>(bytes[1] + h * E, values + row * STRIDE + h * HALF + t * E);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 2 * B; ++e) {
        const int j = U::kBits == 4 || e < E ? t * E + e : HALF + t * E + e - E;
        bytes[1][e] = unit[U::kCodes + U::v_at(j, place)];
      }
    }
    if (!there) continue;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const float s = slot < 0 ? 0.0f : bf16_to_f32(param[kv] & 0xFFFF), m = slot < 0 ? 0.0f : bf16_to_f32(param[kv] >> 16);
      T raw[2 * E];
#pragma unroll
      for (int e = 0; e < 2 * E; ++e) {
        const uint32_t c = U::kBits == 8 ? bytes[kv][e] : kv == 0 ? bytes[0][e / 2] >> 4 * (e & 1) & 15 : bytes[1][e % E] >> 4 * (e / E) & 15;
        raw[e] = from_f32<T>(__builtin_fmaf(s, (float)c, m));  // s c is exact: 16 bits
      }
      T *dst = (T *)a.x[kv] + (int64_t)at * a.token_stride[kv] + (int64_t)head * a.head_stride[kv];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c0 = h * HALF + t * E;
        if (WIDE || c0 + E <= a.dim) {
          copy_row<E * sizeof(T)>(dst + c0, raw + h * E);
        } else {
          const int c = here(c0);
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (c + e < a.dim) dst[c + e] = raw[h * E + e];
        }
      }
    }
  }
}

__global__ void kv_clear_kernel(uint4 *p, int64_t n) {
  int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  for (; i < n; i += (int64_t)gridDim.x * blockDim.x) p[i] = make_uint4(0, 0, 0, 0);
}

// 0: refused, with the error set
static int64_t kv_bytes(const tpuhip_kv_desc *d, const char *what) {
  int rc = TPUHIP_OK;
  int64_t total = 0;
  [&]() -> int {
    TPUHIP_REQUIRE(d, "%s: no descriptor", what);
    TPUHIP_REQUIRE(d->bits == 4 || d->bits == 8, "%s: 4 or 8 bits, not %d", what, d->bits);
    TPUHIP_REQUIRE(kv_padded(d->head_dim), "%s: a head size of 1 to 256, not %d", what, d->head_dim);
    TPUHIP_REQUIRE(d->kv_heads >= 1 && d->kv_heads <= 65535, "%s: %d heads", what, d->kv_heads);
    TPUHIP_REQUIRE(d->page_tokens >= 32 && d->page_tokens % 32 == 0, "%s: pages of a multiple of 32 tokens, not %d", what,
                   d->page_tokens);
    TPUHIP_REQUIRE(d->pages >= 1 && (int64_t)d->pages * d->page_tokens <= INT_MAX, "%s: %d pages of %d tokens", what, d->pages,
                   d->page_tokens);
    const int64_t unit = 2 * kUnitTokens * (kv_padded(d->head_dim) * d->bits / 8 + 4);
    total = (int64_t)d->pages * (d->page_tokens / kUnitTokens) * d->kv_heads * unit;   // below 2^26 * 2^16 * 2^15
    return rc;
  }();
  return total;
}

static bool in_elements(int dtype) { return dtype == TPUHIP_BF16 || dtype == TPUHIP_F16 || dtype == TPUHIP_F32; }

static int rows_args(tpuhip_ctx *ctx, const tpuhip_kv_cache *c, const tpuhip_kv_rows *r, const int32_t *slots, bool output,
                     const char *what, RowsArgs *a) {
  TPUHIP_REQUIRE(ctx && c && r, "%s: NULL argument", what);
  TPUHIP_REQUIRE(c->device == ctx->device, "%s: the cache lies on device %d, the context works on %d", what, c->device, ctx->device);
  TPUHIP_REQUIRE(r->tokens >= 0, "%s: %d tokens", what, r->tokens);
  TPUHIP_REQUIRE(ceil_div64(r->tokens, kUnitTokens) * c->desc.kv_heads * kRowsThreads <= UINT32_MAX, "%s: %d tokens of %d heads in one call",
                 what, r->tokens, c->desc.kv_heads);   // a launch has fewer than 2^32 threads
  TPUHIP_REQUIRE(in_elements(r->dtype), "%s: unknown type %d", what, r->dtype);
  if (r->tokens == 0) return TPUHIP_OK;
  TPUHIP_REQUIRE(r->k && r->v && slots, "%s: NULL argument", what);
  const int size = r->dtype == TPUHIP_F32 ? 4 : 2, dim = c->desc.head_dim, heads = c->desc.kv_heads;
  const int64_t ts[2] = {r->k_token_stride, r->v_token_stride}, hs[2] = {r->k_head_stride, r->v_head_stride};
  void *x[2] = {r->k, r->v};
  for (int i = 0; i < 2; ++i) {
    const char *name = i ? "values" : "keys";
    TPUHIP_REQUIRE(ts[i] >= 0 && hs[i] >= 0 && ts[i] <= INT64_MAX / 8 / r->tokens && hs[i] <= INT64_MAX / 8 / heads,
                   "%s: strides of the %s", what, name);
    TPUHIP_REQUIRE((uintptr_t)x[i] % size == 0, "%s: the %s do not begin at an element", what, name);
    if (output) {   // rows of their own: tokens within a head's stride or heads within a token's
      const bool by_token = (heads == 1 || hs[i] >= dim) && (r->tokens == 1 || ts[i] >= (heads - 1) * hs[i] + dim);
      const bool by_head = (r->tokens == 1 || ts[i] >= dim) && (heads == 1 || hs[i] >= (r->tokens - 1) * ts[i] + dim);
      TPUHIP_REQUIRE(by_token || by_head, "%s: rows of the %s overlap", what, name);
    }
    a->x[i] = x[i];
    a->token_stride[i] = ts[i];
    a->head_stride[i] = hs[i];
  }
  a->wide = dim == c->dp;
  a->data = c->data;
  a->slots = slots;
  a->tokens = r->tokens;
  a->heads = heads;
  a->head_count = FastDiv(heads);
  a->dim = dim;
  a->most = c->desc.pages * c->desc.page_tokens;
  return TPUHIP_OK;
}

// workgroups of a launch
static int64_t rows_blocks(const tpuhip_ctx *ctx, RowsArgs *a) {
  const int64_t blocks = ceil_div64(a->tokens, kUnitTokens) * a->heads;
  a->half = a->tokens >= kUnitTokens && blocks <= 2 * ctx->num_cu ? (int)blocks : 0;
  return a->half ? 2 * blocks : blocks;
}

}  // namespace tpuhip

using namespace tpuhip;

extern "C" {

size_t tpuhip_kv_cache_bytes(const tpuhip_kv_desc *desc) { return (size_t)kv_bytes(desc, "tpuhip_kv_cache_bytes"); }

int tpuhip_kv_cache_create(tpuhip_ctx *ctx, const tpuhip_kv_desc *desc, tpuhip_kv_cache **out) {
  TPUHIP_REQUIRE(ctx && out, "tpuhip_kv_cache_create: NULL argument");
  const int64_t bytes = kv_bytes(desc, "tpuhip_kv_cache_create");
  if (!bytes) return TPUHIP_ERR_INVALID;
  if (int rc = not_captured(ctx, "tpuhip_kv_cache_create")) return rc;
  void *data = nullptr;
  TPUHIP_CHECK_HIP(hipSetDevice(ctx->device));
  if (int rc = attention_workspace(ctx)) return rc;
  if (int rc = tpuhip_malloc(ctx, (size_t)bytes, &data)) return rc;
  launch(ctx, kv_clear_kernel, dim3((unsigned)std::min<int64_t>(ceil_div64(bytes / 16, 256), 8192)), dim3(256), (uint4 *)data, bytes / 16);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);   // the cache may be used from another context, whose stream does not wait for this one
  tpuhip_kv_cache *c = e == hipSuccess ? new (std::nothrow) tpuhip_kv_cache() : nullptr;
  if (!c) {
    (void)tpuhip_free(ctx, data);
    TPUHIP_CHECK_HIP(e);
    return set_error(TPUHIP_ERR_NOMEM, "tpuhip_kv_cache_create: out of host memory");
  }
  c->device = ctx->device;
  c->desc = *desc;
  c->dp = kv_padded(desc->head_dim);
  c->units_per_page = desc->page_tokens / kUnitTokens;
  c->units = (int64_t)desc->pages * c->units_per_page * desc->kv_heads;
  c->unit_bytes = (int)(bytes / c->units);
  c->data = (uint8_t *)data;
  *out = c;
  return TPUHIP_OK;
}

int tpuhip_kv_cache_destroy(tpuhip_ctx *ctx, tpuhip_kv_cache *cache) {
  TPUHIP_REQUIRE(ctx, "tpuhip_kv_cache_destroy: NULL context");
  if (!cache) return TPUHIP_OK;
  if (int rc = not_captured(ctx, "tpuhip_kv_cache_destroy")) return rc;   // a wait would end the recording
  if (int rc = tpuhip_free(ctx, cache->data)) return rc;
  delete cache;
  return TPUHIP_OK;
}

int tpuhip_kv_write(tpuhip_ctx *ctx, tpuhip_kv_cache *cache, const tpuhip_kv_rows *rows, const int32_t *slots) {
  RowsArgs a{};
  if (int rc = rows_args(ctx, cache, rows, slots, false, "tpuhip_kv_write", &a)) return rc;
  if (a.tokens == 0) return TPUHIP_OK;
  TPUHIP_CHECK_HIP(hipSetDevice(ctx->device));
  return kv_dispatch(cache, [&](auto u) -> int {
    using U = decltype(u);
    const int64_t blocks = rows_blocks(ctx, &a);
    const auto pick = [&](auto wide) {
      constexpr bool W = decltype(wide)::value;
      return rows->dtype == TPUHIP_BF16 ? kv_write_kernel<U, Bf16, W>
             : rows->dtype == TPUHIP_F16 ? kv_write_kernel<U, _Float16, W> : kv_write_kernel<U, float, W>;
    };
    const auto kernel = a.wide ? pick(std::true_type{}) : pick(std::false_type{});
    launch(ctx, kernel, dim3((unsigned)blocks), dim3(kRowsThreads), a);
    TPUHIP_CHECK_HIP(hipGetLastError());
    return TPUHIP_OK;
  });
}

int tpuhip_kv_read(tpuhip_ctx *ctx, const tpuhip_kv_cache *cache, const tpuhip_kv_rows *rows, const int32_t *slots) {
  RowsArgs a{};
  if (int rc = rows_args(ctx, cache, rows, slots, true, "tpuhip_kv_read", &a)) return rc;
  if (a.tokens == 0) return TPUHIP_OK;
  TPUHIP_CHECK_HIP(hipSetDevice(ctx->device));
  return kv_dispatch(cache, [&](auto u) -> int {
    using U = decltype(u);
    const int64_t blocks = rows_blocks(ctx, &a);
    const auto pick = [&](auto wide) {
      constexpr bool W = decltype(wide)::value;
      return rows->dtype == TPUHIP_BF16 ? kv_read_kernel<U, Bf16, W>
             : rows->dtype == TPUHIP_F16 ? kv_read_kernel<U, _Float16, W> : kv_read_kernel<U, float, W>;
    };
    const auto kernel = a.wide ? pick(std::true_type{}) : pick(std::false_type{});
    launch(ctx, kernel, dim3((unsigned)blocks), dim3(kRowsThreads), a);
    TPUHIP_CHECK_HIP(hipGetLastError());
    return TPUHIP_OK;
  });
}

}  // extern "C"
