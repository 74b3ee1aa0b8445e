// Products of rows of microscaled 4-bit numbers: y = x w^T (+ bias) (+ residual).
#include "kv_cache.hpp"
#include "mx.hpp"

#include <algorithm>
#include <type_traits>

namespace tpuhip {

struct MxProductArgs {
  const uint8_t *x, *xs, *w, *ws;   // codes and scales: rows of y, columns of y
  int64_t x_stride, xs_stride, w_stride, ws_stride;
  const float *bias;                // NULL: none
  const void *residual;             // NULL: none
  void *y;
  int64_t y_stride, residual_stride;
  int rows, cols, blocks, dtype;
  FastDiv row_count;
  int depth;                        // numbers of a row, where x is elements; x_stride counts those then
  int groups;                       // of a workgroup's waves, each with columns of its own: 2^groups
  int splits, split_chunks;         // of the sums over 512 numbers each, among workgroups: of each tile; of them
  float *part;                      // their sums
  int *counters;                    // of each tile: splits that have ended
};

typedef int int8m __attribute__((ext_vector_type(8)));

// 16 x 16 products of 128 numbers: lane (r, g) of a wave has row r's block g as 16 bytes and its scale as byte S of a dword, and gets rows
// 4g..4g+3 of column r
template <int S>
__device__ __forceinline__ float4m mx_mfma(uint4m a, uint4m b, float4m c, uint32_t sa, uint32_t sb) {
  const int8m va = {(int)a[0], (int)a[1], (int)a[2], (int)a[3]}, vb = {(int)b[0], (int)b[1], (int)b[2], (int)b[3]};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(va, vb, c, 4, 4, S, (int)sa, S, (int)sb);
}
template <int N, int I = 0, typename F>
__device__ __forceinline__ void times(F f) {                   // f of 0 .. N - 1, as constants
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    times<N, I + 1>(f);
  }
}

// Scales 16 chunk .. 16 chunk + 15 of a row.  Past the row's end they are 0, 2^-127: what such numbers of both operands make is below 2^-200, nothing
// in 32 bits, whatever the codes are.
__device__ __forceinline__ uint4m mx_scales16(const uint8_t *row, int chunk, int blocks) {
  typedef uint32_t dword_any __attribute__((aligned(1)));
  typedef uint16_t half_any __attribute__((aligned(1)));
  const uint8_t *at = row + chunk * 16;
  const int rest = blocks - chunk * 16;
  if (rest >= 16) return *(const uint4m_any *)at;
  uint4m v = {0, 0, 0, 0};
  if (rest <= 0) return v;
  uint64_t few = 0;                                            // of the rest, what is beyond eight
  int shift = 0;
  if (rest & 8) {
    const uint2m first = *(const uint2m_any *)at;
    v[0] = first[0], v[1] = first[1];
    at += 8;
  }
  if (rest & 4) {
    few = *(const dword_any *)at;
    at += 4;
    shift = 32;
  }
  if (rest & 2) {
    few |= (uint64_t)*(const half_any *)at << shift;
    at += 2;
    shift += 16;
  }
  if (rest & 1) few |= (uint64_t)*at << shift;
  if (rest & 8)
    v[2] = (uint32_t)few, v[3] = (uint32_t)(few >> 32);
  else
    v[0] = (uint32_t)few, v[1] = (uint32_t)(few >> 32);
  return v;
}
// of them those of blocks 4 s + g, s = 0..3: byte s of a dword
__device__ __forceinline__ uint32_t mx_picked(uint4m v, int g) {
  const uint32_t pick = 0x0C0C0400u + 0x0101u * (uint32_t)g;   // byte g of the second operand, byte g of the first
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(v[3], v[2], pick), __builtin_amdgcn_perm(v[1], v[0], pick), 0x05040100);
}
__device__ __forceinline__ uint32_t mx_scales(const uint8_t *row, int chunk, int blocks, int g) { return mx_picked(mx_scales16(row, chunk, blocks), g); }

// Four neighbours' biases or residuals.  Past the end the last one again: loads without branches, which do not wait for each other.
__device__ __forceinline__ float4m mx_four(const void *x, int64_t row, int n, int cols, int dtype) {
  if (n + 4 <= cols) return mx_load4(x, row + n, dtype);
  float4m v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = mx_load(x, row + min(n + i, cols - 1), dtype);
  return v;
}
template <bool ONCE = false>
__device__ __forceinline__ void mx_put_four(void *y, int64_t row, int n, int cols, int dtype, float4m v) {
  if (n + 4 <= cols) {
    mx_store4<ONCE>(y, row + n, dtype, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < cols) mx_store(y, row + n + i, dtype, v[i]);
  }
}
// A few rows of x, 16 at most: they lie in LDS as codes while a workgroup goes from 16 columns of y (rows of w) to the next.  Its waves take every
// so manieth 512 numbers of the sums, a chunk; w comes from memory as it lies, a chunk ahead, whichever columns that belongs to; the waves' sums meet in LDS,
// added in the waves' order.  Where sums are short, groups of waves have columns of their own.
//   Bound by the reading of w: 65536 columns of 4096 numbers, 143 MB, by a row of float32 take 24.8 us (5.8 TB/s, some of it from the last cache; 29.8
// with a second chunk ahead, which the compiler moves from register to register and waits for, and 28.5 with biases and residuals asked for before the
// sums); 4096 columns, 9 MB, 4.3 us, half of that the chain of x, its blocks' scales, w and the sums.
//   TYPE: of x's elements, which the workgroup quantises for itself, eight numbers a lane; kMxCodes: x is a matrix.
constexpr int kMxCodes = -1, kMxFew = 16;
constexpr int kMxFewPieces = 64;   // of x, 512 numbers of a row each

template <int TYPE>
struct MxRaw {                       // what a lane brings of 512 numbers of a row
  uint4m v[TYPE == TPUHIP_F32 ? 2 : 1];
};

template <int WAVES, int TYPE, bool GROUPS>
__global__ __launch_bounds__(64 * WAVES) void mx_stream_kernel(MxProductArgs a) {
  __shared__ uint4m rows[kMxFewPieces * 17];                   // [chunk][row][17]: 16 blocks of codes, their scales
  __shared__ float4m sums[2][WAVES][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int chunks = (a.blocks + 15) / 16, tiles = (a.cols + 15) / 16, count = a.rows * chunks;
  struct Chunk {
    uint4m w[4];
    uint32_t s;
  };
  const int groups = GROUPS ? a.groups : 0, step = (int)gridDim.x << groups;
  const int per = WAVES >> groups, place = wave & (per - 1), group = (wave << groups) / WAVES;   // waves of a group, which one this is of them
  const auto load = [&](Chunk &c, int tile, int chunk) {
    const int64_t n = min(tile * 16 + r, a.cols - 1);          // past the end, the last row again
    const uint8_t *w = a.w + n * a.w_stride;
#pragma unroll
    for (int s = 0; s < 4; ++s) c.w[s] = *(const uint4m *)(w + (int64_t)min(chunk * 16 + 4 * s + g, a.blocks - 1) * kMxBytes);
    c.s = mx_scales(a.ws + n * a.ws_stride, chunk, a.blocks, g);
  };
  Chunk now;
  int tile = ((int)blockIdx.x << groups) + group;
  // a wave's chunks, of one tile after the other
  const auto load_after = [&](Chunk &c, int &tile, int &chunk) {
    chunk += per;
    if (chunk >= chunks) {
      chunk = place;
      tile += step;
    }
    if (tile < tiles) load(c, tile, chunk);
  };
  int ahead_tile = tile, ahead = place;
  constexpr int BATCH = 4;
  for (int first = wave; first < max(count, 1 + wave); first += BATCH * WAVES) {
    MxRaw<TYPE> raw[BATCH];
    const auto item = [&](int b, int &m, int &chunk) {         // rows of a chunk follow each other
      const int i = first + b * WAVES;
      uint32_t rest = (uint32_t)i;
      chunk = (int)a.row_count.split(rest);
      m = (int)rest;
      return i < count;
    };
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      int m, chunk;
      if (!item(b, m, chunk)) continue;
      if constexpr (TYPE == kMxCodes) {
        const int block = chunk * 16 + lane / 4;
        const bool there = block < a.blocks;
        raw[b].v[0][0] = there ? ((const uint32_t *)(a.x + m * a.x_stride + (int64_t)block * kMxBytes))[lane & 3] : 0;
        raw[b].v[0][1] = there ? a.xs[m * a.xs_stride + block] : 0;
      } else {
        const int col = chunk * 512 + lane * 8;
        const int64_t at = m * a.x_stride + col;
        if (chunk * 512 + 512 <= a.depth) {
          if constexpr (TYPE == TPUHIP_F32) {
            raw[b].v[0] = *(const uint4m_any *)((const float *)a.x + at);
            raw[b].v[1] = *(const uint4m_any *)((const float *)a.x + at + 4);
          } else {
            raw[b].v[0] = *(const uint4m_any *)((const uint16_t *)a.x + at);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const bool there = col + k < a.depth;
            if constexpr (TYPE == TPUHIP_F32)
              raw[b].v[k / 4][k % 4] = there ? ((const uint32_t *)a.x)[at + k] : 0;
            else
              raw[b].v[0][k / 2] = (k % 2 ? raw[b].v[0][k / 2] : 0) | (there ? (uint32_t)((const uint16_t *)a.x)[at + k] : 0u) << 16 * (k % 2);
          }
        }
      }
    }
    if (first == wave && place < chunks) load(now, tile, place);   // behind x, which is waited for first
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      int m, chunk;
      if (!item(b, m, chunk)) continue;
      uint32_t code, byte;
      if constexpr (TYPE == kMxCodes) {
        code = raw[b].v[0][0];
        byte = raw[b].v[0][1];
      } else {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if constexpr (TYPE == TPUHIP_F32) {
            v[k] = __uint_as_float(raw[b].v[k / 4][k % 4]);
          } else {
            const uint32_t pair = raw[b].v[0][k / 2];
            v[k] = TYPE == TPUHIP_BF16 ? __uint_as_float(k % 2 ? pair & 0xFFFF0000u : pair << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)(pair >> 16 * (k % 2)));
          }
        }
        code = mx_quantised8(v, byte);
      }
      uint4m *at = rows + (chunk * a.rows + m) * 17;
      ((uint32_t *)at)[lane] = code;
      if ((lane & 3) == 0) ((uint8_t *)(at + 16))[lane >> 2] = (uint8_t)byte;
    }
  }
  __syncthreads();
  const uint4m *mine = rows + min(r, a.rows - 1) * 17;         // behind the last row it again: its results go nowhere
  for (int turn = 0; tile - group < tiles; tile += step, ++turn) {   // the same number of times for all groups
    float4m acc = {};
    for (int chunk = place; chunk < chunks; chunk += per) {
      Chunk next;
      load_after(next, ahead_tile, ahead);
      const uint4m *x = mine + chunk * a.rows * 17;
      const uint32_t sx = mx_picked(x[16], g);
      times<4>([&](auto s) {
        constexpr int S = decltype(s)::value;
        acc = mx_mfma<S>(now.w[S], x[4 * S + g], acc, now.s, sx);
      });
      now = next;
    }
    sums[turn & 1][wave][lane] = acc;
    __syncthreads();
    // a wave adds them up while the others go on; it is there again before they are written the time after the next
    if (place == (turn & (per - 1))) {
      float4m v = sums[turn & 1][wave - place][lane];
#pragma unroll
      for (int i = 1; i < WAVES; ++i) {
        const float4m more = sums[turn & 1][(wave - place + i) % WAVES][lane];
        if (i < per) v += more;
      }
      const int n = tile * 16 + g * 4;
      if (r < a.rows && n < a.cols) {
        float4m bias = {}, residual = {};
        if (a.bias) bias = mx_four(a.bias, 0, n, a.cols, TPUHIP_F32);
        if (a.residual) residual = mx_four(a.residual, r * a.residual_stride, n, a.cols, a.dtype);
        mx_put_four(a.y, r * a.y_stride, n, a.cols, a.dtype, v + bias + residual);
      }
    }
  }
}

// Many rows of x: a workgroup of WM x WN waves has a tile of BM rows and BN columns of y.  256 numbers of the tile's rows of both operands, a stage, come
// to LDS past the registers, S stages' room in turn; a wave reads the operands of the next 64 numbers while it multiplies those that it has.  Before a
// stage's last products all waves have read it and the next one has come (one barrier a stage), and its room is filled anew.
//   Order in LDS: rows of 128 bytes, block c of a row in place c ^ row / 2 % 8, so that sixteen lanes that read the same block of rows next to each
// other use all 64 banks (with row % 8 each read took twice the time).  Lane (r, g) has blocks 4g..4g + 3 of a stage: its scales are four bytes.
// Scales come by way of registers, two stages' at a time, and lie behind a stage's data: an access to LDS waits for the loads that are on their way to the
// same array, and one to an array that has none for all of them.
//   Bound by what a CU takes in: a small tile's rows of both operands come at 48 of 64 bytes a clock, with the scales, 16 bytes of a line each, more.
// Without a stage's products, or its reads, 64 x 64 tiles take as long (sums of 16384 numbers, 64 rows: 18.7 us; 14.7 without the scales, 11.5 without
// the data).  256 x 256 are bound by products: 8192 x 8192 x 8192 take 282 to 292 us on different cards, 3.8 PFLOP/s, and 270 at best, at a clock of 1.6 GHz
// that the power leaves (products of registers alone, of random numbers: 6.2 PFLOP/s; on a card that took 266 us, 231 without loads, 253 without results).
constexpr int kMxStage = 8;   // blocks of a stage

typedef __attribute__((address_space(3))) uint8_t mx_lds;
typedef float float16m __attribute__((ext_vector_type(16)));

// 32 x 32 products of 64 numbers: lane (r, g) has row r's block g, and gets rows 8 i + 4 g + 0..3, i = 0..3, of column r
template <int S>
__device__ __forceinline__ float16m mx_mfma32(uint4m a, uint4m b, float16m c, uint32_t sa, uint32_t sb) {
  const int8m va = {(int)a[0], (int)a[1], (int)a[2], (int)a[3]}, vb = {(int)b[0], (int)b[1], (int)b[2], (int)b[3]};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(va, vb, c, 4, 4, S, (int)sa, S, (int)sb);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_buffer(const uint8_t *first, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(first), 0, bytes, 0x00020000);
}
// sixteen bytes a lane, from `at` + the lane's `from`, past the registers to LDS, a lane's behind the other's; zeros from behind the buffer's end
__device__ __forceinline__ void mx_to_lds(__amdgpu_buffer_rsrc_t buffer, uint8_t *to, uint32_t from, int at) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer, (mx_lds *)to, 16, (int)from, at, 0, 0);
}

template <int BM, int BN, int WM, int WN, int S>
__global__ __launch_bounds__(64 * WM * WN, S == 2 ? 2 : 1) void mx_tile_kernel(MxProductArgs a) {
  constexpr int WAVES = WM * WN, THREADS = 64 * WAVES, ROWS = BM + BN;
  constexpr int MF = BM / WM / 32, NF = BN / WN / 32, L = ROWS / 8 / WAVES;  // fragments of a wave; pieces of 8 rows that it brings
  constexpr int SR = (ROWS + THREADS - 1) / THREADS;                         // rows whose scales a thread brings
  constexpr int SCALES = ROWS * 128, SIZE = SCALES + ROWS * 16;              // where they lie, and a stage's room
  static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0 && WAVES % 2 == 0 && (S == 2 || (S == 4 && BM < 256)));
  // arrays of their own: the compiler has a read wait for loads into the same one
#define TPUHIP_MX_ROOM(I) __shared__ __attribute__((aligned(128))) uint8_t room##I[S > I ? SIZE : 16]
  TPUHIP_MX_ROOM(0);
  TPUHIP_MX_ROOM(1);
  TPUHIP_MX_ROOM(2);
  TPUHIP_MX_ROOM(3);
#undef TPUHIP_MX_ROOM
  const auto room = [&](auto u) -> uint8_t * {
    constexpr int U = decltype(u)::value % S;
    if constexpr (U == 0) return room0;
    if constexpr (U == 1) return room1;
    if constexpr (U == 2) return room2;
    return room3;
  };
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 31, g = lane >> 5;
  // Tiles: consecutive workgroups go to different XCDs; those of one have neighbouring tiles, four rows of tiles at a time, so that its L2 holds what
  // they share
  const int tiles_m = (a.rows + BM - 1) / BM, tiles_n = (a.cols + BN - 1) / BN;
  const int per = (int)gridDim.x / 8, more = (int)gridDim.x % 8, xcd = (int)blockIdx.x % 8;
  const int work = xcd * per + min(xcd, more) + (int)blockIdx.x / 8, tile = work / a.splits, split = work % a.splits;
  const int group = tile / (4 * tiles_n), in_group = tile % (4 * tiles_n), high = min(4, tiles_m - 4 * group);
  const int m0 = (4 * group + in_group % high) * BM, n0 = in_group / high * BN;
  const int wm = wave % WM * (BM / WM), wn = wave / WM * (BN / WN);
  // What a lane brings of a piece of 8 rows: a row and a block, as an offset from the tile's first row.  Past a row's end, where scales are 0, that is
  // anything: the next row, or zeros behind the last one, which the buffers' sizes end at.
  uint32_t from[L];
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const int row = (i * WAVES + wave) * 8 + (lane >> 3);
    from[i] = (i * WAVES * 8 < BM ? (uint32_t)min(row, a.rows - 1 - m0) * (uint32_t)a.x_stride : (uint32_t)min(row - BM, a.cols - 1 - n0) * (uint32_t)a.w_stride) +
              ((lane & 7) ^ ((wave & 1) * 4 + (lane >> 4))) * kMxBytes;
  }
  const auto bytes = [&](int rows, int64_t stride) { return (uint32_t)(rows - 1) * (uint32_t)stride + (uint32_t)(a.blocks * kMxBytes); };
  const uint8_t *const x0 = a.x + (int64_t)m0 * a.x_stride, *const w0 = a.w + (int64_t)n0 * a.w_stride;
  const uint32_t x_bytes = bytes(min(BM, a.rows - m0), a.x_stride), w_bytes = bytes(min(BN, a.cols - n0), a.w_stride);
  const int chunk0 = split * a.split_chunks, stage0 = chunk0 * 2;             // this one's
  const int stages = min((a.blocks + kMxStage - 1) / kMxStage, stage0 + a.split_chunks * 2) - stage0;
  const auto load = [&](int t, uint8_t *to) {                  // behind the last stage, of nothing; no branch here: products would be moved past it
    const bool there = t < stages;
    const auto x = mx_buffer(x0, there ? x_bytes : 0), w = mx_buffer(w0, there ? w_bytes : 0);
    const int at = there ? (stage0 + t) * (kMxStage * kMxBytes) : 0;
#pragma unroll
    for (int i = 0; i < L; ++i) mx_to_lds(i * WAVES * 8 < BM ? x : w, to + (i * WAVES + wave) * 1024, from[i], at);
  };
  // scales 16 chunk .. 16 chunk + 15 of a thread's rows.  Without a branch: sixteen that there are, and a shift by bytes; rows of fewer have one
  // chunk, whose scales are not brought here.
  const auto scale_row = [&](int row) {
    return row < BM ? a.xs + (int64_t)min(m0 + row, a.rows - 1) * a.xs_stride : a.ws + (int64_t)min(n0 + row - BM, a.cols - 1) * a.ws_stride;
  };
  const uint8_t *scale_rows[SR];
#pragma unroll
  for (int i = 0; i < SR; ++i) scale_rows[i] = a.blocks >= 16 ? scale_row(min(i * THREADS + (int)threadIdx.x, ROWS - 1)) : a.w;
  uint4m next_scales[SR];
  const auto load_scales = [&](int chunk) {
#pragma unroll
    for (int i = 0; i < SR; ++i) next_scales[i] = *(const uint4m_any *)(scale_rows[i] + max(min(chunk * 16, a.blocks - 16), 0));
  };
  const auto put_scales = [&](auto ends, int chunk, uint8_t *to) {   // ends: of a chunk that may reach past the row's end
    const int drop = min(chunk * 16 - min(chunk * 16, a.blocks - 16), 15);
    const uint32_t one = drop & 4 ? ~0u : 0u, two = drop & 8 ? ~0u : 0u, bytes = drop & 3;
    const auto pick = [](uint32_t mask, uint32_t x, uint32_t y) { return (x & mask) | (y & ~mask); };
#pragma unroll
    for (int i = 0; i < SR; ++i) {
      uint4m v = next_scales[i];
      if constexpr (decltype(ends)::value) {
        v = (uint4m){pick(one, v[1], v[0]), pick(one, v[2], v[1]), pick(one, v[3], v[2]), v[3] & ~one};
        v = (uint4m){pick(two, v[2], v[0]), pick(two, v[3], v[1]), v[2] & ~two, v[3] & ~two};
        v = (uint4m){__builtin_amdgcn_alignbyte(v[1], v[0], bytes), __builtin_amdgcn_alignbyte(v[2], v[1], bytes),
                     __builtin_amdgcn_alignbyte(v[3], v[2], bytes), __builtin_amdgcn_alignbyte(0, v[3], bytes)};
      }
      uint32_t *at = (uint32_t *)(to + SCALES) + min(i * THREADS + (int)threadIdx.x, ROWS - 1) * 4;   // some threads have the same row
      at[0] = v[0], at[1] = v[2], at[2] = v[1], at[3] = v[3];
    }
  };
  struct Operands {
    uint4m x[MF], w[NF];
  };
  struct Scales {
    uint32_t x[MF], w[NF];
  };
  Scales sa, sb;                                               // of two stages
  // Two stages' scales of a lane lie next to each other.  A fragment's address is one that the compiler knows nothing of: of neighbours it makes one read
  // of two places, which it does not know to be of this room alone and has wait for all loads (4096 x 16384, 17 rows: 9.5 us, so 8.6).
  int places[MF + NF];
#pragma unroll
  for (int f = 0; f < MF + NF; ++f) {
    places[f] = SCALES + (f < MF ? wm + f * 32 + r : BM + wn + (f - MF) * 32 + r) * 16 + g * 8;
    asm("" : "+v"(places[f]));
  }
  const auto read_scales = [&](const uint8_t *from) {
#pragma unroll
    for (int f = 0; f < MF + NF; ++f) {
      const uint2m v = *(const uint2m *)(from + places[f]);
      (f < MF ? sa.x[f] : sa.w[f - MF]) = v[0];
      (f < MF ? sb.x[f] : sb.w[f - MF]) = v[1];
    }
  };
  const int at_x = (wm + r) * 128, at_w = (BM + wn + r) * 128, at_block = ((4 * g) ^ (r >> 1 & 7)) * 16;   // of step 0; others by ^ 16 step
  const auto read = [&](Operands &o, const uint8_t *from, int s, int f) {   // one of w's fragments and as many parts of x's
#pragma unroll
    for (int i = f * MF / NF; i < (f + 1) * MF / NF; ++i) o.x[i] = *(const uint4m *)(from + at_x + (at_block ^ s * 16) + i * 32 * 128);
    o.w[f] = *(const uint4m *)(from + at_w + (at_block ^ s * 16) + f * 32 * 128);
  };
  float16m acc[NF][MF] = {};
  // multiplies `now` while the operands of step s of a stage are read
  const auto step = [&](auto byte, auto reads, const Scales &sc, const Operands &now, Operands &next, const uint8_t *from, int s) {
    constexpr int B = decltype(byte)::value;
#pragma unroll
    for (int j = 0; j < NF; ++j) {
      if constexpr (decltype(reads)::value) read(next, from, s, j);
#pragma unroll
      for (int i = 0; i < MF; ++i) acc[j][i] = mx_mfma32<B>(now.w[j], now.x[i], acc[j][i], sc.w[j], sc.x[i]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Waits for a stage, of which `behind` loads may still be on their way, and for all waves to have read what they asked for.  vmcnt counts loads in
  // their order; at least so many have to have been issued behind the stage's own.
  const auto turn = [&](auto behind) {
    constexpr int N = decltype(behind)::value;
    static_assert(N < 64);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 0x70);   // vmcnt(N) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // Operands of the multiplied step and of the next.  A wave of one fragment of each has a whole stage's, and reads the next stage's meanwhile: it waits
  // once a stage for LDS, not four times (sums of 16384 numbers, 64 tiles: 32 x 64 14.8 us, by steps 19.1; 64 x 64 17.4 and 22.3).  Of 128 x 128 they
  // would take the registers that hold two steps' products (34.9 us, by stages 39.2).
  constexpr bool WHOLE = S > 2 && MF * NF == 1;
  Operands p[WHOLE ? 4 : 1], q[WHOLE ? 4 : 1];
  load(0, room0);                                              // what is waited for first, first
  const auto first_scales = [&](auto get) {
    const auto of = [&](int row, uint32_t &even, uint32_t &odd) {
      const uint4m v = get(scale_row(row));
      even = g ? v[1] : v[0];
      odd = g ? v[3] : v[2];
    };
#pragma unroll
    for (int f = 0; f < MF; ++f) of(wm + f * 32 + r, sa.x[f], sb.x[f]);
#pragma unroll
    for (int f = 0; f < NF; ++f) of(BM + wn + f * 32 + r, sa.w[f], sb.w[f]);
  };
  if (chunk0 * 16 + 16 <= a.blocks)
    first_scales([&](const uint8_t *row) { return *(const uint4m_any *)(row + chunk0 * 16); });
  else
    first_scales([&](const uint8_t *row) { return mx_scales16(row, chunk0, a.blocks); });
  load_scales(chunk0 + 1);
  __builtin_amdgcn_sched_barrier(0);
  times<S>([&](auto u) {
    if constexpr (decltype(u)::value > 0) load(decltype(u)::value, room(u));
  });
  turn(std::integral_constant<int, (S - 1) * L>{});
#pragma unroll
  for (int k = 0; k < (WHOLE ? 4 : 1); ++k)
#pragma unroll
    for (int f = 0; f < NF; ++f) read(p[k], room0, k, f);
  constexpr std::true_type yes{};
  constexpr std::false_type no{};
  // A stage; MORE: with the loads of the one S behind it; NEXT: there is a next one.  Behind that one's loads come those of S - 2 stages.
  constexpr std::integral_constant<int, (S - 2) * L> rest{};
  const auto stage = [&](auto u, auto behind, auto more, auto next, auto ends, int t) {
    constexpr int U = decltype(u)::value;
    constexpr bool MORE = decltype(more)::value, NEXT = decltype(next)::value;
    uint8_t *const here = room(u), *const there = room(std::integral_constant<int, U + 1>{});
    constexpr std::integral_constant<int, 0> b0{};
    constexpr std::integral_constant<int, 1> b1{};
    constexpr std::integral_constant<int, 2> b2{};
    constexpr std::integral_constant<int, 3> b3{};
    const Scales now = U % 2 ? sb : sa;
    if constexpr (WHOLE) {
      Operands(&mine)[sizeof(p) / sizeof(p[0])] = U % 2 ? q : p, (&others)[sizeof(p) / sizeof(p[0])] = U % 2 ? p : q;
      if constexpr (NEXT) {
        turn(behind);
        if constexpr (U % 2 == 1) read_scales(here);
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int f = 0; f < NF; ++f) read(others[k], there, k, f);
        if constexpr (U % 2 == 0) {
          put_scales(ends, chunk0 + t / 2 + 1, there);
          if constexpr (MORE) load_scales(chunk0 + t / 2 + 2);
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (MORE) load(t + S, here);
      }
      step(b0, no, now, mine[0], others[0], there, 0);
      step(b1, no, now, mine[1], others[1], there, 0);
      step(b2, no, now, mine[2], others[2], there, 0);
      step(b3, no, now, mine[3], others[3], there, 0);
    } else {
      step(b0, yes, now, p[0], q[0], here, 1);
      if constexpr (NEXT && U % 2 == 1) put_scales(ends, chunk0 + t / 2 + 1, here);
      __builtin_amdgcn_sched_barrier(0);
      step(b1, yes, now, q[0], p[0], here, 2);
      step(b2, yes, now, p[0], q[0], here, 3);
      if constexpr (NEXT) {
        turn(behind);
        if constexpr (U % 2 == 1) {
          read_scales(here);
          if constexpr (MORE) load_scales(chunk0 + t / 2 + 2);   // before the data: what is in registers has come when the data before it have
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (MORE) load(t + S, here);
      }
      step(b3, next, now, q[0], p[0], there, 0);
    }
  };
  constexpr std::integral_constant<int, 0> u0{};
  constexpr std::integral_constant<int, 1> u1{};
  // No way out of a loop in between: the compiler would have it wait for loads on that way.
  int t = 0;
  if constexpr (S == 2) {                                      // in pairs; behind the last stage come scales of 0
    for (; t + 2 < stages; t += 2) {
      stage(u0, rest, yes, yes, yes, t);
      stage(u1, rest, yes, yes, yes, t + 1);
    }
    stage(u0, rest, no, yes, yes, t);
    if (BM >= 256 || t + 1 < stages) stage(u1, rest, no, no, yes, t + 1);   // of the largest tiles always: a way around it costs them registers
  } else {
    // The loop ends before a chunk that may reach past a row's end is put, as a wave has a SIMD to itself where tiles are few: 64 x 64, sums of 16384
    // numbers, 64 tiles: 16.2 us, with the shifts of the ends in it 17.6; 128 x 128 31.6 and 35.0.  Up to S + 2 stages are left then, of S that have been
    // asked for (those that there are not: zeros).
    for (; t + S + 3 <= stages; t += S) times<S>([&](auto u) { stage(u, rest, yes, yes, no, t + decltype(u)::value); });
    times<S + 2>([&](auto u) {
      constexpr int U = decltype(u)::value;
      constexpr std::integral_constant<int, (U < 2 ? S - 2 : U < S ? S - U : 0) * L> behind{};
      if (t + U < stages) stage(u, behind, std::bool_constant<(U < 2)>{}, yes, yes, t + U);
    });
  }
  turn(std::integral_constant<int, 0>{});                      // nothing is on its way to LDS any more
  if (a.splits > 1) {
    // Splits meet in memory, past the caches that a device's XCDs have of their own, as their lanes have them; the last of a tile's to end adds them
    // in their order
    constexpr int PARTS = NF * MF * 8;                         // pairs of a lane
    const int64_t between = (int64_t)PARTS * THREADS;
    uint64_t *part = (uint64_t *)a.part + (int64_t)tile * a.splits * between + threadIdx.x;
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int k = 0; k < 8; ++k)
          __hip_atomic_store(part + split * between + ((j * MF + i) * 8 + k) * THREADS,
                             __builtin_bit_cast(uint64_t, (float2m){acc[j][i][2 * k], acc[j][i][2 * k + 1]}), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __shared__ int last;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
      const int before = __hip_atomic_fetch_add(a.counters + tile, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      last = before == a.splits - 1;
      if (last) __hip_atomic_store(a.counters + tile, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);   // for the next call
    }
    __syncthreads();
    if (!last) return;
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
      for (int i = 0; i < MF; ++i) acc[j][i] = (float16m){};
    constexpr int AT_ONCE = NF * MF == 1 ? 4 : NF * MF <= 2 ? 2 : 1;   // splits whose sums are on their way together (one by one: 4.5 us for four of 64 x 64)
    for (int p0 = 0; p0 < a.splits; p0 += AT_ONCE) {
      float2m v[AT_ONCE][NF][MF][8];
#pragma unroll
      for (int p = 0; p < AT_ONCE; ++p)
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
          for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k)
              v[p][j][i][k] = __builtin_bit_cast(float2m, __hip_atomic_load(part + min(p0 + p, a.splits - 1) * between + ((j * MF + i) * 8 + k) * THREADS,
                                                                            __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
#pragma unroll
      for (int p = 0; p < AT_ONCE; ++p)
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
          for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
              for (int h = 0; h < 2; ++h) acc[j][i][2 * k + h] += p0 + p < a.splits ? v[p][j][i][k][h] : 0.0f;
    }
  }
  // Results go through LDS, a wave's by itself, 32 rows at a time: then a lane has four neighbours of a row, the same ones of every row, and FOURS lanes
  // have a row of the wave's.  Four numbers c of row m lie in place c ^ key(m).
  constexpr int FOURS = NF * 8, PASS = 64 / FOURS, PASSES = 32 / PASS;
  constexpr int HERE = WAVES * 32 * FOURS * 16 <= ROWS * 128 ? WAVES : WAVES / 2;   // waves that a room is large enough for
  static_assert(HERE * 32 * FOURS * 16 <= ROWS * 128);
  float4m *mine = (float4m *)(wave < HERE ? room0 : room1) + wave % HERE * 32 * FOURS;
  const auto key = [](int row) { return FOURS == 8 ? row >> 1 & 7 : row & (FOURS < 16 ? FOURS - 1 : 15); };   // sixteen rows in all banks
  const int four = lane % FOURS, row0 = lane / FOURS, n = n0 + wn + 4 * four;
  const float4m bias = a.bias ? mx_four(a.bias, 0, min(n, a.cols - 1), a.cols, TPUHIP_F32) : (float4m){0, 0, 0, 0};
  const auto results = [&](auto type) {
    constexpr int TYPE = decltype(type)::value;
#pragma unroll
    for (int i = 0; i < MF; ++i) {
#pragma unroll
      for (int j = 0; j < NF; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mine[r * FOURS + ((j * 8 + 2 * k + g) ^ key(r))] = (float4m){acc[j][i][4 * k], acc[j][i][4 * k + 1], acc[j][i][4 * k + 2], acc[j][i][4 * k + 3]};
      __builtin_amdgcn_wave_barrier();
      float4m v[PASSES];
#pragma unroll
      for (int k = 0; k < PASSES; ++k) {
        const int row = k * PASS + row0;
        v[k] = mine[row * FOURS + (four ^ key(row))];
      }
      __builtin_amdgcn_wave_barrier();
      const int first = m0 + wm + i * 32 + row0;
      if (n >= a.cols) continue;
#pragma unroll
      for (int k = 0; k < PASSES; ++k) v[k] += bias;
      if (a.residual) {
        float4m more[PASSES];
#pragma unroll
        for (int k = 0; k < PASSES; ++k) more[k] = mx_four(a.residual, (int64_t)min(first + k * PASS, a.rows - 1) * a.residual_stride, n, a.cols, TYPE);
#pragma unroll
        for (int k = 0; k < PASSES; ++k) v[k] += more[k];
      }
#pragma unroll
      for (int k = 0; k < PASSES; ++k)
        if (first + k * PASS < a.rows) mx_put_four<(BM >= 256)>(a.y, (int64_t)(first + k * PASS) * a.y_stride, n, a.cols, TYPE, v[k]);
    }
  };
  if (a.dtype == TPUHIP_BF16)
    results(std::integral_constant<int, TPUHIP_BF16>{});
  else if (a.dtype == TPUHIP_F16)
    results(std::integral_constant<int, TPUHIP_F16>{});
  else
    results(std::integral_constant<int, TPUHIP_F32>{});
}

static int mx_product_args(tpuhip_ctx *ctx, const tpuhip_mx_product_desc *d, const tpuhip_mx_matrix *x, const tpuhip_mx_matrix *w, void *y,
                           const char *what, MxProductArgs *a) {
  TPUHIP_REQUIRE(ctx && d, "%s: NULL argument", what);
  if (int rc = mx_check(x, "x", what)) return rc;
  if (int rc = mx_check(w, "w", what)) return rc;
  TPUHIP_REQUIRE(x->cols == w->cols, "%s: x has %d columns, w %d", what, x->cols, w->cols);
  TPUHIP_REQUIRE(w->rows >= 1, "%s: w without rows", what);
  if (int rc = mx_check_rows(x->rows, w->rows, y, d->dtype, d->y_stride, true, "y", what)) return rc;
  if (d->residual)
    if (int rc = mx_check_rows(x->rows, w->rows, d->residual, d->dtype, d->residual_stride, false, "the residual", what)) return rc;
  TPUHIP_REQUIRE((uintptr_t)d->bias % 4 == 0, "%s: the bias does not begin at an element", what);
  TPUHIP_REQUIRE(x->rows <= 1 << 30 && w->rows <= 1 << 30, "%s: %d rows, %d columns", what, x->rows, w->rows);
  for (const tpuhip_mx_matrix *m : {x, w})                     // a tile's rows are reached by 32 bits
    TPUHIP_REQUIRE(m->rows == 1 || m->codes_stride < 1 << 24, "%s: rows of codes lie %lld bytes apart", what, (long long)m->codes_stride);
  *a = MxProductArgs{};
  a->x = (const uint8_t *)x->codes;
  a->xs = (const uint8_t *)x->scales;
  a->w = (const uint8_t *)w->codes;
  a->ws = (const uint8_t *)w->scales;
  a->x_stride = x->codes_stride;
  a->xs_stride = x->scales_stride;
  a->w_stride = w->codes_stride;
  a->ws_stride = w->scales_stride;
  a->bias = d->bias;
  a->residual = d->residual;
  a->y = y;
  a->y_stride = d->y_stride;
  a->residual_stride = d->residual_stride;
  a->rows = x->rows;
  a->cols = w->rows;
  a->row_count = FastDiv(std::max(x->rows, 1));
  a->blocks = mx_blocks(x->cols);
  a->dtype = d->dtype;
  return TPUHIP_OK;
}

// Forms of the tile kernel, and what a call takes in each, in microseconds: some for the first loads and the results, and a stage as much as `low` with one
// workgroup, `one` with one on each CU and `full` with `at_once` of them, which is as many as have room; more come in turns.  Measured | as worked out
// here, with sums of 4096 numbers (16 stages):
//   32 x 64     64 .. 256 tiles  6.1   6.8 | 6.3  6.6     512   9.8 | 10.4
//   64 x 64     64 .. 256        6.9   8.2 | 7.1  7.8     512  13.3 | 13.1     1024  21.9 | 23.4
//   64 x 128    32 .. 256        9.4  12.3 | 9.4 11.9     512  21.5 | 23.9
//   128 x 128   32 .. 256       12.2  17.5 | 12.5 15.4
//   128 x 128   128 .. 256      15.0  18.2 | 16.7 17.5    512  28.4 | 28.8     1032  60.4 | 62.8
//   256 x 128   32 .. 256       19.1  25.3 | 19.5 24.0    688  68.0 | 70.3
//   256 x 256   64 .. 256       29.9  43.0 | 29.7 42.3    688  115  | 121      1024 (32 stages)  282 | 300
// Over 156 sizes of bfloat16 results what is chosen takes 1.2 % more than the quickest form in the mean and 15.5 % at the worst, with results of
// float32, biases and residuals 1.5 % and 28.6 %.
struct MxForm {
  int rows, cols, at_once;
  float base, low, one, full;
};
constexpr MxForm kMxForms[] = {{32, 64, 2, 3.4f, 0.17f, 0.20f, 0.31f},   {64, 64, 2, 3.5f, 0.21f, 0.27f, 0.47f},   {64, 128, 1, 4.1f, 0.31f, 0.49f, 0.49f},
                               {128, 128, 1, 5.2f, 0.43f, 0.64f, 0.64f}, {128, 128, 2, 6.0f, 0.62f, 0.72f, 1.20f}, {256, 128, 1, 6.4f, 0.78f, 1.10f, 1.10f},
                               {256, 256, 1, 9.5f, 1.00f, 2.05f, 2.05f}};
constexpr int kMxFormCount = sizeof(kMxForms) / sizeof(kMxForms[0]);

struct MxChoice {
  int form, splits;
};
// Sums in parts cost their joining, measured in two and in four parts: 32 x 64 tiles 2.1 and 3.6 us, 64 x 64 2.9 and 4, 64 x 128 3.6 and 5.3, 128 x 128 6.6
// and 10.5.  bytes: that a result and what it is added to take, which a CU moves 40 KB a microsecond of; two are in the table above.  777 x 2050 x 4999 of
// float32 with a residual, 8 bytes: 128 x 128 22.9 us, 256 x 128 23.7; of 2 bytes 18.8 and 17.5.
static MxChoice mx_choose(int64_t rows, int64_t cols, int blocks, int bytes, int num_cu) {
  MxChoice best = {0, 1};
  float least = 0;
  const int stages = (blocks + kMxStage - 1) / kMxStage;
  for (int f = 0; f < kMxFormCount; ++f) {
    const MxForm &form = kMxForms[f];
    const int64_t tiles = ceil_div64(rows, form.rows) * ceil_div64(cols, form.cols), room = (int64_t)form.at_once * num_cu;
    for (int splits = 1; splits <= 8 && (splits == 1 || (form.rows < 256 && tiles * splits <= num_cu && splits * 2 <= stages)); splits *= 2) {
      const int64_t whole = tiles * splits / room, rest = tiles * splits % room;
      const float load = (float)rest / num_cu, size = form.rows * form.cols / 4096.0f;
      const float last = load <= 1 ? form.low + (form.one - form.low) * load : form.one + (form.full - form.one) * (load - 1);
      const float each = whole * form.full + (rest ? last : 0.0f);
      const float join = splits > 1 ? 0.8f + 0.4f * splits + size * (0.7f + 0.3f * splits) : 0.0f;
      const float loads = (float)tiles * splits / num_cu;
      const float starts = form.at_once == 1 ? whole + (rest != 0) : loads <= 1 ? 1 : 1.6f + 0.4f * std::max(loads - 2, 0.0f);   // with others at work meanwhile
      const float moves = (bytes - 2) * form.rows * form.cols / 40000.0f * (form.at_once == 1 ? starts : std::max(1.3f * loads, 1.0f));
      const float cost = form.base * starts + each * ((stages + splits - 1) / splits) + join + moves;
      if ((f == 0 && splits == 1) || cost < least) {
        least = cost;
        best = {f, splits};
      }
    }
  }
  return best;
}

// Workgroups whose tiles are too few for the device share the sums of each
template <int BM, int BN, int WM, int WN, int S>
static int mx_launch_tiles(tpuhip_ctx *ctx, MxProductArgs a, int splits) {
  const int64_t tiles = ceil_div64(a.rows, BM) * ceil_div64(a.cols, BN);
  TPUHIP_REQUIRE(tiles <= UINT32_MAX / (64 * WM * WN), "a product of %d rows and %d columns in one call", a.rows, a.cols);   // a launch has fewer than 2^32 threads
  const int chunks = (a.blocks + 15) / 16;
  if (splits > 1 && (!ctx->join || tiles > kCounters || tiles * splits * BM * BN * 4 > (int64_t)kJoinBytes)) splits = 1;
  a.split_chunks = (int)ceil_div64(chunks, splits);
  a.splits = (int)ceil_div64(chunks, a.split_chunks);
  a.counters = (int *)ctx->join;
  a.part = (float *)((char *)ctx->join + kCounters * 4);
  launch(ctx, mx_tile_kernel<BM, BN, WM, WN, S>, dim3((unsigned)(tiles * a.splits)), dim3(64 * WM * WN), a);
  TPUHIP_CHECK_HIP(hipGetLastError());
  return TPUHIP_OK;
}

static int64_t mx_chunks(const MxProductArgs &a) { return (a.blocks + 15) / 16; }

// Rows of x that every workgroup quantises or copies for itself, 512 numbers of a row at a time: from some number of those on, tiles, and quantising x
// in a launch of its own for them, are quicker.  x, w of 4096 x 4096: 1 row of bfloat16 4.4 us and 7.9 in tiles, 4 rows 5.3 and 7.9, 8 rows (64 pieces)
// 7.0 and 8.3, 12 rows 8.8 and 8.4; 3 rows of 16384 (96) 12.4 and 12.6; x in 4 bits: 1 row 4.1 and 5.7, 4 rows (32) 5.1 and 5.6, 8 rows 6.4 and 5.8.
static bool mx_streams(const MxProductArgs &a, int type) {
  return a.rows <= kMxFew && a.rows * mx_chunks(a) <= (type == kMxCodes ? kMxFewPieces / 2 : kMxFewPieces);
}

// Up to two workgroups a CU, each of which goes from columns to columns: of 16384 columns one row takes 9.1 us so, 10.0 with four a CU.  Eight waves
// where sums are long (16384 numbers: 10.7 us, with four 12.3) or columns many (65536: 24.8 and 30.1), otherwise four (4096 x 4096: 4.3 us, with eight 4.6).
// Groups where some waves would have nothing and there are columns for all: 3 rows x 224 x 44346 4.5 us, with one group 7.2; 4 x 512 x 65536 5.8 and 8.5.
template <int WAVES>
static int mx_launch_stream(tpuhip_ctx *ctx, MxProductArgs a, int type) {
  const int64_t columns = ceil_div64(a.cols, 16);
  while (mx_chunks(a) << (a.groups + 1) <= WAVES && columns > (int64_t)2 * ctx->num_cu << a.groups) ++a.groups;
  const int64_t tiles = ceil_div64(columns, 1 << a.groups), turns = ceil_div64(tiles, 2 * ctx->num_cu);
  const auto kernel = [&](auto groups) {
    constexpr bool GROUPS = decltype(groups)::value;
    return type == kMxCodes ? mx_stream_kernel<WAVES, kMxCodes, GROUPS> : type == TPUHIP_BF16 ? mx_stream_kernel<WAVES, TPUHIP_BF16, GROUPS>
           : type == TPUHIP_F16 ? mx_stream_kernel<WAVES, TPUHIP_F16, GROUPS> : mx_stream_kernel<WAVES, TPUHIP_F32, GROUPS>;
  };
  launch(ctx, a.groups ? kernel(std::true_type{}) : kernel(std::false_type{}), dim3((unsigned)ceil_div64(tiles, turns)), dim3(64 * WAVES), a);
  TPUHIP_CHECK_HIP(hipGetLastError());
  return TPUHIP_OK;
}

// type: of x's elements, where mx_streams() takes those, or kMxCodes: x is a matrix
static int mx_multiply(tpuhip_ctx *ctx, const MxProductArgs &a, int type) {
  // with any product, not with the first in parts: that one may be recorded, and would be in one part where the same call by itself is in several
  if (int rc = attention_workspace(ctx)) return rc;
  if (mx_streams(a, type)) return mx_chunks(a) > 8 || a.cols > 128 * ctx->num_cu ? mx_launch_stream<8>(ctx, a, type) : mx_launch_stream<4>(ctx, a, type);
  const MxChoice c = mx_choose(a.rows, a.cols, a.blocks, mx_size(a.dtype) * (a.residual ? 2 : 1), ctx->num_cu);
  switch (c.form) {
    case 0: return mx_launch_tiles<32, 64, 1, 2, 4>(ctx, a, c.splits);
    case 1: return mx_launch_tiles<64, 64, 2, 2, 4>(ctx, a, c.splits);
    case 2: return mx_launch_tiles<64, 128, 1, 4, 4>(ctx, a, c.splits);
    case 3: return mx_launch_tiles<128, 128, 2, 2, 4>(ctx, a, c.splits);
    case 4: return mx_launch_tiles<128, 128, 2, 2, 2>(ctx, a, c.splits);
    case 5: return mx_launch_tiles<256, 128, 4, 2, 2>(ctx, a, c.splits);
    default: return mx_launch_tiles<256, 256, 2, 4, 2>(ctx, a, c.splits);
  }
}

}  // namespace tpuhip

using namespace tpuhip;

extern "C" {

int tpuhip_mx_product(tpuhip_ctx *ctx, const tpuhip_mx_product_desc *desc, const tpuhip_mx_matrix *x, const tpuhip_mx_matrix *w, void *y) {
  MxProductArgs a;
  if (int rc = mx_product_args(ctx, desc, x, w, y, "tpuhip_mx_product", &a)) return rc;
  if (a.rows == 0) return TPUHIP_OK;
  TPUHIP_CHECK_HIP(hipSetDevice(ctx->device));
  return mx_multiply(ctx, a, kMxCodes);
}

int tpuhip_mx_linear(tpuhip_ctx *ctx, const tpuhip_mx_product_desc *desc, const void *x, int x_dtype, int64_t x_stride,
                     const tpuhip_mx_matrix *room, const tpuhip_mx_matrix *w, void *y) {
  const char *what = "tpuhip_mx_linear";
  MxProductArgs a;
  if (int rc = mx_product_args(ctx, desc, room, w, y, what, &a)) return rc;
  if (int rc = mx_check_rows(a.rows, room->cols, x, x_dtype, x_stride, false, "x", what)) return rc;
  if (a.rows == 0) return TPUHIP_OK;
  TPUHIP_CHECK_HIP(hipSetDevice(ctx->device));
  if (mx_streams(a, x_dtype)) {                                // quantised on the way
    a.x = (const uint8_t *)x;
    a.x_stride = x_stride;
    a.depth = room->cols;
    return mx_multiply(ctx, a, x_dtype);
  }
  if (int rc = mx_quantize(ctx, room, x, x_dtype, x_stride, what)) return rc;
  return mx_multiply(ctx, a, kMxCodes);
}

}  // extern "C"
