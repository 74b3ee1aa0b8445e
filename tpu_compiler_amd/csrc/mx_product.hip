// Products of rows of microscaled 4-bit numbers: y = x w^T (+ bias) (+ residual).
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
};

typedef int int8m __attribute__((ext_vector_type(8)));

// 16 x 16 products of 128 numbers: lane (r, g) of a wave has row r's block g as 16 bytes and its scale as byte S of a dword, and gets rows
// 4g..4g+3 of column r
template <int S>
__device__ __forceinline__ float4m mx_mfma(uint4m a, uint4m b, float4m c, uint32_t sa, uint32_t sb) {
  const int8m va = {(int)a[0], (int)a[1], (int)a[2], (int)a[3]}, vb = {(int)b[0], (int)b[1], (int)b[2], (int)b[3]};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(va, vb, c, 4, 4, S, (int)sa, S, (int)sb);
}
template <typename F>
__device__ __forceinline__ void four_times(F f) {
  f(std::integral_constant<int, 0>{});
  f(std::integral_constant<int, 1>{});
  f(std::integral_constant<int, 2>{});
  f(std::integral_constant<int, 3>{});
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
__device__ __forceinline__ uint32_t mx_scales(const uint8_t *row, int chunk, int blocks, int g) {
  const uint4m v = mx_scales16(row, chunk, blocks);
  const uint32_t pick = 0x0C0C0400u + 0x0101u * (uint32_t)g;   // byte g of the second operand, byte g of the first
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(v[3], v[2], pick), __builtin_amdgcn_perm(v[1], v[0], pick), 0x05040100);
}

// four neighbours of a row of y
__device__ __forceinline__ void mx_result(const MxProductArgs &a, int m, int n, float4m v) {
  const int64_t from = (int64_t)m * a.residual_stride + n, to = (int64_t)m * a.y_stride + n;
  if (n + 4 <= a.cols) {
    if (a.bias) v += mx_load4(a.bias, n, TPUHIP_F32);
    if (a.residual) v += mx_load4(a.residual, from, a.dtype);
    mx_store4(a.y, to, a.dtype, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n + i >= a.cols) return;
    if (a.bias) v[i] += a.bias[n + i];
    if (a.residual) v[i] += mx_load(a.residual, from + i, a.dtype);
    mx_store(a.y, to + i, a.dtype, v[i]);
  }
}

// Few rows of x: a workgroup has 16 NT columns of y (rows of w) and 16 MT rows; its waves take every so manieth 512 numbers of the sums, operands
// come from memory as they lie, and the waves' sums meet in LDS, added in the waves' order.
template <int NT, int MT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void mx_stream_kernel(MxProductArgs a) {
  __shared__ float4m sums[WAVES][NT * MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int n0 = (int)blockIdx.x * 16 * NT, m0 = (int)blockIdx.y * 16 * MT;
  const uint8_t *w[NT], *ws[NT], *x[MT], *xs[MT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {                               // past the end, the last row again
    const int64_t n = min(n0 + 16 * j + r, a.cols - 1);
    w[j] = a.w + n * a.w_stride;
    ws[j] = a.ws + n * a.ws_stride;
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t m = min(m0 + 16 * i + r, a.rows - 1);
    x[i] = a.x + m * a.x_stride;
    xs[i] = a.xs + m * a.xs_stride;
  }
  float4m acc[NT][MT] = {};
  for (int chunk = wave; chunk * 16 < a.blocks; chunk += WAVES) {
    uint32_t sw[NT], sx[MT];
#pragma unroll
    for (int j = 0; j < NT; ++j) sw[j] = mx_scales(ws[j], chunk, a.blocks, g);
#pragma unroll
    for (int i = 0; i < MT; ++i) sx[i] = mx_scales(xs[i], chunk, a.blocks, g);
    four_times([&](auto s) {
      constexpr int S = decltype(s)::value;
      const int64_t at = (int64_t)min(chunk * 16 + 4 * S + g, a.blocks - 1) * kMxBytes;
      uint4m vw[NT], vx[MT];
#pragma unroll
      for (int j = 0; j < NT; ++j) vw[j] = *(const uint4m *)(w[j] + at);
#pragma unroll
      for (int i = 0; i < MT; ++i) vx[i] = *(const uint4m *)(x[i] + at);
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[j][i] = mx_mfma<S>(vw[j], vx[i], acc[j][i], sw[j], sx[i]);
    });
  }
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) sums[wave][j * MT + i][lane] = acc[j][i];
  __syncthreads();
  for (int k = threadIdx.x; k < NT * MT * 64; k += 64 * WAVES) {
    float4m v = sums[0][k / 64][k % 64];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) v += sums[i][k / 64][k % 64];
    const int m = m0 + k / 64 % MT * 16 + k % 16, n = n0 + k / 64 / MT * 16 + k % 64 / 16 * 4;
    if (m < a.rows && n < a.cols) mx_result(a, m, n, v);
  }
}

// Many rows of x: a workgroup of WM x WN waves has a tile of BM rows and BN columns of y.  256 numbers of the tile's rows
// of both operands, a stage, come to LDS past the registers while the stage before is multiplied; a wave reads the operands of the next 64
// numbers while it multiplies those that it has, so that the matrix unit waits for neither, and there is one barrier a stage.
//   Order in LDS: rows of 128 bytes, block c of a row in place c ^ row / 2 % 8, so that sixteen lanes that read the same block of rows next to each
// other use all 64 banks (with row % 8 each read took twice the time).  Lane (r, g) has blocks 4g..4g + 3 of a stage: its scales are four bytes, a dword in LDS.
constexpr int kMxStage = 8;   // blocks of a stage

typedef __attribute__((address_space(1))) const uint8_t mx_global;
typedef __attribute__((address_space(3))) uint8_t mx_lds;
typedef float float16m __attribute__((ext_vector_type(16)));

// 32 x 32 products of 64 numbers: lane (r, g) has row r's block g, and gets rows 8 i + 4 g + 0..3, i = 0..3, of column r
template <int S>
__device__ __forceinline__ float16m mx_mfma32(uint4m a, uint4m b, float16m c, uint32_t sa, uint32_t sb) {
  const int8m va = {(int)a[0], (int)a[1], (int)a[2], (int)a[3]}, vb = {(int)b[0], (int)b[1], (int)b[2], (int)b[3]};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(va, vb, c, 4, 4, S, (int)sa, S, (int)sb);
}

template <int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void mx_tile_kernel(MxProductArgs a) {
  constexpr int WAVES = WM * WN, THREADS = 64 * WAVES, ROWS = BM + BN;
  constexpr int MF = BM / WM / 32, NF = BN / WN / 32, L = ROWS / 8 / WAVES;  // fragments of a wave; pieces of 8 rows that it brings
  constexpr int SR = ROWS / THREADS;                                         // rows whose scales a thread brings
  static_assert(ROWS % THREADS == 0 && BM % (8 * WAVES) == 0 && WAVES % 2 == 0 && MF % NF == 0);
  __shared__ __attribute__((aligned(128))) uint8_t stage0[ROWS * 128];
  __shared__ __attribute__((aligned(128))) uint8_t stage1[ROWS * 128];
  __shared__ uint32_t scales[2][4][ROWS];                      // of two stages, four bytes each: [of which two][stage, g][row]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 31, g = lane >> 5;
  // Tiles: consecutive workgroups go to different XCDs; those of one have neighbouring tiles, four rows of tiles at a time, so that its L2 holds what
  // they share
  const int tiles_m = (a.rows + BM - 1) / BM, tiles_n = (a.cols + BN - 1) / BN, tiles = tiles_m * tiles_n;
  const int per = tiles / 8, more = tiles % 8, xcd = (int)blockIdx.x % 8;
  const int tile = xcd * per + min(xcd, more) + (int)blockIdx.x / 8;
  const int group = tile / (4 * tiles_n), in_group = tile % (4 * tiles_n), high = min(4, tiles_m - 4 * group);
  const int m0 = (4 * group + in_group % high) * BM, n0 = in_group / high * BN;
  const int wm = wave % WM * (BM / WM), wn = wave / WM * (BN / WN);
  // what a lane brings of a piece of 8 rows: a row, as an offset from the tile's first row, and a block
  uint32_t from[L];
#pragma unroll
  for (int i = 0; i < L; ++i) {
    const int row = (i * WAVES + wave) * 8 + (lane >> 3);
    from[i] = i * WAVES * 8 < BM ? (uint32_t)min(row, a.rows - 1 - m0) * (uint32_t)a.x_stride : (uint32_t)min(row - BM, a.cols - 1 - n0) * (uint32_t)a.w_stride;
  }
  const int block = (lane & 7) ^ ((wave & 1) * 4 + (lane >> 4));
  const uint8_t *x0 = a.x + (int64_t)m0 * a.x_stride, *w0 = a.w + (int64_t)n0 * a.w_stride;
  const int stages = (a.blocks + kMxStage - 1) / kMxStage;
  const auto load = [&](int t, uint8_t *stage) {
    t = min(t, stages - 1);                                    // no branch here: products would be moved past it
    const uint32_t at = (uint32_t)(min(block, a.blocks - 1 - t * kMxStage) * kMxBytes);   // past the row's end, its last block again: its scales are 0
#pragma unroll
    for (int i = 0; i < L; ++i)
      __builtin_amdgcn_global_load_lds((mx_global *)((i * WAVES * 8 < BM ? x0 : w0) + t * (kMxStage * kMxBytes) + (from[i] + at)),
                                       (mx_lds *)(stage + (i * WAVES + wave) * 1024), 16, 0, 0);
  };
  const uint8_t *scale_rows[SR];
#pragma unroll
  for (int i = 0; i < SR; ++i) {
    const int row = i * THREADS + threadIdx.x;
    scale_rows[i] = row < BM ? a.xs + (int64_t)min(m0 + row, a.rows - 1) * a.xs_stride : a.ws + (int64_t)min(n0 + row - BM, a.cols - 1) * a.ws_stride;
  }
  uint4m next_scales[SR];
  const auto load_scales = [&](int chunk) {                    // of the last stages they may be others': see below
#pragma unroll
    for (int i = 0; i < SR; ++i) next_scales[i] = *(const uint4m_any *)(scale_rows[i] + min(chunk * 16, a.blocks - 16));
  };
  const auto put_scales = [&](int chunk) {
#pragma unroll
    for (int i = 0; i < SR; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) scales[chunk & 1][k][i * THREADS + threadIdx.x] = next_scales[i][k];
  };
  struct Operands {
    uint4m x[MF], w[NF];
  };
  struct Scales {
    uint32_t x[MF], w[NF];
  };
  const auto read_scales = [&](Scales &s, int t) {
    const uint32_t *at = scales[t >> 1 & 1][(t & 1) * 2 + g];
#pragma unroll
    for (int f = 0; f < MF; ++f) s.x[f] = at[wm + f * 32 + r];
#pragma unroll
    for (int f = 0; f < NF; ++f) s.w[f] = at[BM + wn + f * 32 + r];
  };
  const int at_x = (wm + r) * 128, at_w = (BM + wn + r) * 128, at_block = ((4 * g) ^ (r >> 1 & 7)) * 16;   // of step 0; others by ^ 16 step
  const auto read = [&](Operands &o, const uint8_t *stage, int s, int f) {   // one of w's fragments and as many parts of x's
#pragma unroll
    for (int i = f * MF / NF; i < (f + 1) * MF / NF; ++i) o.x[i] = *(const uint4m *)(stage + at_x + (at_block ^ s * 16) + i * 32 * 128);
    o.w[f] = *(const uint4m *)(stage + at_w + (at_block ^ s * 16) + f * 32 * 128);
  };
  float16m acc[NF][MF] = {};
  // multiplies `now` while the operands of step s of a stage are read
  const auto step = [&](auto byte, auto reads, const Scales &sc, const Operands &now, Operands &next, const uint8_t *stage, int s) {
    constexpr int S = decltype(byte)::value;
#pragma unroll
    for (int j = 0; j < NF; ++j) {
      if constexpr (decltype(reads)::value) read(next, stage, s, j);
#pragma unroll
      for (int i = 0; i < MF; ++i) acc[j][i] = mx_mfma32<S>(now.w[j], now.x[i], acc[j][i], sc.w[j], sc.x[i]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  constexpr std::integral_constant<int, 0> b0{};
  constexpr std::integral_constant<int, 1> b1{};
  constexpr std::integral_constant<int, 2> b2{};
  constexpr std::integral_constant<int, 3> b3{};
  Operands p, q;
  Scales sa, sb;                                               // of two stages
  load(0, stage0);
  load_scales(0);                                              // there are sixteen at least
  put_scales(0);
  __builtin_amdgcn_s_waitcnt(0x0F70);                          // vmcnt(0)
  __syncthreads();
  read_scales(sa, 0);                                          // before loads into LDS are on their way: the compiler has it wait for them
  read_scales(sb, 1);
  load(1, stage1);
#pragma unroll
  for (int f = 0; f < NF; ++f) read(p, stage0, 0, f);
  const auto two_stages = [&](auto last, int chunk) {
    constexpr bool LAST = decltype(last)::value;
    const int t = chunk * 2;
    if (!LAST) load_scales(chunk + 1);
    step(b0, std::true_type{}, sa, p, q, stage0, 1);
    step(b1, std::true_type{}, sa, q, p, stage0, 2);
    step(b2, std::true_type{}, sa, p, q, stage0, 3);
    __builtin_amdgcn_s_waitcnt(0x0F70);
    __syncthreads();                                           // the next stage is there, this one has been read
    if (!LAST) load(t + 2, stage0);
    step(b3, std::true_type{}, sa, q, p, stage1, 0);
    if (!LAST) put_scales(chunk + 1);
    step(b0, std::true_type{}, sb, p, q, stage1, 1);
    step(b1, std::true_type{}, sb, q, p, stage1, 2);
    step(b2, std::true_type{}, sb, p, q, stage1, 3);
    __builtin_amdgcn_s_waitcnt(0x0F70);
    __syncthreads();
    const Scales now = sb;
    if (!LAST) {
      read_scales(sa, t + 2);
      read_scales(sb, t + 3);
      load(t + 3, stage1);
    }
    step(b3, std::bool_constant<!LAST>{}, now, q, p, stage0, 0);
  };
  const int chunks = (stages + 1) / 2;
  for (int chunk = 0; chunk < chunks - 1; ++chunk) two_stages(std::false_type{}, chunk);
  if (a.blocks % 16) {                                         // the last scales, zeros past the end; out of the loop, as products would be moved past a branch
#pragma unroll
    for (int i = 0; i < SR; ++i) next_scales[i] = mx_scales16(scale_rows[i], chunks - 1, a.blocks);
    __syncthreads();                                           // those that are there have been read
    put_scales(chunks - 1);
    __syncthreads();
    read_scales(sa, chunks * 2 - 2);
    read_scales(sb, chunks * 2 - 1);
  }
  two_stages(std::true_type{}, chunks - 1);
  // Results go through LDS, a wave's by itself, 32 rows at a time: then a lane has four neighbours of a row, the same ones of every row, and FOURS lanes
  // have a row of the wave's.  Four numbers c of row m lie in place c ^ m % 16.  All loads into LDS have been waited for, and all waves have read the last
  // stage.
  constexpr int FOURS = NF * 8, PASS = 64 / FOURS, PASSES = 32 / PASS;
  static_assert(WAVES * 32 * FOURS * 16 <= ROWS * 128);
  float4m *mine = (float4m *)stage0 + wave * 32 * FOURS;
  const int four = lane % FOURS, row0 = lane / FOURS, n = n0 + wn + 4 * four;
  const float4m bias = a.bias && n + 4 <= a.cols ? mx_load4(a.bias, n, TPUHIP_F32) : (float4m){0, 0, 0, 0};
  const auto results = [&](auto type) {
    constexpr int TYPE = decltype(type)::value;
#pragma unroll
    for (int i = 0; i < MF; ++i) {
#pragma unroll
      for (int j = 0; j < NF; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mine[r * FOURS + ((j * 8 + 2 * k + g) ^ (r & 15))] = (float4m){acc[j][i][4 * k], acc[j][i][4 * k + 1], acc[j][i][4 * k + 2], acc[j][i][4 * k + 3]};
      __builtin_amdgcn_wave_barrier();
      float4m v[PASSES];
#pragma unroll
      for (int k = 0; k < PASSES; ++k) {
        const int row = k * PASS + row0;
        v[k] = mine[row * FOURS + (four ^ (row & 15))];
      }
      __builtin_amdgcn_wave_barrier();
      const int first = m0 + wm + i * 32 + row0;
      if (n + 4 <= a.cols) {
#pragma unroll
        for (int k = 0; k < PASSES; ++k) v[k] += bias;
        if (a.residual)
#pragma unroll
          for (int k = 0; k < PASSES; ++k)
            if (first + k * PASS < a.rows) v[k] += mx_load4(a.residual, (int64_t)(first + k * PASS) * a.residual_stride + n, TYPE);
#pragma unroll
        for (int k = 0; k < PASSES; ++k)
          if (first + k * PASS < a.rows) mx_store4(a.y, (int64_t)(first + k * PASS) * a.y_stride + n, TYPE, v[k]);
      } else if (n < a.cols) {
#pragma unroll
        for (int k = 0; k < PASSES; ++k)
          if (first + k * PASS < a.rows) mx_result(a, first + k * PASS, n, v[k]);
      }
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
  // a launch has fewer than 2^32 threads by the columns, and 65535 workgroups by the rows
  TPUHIP_REQUIRE(x->rows <= 16 * 65535 && w->rows <= 1 << 26, "%s: %d rows of %d columns in one call", what, x->rows, w->rows);
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
  a->blocks = mx_blocks(x->cols);
  a->dtype = d->dtype;
  return TPUHIP_OK;
}

template <int BM, int BN, int WM, int WN>
static void mx_launch_tiles(tpuhip_ctx *ctx, const MxProductArgs &a) {
  launch(ctx, mx_tile_kernel<BM, BN, WM, WN>, dim3((unsigned)(ceil_div64(a.rows, BM) * ceil_div64(a.cols, BN))), dim3(64 * WM * WN), a);
}

static int mx_multiply(tpuhip_ctx *ctx, const MxProductArgs &a) {
  if (a.rows > 128 && a.blocks >= 16) {
    if (ceil_div64(a.rows, 256) * ceil_div64(a.cols, 256) >= ctx->num_cu / 2)
      mx_launch_tiles<256, 256, 2, 4>(ctx, a);
    else
      mx_launch_tiles<128, 128, 2, 2>(ctx, a);
    TPUHIP_CHECK_HIP(hipGetLastError());
    return TPUHIP_OK;
  }
  launch(ctx, mx_stream_kernel<1, 1, 8>, dim3((unsigned)ceil_div64(a.cols, 16), (unsigned)ceil_div64(a.rows, 16)), dim3(512), a);
  TPUHIP_CHECK_HIP(hipGetLastError());
  return TPUHIP_OK;
}

}  // namespace tpuhip

using namespace tpuhip;

extern "C" {

int tpuhip_mx_product(tpuhip_ctx *ctx, const tpuhip_mx_product_desc *desc, const tpuhip_mx_matrix *x, const tpuhip_mx_matrix *w, void *y) {
  MxProductArgs a;
  if (int rc = mx_product_args(ctx, desc, x, w, y, "tpuhip_mx_product", &a)) return rc;
  if (a.rows == 0) return TPUHIP_OK;
  TPUHIP_CHECK_HIP(hipSetDevice(ctx->device));
  return mx_multiply(ctx, a);
}

int tpuhip_mx_linear(tpuhip_ctx *ctx, const tpuhip_mx_product_desc *desc, const void *x, int x_dtype, int64_t x_stride,
                     const tpuhip_mx_matrix *room, const tpuhip_mx_matrix *w, void *y) {
  const char *what = "tpuhip_mx_linear";
  MxProductArgs a;
  if (int rc = mx_product_args(ctx, desc, room, w, y, what, &a)) return rc;
  if (int rc = mx_check_rows(a.rows, room->cols, x, x_dtype, x_stride, false, "x", what)) return rc;
  if (a.rows == 0) return TPUHIP_OK;
  TPUHIP_CHECK_HIP(hipSetDevice(ctx->device));
  if (int rc = mx_quantize(ctx, room, x, x_dtype, x_stride, what)) return rc;
  return mx_multiply(ctx, a);
}

}  // extern "C"
