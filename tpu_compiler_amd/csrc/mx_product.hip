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

// The scales of a lane for 512 numbers of its row, blocks 16 chunk + 4 s + g, s = 0..3: byte s of a dword.  Past the row's end they are 0, 2^-127:
// what such numbers of both operands make is below 2^-200, nothing in 32 bits, whatever the codes are.
__device__ __forceinline__ uint32_t mx_scales(const uint8_t *row, int chunk, int blocks, int g) {
  const uint8_t *at = row + chunk * 16;
  if (chunk * 16 + 16 <= blocks) {
    const uint4m v = *(const uint4m_any *)at;
    const uint32_t pick = 0x0C0C0400u + 0x0101u * (uint32_t)g;   // byte g of the second operand, byte g of the first
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(v[3], v[2], pick), __builtin_amdgcn_perm(v[1], v[0], pick), 0x05040100);
  }
  uint32_t v = 0;
#pragma unroll
  for (int s = 0; s < 4; ++s)
    if (chunk * 16 + 4 * s + g < blocks) v |= (uint32_t)at[4 * s + g] << 8 * s;
  return v;
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

static int mx_multiply(tpuhip_ctx *ctx, const MxProductArgs &a) {
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
