// Rows into microscaled 4-bit numbers and back.
#include "mx.hpp"

namespace tpuhip {

struct MxRowsArgs {
  uint8_t *codes, *scales;
  void *x;
  int64_t codes_stride, scales_stride, x_stride;
  FastDiv row_blocks;           // blocks of a row
  uint32_t blocks;              // of all rows
  int cols, dtype;
};

// Four threads a block, eight numbers each: one or two loads of 16 bytes, a wave's next to each other, and two exchanges between neighbouring lanes for
// the block's largest size.  Bound by memory: 8192 x 8192 of bfloat16, 170 MB, are quantised in 31 us (5.5 TB/s, some of it from the last cache), 37
// where the caches are full of another kernel's results, and read back in 27; 4999 x 2050 of float32, parts of longer rows that begin anywhere, 46 MB, take
// 9.4 and 11.6 us; a row of 4096 1.5 and 1.9, latency.
constexpr int kMxThreads = 256, kMxThreadsBlock = 4;

__global__ __launch_bounds__(kMxThreads) void mx_quantize_kernel(MxRowsArgs a) {
  const uint32_t at = blockIdx.x * (kMxThreads / kMxThreadsBlock) + threadIdx.x / kMxThreadsBlock, t = threadIdx.x % kMxThreadsBlock;
  if (at >= a.blocks) return;                                  // the four threads of a block together
  uint32_t block = at;
  const int64_t row = a.row_blocks.split(block);
  const int col = (int)(block * kMxBlock + t * 8);
  float v[8];
  if (col + 8 <= a.cols) {
    mx_load8(a.x, row * a.x_stride + col, a.dtype, v);
  } else {
    // the row's last number in the place of those that are not there: loads without branches, which do not wait for each other
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = mx_load(a.x, row * a.x_stride + min(col + i, a.cols - 1), a.dtype);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < a.cols ? v[i] : 0.0f;
  }
  uint32_t byte;
  *(uint32_t *)(a.codes + row * a.codes_stride + (int64_t)block * kMxBytes + t * 4) = mx_quantised8(v, byte);
  if (t == 0) a.scales[row * a.scales_stride + block] = (uint8_t)byte;
}

__global__ __launch_bounds__(kMxThreads) void mx_read_kernel(MxRowsArgs a) {
  const uint32_t at = blockIdx.x * (kMxThreads / kMxThreadsBlock) + threadIdx.x / kMxThreadsBlock, t = threadIdx.x % kMxThreadsBlock;
  if (at >= a.blocks) return;
  uint32_t block = at;
  const int64_t row = a.row_blocks.split(block);
  const int col = (int)(block * kMxBlock + t * 8);
  const uint32_t c = *(const uint32_t *)(a.codes + row * a.codes_stride + (int64_t)block * kMxBytes + t * 4);
  const float scale = mx_scale(a.scales[row * a.scales_stride + block]);
  float v[8];
  const auto pair = [&](int i, float2m p) { v[2 * i] = p[0], v[2 * i + 1] = p[1]; };
  pair(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0));
  pair(1, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1));
  pair(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2));
  pair(3, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3));
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= scale;                   // exact, past 2^128 infinite
  const int64_t to = row * a.x_stride + col;
  if (col + 8 <= a.cols) {
    mx_store4(a.x, to, a.dtype, (float4m){v[0], v[1], v[2], v[3]});
    mx_store4(a.x, to + 4, a.dtype, (float4m){v[4], v[5], v[6], v[7]});
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (col + i < a.cols) mx_store(a.x, to + i, a.dtype, v[i]);
  }
}

int mx_check(const tpuhip_mx_matrix *m, const char *name, const char *what) {
  TPUHIP_REQUIRE(m, "%s: NULL argument", what);
  TPUHIP_REQUIRE(m->rows >= 0 && m->cols >= 1, "%s: %s of %d rows, %d columns", what, name, m->rows, m->cols);
  TPUHIP_REQUIRE(m->cols <= 1 << 24, "%s: %s of %d columns", what, name, m->cols);
  if (m->rows == 0) return TPUHIP_OK;
  const int blocks = mx_blocks(m->cols);
  TPUHIP_REQUIRE(m->codes && m->scales, "%s: NULL argument", what);
  TPUHIP_REQUIRE((uintptr_t)m->codes % kMxBytes == 0, "%s: codes of %s do not begin at a multiple of %d bytes", what, name, kMxBytes);
  const int64_t most = INT64_MAX / 8 / m->rows;
  TPUHIP_REQUIRE(m->codes_stride % kMxBytes == 0 && (m->rows == 1 || m->codes_stride >= (int64_t)blocks * kMxBytes) && m->codes_stride >= 0 &&
                     m->codes_stride <= most,
                 "%s: rows of %s's codes lie %lld bytes apart", what, name, (long long)m->codes_stride);
  TPUHIP_REQUIRE((m->rows == 1 || m->scales_stride >= blocks) && m->scales_stride >= 0 && m->scales_stride <= most,
                 "%s: rows of %s's scales lie %lld bytes apart", what, name, (long long)m->scales_stride);
  return TPUHIP_OK;
}

int mx_check_rows(int rows, int cols, const void *x, int dtype, int64_t stride, bool output, const char *name, const char *what) {
  TPUHIP_REQUIRE(mx_elements(dtype), "%s: %s of unknown type %d", what, name, dtype);
  if (rows == 0) return TPUHIP_OK;
  TPUHIP_REQUIRE(x, "%s: NULL argument", what);
  TPUHIP_REQUIRE((uintptr_t)x % mx_size(dtype) == 0, "%s: %s does not begin at an element", what, name);
  TPUHIP_REQUIRE(stride >= 0 && stride <= INT64_MAX / 8 / rows && (!output || rows == 1 || stride >= cols), "%s: rows of %s lie %lld elements apart",
                 what, name, (long long)stride);
  return TPUHIP_OK;
}

static int mx_rows(tpuhip_ctx *ctx, const tpuhip_mx_matrix *m, const void *x, int dtype, int64_t x_stride, bool read, const char *what) {
  TPUHIP_REQUIRE(ctx, "%s: NULL argument", what);
  if (int rc = mx_check(m, "the matrix", what)) return rc;
  if (int rc = mx_check_rows(m->rows, m->cols, x, dtype, x_stride, read, "x", what)) return rc;
  if (m->rows == 0) return TPUHIP_OK;
  MxRowsArgs a{};
  const int64_t blocks = (int64_t)m->rows * mx_blocks(m->cols);
  TPUHIP_REQUIRE(ceil_div64(blocks, kMxThreads / kMxThreadsBlock) <= UINT32_MAX / kMxThreads,   // a launch has fewer than 2^32 threads
                 "%s: %d rows of %d columns in one call", what, m->rows, m->cols);
  a.codes = (uint8_t *)m->codes;
  a.scales = (uint8_t *)m->scales;
  a.x = const_cast<void *>(x);
  a.codes_stride = m->codes_stride;
  a.scales_stride = m->scales_stride;
  a.x_stride = x_stride;
  a.row_blocks = FastDiv(mx_blocks(m->cols));
  a.blocks = (uint32_t)blocks;
  a.cols = m->cols;
  a.dtype = dtype;
  TPUHIP_CHECK_HIP(hipSetDevice(ctx->device));
  launch(ctx, read ? mx_read_kernel : mx_quantize_kernel, dim3((unsigned)ceil_div64(blocks, kMxThreads / kMxThreadsBlock)), dim3(kMxThreads), a);
  TPUHIP_CHECK_HIP(hipGetLastError());
  return TPUHIP_OK;
}

int mx_quantize(tpuhip_ctx *ctx, const tpuhip_mx_matrix *m, const void *x, int dtype, int64_t x_stride, const char *what) {
  return mx_rows(ctx, m, x, dtype, x_stride, false, what);
}

}  // namespace tpuhip

using namespace tpuhip;

extern "C" {

int tpuhip_mx_quantize(tpuhip_ctx *ctx, const tpuhip_mx_matrix *m, const void *x, int dtype, int64_t x_stride) {
  return mx_rows(ctx, m, x, dtype, x_stride, false, "tpuhip_mx_quantize");
}

int tpuhip_mx_read(tpuhip_ctx *ctx, const tpuhip_mx_matrix *m, void *x, int dtype, int64_t x_stride) {
  return mx_rows(ctx, m, x, dtype, x_stride, true, "tpuhip_mx_read");
}

}  // extern "C"
