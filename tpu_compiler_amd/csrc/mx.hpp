// Rows of microscaled 4-bit floating point numbers: blocks of 32 with a scale 2^e, shared by the kernels that make, read and multiply them.
//
// A block's scale is a byte e + 127 (255: NaN), its codes are 16 bytes, two a byte, even columns in the low halves: sign, two bits of exponent,
// one of fraction, that is 0, 0.5, 1, 1.5, 2, 3, 4, 6.  v_mfma_scale_f32_16x16x128_f8f6f4 takes 16 bytes of a row's codes, a block, from each
// lane and the byte of its scale, so that codes are operands as they lie in memory, row by row, and nothing is laid out anew.
#pragma once

#include "common.hpp"

namespace tpuhip {

constexpr int kMxBlock = 32, kMxBytes = 16;   // numbers of a block, bytes of their codes

constexpr bool mx_elements(int dtype) { return dtype == TPUHIP_BF16 || dtype == TPUHIP_F16 || dtype == TPUHIP_F32; }
constexpr int mx_size(int dtype) { return dtype == TPUHIP_F32 ? 4 : 2; }
constexpr int mx_blocks(int cols) { return cols / kMxBlock + (cols % kMxBlock != 0); }

// refuses a matrix that is none
int mx_check(const tpuhip_mx_matrix *m, const char *name, const char *what);
// mx_quantize.hip: the launch of tpuhip_mx_quantize, its arguments checked
int mx_quantize(tpuhip_ctx *ctx, const tpuhip_mx_matrix *m, const void *x, int dtype, int64_t x_stride, const char *what);
// refuses rows of elements that are none
int mx_check_rows(int rows, int cols, const void *x, int dtype, int64_t stride, bool output, const char *name, const char *what);

typedef float float2m __attribute__((ext_vector_type(2)));
typedef float float4m __attribute__((ext_vector_type(4)));
typedef uint32_t uint2m __attribute__((ext_vector_type(2)));
typedef uint32_t uint4m __attribute__((ext_vector_type(4)));
// rows begin at any element, scales at any byte: memory takes any address
typedef uint32_t uint4m_any __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t uint2m_any __attribute__((ext_vector_type(2), aligned(1)));

// The scale of a block whose largest size is `top`, as its byte: the exponent's bits less those of 4, the largest code's power of two.  The
// smallest is 2^-127, which zeros have too.  A block that holds an infinity or a NaN is a NaN as a whole: 255.
__device__ __forceinline__ uint32_t mx_scale_byte(float top) {
  const int e = (int)(__float_as_uint(top) >> 23 & 0xFF);
  return e == 255 ? 255u : (uint32_t)max(e - 2, 0);
}
// 2^(byte - 127), and of 255 a NaN
__device__ __forceinline__ float mx_scale(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7FC00000u : byte << 23);
}
// Eight numbers over a scale as codes, to nearest, ties to even, the largest one for what is beyond: as the conversion rounds, in bfloat16, float16
// and float32 the same (all ties, neighbours, subnormal numbers and scales compared with the definition).
__device__ __forceinline__ uint32_t mx_codes8(const float (&v)[8], float scale) {
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], scale, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], scale, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], scale, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], scale, 3);
  return c;
}

// The codes of eight of a block's numbers, which four neighbouring lanes share, and the block's scale
template <int CTRL>
__device__ __forceinline__ float mx_dpp_max(float v) {
  return __builtin_elementwise_maximum(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true)));
}
__device__ __forceinline__ uint32_t mx_quantised8(const float (&v)[8], uint32_t &byte) {
  float top = 0;                                               // a NaN stays
#pragma unroll
  for (int i = 0; i < 8; ++i) top = __builtin_elementwise_maximum(top, __builtin_fabsf(v[i]));
  byte = mx_scale_byte(mx_dpp_max<0x4E>(mx_dpp_max<0xB1>(top)));
  const uint32_t c = mx_codes8(v, mx_scale(byte == 255 ? 127 : byte));
  return byte == 255 ? 0u : c;
}

__device__ __forceinline__ float mx_load(const void *x, int64_t i, int dtype) {
  if (dtype == TPUHIP_F32) return ((const float *)x)[i];
  const uint16_t b = ((const uint16_t *)x)[i];
  return dtype == TPUHIP_BF16 ? __uint_as_float((uint32_t)b << 16) : (float)__builtin_bit_cast(_Float16, b);
}
__device__ __forceinline__ uint32_t mx_half(float v, int dtype) {
  return dtype == TPUHIP_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)v) : __builtin_bit_cast(uint16_t, (_Float16)v);
}
__device__ __forceinline__ void mx_store(void *x, int64_t i, int dtype, float v) {
  if (dtype == TPUHIP_F32)
    ((float *)x)[i] = v;
  else
    ((uint16_t *)x)[i] = (uint16_t)mx_half(v, dtype);
}
// eight neighbours
__device__ __forceinline__ void mx_load8(const void *x, int64_t i, int dtype, float (&v)[8]) {
  if (dtype == TPUHIP_F32) {
    const uint4m a = *(const uint4m_any *)((const float *)x + i), b = *(const uint4m_any *)((const float *)x + i + 4);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = __uint_as_float(a[k]), v[4 + k] = __uint_as_float(b[k]);
    return;
  }
  const uint4m a = *(const uint4m_any *)((const uint16_t *)x + i);
  if (dtype == TPUHIP_BF16) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[2 * k] = __uint_as_float(a[k] << 16), v[2 * k + 1] = __uint_as_float(a[k] & 0xFFFF0000u);
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[2 * k] = (float)__builtin_bit_cast(_Float16, (uint16_t)a[k]);
      v[2 * k + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(a[k] >> 16));
    }
  }
}
// ONCE: past the L2 as far as that goes, which operands need more.  Large products end their tiles at the same time: 8192 x 8192 x 8192 took 266 us so
// and 276 otherwise, in turn on one card.
template <bool ONCE = false>
__device__ __forceinline__ void mx_store4(void *x, int64_t i, int dtype, float4m v) {
  if (dtype == TPUHIP_F32) {
    uint4m_any *to = (uint4m_any *)((float *)x + i);
    const uint4m_any a = __builtin_bit_cast(uint4m_any, v);
    if constexpr (ONCE)
      __builtin_nontemporal_store(a, to);
    else
      *to = a;
  } else {
    uint2m_any *to = (uint2m_any *)((uint16_t *)x + i);
    const uint2m_any a = {mx_half(v[0], dtype) | mx_half(v[1], dtype) << 16, mx_half(v[2], dtype) | mx_half(v[3], dtype) << 16};
    if constexpr (ONCE)
      __builtin_nontemporal_store(a, to);
    else
      *to = a;
  }
}
__device__ __forceinline__ float4m mx_load4(const void *x, int64_t i, int dtype) {
  float4m v;
  if (dtype == TPUHIP_F32) {
    const uint4m a = *(const uint4m_any *)((const float *)x + i);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = __uint_as_float(a[k]);
    return v;
  }
  const uint2m a = *(const uint2m_any *)((const uint16_t *)x + i);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint16_t b = (uint16_t)(a[k >> 1] >> 16 * (k & 1));
    v[k] = dtype == TPUHIP_BF16 ? __uint_as_float((uint32_t)b << 16) : (float)__builtin_bit_cast(_Float16, b);
  }
  return v;
}

}  // namespace tpuhip
