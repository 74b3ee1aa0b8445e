// The key/value cache in 4 or 8 bits: its memory, rows on their way into it and out of it.
#include "kv_cache.hpp"

#include <algorithm>
#include <climits>
#include <new>

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

// E elements from or to memory that is aligned to a dword
typedef uint32_t dwords4 __attribute__((ext_vector_type(4), aligned(4)));
template <int BYTES>
__device__ __forceinline__ void copy_dwords(void *dst, const void *src) {
  static_assert(BYTES % 4 == 0);
  constexpr int full = BYTES / 16;
#pragma unroll
  for (int i = 0; i < full; ++i) ((dwords4 *)dst)[i] = ((const dwords4 *)src)[i];
#pragma unroll
  for (int i = full * 4; i < BYTES / 4; ++i) ((uint32_t *)dst)[i] = ((const uint32_t *)src)[i];
}

struct RowsArgs {
  uint8_t *data;
  const int32_t *slots;
  void *x[2];                   // keys, values
  int64_t token_stride[2], head_stride[2];
  int tokens, heads, dim, most; // slots below `most` exist
  int wide;                     // rows begin at dwords
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

// the slots of the workgroup's rows, and whether they are a unit's tokens in order
__device__ __forceinline__ bool load_slots(const RowsArgs &a, int first, int (&slot)[kUnitTokens]) {
  const int tid = threadIdx.x;
  int mine = -1;
  if (tid < kUnitTokens && first + tid < a.tokens) mine = a.slots[first + tid];
  if ((unsigned)mine >= (unsigned)a.most) mine = -1;
  if (tid < kUnitTokens) slot[tid] = mine;
  __syncthreads();
  const int s0 = slot[0];
  const bool in_order = s0 >= 0 && (s0 & 31) == 0 && slot[tid & 31] == s0 + (tid & 31);
  return __syncthreads_and(in_order);
}

template <typename U, typename T>
__global__ __launch_bounds__(kRowsThreads) void kv_write_kernel(RowsArgs a) {
  constexpr int E = U::kDim / 16, HALF = U::kDim / 2;
  __shared__ __attribute__((aligned(16))) uint8_t unit[U::kBytes];
  __shared__ int slot[kUnitTokens];
  const int first = blockIdx.x * kUnitTokens, head = blockIdx.y;
  const int t = threadIdx.x & (kRowThreads - 1), row = threadIdx.x / kRowThreads;
  const bool in_order = load_slots(a, first, slot);
  const int my_slot = slot[row];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    float x[2 * E];
    if (my_slot >= 0) {
      const T *src = (const T *)a.x[kv] + (int64_t)(first + row) * a.token_stride[kv] + (int64_t)head * a.head_stride[kv];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c0 = h * HALF + t * E;
        T raw[E];
        if (a.wide && c0 + E <= a.dim) {
          copy_dwords<E * sizeof(T)>(raw, src + c0);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) raw[e] = src[min(c0 + e, a.dim - 1)];   // what is past the end repeats the last one
        }
#pragma unroll
        for (int e = 0; e < E; ++e) x[h * E + e] = to_f32(raw[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 2 * E; ++e) x[e] = 0;
    }
    float lo = x[0], hi = x[0], bad = 0;
#pragma unroll
    for (int e = 0; e < 2 * E; ++e) {
      lo = fminf(lo, x[e]);
      hi = fmaxf(hi, x[e]);
      bad = fabsf(x[e]) <= __FLT_MAX__ ? bad : 1.0f;   // an infinity or a NaN
    }
    lo = over8(lo, [](float p, float q) { return fminf(p, q); });
    hi = over8(hi, [](float p, float q) { return fmaxf(p, q); });
    bad = over8(bad, [](float p, float q) { return fmaxf(p, q); });
    uint32_t mb = bf16_down(lo);
    const float m = bf16_to_f32(mb);
    const float step = (hi - m) / (float)U::kLevels;
    uint32_t sb = 0x8000u ^ bf16_down(-step);
    float s = bf16_to_f32(sb);
    if (bad != 0 || !(s <= __FLT_MAX__)) {
      mb = 0x7FC0;
      sb = 0;
      s = 0;
    } else if (s < 0x1p-126f) {
      sb = 0;
      s = 0;
    }
    // c = rint((x - m) / s), the quotient rounded as a division rounds it (ties of bfloat16 numbers are common): a product with the
    // inverse and one step of correction, at a scale where neither the inverse nor the remainder leaves the normal numbers
    const float scale = s > 0x1p100f ? 0x1p-64f : s < 0x1p-90f ? 0x1p64f : 1.0f;
    const float ss = s * scale, inv = s > 0 ? 1.0f / ss : 0.0f;
    uint32_t c[2 * E];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float d = (x[h * E + e] - m) * scale;
        const float q0 = d * inv;
        const float q = __builtin_fmaf(__builtin_fmaf(-q0, ss, d), inv, q0);
        const int v = (int)fminf(fmaxf(rintf(q), 0.0f), (float)U::kLevels);
        c[h * E + e] = s > 0 && h * HALF + t * E + e < a.dim ? v : 0;
      }
    uint8_t *codes = unit + kv * U::kCodes;
    if (kv == 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint8_t *at = codes + row * U::kRow + (h * HALF + t * E) * U::kBits / 8;
#pragma unroll
        for (int b = 0; b < E * U::kBits / 8; ++b)
          at[b] = U::kBits == 4 ? c[h * E + 2 * b] | c[h * E + 2 * b + 1] << 4 : c[h * E + b];
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if constexpr (U::kBits == 4) {
          codes[U::v_at(t * E + e, row)] = c[e] | c[E + e] << 4;
        } else {
          codes[U::v_at(t * E + e, row)] = c[e];
          codes[U::v_at(HALF + t * E + e, row)] = c[E + e];
        }
      }
    }
    if (t == 0) ((uint32_t *)(unit + U::kParams))[kv * kUnitTokens + row] = mb << 16 | sb;
  }
  __syncthreads();
  if (in_order) {
    uint4 *dst = (uint4 *)(a.data + ((int64_t)(slot[0] >> 5) * a.heads + head) * U::kBytes);
    for (int i = threadIdx.x; i < U::kBytes / 16; i += kRowsThreads) dst[i] = ((const uint4 *)unit)[i];
    return;
  }
  if (my_slot < 0) return;
  uint8_t *dst = a.data + ((int64_t)(my_slot >> 5) * a.heads + head) * U::kBytes;
  const int place = my_slot & 31;
  // keys: a row's bytes lie together
  constexpr int kBytes = U::kRow / kRowThreads;
  {
    uint8_t *to = dst + place * U::kRow + t * kBytes;
    const uint8_t *from = unit + row * U::kRow + t * kBytes;
    if constexpr (kBytes % 4 == 0) {
      copy_dwords<kBytes>(to, from);
    } else {
#pragma unroll
      for (int b = 0; b < kBytes; b += 2) *(uint16_t *)(to + b) = *(const uint16_t *)(from + b);
    }
  }
  if (t < 2) ((uint32_t *)(dst + U::kParams))[t * kUnitTokens + place] = ((const uint32_t *)(unit + U::kParams))[t * kUnitTokens + row];
  // values: a byte in each column, or dwords where the four tokens of one are all here
  const uint8_t *values = unit + U::kCodes;
  dst += U::kCodes;
  const int in4 = place & 3, lead = row - in4;
  bool four = lead >= 0 && lead + 3 < kUnitTokens;
  if (four)
    for (int i = 0; i < 4; ++i) four &= slot[lead + i] == my_slot - in4 + i;
  if (four) {
    for (int j = in4 * kRowThreads + t; j < U::kRow; j += 4 * kRowThreads)
      *(uint32_t *)(dst + U::v_at(j, place & ~3)) = values[U::v_at(j, lead)] | values[U::v_at(j, lead + 2)] << 8 |
                                                    values[U::v_at(j, lead + 1)] << 16 | (uint32_t)values[U::v_at(j, lead + 3)] << 24;
  } else {
    for (int j = t; j < U::kRow; j += kRowThreads) dst[U::v_at(j, place)] = values[U::v_at(j, row)];
  }
}

template <typename U, typename T>
__global__ __launch_bounds__(kRowsThreads) void kv_read_kernel(RowsArgs a) {
  constexpr int E = U::kDim / 16, HALF = U::kDim / 2;
  __shared__ __attribute__((aligned(16))) uint8_t values[U::kCodes];
  __shared__ int slot[kUnitTokens];
  const int first = blockIdx.x * kUnitTokens, head = blockIdx.y;
  const int t = threadIdx.x & (kRowThreads - 1), row = threadIdx.x / kRowThreads;
  const bool in_order = load_slots(a, first, slot);
  const int my_slot = slot[row];
  const int place = my_slot & 31;
  const uint8_t *unit = a.data + ((int64_t)(my_slot >> 5) * a.heads + head) * U::kBytes;
  if (in_order) {
    for (int i = threadIdx.x; i < U::kCodes / 16; i += kRowsThreads) ((uint4 *)values)[i] = ((const uint4 *)(unit + U::kCodes))[i];
    __syncthreads();
  }
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    T raw[2 * E];
    if (my_slot >= 0) {
      const uint32_t param = ((const uint32_t *)(unit + U::kParams))[kv * kUnitTokens + place];
      const float s = bf16_to_f32(param & 0xFFFF), m = bf16_to_f32(param >> 16);
      uint32_t c[2 * E];
      if (kv == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint8_t *at = unit + place * U::kRow + (h * HALF + t * E) * U::kBits / 8;
          uint8_t byte[E * U::kBits / 8];
          if constexpr (sizeof(byte) % 4 == 0) {
            copy_dwords<sizeof(byte)>(byte, at);
          } else {
#pragma unroll
            for (int b = 0; b < (int)sizeof(byte); ++b) byte[b] = at[b];
          }
#pragma unroll
          for (int e = 0; e < E; ++e) c[h * E + e] = U::kBits == 4 ? byte[e / 2] >> 4 * (e & 1) & 15 : byte[e];
        }
      } else {
        const uint8_t *from = in_order ? values : unit + U::kCodes;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if constexpr (U::kBits == 4) {
            const uint32_t b = from[U::v_at(t * E + e, place)];
            c[e] = b & 15;
            c[E + e] = b >> 4;
          } else {
            c[e] = from[U::v_at(t * E + e, place)];
            c[E + e] = from[U::v_at(HALF + t * E + e, place)];
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 2 * E; ++e) raw[e] = from_f32<T>(__builtin_fmaf(s, (float)c[e], m));   // s c is exact: 16 bits
    } else {
#pragma unroll
      for (int e = 0; e < 2 * E; ++e) raw[e] = from_f32<T>(0.0f);
    }
    if (first + row >= a.tokens) continue;
    T *dst = (T *)a.x[kv] + (int64_t)(first + row) * a.token_stride[kv] + (int64_t)head * a.head_stride[kv];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int c0 = h * HALF + t * E;
      if (a.wide && c0 + E <= a.dim) {
        copy_dwords<E * sizeof(T)>(dst + c0, raw + h * E);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (c0 + e < a.dim) dst[c0 + e] = raw[h * E + e];
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
  TPUHIP_REQUIRE(in_elements(r->dtype), "%s: unknown type %d", what, r->dtype);
  if (r->tokens == 0) return TPUHIP_OK;
  TPUHIP_REQUIRE(r->k && r->v && slots, "%s: NULL argument", what);
  const int size = r->dtype == TPUHIP_F32 ? 4 : 2, dim = c->desc.head_dim, heads = c->desc.kv_heads;
  const int64_t ts[2] = {r->k_token_stride, r->v_token_stride}, hs[2] = {r->k_head_stride, r->v_head_stride};
  void *x[2] = {r->k, r->v};
  a->wide = 1;
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
    if ((uintptr_t)x[i] % 4 || ts[i] * size % 4 || hs[i] * size % 4) a->wide = 0;
    a->x[i] = x[i];
    a->token_stride[i] = ts[i];
    a->head_stride[i] = hs[i];
  }
  a->data = c->data;
  a->slots = slots;
  a->tokens = r->tokens;
  a->heads = heads;
  a->dim = dim;
  a->most = c->desc.pages * c->desc.page_tokens;
  return TPUHIP_OK;
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
  const hipError_t e = hipGetLastError();
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
  if (int rc = tpuhip_free(ctx, cache->data)) return rc;
  delete cache;
  return TPUHIP_OK;
}

int tpuhip_kv_write(tpuhip_ctx *ctx, tpuhip_kv_cache *cache, const tpuhip_kv_rows *rows, const int32_t *slots) {
  RowsArgs a{};
  if (int rc = rows_args(ctx, cache, rows, slots, false, "tpuhip_kv_write", &a)) return rc;
  if (a.tokens == 0) return TPUHIP_OK;
  return kv_dispatch(cache, [&](auto u) -> int {
    using U = decltype(u);
    const auto kernel = rows->dtype == TPUHIP_BF16 ? kv_write_kernel<U, Bf16>
                        : rows->dtype == TPUHIP_F16 ? kv_write_kernel<U, _Float16> : kv_write_kernel<U, float>;
    launch(ctx, kernel, dim3((unsigned)ceil_div64(a.tokens, kUnitTokens), (unsigned)a.heads), dim3(kRowsThreads), a);
    TPUHIP_CHECK_HIP(hipGetLastError());
    return TPUHIP_OK;
  });
}

int tpuhip_kv_read(tpuhip_ctx *ctx, const tpuhip_kv_cache *cache, const tpuhip_kv_rows *rows, const int32_t *slots) {
  RowsArgs a{};
  if (int rc = rows_args(ctx, cache, rows, slots, true, "tpuhip_kv_read", &a)) return rc;
  if (a.tokens == 0) return TPUHIP_OK;
  return kv_dispatch(cache, [&](auto u) -> int {
    using U = decltype(u);
    const auto kernel = rows->dtype == TPUHIP_BF16 ? kv_read_kernel<U, Bf16>
                        : rows->dtype == TPUHIP_F16 ? kv_read_kernel<U, _Float16> : kv_read_kernel<U, float>;
    launch(ctx, kernel, dim3((unsigned)ceil_div64(a.tokens, kUnitTokens), (unsigned)a.heads), dim3(kRowsThreads), a);
    TPUHIP_CHECK_HIP(hipGetLastError());
    return TPUHIP_OK;
  });
}

}  // extern "C"
