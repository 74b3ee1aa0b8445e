// Attention to a key/value cache of 4 or 8 bits.
#include "kv_cache.hpp"

#include <climits>
#include <cmath>

namespace tpuhip {

struct AttentionArgs {
  const uint8_t *data;
  const int32_t *q_starts, *kv_lens, *table;
  const uint16_t *q;
  uint16_t *out;
  int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;
  int heads, kv_heads, dim, pages, units_per_page, table_stride;
  int total_q, max_q, max_kv, window, sinks, bf16;
  float scale;
};

__device__ __forceinline__ float load16(uint16_t b, int bf16) {
  return bf16 ? bf16_to_f32(b) : (float)__builtin_bit_cast(_Float16, b);
}
__device__ __forceinline__ uint16_t store16(float v, int bf16) {
  return bf16 ? __builtin_bit_cast(uint16_t, (__bf16)v) : __builtin_bit_cast(uint16_t, (_Float16)v);
}

// One wave a query and head: a lane a token for the scores, a lane a channel (or DP/64 of them) for the sums.
template <typename U>
__global__ __launch_bounds__(64) void kv_attention_kernel(AttentionArgs a) {
  __shared__ float q[U::kDim], weight[64], bias[64];
  __shared__ const uint8_t *unit_of[2];
  const int lane = threadIdx.x, head = blockIdx.y, seq = blockIdx.z, kvh = head / (a.heads / a.kv_heads);
  const int begin = min(max(a.q_starts[seq], 0), a.total_q), end = min(max(a.q_starts[seq + 1], begin), a.total_q);
  const int n = min(end - begin, a.max_q), kv_len = min(max(a.kv_lens[seq], 0), a.max_kv);
  const int i = blockIdx.x;
  if (i >= n) return;
  const int p = kv_len - n + i;
  const uint16_t *qs = a.q + (int64_t)(begin + i) * a.q_token_stride + (int64_t)head * a.q_head_stride;
  float q_sum = 0;
  for (int c = lane; c < U::kDim; c += 64) {
    q[c] = c < a.dim ? load16(qs[c], a.bf16) : 0;
    q_sum += q[c];
  }
  for (int d = 1; d < 64; d <<= 1) q_sum += __shfl_xor(q_sum, d);
  float top = -INFINITY, total = 0, acc[U::kDim / 64 + 1] = {};
  for (int t0 = 0; t0 <= p; t0 += 64) {
    __syncthreads();
    if (lane < 2) {
      const int block = t0 / kUnitTokens + lane;
      const uint8_t *u = nullptr;
      if (block * kUnitTokens <= p) {
        const int page = a.table[(int64_t)seq * a.table_stride + block / a.units_per_page];
        if ((unsigned)page < (unsigned)a.pages)
          u = a.data + (((int64_t)page * a.units_per_page + block % a.units_per_page) * a.kv_heads + kvh) * U::kBytes;
      }
      unit_of[lane] = u;
    }
    __syncthreads();
    const int t = t0 + lane, place = t & 31;
    const uint8_t *u = unit_of[lane >> 5];
    const bool seen = u && t <= p && (!a.window || t > p - a.window || t < a.sinks);
    float x = -INFINITY, step = 0, offset = 0;
    if (seen) {
      float dot = 0;
      for (int c = 0; c < U::kDim; ++c) {
        const uint8_t b = u[place * U::kRow + c * U::kBits / 8];
        dot += q[c] * (float)(U::kBits == 4 ? b >> 4 * (c & 1) & 15 : b);
      }
      const uint32_t kp = ((const uint32_t *)(u + U::kParams))[place], vp = ((const uint32_t *)(u + U::kParams))[32 + place];
      x = (bf16_to_f32(kp & 0xFFFF) * dot + bf16_to_f32(kp >> 16) * q_sum) * a.scale;
      step = bf16_to_f32(vp & 0xFFFF);
      offset = bf16_to_f32(vp >> 16);
    }
    float most = x;
    for (int d = 1; d < 64; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
    const float now = fmaxf(top, most);
    const float old = now == top ? 1.0f : expf(top - now);
    const float w = seen ? expf(x - now) : 0;
    float sum = w;
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
    top = now;
    total = total * old + sum;
    weight[lane] = w * step;
    bias[lane] = w * offset;
    __syncthreads();
    for (int k = 0, c = lane; c < U::kDim; c += 64, ++k) {
      float v = acc[k] * old;
      const int half = U::kDim / 2, j = U::kBits == 4 && c >= half ? c - half : c;
      for (int s = 0; s < 64; ++s) {
        if (!unit_of[s >> 5]) continue;
        const uint8_t b = unit_of[s >> 5][U::kCodes + U::v_at(j, s & 31)];
        v += weight[s] * (float)(U::kBits == 4 ? (c >= half ? b >> 4 : b & 15) : b) + bias[s];
      }
      acc[k] = v;
    }
  }
  uint16_t *out = a.out + (int64_t)(begin + i) * a.out_token_stride + (int64_t)head * a.out_head_stride;
  for (int k = 0, c = lane; c < a.dim; c += 64, ++k) out[c] = store16(total != 0 ? acc[k] / total : 0, a.bf16);
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
  a.kv_heads = kv_heads;
  a.dim = dim;
  a.pages = cache->desc.pages;
  a.units_per_page = cache->units_per_page;
  a.table_stride = d->table_stride;
  a.total_q = d->total_q;
  a.max_q = d->max_q < d->total_q ? d->max_q : d->total_q;
  a.max_kv = d->max_kv;
  a.window = d->window;
  a.sinks = d->sinks;
  a.bf16 = d->dtype == TPUHIP_BF16;
  a.scale = d->scale;
  return kv_dispatch(cache, [&](auto u) -> int {
    using U = decltype(u);
    launch(ctx, kv_attention_kernel<U>, dim3((unsigned)a.max_q, (unsigned)a.heads, (unsigned)d->n_seq), dim3(64), a);
    TPUHIP_CHECK_HIP(hipGetLastError());
    return TPUHIP_OK;
  });
}

}  // extern "C"
