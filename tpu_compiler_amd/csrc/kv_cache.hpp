// The key/value cache: what a page holds and where, shared by the kernels that write, read and attend to it.
//
// A row (one token's keys or values of one head, D numbers) is held as integers c of `bits` bits with an offset m and a step s, both
// bfloat16, and stands for m + s c.  32 tokens of a head, a unit, lie together:
//
//   K codes   32 x kRow bytes, token by token: byte i holds channels 2i (low half) and 2i + 1, or channel i of 8 bits
//   V codes   32 x kRow bytes, byte column by byte column: column j holds channels j (low half) and j + DP/2, or channel j
//   K params  32 dwords, s in the low half and m in the high one;  V params likewise
//
// The attention kernel multiplies keys as a matrix of tokens x channels and values as one of channels x tokens, both of them the left
// operand of v_mfma_f32_16x16x32, of which a lane holds eight consecutive elements of a row.  With keys by token and values by column,
// a wave reads both straight from memory into the lanes that use them, sixteen bytes a lane, and nothing passes through LDS.  DP is D
// rounded up to a size that the kernels are made for; what is added holds zeros.
#pragma once

#include "common.hpp"

struct tpuhip_kv_cache {
  int device;
  tpuhip_kv_desc desc;
  int dp;              // padded head size
  int units_per_page;
  int64_t units;       // of all pages and heads
  int unit_bytes;
  uint8_t *data;
};

namespace tpuhip {

constexpr int kUnitTokens = 32;

template <int DP, int BITS>
struct KvUnit {
  static_assert(DP % 32 == 0 && (BITS == 4 || BITS == 8));
  static constexpr int kDim = DP, kBits = BITS;
  static constexpr int kLevels = (1 << BITS) - 1;
  static constexpr int kRow = DP * BITS / 8;          // bytes of a row's codes
  static constexpr int kCodes = kUnitTokens * kRow;   // of a unit's keys, and of its values
  static constexpr int kParams = 2 * kCodes;          // where the params begin
  static constexpr int kBytes = kParams + 2 * kUnitTokens * 4;
  static constexpr int kBlocks = kRow / 16;           // of 16 byte columns
  static constexpr bool kPaired = kBlocks % 2 == 0;   // a lane's bytes of two blocks lie together: 16, else 8

  // the byte of column j, token t among the values' codes.  Lane (t / 4 % 4, j % 16) of a wave holds the tokens 4g..4g+3 and
  // 16+4g..16+4g+3 of a column; of four tokens the middle two change places, so that every other byte, masked out of a dword, is a
  // pair of neighbours.
  static __host__ __device__ constexpr int v_at(int j, int t) {
    const int block = j >> 4, lane = (t >> 2 & 3) * 16 + (j & 15), half = t >> 4, r = t & 3;
    const int in4 = (r >> 1) | (r & 1) << 1;
    return kPaired ? (block >> 1) * 1024 + lane * 16 + (block & 1) * 8 + half * 4 + in4
                   : block * 512 + lane * 8 + half * 4 + in4;
  }
};

// head sizes the kernels are made for; 0: none
constexpr int kv_padded(int dim) {
  return dim < 1 ? 0 : dim <= 64 ? 64 : dim <= 96 ? 96 : dim <= 128 ? 128 : dim <= 192 ? 192 : dim <= 256 ? 256 : 0;
}

// f(KvUnit<DP, BITS>{}) for a cache's sizes
template <typename F>
int kv_dispatch(const tpuhip_kv_cache *c, F f) {
#define TPUHIP_KV_CASE(DP)                                     \
  case DP:                                                     \
    return c->desc.bits == 4 ? f(KvUnit<DP, 4>{}) : f(KvUnit<DP, 8>{});
  switch (c->dp) {
    TPUHIP_KV_CASE(64)
    TPUHIP_KV_CASE(96)
    TPUHIP_KV_CASE(128)
    TPUHIP_KV_CASE(192)
    TPUHIP_KV_CASE(256)
  }
#undef TPUHIP_KV_CASE
  return set_error(TPUHIP_ERR_INVALID, "kv cache: no kernels for a head size of %d", c->desc.head_dim);
}

// kv_attention.hip: makes ctx->join if it can
int attention_workspace(tpuhip_ctx *ctx);

__device__ __forceinline__ float bf16_to_f32(uint32_t b) { return __uint_as_float(b << 16); }

}  // namespace tpuhip
