// The key/value cache in 8 bits, as the kernels see it. Block: 16, 32 or 64 tokens of one
// key/value head. K codes [blocks][heads][tokens][dim], V codes [blocks][heads][dim][tokens]
// (the product with the probabilities sums over tokens, and its operand wants them side by
// side), one f32 scale for each (block, head) of either: value = code * scale.
#pragma once

#include "sequences.cuh"

namespace b200 {
namespace {

struct Cache {
  int8_t *k_codes, *v_codes;
  float *k_scales, *v_scales;
  int64_t blocks;
  int32_t heads, dim, tokens, token_bits;  // tokens of a block = 1 << token_bits
};

struct Table {
  const int32_t* blocks;  // [batch][width], rows `stride` apart
  int64_t stride;
  int32_t width;
};

// The cache's block that holds `page` of sequence b, or -1 (and a status bit).
__device__ __forceinline__ int64_t block_of(const Cache& c, const Table& t, int32_t b, int64_t page, int32_t* status) {
  int64_t block = -1;
  if (page >= 0 && page < t.width) block = t.blocks[b * t.stride + page];
  if (block < 0 || block >= c.blocks) {
    if (status) atomicOr(status, kErrBlocks);
    return -1;
  }
  return block;
}

inline bool valid_cache(const b200_kv_cache* c) {
  return c->blocks >= 0 && c->heads >= 1 && c->heads <= 65535 && (c->dim == 64 || c->dim == 128) &&
         (c->block_tokens == 16 || c->block_tokens == 32 || c->block_tokens == 64);
}
inline bool cache_pointers(const b200_kv_cache* c) { return c->k_codes && c->v_codes && c->k_scales && c->v_scales; }
inline bool cache_aligned(const b200_kv_cache* c) {
  return aligned(c->k_codes, 16) && aligned(c->v_codes, 16) && aligned(c->k_scales, 4) && aligned(c->v_scales, 4);
}
inline Cache device_cache(const b200_kv_cache* c) {
  return Cache{static_cast<int8_t*>(c->k_codes), static_cast<int8_t*>(c->v_codes),
               c->k_scales,                      c->v_scales,
               c->blocks,                        c->heads,
               c->dim,                           c->block_tokens,
               c->block_tokens == 16 ? 4 : (c->block_tokens == 32 ? 5 : 6)};
}

}  // namespace
}  // namespace b200
