// The 4-bit key/value cache in memory.
//
// Tokens live in pages of P (16 .. 256, a power of two) slots; slot = page * P + offset. One row is the D
// elements of one token and key/value head: D/2 bytes of codes and the pair (lo, hi), its smallest and
// largest element, both exact in the cache's 16-bit type. An element's value is lo + code * (hi - lo) / 15.
//   codes [pages, heads, P * D/2 bytes], pairs [pages, heads, P] of 4 bytes (lo in the low half).
// Keys: a token's row is D/2 contiguous bytes, nibble n of 32-bit word w is element 8 w + n.
// Values: 16 tokens x 64 elements form a block of 512 bytes, (P/16, D/64) blocks per page and head. Token s of
// the block and word g (elements 8 g .. 8 g + 7) lie at byte ((s / 4) * 8 + g) * 16 + (s % 4) * 4: a 16-byte
// load holds the same eight elements of four consecutive tokens, as a product that sums over tokens wants
// them, and a token still owns its 32-bit words (concurrent writers touch different words).
#pragma once

#include "common.cuh"

namespace b200lut {

struct CacheView {
  uint8_t *k, *v;              // codes
  uint32_t *k_pair, *v_pair;
  int n_pages, heads, page_log2, D;
};

// Byte offsets of a (page, head) in the codes and of a token's pair.
__host__ __device__ inline long long cache_codes_at(long long page, int head, int heads, int page_log2, int D) {
  return ((page * heads + head) << page_log2) * (D / 2);
}
__host__ __device__ inline long long cache_pair_at(long long page, int head, int heads, int page_log2, int offset) {
  return ((page * heads + head) << page_log2) + offset;
}
// Byte offset of 32-bit word w of token `offset` inside a (page, head).
__host__ __device__ inline int key_word_at(int offset, int w, int D) { return offset * (D / 2) + 4 * w; }
__host__ __device__ inline int value_word_at(int offset, int w, int D) {
  const int s = offset & 15;
  return ((offset >> 4) * (D / 64) + (w >> 3)) * 512 + ((s >> 2) * 8 + (w & 7)) * 16 + (s & 3) * 4;
}

// What a row's pair says: value = lo + code * step.
template <typename T>
__device__ __forceinline__ float2 lo_step(uint32_t pair) {
  const float lo = DType<T>::to_float(uint16_t(pair & 0xFFFFu)), hi = DType<T>::to_float(uint16_t(pair >> 16));
  return make_float2(lo, (hi - lo) * (1.f / 15.f));
}

int check_cache(const b200lut_kv_cache* c, const char* who, CacheView* v);

}  // namespace b200lut
