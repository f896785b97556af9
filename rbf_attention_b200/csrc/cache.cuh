// Layout of the paged 8-bit cache, shared by the kernels that write it (cache_write.cu) and attend over it (cache_attn.cu).
//
// A pool is (pages, H, cache_page_bytes(P)) bytes: a page holds 256 tokens of H heads, P (64 or 128) columns each. A head's
// part is a header of 16 fp32 pairs (key scale, value scale), one per block of 16 tokens, and 18 slots of 32 * P bytes.
// Slots 0 to 15 hold blocks that are complete: code + 128 as a byte, value = code * scale, scale = largest magnitude / 127.
// Slots 16 and 17 hold the keys and the values of the block that is not complete yet as they came, 16 rows of P 16-bit
// numbers: a block is rounded once, when its last token arrives, so what the cache holds depends on the tokens and not on the
// portions they came in, and a copy of a page is a copy of everything.
//
// Inside a slot the bytes stand in the order in which a warp's lanes take them as operands of mma.m16n8k16, 16 bytes per lane
// and 512 per warp-wide load, so that loads are dense and nothing is transposed:
//   keys:   chunk (dims / 64) * 2 + half, lane (g, t): row g of the half, dims 64 * (chunk / 2) + 16 t ... + 15.
//           Row g of half h is token 4 (g / 2) + 2 h + g % 2, so that the scores' rows are the values' k index as they are;
//   values: chunk dims / 32, lane (g, t): four words, word i = dim 32 * chunk + 4 g + i of tokens 4 t ... 4 t + 3.
#pragma once

#include <stdint.h>

namespace rbf {

constexpr int kPageTokens = 256;
constexpr int kBlockTokens = 16;                                // tokens that share a scale
constexpr int kPageBlocks = kPageTokens / kBlockTokens;
constexpr int kPageHeader = kPageBlocks * 8;
constexpr float kSmallestHeld = 1e-30f;                         // blocks whose largest magnitude is below it are held as zeros

constexpr int cache_columns(int D) { return D <= 64 ? 64 : 128; }
constexpr int cache_slot_bytes(int P) { return 32 * P; }
constexpr int cache_page_bytes(int P) { return kPageHeader + (kPageBlocks + 2) * cache_slot_bytes(P); }

// A sequence's tokens: `held` before the call's new ones, `fresh` of those, both within what its row of the page table spans.
struct CacheSpan {
  int held, fresh;
};
__device__ __forceinline__ CacheSpan cache_span(const int* lengths, const int* fresh, int b, int T, int max_pages) {
  const int64_t room = static_cast<int64_t>(max_pages) * kPageTokens;
  const int64_t cap = room < 0x7fffff00 ? room : 0x7fffff00;
  int64_t n = lengths[b];
  n = n < 0 ? 0 : n > cap ? cap : n;
  int64_t f = fresh != nullptr ? fresh[b] : T;
  f = f < 0 ? 0 : f > T ? T : f;
  return {static_cast<int>(n), static_cast<int>(f < cap - n ? f : cap - n)};
}

// A head's part of the page that holds token `position` of sequence b, or null: a page number outside the pool is not followed.
__device__ __forceinline__ const uint8_t* cache_page(const uint8_t* pages, const int* table, int b, int max_pages, int num_pages,
                                                     int H, int h, int page_bytes, int position) {
  const int column = position / kPageTokens;
  if (column >= max_pages) return nullptr;
  const int id = table[static_cast<int64_t>(b) * max_pages + column];
  if (id < 0 || id >= num_pages) return nullptr;
  return pages + (static_cast<int64_t>(id) * H + h) * page_bytes;
}

}  // namespace rbf
