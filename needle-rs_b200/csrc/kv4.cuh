// kv4.cuh — the cache of keys and values in 4 bits: its layout, and the
// requests of a call.
//
// A page holds page_tokens tokens of one request, for each KV head one after
// another in tiles of 16 tokens.  A tile is 640 bytes for each group of 32
// dimensions (NG groups: head_dim rounded up):
//   K codes  [NG][32][2] words    V codes [NG][32][2] words
//   K scales [NG][8][2], minima [NG][8][2]: f16 of rows r and r + 8
//   V scales and minima [NG][4][2][4]: f16 of tokens 4 q .. 4 q + 3
// The order inside is that of the operands of a 16 x 8 x 16 matrix
// instruction, so that a lane fetches what it multiplies in 8 bytes and needs no
// shuffle, and a token's codes share no byte with another's:
//   K as its rows (16 tokens) by dimensions: lane 4 r + q has tokens m = r and
//   m = r + 8, words of 8 dimensions 32 g + 8 q .., where token t is row
//   m = 2 (t / 4) + t % 2 + 8 (t / 2 % 2) and dimension d of a word sits in
//   nibble d / 2 + 4 (d % 2): a mask leaves a pair of neighbours in the
//   halves of a word.
//   V transposed (dimensions by 16 tokens): lane 4 r + q has dimensions
//   32 g + 4 r .. + 3 of tokens 4 q, 4 q + 1 (low and high half of word 0)
//   and 4 q + 2, 4 q + 3 (word 1), a nibble each.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "ops.h"

namespace ndl {
namespace kv4 {

constexpr int kTokens = 16, kGroup = 32;
constexpr int kMaxTokens = 1 << 30;  // of a request
constexpr float kLargest = 32768.0f;  // magnitudes above it do not fit: 15 steps of f16 from there may pass f16's range

__host__ __device__ constexpr int tile_bytes(int ng) { return 640 * ng; }
// Offsets inside a tile.
__host__ __device__ constexpr int v_codes(int ng) { return 256 * ng; }
__host__ __device__ constexpr int k_params(int ng) { return 512 * ng; }
__host__ __device__ constexpr int v_params(int ng) { return 576 * ng; }

__host__ __device__ __forceinline__ int row_of(int t) { return 2 * (t >> 2) + (t & 1) + 8 * ((t >> 1) & 1); }
// Word (4 bytes) of dimensions 32 g + 8 q .. of token t's key.
__host__ __device__ __forceinline__ int k_word(int t, int g, int q) {
  const int m = row_of(t);
  return ((g * 32 + (m & 7) * 4 + q) * 2 + (m >> 3)) * 4;
}
// Half word (2 bytes) of dimensions 32 g + 4 r .. of token t's value.
__host__ __device__ __forceinline__ int v_half(int ng, int t, int g, int r) {
  return v_codes(ng) + ((g * 32 + r * 4 + (t >> 2)) * 2 + ((t >> 1) & 1)) * 4 + (t & 1) * 2;
}
__host__ __device__ __forceinline__ int k_param(int ng, int t, int g, int which) {
  const int m = row_of(t);
  return k_params(ng) + (((which * ng + g) * 8 + (m & 7)) * 2 + (m >> 3)) * 2;
}
__host__ __device__ __forceinline__ int v_param(int ng, int t, int g, int which) {
  return v_params(ng) + (((g * 4 + (t >> 2)) * 2 + which) * 4 + (t & 3)) * 2;
}

// A request of a call.
struct Seq {
  int row0, n, len;  // its rows of the operands, tokens in its cache
};

// Request i; one whose numbers do not fit the operands has no rows and no
// tokens, and the plan's flag says so.  `inside`: its rows are its last tokens.
__host__ __device__ __forceinline__ Seq sequence(const Kv4Rows &b, const Kv4Shape &s, int i, bool inside, int *bad) {
  const int a = b.row_start[i], e = b.row_start[i + 1], len = b.kv_len[i];
  const bool ok = a >= 0 && a <= e && e <= b.rows && e - a <= b.max_new && len >= 0 && len <= kMaxTokens && len <= (int64_t)b.width * s.page_tokens &&
                  !(inside && e - a > len);
  if (!ok) *bad = 1;
  return ok ? Seq{a, e - a, len} : Seq{0, 0, 0};
}

// Which page holds tile `t` (of 16 tokens) of request i's cache, as its table says, and the tile's number in it.  A load: what is
// done with it can wait a while.
struct Page {
  int page, in;
};
__host__ __device__ __forceinline__ Page page_of(const Kv4Rows &b, const Kv4Shape &s, int i, int t) {
  const int per = s.page_tokens / kTokens, n = (int)(((uint64_t)(uint32_t)t * s.per_inverse) >> 38);  // t / per
  return Page{b.table[(int64_t)i * b.width + n], t - n * per};
}
// Where that tile begins for a KV head, in units of 128 bytes; kNoPlace (flag set) where there is no such page.
constexpr uint32_t kNoPlace = 0xffffffffu;
__host__ __device__ __forceinline__ uint32_t place_of(const Kv4Shape &s, const Page &p, int kvh, int *bad) {
  if (p.page < 0 || p.page >= s.n_pages) {
    *bad = 1;
    return kNoPlace;
  }
  const int per = s.page_tokens / kTokens;
  return (uint32_t)(((int64_t)p.page * s.page_bytes + ((int64_t)kvh * per + p.in) * tile_bytes(s.ng)) >> 7);
}
// The same as an address, or NULL.
__host__ __device__ __forceinline__ uint8_t *tile_at(uint8_t *pages, const Kv4Rows &b, const Kv4Shape &s, int i, int t, int kvh,
                                                     int *bad) {
  const uint32_t p = place_of(s, page_of(b, s, i, t), kvh, bad);
  return p == kNoPlace ? nullptr : pages + (int64_t)p * 128;
}

}  // namespace kv4
}  // namespace ndl
