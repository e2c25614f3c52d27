// Where the values of a paged 4-bit cache lie: index arithmetic shared by the kernels, the host's checks and the tests (plain C++).
//
// A pool is `pages` pages; a page holds, for each key/value head, `page` tokens in tiles of 16.  A tile is
//   K codes [8 dim bytes] | K scales [dim bytes] | (Q4_1: K minima [dim bytes]) | the same for V
// and its order inside is that of the operands of 16 x 8 x 16 matrix products, so that a lane (g = lane / 4, t = lane % 4) of the
// attention kernels gets its share by 16-byte loads and unpacks it by masks alone:
//   codes   512 bytes for every 64 dims (chunk c); a lane's 16 bytes are four words j of eight 4-bit codes n
//     K     token g + 8 (j / 2), block of 32 dims 2 c + j % 2, dim 8 t + n of the block
//     V     token 2 t + j % 2 + 8 (j / 2), block 2 c + n / 4, dim 4 g + n % 4 of the block
//   scales  fp16 [t][block][j], token 2 t + j % 2 + 8 (j / 2)
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define CB_HD __host__ __device__ __forceinline__
#else
#define CB_HD inline
#endif

namespace cb {

struct Kv4Shape {
  int kv_heads, dim, q41, page;
  int64_t pages;
};

CB_HD int kv4_part_bytes(const Kv4Shape &s) { return (s.q41 ? 10 : 9) * s.dim; }   // K or V of a tile
CB_HD int kv4_tile_bytes(const Kv4Shape &s) { return 2 * kv4_part_bytes(s); }
CB_HD int64_t kv4_page_bytes(const Kv4Shape &s) { return (int64_t)s.kv_heads * (s.page / 16) * kv4_tile_bytes(s); }
// whether a page number of a table may be followed
CB_HD bool kv4_page_ok(const Kv4Shape &s, int64_t page_id) { return page_id >= 0 && page_id < s.pages; }
// first byte of the tile of `token_in_page` of a head
CB_HD int64_t kv4_tile_at(const Kv4Shape &s, int64_t page_id, int head, int token_in_page) {
  return page_id * kv4_page_bytes(s) + (int64_t)(head * (s.page / 16) + token_in_page / 16) * kv4_tile_bytes(s);
}
// inside K's (V's) part of a tile: byte that holds the code of (token, dim), tokens 0..15; the odd of its two codes is in the high half
CB_HD int kv4_k_byte(int token, int dim) {
  const int block = dim / 32, within = dim % 32;
  return block / 2 * 512 + (token % 8 * 4 + within / 8) * 16 + (token / 8 * 2 + block % 2) * 4 + within % 8 / 2;
}
CB_HD int kv4_v_byte(int token, int dim) {
  const int block = dim / 32, within = dim % 32;
  return block / 2 * 512 + (within / 4 * 4 + token % 8 / 2) * 16 + (token / 8 * 2 + token % 2) * 4 + block % 2 * 2 + within % 4 / 2;
}
// index of a block's scale among the part's halves (the minima follow, dim / 2 halves on)
CB_HD int kv4_scale_index(int token, int block, int dim) { return (token % 8 / 2 * (dim / 32) + block) * 4 + token / 8 * 2 + token % 2; }

}  // namespace cb
