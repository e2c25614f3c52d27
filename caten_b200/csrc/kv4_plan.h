// How a call of attention over the 4-bit cache is cut, and the workspace that it needs: shared by the host's code and the tests (plain C++).
#pragma once

#include <stdint.h>

#include <algorithm>

#include "kv4_layout.h"

namespace cb {

// Rows (tokens x the query heads that share a key head) of a unit of each kernel, and warps of a block.
constexpr int K2_ROWS = 4, K4_ROWS = 8, K3_ROWS = 128;
constexpr int K1_WARPS = 4, K2_WARPS = 4;                            // 1 or 4 of them share a unit
CB_HD constexpr int k4_warps(bool shared) { return shared ? 8 : 4; }
constexpr int K4_GROUP = 64;       // tokens at a time with single rows
constexpr int KJ_PARTS = 1024;     // at most, of a call
// units (K4: blocks) that fill the SMs, by the warps that share one; K4: as many as that are left whole
constexpr int64_t K1_FILL = 148 * 20, K2_FILL = 148 * 48, K3_FILL = 148, K4_FILL = 148 * 12, K4_WHOLE = 148 * 4;

struct Kv4Heads {
  int dim, kv_heads;
  int64_t group;   // query heads of a key head
};

// How a call is cut: row tiles, and parts of the tokens where row tiles alone leave SMs idle.  By sizes that the host knows.
struct Kv4Plan {
  int64_t units;   // row tiles of all sequences and key heads
  int tile_rows, row_tiles, parts, part_tokens, warps;
};
// Whether rows are enough for tiles of 128: 48 a sequence and key head on the average, and 1e8 products of all, below which that kernel's start costs more
// than it saves.  us in tiles of 8 rows and of 128: 32 rows over 2000 tokens (16 sequences, 8 key heads of 128) 94 and 120, 48 over 300 (64 sequences) 97
// and 82; 8 prompts of 64, 8 heads of 128, 9.0 and 11.5, one of 256, 12 heads of 64, 10.1 and 17.0; 600 over 2000, 32 heads of 128 over 8, 271 and 127.
inline bool kv4_prompts(const Kv4Heads &h, int64_t batch, int64_t rows, int64_t max_length) {
  return h.dim <= 128 && rows * h.group >= 48 * batch && (double)rows * (double)(h.kv_heads * h.group) * (double)max_length * h.dim >= 1e8;
}
// Of arguments that were checked; false: too many rows.
inline bool kv4_plan_of(const Kv4Heads &h, int64_t batch, int64_t rows, int64_t max_new, int64_t max_length, Kv4Plan *p) {
  p->tile_rows = max_new * h.group == 1 ? 1 : max_new * h.group <= K2_ROWS ? K2_ROWS : kv4_prompts(h, batch, rows, max_length) ? K3_ROWS : K4_ROWS;
  p->row_tiles = (int)((max_new * h.group + p->tile_rows - 1) / p->tile_rows);
  if (batch && (int64_t)h.kv_heads * p->row_tiles > 0x7fffffff / batch) return false;
  p->units = batch * h.kv_heads * p->row_tiles;
  const int64_t groups = (max_length + K4_GROUP - 1) / K4_GROUP;
  int64_t fill, blocks, shares;   // units of work that fill the SMs; units without parts; warps over whom a unit's tokens are dealt
  if (p->tile_rows == 1) {
    // A warp each where that is enough (20 warps an SM), and for up to four groups already with four an SM: a second and third warp would have one group
    // or none (592 of 128 dims: 200 tokens 8.4 us and 10.1, 400 15.4 and 13.5; 2000: 100 tokens 12.2 and 22).  Otherwise four.
    p->warps = p->units >= 148 * 16 || (groups <= 4 && p->units >= 148 * 4) ? 1 : K1_WARPS;
    fill = K1_FILL / p->warps; blocks = p->units; shares = p->warps;
  } else if (p->tile_rows == K2_ROWS) {
    // (likewise, with a stage half as long: 1184, 200 tokens 19 us and 24; 592, 200 tokens 15.5 and 13)
    p->warps = p->units >= 148 * 16 || (groups <= 4 && p->units >= 148 * 8) ? 1 : K2_WARPS;
    fill = K2_FILL / p->warps; blocks = p->units; shares = p->warps;
  } else if (p->tile_rows == K3_ROWS) {
    p->warps = 1;
    fill = K3_FILL; blocks = p->units; shares = 1;   // (152 tiles over 2000 tokens, 600 rows of 32 heads over 8: 135 us whole, 156 in three parts)
  } else {
    p->warps = p->row_tiles >= 4 ? 4 : p->row_tiles >= 2 ? 2 : 1;
    fill = K4_FILL; blocks = p->units / p->row_tiles * ((p->row_tiles + p->warps - 1) / p->warps); shares = k4_warps(p->warps == 4) / p->warps;
  }
  // (blocks of several rows that fill the SMs as they are would only add the join: 5 prompts of up to 333 tokens in such tiles 116 -> 136 us)
  int64_t parts = !blocks || (p->tile_rows == K4_ROWS && blocks >= K4_WHOLE) ? 1 : (fill + blocks - 1) / blocks;
  // A part gives each warp two groups at least.  Single rows of up to four groups a warp are left whole: two groups less take no longer than the join
  // and its launch (25 heads x 700 tokens 7.2 us in parts, 5.3 whole; 1000 7.2 and 6.2; 1500 7.4 and 7.9).
  const bool whole = p->tile_rows == 1 && groups <= 4 * shares;
  // Blocks of two to four rows that fill three quarters of their places on the SMs are cut into no less than eight groups a warp (64 sequences of 8
  // key heads: 700 tokens 35 us in parts, 25 whole; 10000 229 and 248, with uneven lengths 164 and 220).
  const bool coarse = p->tile_rows == K2_ROWS && blocks >= 148 * 3;
  const int64_t most = whole ? 1 : coarse ? groups / (8 * shares) : (groups + 2 * shares - 1) / (2 * shares);
  if (parts > most) parts = most;
  if (parts > KJ_PARTS) parts = KJ_PARTS;
  if (parts < 1) parts = 1;
  const int64_t each = groups ? (groups + parts - 1) / parts : 1;
  p->part_tokens = (int)(each * K4_GROUP);
  p->parts = (int)(groups ? (groups + each - 1) / each : 1);
  if (p->units * p->parts > 0x7fffffff / std::max(K4_ROWS, p->tile_rows)) return false;
  return true;
}

// Bytes that the parts of a call's rows take.
inline int64_t kv4_plan_bytes(const Kv4Plan &p, int dim) { return p.parts > 1 ? p.units * p.parts * p.tile_rows * (dim + 2) * (int64_t)sizeof(float) : 0; }

// Bytes that are enough for every call of these heads whose sizes are at most these: a smaller call may be cut into more parts, or take another kernel.
// Each kernel's parts are at most its units times the parts that max_length allows, and units that do not fill the SMs are cut into no more than
// fill them: parts = ceil(fill / units), so units x parts < fill + units < 2 fill.
inline int64_t kv4_work_bound(const Kv4Heads &h, int64_t batch, int64_t max_new, int64_t max_length) {
  const int64_t heads = batch * h.kv_heads, groups = (max_length + K4_GROUP - 1) / K4_GROUP, rows = max_new * h.group;
  auto of = [&](int64_t tile_rows, int64_t units, int64_t each, int64_t most) {   // each: groups of a part, at least
    const int64_t parts = std::min<int64_t>(KJ_PARTS, (groups + each - 1) / each);
    return parts > 1 ? std::min(units * parts, most) * tile_rows : 0;
  };
  int64_t most = 0;
  if (h.group == 1 && groups > 4) most = std::max(most, of(1, heads, 2, 2 * K1_FILL));
  if (h.group <= K2_ROWS && rows > 1) most = std::max(most, of(K2_ROWS, heads, 2, 2 * K2_FILL));
  if (rows > K2_ROWS) most = std::max(most, of(K4_ROWS, heads * ((rows + K4_ROWS - 1) / K4_ROWS), 4, 4 * (K4_FILL + K4_WHOLE)));   // (four units a block at most)
  if (rows > K2_ROWS && h.dim <= 128) most = std::max(most, of(K3_ROWS, heads * ((rows + K3_ROWS - 1) / K3_ROWS), 2, 2 * K3_FILL));
  return std::max<int64_t>(16, most * (h.dim + 2) * (int64_t)sizeof(float));
}

}  // namespace cb
