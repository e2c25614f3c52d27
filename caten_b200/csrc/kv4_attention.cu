// Attention over a paged 4-bit cache: o = sum_t softmax_t(scale q . k_t) v_t over the tokens that a query sees, keys and values
// d code + m (Q4_0: m = -8 d) in blocks of 32 dims.
//
// Both products run as 16 x 8 x 16 matrix products on fp16 operands, in which code - 8 is exact: four bits or-ed into 1024 (or, four bits up, 64
// in sixteenths) and 1032 (72) taken off, two codes at a time.  (Masked where they stand, as subnormal halves, codes need no second instruction, but
// the tensor cores align products by the operands' exponent fields, so the ten leading zeros are lost from their 24 bits: errors of 1e-5.)  The other
// operand is split in two halves (22 bits): q, scaled to the top of fp16's range by a power of two, in rows r and r + 8 of the first product, whose sums
// are added; p d in two of the second.  Scales and minima stay outside the products, in fp32:
//   score(r, t) = sum over blocks of d_t,b (q_r . (codes - 8)) + n_t,b sum(q_r)          out(r, j) = sum_t (p_rt d_t,b) (code_tj - 8) + sum_t p_rt n_t,b
// with n = 0 (Q4_0) or the minimum + 8 d (Q4_1).  From the middle of the codes, because a sum of thousands of p d code is many times what is left when
// 8 p d is taken off it, and so is its error (100001 tokens: 3e-4).
// (So in the kernels for up to 48 rows; the one for prompts multiplies the scales in before.)
// A warp has 8 rows (tokens x the heads that share a key head; kernels for one row and for two to four follow, and one for tiles of 128) and takes 64 or
// 32 tokens at a time: running maximum and sum of the softmax per row, the group's p d times a power of two for each row and block of 32 dims that
// brings its largest near the top of fp16 (so what a row does not see, what has no probability and what other dims hold cost it no bits), and the sums
// joined to the running ones in fp32.
#include <algorithm>

#include "common.cuh"
#include "kv4.cuh"
#include "kv4_plan.h"
#include "kv4_ring.h"
#include "tcgen05.cuh"

namespace cb {

__host__ __device__ constexpr int K4_TILES(int chunks) { return chunks == 1 ? 4 : 2; }   // 16 tokens at a time with several

struct Kv4AttnArgs {
  const float *q;
  const uint8_t *pool;
  const int *table, *lengths, *starts;
  float *out, *part;
  int *status;
  int64_t ldq, rows;
  Kv4Shape s;
  int heads, group, max_pages, max_new, max_length, batch;
  int row_tiles, parts, part_tokens;
  int tile_rows;   // 1, 4, 8 or 128: which kernel
  int warps;       // 1 and 4 rows: warps that share a unit; 8: row tiles of a block
  float scale;
};

// rows of a sequence and how far they see; what a plan's device memory says is checked against the call's arguments here
struct Kv4Seq {
  int64_t first;   // row of q and out
  int count, length;
};
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4AttnArgs &a, int b, bool tells) {
  Kv4Seq q;
  q.first = a.starts ? a.starts[b] : b;
  const int64_t end = a.starts ? a.starts[b + 1] : b + 1;
  const int length = a.lengths[b];
  q.count = (int)(end - q.first);
  q.length = length;
  if (q.first < 0 || end < q.first || end > a.rows || end - q.first > a.max_new) {
    if (tells) report_bad_index(a.status, 44, b);
    q.count = 0;
  }
  if (length < 0 || length > a.max_length) {
    if (tells) report_bad_index(a.status, 45, length);
    q.length = length < 0 ? 0 : a.max_length;
  }
  return q;
}

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack_half_lo(float a, float b, uint32_t hi) {
  const float2 h = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
  return pack_half(a - h.x, b - h.y);
}
// code - 8 of the low four bits of both halves of w; of the next four
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) {
  uint32_t r;
  asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"((w & 0x000f000fu) | 0x64006400u), "r"(0x64086408u));   // 1024 + c - 1032
  return r;
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"((w & 0x00f000f0u) | 0x64006400u), "r"(0x2c002c00u), "r"(0xd480d480u));   // (1024 + 16 c) / 16 - 72
  return r;
}
__device__ __forceinline__ float2 half_pair(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
__device__ __forceinline__ float warp_max(float x) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}

// halves that are infinite or NaN made 0
__device__ __forceinline__ uint32_t finite_halves(uint32_t w) {
  return w & (((w & 0x7c00u) == 0x7c00u ? 0u : 0xffffu) | ((w & 0x7c000000u) == 0x7c000000u ? 0u : 0xffff0000u));
}
// keeps a rare branch a branch: as selects, its instructions would be everybody's
__device__ __forceinline__ void keep_branch() { asm volatile(""); }
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// power of two 2^(k - floor(log2 x)), for all of fp32's normal range (x of 2^127: 2^(k - 127)); at most 2^113, so that its reciprocal is normal too; 1 for zero
__device__ __forceinline__ float to_top(float x, int k = 14) {
  const int e = (int)(__float_as_uint(x) >> 23 & 0xff);
  if (x == 0.0f) return 1.0f;
  return __uint_as_float((uint32_t)min(254 + k - e, 240) << 23);
}

// the same for x >= 0, with 2^113 for zero; the inverse of such a power; the largest magnitude (NaN is passed over)
__device__ __forceinline__ float to_top_of(float x, int k = 14) { return __uint_as_float((uint32_t)min(254 + k - (int)(__float_as_uint(x) >> 23 & 0xff), 240) << 23); }
__device__ __forceinline__ float inverse_power(float x) { return __uint_as_float(0x7f000000u - __float_as_uint(x)); }
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float r;
  asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ float max_abs_nan(float a, float b, float c) {   // (NaN stays)
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A block's warps (four, eight where they make operands) are `row_warps` row tiles (one or two, then four) times two or four shares of the tokens.  The
// warps of a share work on one ring of two stages of 64 or 32 tokens, which bulk copies fill while the other is read (each stage is read by all its
// warps before it is filled again).
// With four row tiles (SHARED) the warps first turn a stage's codes into operands and its scales into floats, a quarter each, in shared memory: of the
// instructions of 16 tokens and a block of 32 dims, a hundred, that is nearly half, and each warp would do it for itself (5 prompts of 167 to 333
// tokens, 16 heads over 4 of 128: 130 us; they go in tiles of 128 rows now).
template <int NC, bool Q41, bool SHARED>
__global__ void __launch_bounds__(k4_warps(SHARED) * 32, SHARED ? (NC <= 2 ? 2 : 1) : NC == 1 ? 4 : NC == 2 ? 3 : 2) kv4_attention_kernel(const Kv4AttnArgs a) {
  constexpr int NB = 2 * NC, D = 64 * NC, PART = (Q41 ? 10 : 9) * D, TILE = 2 * PART, TILES = K4_TILES(NC), GROUP = 16 * TILES, STAGE = TILES * TILE;
  constexpr int WARPS = k4_warps(SHARED), PER_TILE = 16 * NB;   // (floats of a kind of a tile)
  constexpr int KINDS = Q41 ? 4 : 2;   // SHARED: scales of K and V, and minima + 8 d
  constexpr int OPS = TILES * NC * 8 * 512, FLOATS = TILES * KINDS * PER_TILE * 4, SHARE = 2 * STAGE + (SHARED ? OPS + FLOATS : 0);   // bytes
  __shared__ float sm[WARPS][K4_ROWS], sl[WARPS][K4_ROWS];
  __shared__ uint64_t bars[WARPS][2];
  __shared__ int gave_up[WARPS], never;           // (never: not set by anyone)
  __shared__ unsigned present[WARPS][2];          // of a share: tiles of each stage
  extern __shared__ __align__(128) uint8_t ring[];   // two stages a share (SHARED: then its operands); behind the last group, the warps' sums
  pdl_enter();
  const int lane = threadIdx.x & 31, warp = warp_index(), g = lane >> 2, t = lane & 3;
  const int row_warps = a.warps, shares = WARPS / row_warps, share = warp / row_warps, sub = warp % row_warps;
  int64_t u = blockIdx.x;
  const int part = (int)(u % a.parts); u /= a.parts;
  const int row_groups = (a.row_tiles + row_warps - 1) / row_warps;
  const int rg = row_groups - 1 - (int)(u % row_groups); u /= row_groups;   // (later rows see more: they start first)
  const int head = (int)(u % a.s.kv_heads);
  const int b = (int)(u / a.s.kv_heads);
  const Kv4Seq seq = kv4_seq(a, b, threadIdx.x == 0 && part == 0 && rg == 0 && head == 0);
  const int count = seq.count * a.group;   // rows of this key head
  if (rg * row_warps * K4_ROWS >= count) return;
  // row r: token r / group, query head head * group + r % group
  const int rt = rg * row_warps + sub, r = rt * K4_ROWS + g, tok = r / a.group;
  auto sees_of = [&](int row) { return row < count ? max(0, seq.length - seq.count + row / a.group + 1) : 0; };   // tokens before and at its position
  const int sees = sees_of(r), least = sees_of(rt * K4_ROWS), most = sees_of(min(count, rt * K4_ROWS + K4_ROWS) - 1);   // (least: 0 for a tile without rows)
  const int reach = sees_of(min(count, (rg + 1) * row_warps * K4_ROWS) - 1);   // of the block
  const int t0 = part * a.part_tokens, t1 = min(reach, t0 + a.part_tokens);
  if (t0 >= t1 && part > 0) return;
  const bool mine = rt * K4_ROWS < count;

  const uint32_t bar = smem_u32(&bars[share][0]);
  uint8_t *const stages = ring + share * SHARE;
  const int *table = a.table + (int64_t)b * a.max_pages;
  const int64_t page_bytes = kv4_page_bytes(a.s);
  const int tile_shift = a.s.page == 16 ? 0 : a.s.page == 32 ? 1 : a.s.page == 64 ? 2 : 3;   // tiles of a page, log2
  const int first = t0 + share * GROUP, step = shares * GROUP;
  // by the share's first warp, lanes over tiles: what can be followed is copied, the rest counts for nothing
  auto page_at = [&](int base) { return lane < TILES && base + 16 * lane < t1 ? table[((base >> 4) + lane) >> tile_shift] : -1; };
  auto issue = [&](int base, int id, int stage) {
    const bool wanted = lane < TILES && base + 16 * lane < t1, good = wanted && kv4_page_ok(a.s, id);
    if (wanted && !good) report_bad_index(a.status, 46, id);
    const unsigned there = __ballot_sync(0xffffffffu, good);
    if (lane == 0) {
      present[share][stage] = there;
      mbar_expect_tx(bar + 8 * stage, __popc(there) * TILE);   // (its arrival publishes `present`)
    }
    __syncwarp();
    if (good) bulk_load(smem_u32(stages) + stage * STAGE + lane * TILE,
                        a.pool + id * page_bytes + ((int64_t)(head << tile_shift) + (((base >> 4) + lane) & ((1 << tile_shift) - 1))) * TILE, TILE, bar + 8 * stage);
  };
  int id_next = -1;
  if (sub == 0) {
    if (lane == 0) {
      mbar_init(bar, 1);
      mbar_init(bar + 8, 1);
      gave_up[share] = never = 0;
      fence_proxy_async();
    }
    __syncwarp();
    if (first < t1) issue(first, page_at(first), 0);
    if (first + step < t1) issue(first + step, page_at(first + step), 1);
    id_next = page_at(first + 2 * step);
  }

  // q as the first product's operand: a block's two steps, {dims 8t + 0, 4 | 8t + 1, 5} and {2, 6 | 3, 7}; hi in rows g, lo in rows g + 8
  uint32_t qa[NB][2][4];
  float qsum[NB];   // Q4_1: sum(q) of a block
  float factor;
  {
    const float *q = a.q + (seq.first + tok) * a.ldq + (int64_t)(head * a.group + r % a.group) * D + 8 * t;
    float x[NB][8], top = 0.0f;
#pragma unroll
    for (int k = 0; k < NB; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[k][j] = r < count ? q[32 * k + j] : 0.0f;
        top = fmaxf(top, fabsf(x[k][j]));
      }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float up = to_top(top);
    factor = a.scale * 1.4426950408889634f * (1.0f / up);
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[k][j] *= up;
        sum += x[k][j];
      }
      if (Q41) {
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        qsum[k] = sum;
      }
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        qa[k][st][0] = pack_half(x[k][2 * st], x[k][2 * st + 4]);
        qa[k][st][1] = pack_half_lo(x[k][2 * st], x[k][2 * st + 4], qa[k][st][0]);
        qa[k][st][2] = pack_half(x[k][2 * st + 1], x[k][2 * st + 5]);
        qa[k][st][3] = pack_half_lo(x[k][2 * st + 1], x[k][2 * st + 5], qa[k][st][2]);
      }
    }
  }

  float run_max = -INFINITY, run_sum = 0.0f;   // of row g (run_sum: this lane's tokens)
  float off[Q41 ? NB : 1];                     // Q4_1: sums of p (m + 8 d) of a block, row g, this lane's tokens
  float o[NB][2][4];                           // rows 2t, 2t + 1; dims 4g + {0, 1} and 4g + {2, 3} of a block
#pragma unroll
  for (int k = 0; k < NB; ++k) {
    if (Q41) off[k] = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[k][i >> 2][i & 3] = 0.0f;
  }
  // SHARED: operands of a stage [tile][chunk][K: block, token half | V: block, dims][lane], then scales of K and of V as floats, and Q4_1's minima + 8 d
  uint4 *const ops = reinterpret_cast<uint4 *>(stages + 2 * STAGE);
  float *const floats = reinterpret_cast<float *>(stages + 2 * STAGE + OPS);
  __syncthreads();   // the barriers are there
  // scales of tokens 2t, 2t + 1, 2t + 8, 2t + 9, and Q4_1's minima + 8 d
  auto scales_of = [](const uint8_t *at, float (&d)[4], float (&n)[4]) {
    const uint2 d2 = *reinterpret_cast<const uint2 *>(at);
    const float2 d01 = half_pair(d2.x), d23 = half_pair(d2.y);
    d[0] = d01.x; d[1] = d01.y; d[2] = d23.x; d[3] = d23.y;
    if (Q41) {
      const uint2 m2 = *reinterpret_cast<const uint2 *>(at + D);
      const float2 m01 = half_pair(m2.x), m23 = half_pair(m2.y);
      n[0] = fmaf(8.0f, d[0], m01.x); n[1] = fmaf(8.0f, d[1], m01.y); n[2] = fmaf(8.0f, d[2], m23.x); n[3] = fmaf(8.0f, d[3], m23.y);
    }
  };
  int stage = 0;
  uint32_t phase = 0;
  bool ok = true;
  for (int base = first; base < t1; base += step) {
    // (a wait that runs out does not leave the loop: the share's warps meet below as often as each other)
    if (ok && !mbar_wait(bar + 8 * stage, phase, &gave_up[share])) {
      ok = false;
      if (lane == 0) {
        gave_up[share] = 1;
        atomicCAS(a.status, 0, DEV_WAIT_TIMEOUT);
        a.status[1] = 48;
      }
      if (sub == 0)
        ring_land(stage, phase, base + step < t1, [&](int s, uint32_t p) {
          mbar_wait_thread(bar + 8 * s, p, &never);
        });
    }
    if (SHARED && ok) {
      const uint8_t *tiles = stages + stage * STAGE;
      const unsigned there = present[share][stage];
#pragma unroll
      for (int unit0 = 0; unit0 < TILES * NC * 2; unit0 += 4) {
        const int unit = unit0 + sub, i = unit / (2 * NC), c = unit % NC;
        const bool of_k = unit / NC % 2 == 0;
        const uint4 w = *reinterpret_cast<const uint4 *>(tiles + i * TILE + (of_k ? 0 : PART) + c * 512 + lane * 16);
        uint4 *dst = ops + ((i * NC + c) * 8 + (of_k ? 0 : 4)) * 32 + lane;
        if (of_k) {   // tokens 0..7 and 8..15 of the even and of the odd block
          const uint32_t x[4] = {w.x, w.z, w.y, w.w};
#pragma unroll
          for (int n = 0; n < 4; ++n) dst[n * 32] = make_uint4(codes_lo(x[n]), codes_hi(x[n]), codes_lo(x[n] >> 8), codes_hi(x[n] >> 8));
        } else {      // of the even and of the odd block, tokens 2t, 2t + 1 and 2t + 8, 2t + 9
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const uint32_t x = __byte_perm(w.x, w.y, n ? 0x7632 : 0x5410), y = __byte_perm(w.z, w.w, n ? 0x7632 : 0x5410);
            dst[2 * n * 32] = make_uint4(codes_lo(x), codes_hi(x), codes_lo(y), codes_hi(y));
            dst[(2 * n + 1) * 32] = make_uint4(codes_lo(x >> 8), codes_hi(x >> 8), codes_lo(y >> 8), codes_hi(y >> 8));
          }
        }
      }
      for (int j = sub * 32 + lane; j < TILES * KINDS * PER_TILE / 2; j += 128) {
        const int i = j / (KINDS * PER_TILE / 2), rest = j % (KINDS * PER_TILE / 2), kind = rest / (PER_TILE / 2), pair = rest % (PER_TILE / 2);
        const uint8_t *at = tiles + i * TILE + (kind & 1) * PART + 8 * D + pair * 4;
        float2 x = half_pair(*reinterpret_cast<const uint32_t *>(at));
        if (kind >= 2) {
          const float2 m = half_pair(*reinterpret_cast<const uint32_t *>(at + D));
          x = make_float2(fmaf(8.0f, x.x, m.x), fmaf(8.0f, x.y, m.y));
        }
        *reinterpret_cast<float2 *>(floats + (i * KINDS + kind) * PER_TILE + pair * 2) = x;
      }
    }
    if (SHARED) asm volatile("bar.sync %0, 128;" ::"r"(1 + share) : "memory");
    if (ok && mine && base < most) {
      const uint8_t *tiles = stages + stage * STAGE;
      const unsigned there = present[share][stage];
      const bool clean = base + GROUP <= least && there == (1u << TILES) - 1u;   // every row sees every token
      float s[TILES][4];
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        const uint8_t *tile = tiles + i * TILE;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          uint4 w = make_uint4(0, 0, 0, 0);
          if (!SHARED) w = *reinterpret_cast<const uint4 *>(tile + c * 512 + lane * 16);
          const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int blk = 2 * c + k;
            const uint8_t *sc = tile + 8 * D + (t * NB + blk) * 8;
            float d[4], off_k[4];
            if (SHARED) {
              const float4 x = *reinterpret_cast<const float4 *>(floats + i * KINDS * PER_TILE + (t * NB + blk) * 4);
              d[0] = x.x; d[1] = x.y; d[2] = x.z; d[3] = x.w;
              if (Q41) {
                const float4 y = *reinterpret_cast<const float4 *>(floats + (i * KINDS + 2) * PER_TILE + (t * NB + blk) * 4);
                off_k[0] = y.x; off_k[1] = y.y; off_k[2] = y.z; off_k[3] = y.w;
              }
            } else {
              scales_of(sc, d, off_k);
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {   // tokens 0..7, 8..15
              uint4 op;
              if (SHARED) {
                op = ops[((i * NC + c) * 8 + 2 * k + n) * 32 + lane];
              } else {
                const uint32_t lo = words[2 * n + k], hi = lo >> 8;
                op = make_uint4(codes_lo(lo), codes_hi(lo), codes_lo(hi), codes_hi(hi));
              }
              float p[4] = {0.f, 0.f, 0.f, 0.f};
              mma_16816(p, qa[blk][0], op.x, op.y);
              mma_16816(p, qa[blk][1], op.z, op.w);
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const int e = 2 * n + j;
                if (Q41) acc[e] = fmaf(off_k[e], qsum[blk], acc[e]);   // (d code + m = d (code - 8) + (m + 8 d), which cancel before they are summed)
                acc[e] = fmaf(d[e], p[j] + p[2 + j], acc[e]);
              }
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[i][e] = acc[e] * factor;
        }
        if (!clean) {
          keep_branch();
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int at = base + 16 * i + 2 * t + (e & 1) + 8 * (e >> 1);
            if (at >= sees || at >= t1 || !(there >> i & 1)) s[i][e] = -INFINITY;
          }
        }
      }
      float top = run_max;
#pragma unroll
      for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, s[i][e]);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float ref = top == -INFINITY ? 0.0f : top;
      const float corr = exp2_fast(run_max - ref);   // (-inf: 0)
      run_max = top;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[i][e] = exp2_fast(s[i][e] - ref);
          sum += s[i][e];
        }
      run_sum = fmaf(run_sum, corr, sum);
      if (__any_sync(0xffffffffu, corr != 1.0f)) {   // (in a long history nearly never)
        keep_branch();
        const float corr0 = __shfl_sync(0xffffffffu, corr, 8 * t), corr1 = __shfl_sync(0xffffffffu, corr, 8 * t + 4);
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          if (Q41) off[k] *= corr;
#pragma unroll
          for (int i = 0; i < 8; ++i) o[k][i >> 2][i & 3] *= i & 1 ? corr1 : corr0;
        }
      }
      // values
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        uint4 w[TILES];
#pragma unroll
        for (int i = 0; i < TILES; ++i)
          if (!SHARED) w[i] = *reinterpret_cast<const uint4 *>(tiles + i * TILE + PART + c * 512 + lane * 16);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int blk = 2 * c + k;
          // p d, times a power of two that brings the row's largest of this block near the top of fp16
          float pd[TILES][4], largest = 0.0f, add = 0.0f;
#pragma unroll
          for (int i = 0; i < TILES; ++i) {
            float d[4], n[4], pn[4];
            if (SHARED) {
              const float4 x = *reinterpret_cast<const float4 *>(floats + (i * KINDS + 1) * PER_TILE + (t * NB + blk) * 4);
              d[0] = x.x; d[1] = x.y; d[2] = x.z; d[3] = x.w;
              if (Q41) {
                const float4 y = *reinterpret_cast<const float4 *>(floats + (i * KINDS + 3) * PER_TILE + (t * NB + blk) * 4);
                n[0] = y.x; n[1] = y.y; n[2] = y.z; n[3] = y.w;
              }
            } else {
              scales_of(tiles + i * TILE + PART + 8 * D + (t * NB + blk) * 8, d, n);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              pd[i][e] = s[i][e] * d[e];
              if (Q41) pn[e] = s[i][e] * n[e];
            }
            if (!clean) {   // (0 times what a scale behind the last token, or of a token that the row does not see, may be)
              keep_branch();
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (base + 16 * i + 2 * t + (e & 1) + 8 * (e >> 1) >= min(sees, t1) || !(there >> i & 1)) pd[i][e] = pn[e] = 0.0f;
            }
            if (Q41) add += (pn[0] + pn[1]) + (pn[2] + pn[3]);
            largest = max_abs(largest, pd[i][0], pd[i][1]);
            largest = max_abs(largest, pd[i][2], pd[i][3]);
          }
          if (Q41) off[blk] += add;
          largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
          largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
          const float up = to_top_of(largest), down = inverse_power(up);
          const float down0 = __shfl_sync(0xffffffffu, down, 8 * t), down1 = __shfl_sync(0xffffffffu, down, 8 * t + 4);
          float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
          for (int i = 0; i < TILES; ++i) {
            const float x0 = pd[i][0] * up, x1 = pd[i][1] * up, x2 = pd[i][2] * up, x3 = pd[i][3] * up;
            const uint32_t h0 = pack_half(x0, x1), h1 = pack_half(x2, x3), l0 = pack_half_lo(x0, x1, h0), l1 = pack_half_lo(x2, x3, h1);
            uint4 va, vb;
            if (SHARED) {
              va = ops[((i * NC + c) * 8 + 4 + 2 * k) * 32 + lane];
              vb = ops[((i * NC + c) * 8 + 5 + 2 * k) * 32 + lane];
            } else {
              const uint32_t x = __byte_perm(w[i].x, w[i].y, k ? 0x7632 : 0x5410), y = __byte_perm(w[i].z, w[i].w, k ? 0x7632 : 0x5410);
              va = make_uint4(codes_lo(x), codes_hi(x), codes_lo(y), codes_hi(y));
              vb = make_uint4(codes_lo(x >> 8), codes_hi(x >> 8), codes_lo(y >> 8), codes_hi(y >> 8));
            }
            const uint32_t a0[4] = {va.x, va.y, va.z, va.w}, a1[4] = {vb.x, vb.y, vb.z, vb.w};
            mma_16816(acc[0], a0, h0, h1);
            mma_16816(acc[0], a0, l0, l1);
            mma_16816(acc[1], a1, h0, h1);
            mma_16816(acc[1], a1, l0, l1);
          }
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[blk][n][e] = fmaf(acc[n][e], e & 1 ? down1 : down0, o[blk][n][e]);
        }
      }
    }
    // the stage has been read by all the share's warps
    if (row_warps > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + share), "r"(32 * row_warps) : "memory");
    else __syncwarp();
    if (sub == 0 && ok && base + 2 * step < t1) {
      issue(base + 2 * step, id_next, stage);
      id_next = page_at(base + 3 * step);
    }
    phase ^= stage;
    stage ^= 1;
  }

  // the warp's sums: over the four lanes of a row, then the blocks' constant parts to the lanes that hold the outputs
  run_sum += __shfl_xor_sync(0xffffffffu, run_sum, 1);
  run_sum += __shfl_xor_sync(0xffffffffu, run_sum, 2);
  if (Q41)
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      off[k] += __shfl_xor_sync(0xffffffffu, off[k], 1);
      off[k] += __shfl_xor_sync(0xffffffffu, off[k], 2);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float add = __shfl_sync(0xffffffffu, off[k], 8 * t + 4 * j);
        o[k][0][j] += add; o[k][0][2 + j] += add; o[k][1][j] += add; o[k][1][2 + j] += add;
      }
    }
  float *so = reinterpret_cast<float *>(ring) + warp * K4_ROWS * D;   // [row][D]
  if (__syncthreads_or(!ok)) return;   // no stage is read or filled any more; what did not come is nobody's output
#pragma unroll
  for (int k = 0; k < NB; ++k) {
    float *dst = so + 2 * t * D + 32 * k + 4 * g;
    *reinterpret_cast<float4 *>(dst) = make_float4(o[k][0][0], o[k][0][2], o[k][1][0], o[k][1][2]);
    *reinterpret_cast<float4 *>(dst + D) = make_float4(o[k][0][1], o[k][0][3], o[k][1][1], o[k][1][3]);
  }
  if (t == 0) { sm[warp][g] = run_max; sl[warp][g] = run_sum; }
  __syncthreads();
  if (share > 0 || !mine) return;
  const int64_t tile_of = ((int64_t)b * a.s.kv_heads + head) * a.row_tiles + rt;
#pragma unroll
  for (int j = 0; j < 2; ++j) {   // rows 2t and 2t + 1
    const int row = 2 * t + j, rr = rt * K4_ROWS + row;
    float top = sm[warp][row];
    for (int w = 1; w < shares; ++w) top = fmaxf(top, sm[warp + w * row_warps][row]);
    const float ref = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    float4 x[NB];
#pragma unroll
    for (int k = 0; k < NB; ++k) x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < shares; ++w) {
      const float e = exp2_fast(sm[warp + w * row_warps][row] - ref);
      sum = fmaf(sl[warp + w * row_warps][row], e, sum);
      const float *src = so + (w * row_warps * K4_ROWS + row) * D + 4 * g;
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const float4 y = *reinterpret_cast<const float4 *>(src + 32 * k);
        x[k].x = fmaf(y.x, e, x[k].x); x[k].y = fmaf(y.y, e, x[k].y); x[k].z = fmaf(y.z, e, x[k].z); x[k].w = fmaf(y.w, e, x[k].w);
      }
    }
    if (rr >= count) continue;
    float *dst = a.parts == 1 ? a.out + (seq.first + rr / a.group) * (int64_t)a.heads * D + (int64_t)(head * a.group + rr % a.group) * D
                              : a.part + ((tile_of * a.parts + part) * K4_ROWS + row) * (D + 2);
    const float scale = a.parts > 1 ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      float *p = dst + 32 * k + 4 * g;
      p[0] = x[k].x * scale; p[1] = x[k].y * scale; p[2] = x[k].z * scale; p[3] = x[k].w * scale;
    }
    if (a.parts > 1 && g == 0) { dst[D] = top; dst[D + 1] = sum; }
  }
}

// ---- two to four rows -------------------------------------------------------------------------------
// Key heads shared by two to four query heads, or as many tokens of one: with codes as the first operand (16 tokens) and the rows in the eight
// columns, halves side by side (column 2 r + h), nothing is empty: half the products of the kernel above, a score in one lane (row t, tokens g and
// g + 8), half the softmax; in the second product columns 2 r + h again, whose two sums a lane has both.  Each warp has a ring of its own.
// p d is scaled for each row, group and block of 32 dims by what the largest of them needs: a row's bits do not depend on tokens that it does not see, or
// that have no probability, nor on other dims.  The lanes of a row's two columns have two of a lane's four tokens each, make both halves of theirs and
// exchange one.
// Bound by instructions (unpacking, two roundings of p d).  4 heads to a key head of 128, Q4_0: 256 sequences of 768 tokens 71 us, 3 of 20000 to 100001
// 102 (in warps of 8 rows 167); Q4_1 79 and 111; 32 heads over 16 key heads of 256, 8 sequences of 580 to 2900 49 and 54.  (One power of two for a group, from
// the scales alone: 70 and 99, 80 and 110, 47 and 52, and values of 1e-4 beside 1e5 off by 4e-3 of themselves.)

template <int NC, bool Q41>
__global__ void __launch_bounds__(K2_WARPS * 32, NC <= 2 ? 4 : 2) kv4_attention_few_kernel(const Kv4AttnArgs a) {
  constexpr int NB = 2 * NC, D = 64 * NC, PART = (Q41 ? 10 : 9) * D, TILE = 2 * PART, TILES = K4_TILES(NC), GROUP = 16 * TILES, STAGE = TILES * TILE;
  __shared__ float sm[K2_WARPS][K2_ROWS], sl[K2_WARPS][K2_ROWS];
  __shared__ uint64_t bars[K2_WARPS][2];
  __shared__ int gave_up[K2_WARPS];
  extern __shared__ __align__(128) uint8_t ring[];   // two stages a warp; behind the last group, the warps' sums
  pdl_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int share = a.warps, first_warp = warp / share * share;
  int64_t u = (int64_t)blockIdx.x * (K2_WARPS / share) + warp / share;
  const int part = (int)(u % a.parts); u /= a.parts;
  const int64_t tile_of = u;
  const int rt = (int)(u % a.row_tiles); u /= a.row_tiles;
  const int head = (int)(u % a.s.kv_heads);
  const int64_t b = u / a.s.kv_heads;
  Kv4Seq seq = {0, 0, 0};
  if (b < a.batch) seq = kv4_seq(a, (int)b, lane == 0 && warp == first_warp && part == 0 && rt == 0 && head == 0);
  const int count = seq.count * a.group, r0 = rt * K2_ROWS;
  auto sees_of = [&](int row) { return row < count ? max(0, seq.length - seq.count + row / a.group + 1) : 0; };   // tokens before and at its position
  const int sees = sees_of(r0 + t), sees_col = sees_of(r0 + (g >> 1)), least = sees_of(r0), most = sees_of(min(count, r0 + K2_ROWS) - 1);
  const int t0 = part * a.part_tokens, t1 = r0 < count ? min(most, t0 + a.part_tokens) : 0;
  const bool live = r0 < count && (t0 < t1 || part == 0);

  float run_max = -INFINITY, run_sum = 0.0f;   // of row t (run_sum: this lane's tokens)
  float off[Q41 ? NB : 1];                     // Q4_1: sums of p (m + 8 d) of a block, the column's row, this lane's tokens
  float o[NB][2][4];                                            // columns 2t, 2t + 1; dims 4g + {0 | 1} and 4g + {2 | 3} of a block
#pragma unroll
  for (int k = 0; k < NB; ++k) {
    if (Q41) off[k] = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[k][i >> 2][i & 3] = 0.0f;
  }

  const int first = t0 + (warp - first_warp) * GROUP, step = share * GROUP;
  uint8_t *const mine = ring + warp * 2 * STAGE;
  bool ok = true;   // the copies came
  if (live && first < t1) {
    const uint32_t bar = smem_u32(&bars[warp][0]), dst = smem_u32(mine);
    if (lane == 0) {
      mbar_init(bar, 1);
      mbar_init(bar + 8, 1);
      gave_up[warp] = 0;
      fence_proxy_async();
    }
    __syncwarp();
    const int *table = a.table + b * a.max_pages;
    const int64_t page_bytes = kv4_page_bytes(a.s);
    const int tile_shift = a.s.page == 16 ? 0 : a.s.page == 32 ? 1 : a.s.page == 64 ? 2 : 3;   // tiles of a page, log2
    auto page_at = [&](int base) { return lane < TILES && base + 16 * lane < t1 ? table[((base >> 4) + lane) >> tile_shift] : -1; };
    auto issue = [&](int base, int id, int stage) -> unsigned {   // lanes over tiles: what can be followed is copied, the rest counts for nothing
      const bool wanted = lane < TILES && base + 16 * lane < t1, good = wanted && kv4_page_ok(a.s, id);
      if (wanted && !good) report_bad_index(a.status, 46, id);
      const unsigned there = __ballot_sync(0xffffffffu, good);
      if (lane == 0) mbar_expect_tx(bar + 8 * stage, __popc(there) * TILE);
      __syncwarp();
      if (good) bulk_load(dst + stage * STAGE + lane * TILE,
                          a.pool + id * page_bytes + ((int64_t)(head << tile_shift) + (((base >> 4) + lane) & ((1 << tile_shift) - 1))) * TILE, TILE, bar + 8 * stage);
      return there;
    };
    unsigned there_now = issue(first, page_at(first), 0), there_next = 0;
    if (first + step < t1) there_next = issue(first + step, page_at(first + step), 1);
    int id_next = page_at(first + 2 * step);

    // q: this lane's column (row g / 2, half g % 2); dims {0, 4 | 1, 5} and {2, 6 | 3, 7} of the lane's eight in each block
    uint32_t qb[NB][4];
    float qsum[NB];   // Q4_1: sum(q) of a block, row t
    float factor;
    {
      const int r = r0 + (g >> 1);
      const float *q = a.q + (seq.first + r / a.group) * a.ldq + (int64_t)(head * a.group + r % a.group) * D + 8 * t;
      float top = 0.0f;
      if (r < count)
#pragma unroll
        for (int k = 0; k < NB; ++k)
#pragma unroll
          for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(q[32 * k + j]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const float up = to_top(top);
      factor = __shfl_sync(0xffffffffu, a.scale * 1.4426950408889634f * (1.0f / up), 8 * t);
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        float y[8], sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float z = r < count ? q[32 * k + j] * up : 0.0f, hi = __half2float(__float2half_rn(z));
          sum += z;
          y[j] = g & 1 ? z - hi : hi;
        }
        if (Q41) {
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          qsum[k] = __shfl_sync(0xffffffffu, sum, 8 * t);
        }
        qb[k][0] = pack_half(y[0], y[4]);
        qb[k][1] = pack_half(y[1], y[5]);
        qb[k][2] = pack_half(y[2], y[6]);
        qb[k][3] = pack_half(y[3], y[7]);
      }
    }
    int stage = 0, base = first;
    uint32_t phase = 0;
    for (; base < t1; base += step) {
      ok = mbar_wait(bar + 8 * stage, phase, &gave_up[warp]);
      if (!ok) break;
      const uint8_t *tiles = mine + stage * STAGE;
      const unsigned there = there_now;
      const bool clean = base + GROUP <= least && there == (1u << TILES) - 1u;   // every row sees every token
      float s[TILES][2];
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        const uint8_t *tile = tiles + i * TILE;
        float x0 = 0.0f, x1 = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const uint4 w = *reinterpret_cast<const uint4 *>(tile + c * 512 + lane * 16);   // tokens g (x, y) and g + 8 (z, w); even and odd block
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int blk = 2 * c + k;
            const uint32_t x = k ? w.y : w.x, y = k ? w.w : w.z;
            const uint32_t a0[4] = {codes_lo(x), codes_lo(y), codes_hi(x), codes_hi(y)};
            const uint32_t a1[4] = {codes_lo(x >> 8), codes_lo(y >> 8), codes_hi(x >> 8), codes_hi(y >> 8)};
            float p[4] = {0.f, 0.f, 0.f, 0.f};
            mma_16816(p, a0, qb[blk][0], qb[blk][1]);
            mma_16816(p, a1, qb[blk][2], qb[blk][3]);
            const uint8_t *sc = tile + 8 * D + ((g >> 1) * NB + blk) * 8;
            const uint2 d2 = *reinterpret_cast<const uint2 *>(sc);
            const float2 d = half_pair(__byte_perm(d2.x, d2.y, g & 1 ? 0x7632 : 0x5410));
            if (Q41) {
              const uint2 m2 = *reinterpret_cast<const uint2 *>(sc + D);
              const float2 m = half_pair(__byte_perm(m2.x, m2.y, g & 1 ? 0x7632 : 0x5410));
              x0 = fmaf(fmaf(8.0f, d.x, m.x), qsum[blk], x0);   // (as above)
              x1 = fmaf(fmaf(8.0f, d.y, m.y), qsum[blk], x1);
            }
            x0 = fmaf(d.x, p[0] + p[1], x0);
            x1 = fmaf(d.y, p[2] + p[3], x1);
          }
        }
        s[i][0] = x0 * factor;
        s[i][1] = x1 * factor;
        if (!clean) {   // what stands behind the last token may be anything
          keep_branch();
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (base + 16 * i + g + 8 * e >= min(sees, t1) || !(there >> i & 1)) s[i][e] = -INFINITY;
        }
      }
      float top = run_max;
#pragma unroll
      for (int i = 0; i < TILES; ++i) top = fmaxf(top, fmaxf(s[i][0], s[i][1]));
#pragma unroll
      for (int k = 4; k < 32; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
      const float ref = top == -INFINITY ? 0.0f : top;
      const float corr = exp2_fast(run_max - ref);   // (-inf: 0)
      run_max = top;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s[i][e] = exp2_fast(s[i][e] - ref);
          sum += s[i][e];
        }
      run_sum = fmaf(run_sum, corr, sum);
      // p of the column's row: tokens 2t, 2t + 1 in an even column, 2t + 8, 2t + 9 in an odd one, which makes both halves of theirs
      float p[TILES][2];
#pragma unroll
      for (int i = 0; i < TILES; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float even = __shfl_sync(0xffffffffu, s[i][0], 8 * t + 4 * e + (g >> 1)), odd = __shfl_sync(0xffffffffu, s[i][1], 8 * t + 4 * e + (g >> 1));
          p[i][e] = g & 1 ? odd : even;
        }
      if (__any_sync(0xffffffffu, corr != 1.0f)) {   // (in a long history nearly never)
        keep_branch();
        const float corr_col = __shfl_sync(0xffffffffu, corr, g >> 1);
#pragma unroll
        for (int k = 0; k < NB; ++k) {
          if (Q41) off[k] *= corr_col;
#pragma unroll
          for (int i = 0; i < 8; ++i) o[k][i >> 2][i & 3] *= corr;
        }
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        uint4 w[TILES];
#pragma unroll
        for (int i = 0; i < TILES; ++i) w[i] = *reinterpret_cast<const uint4 *>(tiles + i * TILE + PART + c * 512 + lane * 16);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int blk = 2 * c + k;
          float pd[TILES][2], most = 0.0f, add = 0.0f;
#pragma unroll
          for (int i = 0; i < TILES; ++i) {
            const uint8_t *sc = tiles + i * TILE + PART + 8 * D + (t * NB + blk) * 8 + 4 * (g & 1);
            const float2 d = half_pair(*reinterpret_cast<const uint32_t *>(sc));
            float2 n = make_float2(0.f, 0.f);
            if (Q41) {
              const float2 m = half_pair(*reinterpret_cast<const uint32_t *>(sc + D));
              n = make_float2(fmaf(8.0f, d.x, m.x), fmaf(8.0f, d.y, m.y));
            }
            float pn[2] = {p[i][0] * n.x, p[i][1] * n.y};
            pd[i][0] = p[i][0] * d.x;
            pd[i][1] = p[i][1] * d.y;
            if (!clean) {   // (0 times what a scale behind the last token, or of a token that the row does not see, may be)
              keep_branch();
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (base + 16 * i + 2 * t + 8 * (g & 1) + e >= min(sees_col, t1) || !(there >> i & 1)) pd[i][e] = pn[e] = 0.0f;
            }
            if (Q41) add += pn[0] + pn[1];
            most = max_abs(most, pd[i][0], pd[i][1]);
          }
          if (Q41) off[blk] += add;
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
          most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 4));
          const float up = to_top_of(most), down = __shfl_sync(0xffffffffu, inverse_power(up), 8 * t);
          float acc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
          for (int i = 0; i < TILES; ++i) {
            const float x0 = pd[i][0] * up, x1 = pd[i][1] * up;
            const uint32_t hi = pack_half(x0, x1), lo = pack_half_lo(x0, x1, hi), other = __shfl_xor_sync(0xffffffffu, g & 1 ? hi : lo, 4);
            const uint32_t b0 = g & 1 ? other : hi, b1 = g & 1 ? lo : other;   // upper halves in the even column, lower ones in the odd
            const uint32_t x = __byte_perm(w[i].x, w[i].y, k ? 0x7632 : 0x5410), y = __byte_perm(w[i].z, w[i].w, k ? 0x7632 : 0x5410);
            const uint32_t a0[4] = {codes_lo(x), codes_hi(x), codes_lo(y), codes_hi(y)};
            const uint32_t a1[4] = {codes_lo(x >> 8), codes_hi(x >> 8), codes_lo(y >> 8), codes_hi(y >> 8)};
            mma_16816(acc[0], a0, b0, b1);
            mma_16816(acc[1], a1, b0, b1);
          }
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[blk][n][e] = fmaf(acc[n][e], down, o[blk][n][e]);
        }
      }
      __syncwarp();   // the stage has been read
      there_now = there_next;
      if (base + 2 * step < t1) {
        there_next = issue(base + 2 * step, id_next, stage);
        id_next = page_at(base + 3 * step);
      }
      phase ^= stage;
      stage ^= 1;
    }
    if (!ok) {
      if (lane == 0) {
        atomicCAS(a.status, 0, DEV_WAIT_TIMEOUT);
        a.status[1] = 49;
      }
      ring_land(stage, phase, base + step < t1, [&](int s, uint32_t p) {   // (with a flag that nobody raises)
        mbar_wait_thread(bar + 8 * s, p, &gave_up[warp]);
      });
    }
  }

  // row t: its sum over the lanes of its tokens; its outputs, halves together: four dims of a block a lane
#pragma unroll
  for (int k = 4; k < 32; k <<= 1) run_sum += __shfl_xor_sync(0xffffffffu, run_sum, k);
  float4 x[NB];
#pragma unroll
  for (int k = 0; k < NB; ++k) {
    float add = 0.0f;
    if (Q41) {
      off[k] += __shfl_xor_sync(0xffffffffu, off[k], 1);
      off[k] += __shfl_xor_sync(0xffffffffu, off[k], 2);
      off[k] += __shfl_xor_sync(0xffffffffu, off[k], 4);
      add = __shfl_sync(0xffffffffu, off[k], 8 * t);
    }
    x[k] = make_float4(o[k][0][0] + o[k][0][1] + add, o[k][0][2] + o[k][0][3] + add, o[k][1][0] + o[k][1][1] + add, o[k][1][2] + o[k][1][3] + add);
  }
  float top = run_max, sum = run_sum;
  if (share > 1) {
    float *so = reinterpret_cast<float *>(ring);   // [warp][row][D], each inside the warp's own stages
    constexpr int STRIDE = 2 * STAGE / (int)sizeof(float);
    static_assert(STRIDE >= K2_ROWS * D, "the warps' sums fit their rings");
#pragma unroll
    for (int k = 0; k < NB; ++k) *reinterpret_cast<float4 *>(so + warp * STRIDE + t * D + 32 * k + 4 * g) = x[k];
    if (g == 0) { sm[warp][t] = run_max; sl[warp][t] = run_sum; }
    if (__syncthreads_or(!ok)) return;   // (the block is one unit's; what did not come is nobody's output)
    if (warp != first_warp) return;
    for (int w = warp + 1; w < warp + share; ++w) top = fmaxf(top, sm[w][t]);
    const float ref = top == -INFINITY ? 0.0f : top;
    sum = 0.0f;
#pragma unroll
    for (int k = 0; k < NB; ++k) x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = warp; w < warp + share; ++w) {
      const float e = exp2_fast(sm[w][t] - ref);
      sum = fmaf(sl[w][t], e, sum);
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const float4 y = *reinterpret_cast<const float4 *>(so + w * STRIDE + t * D + 32 * k + 4 * g);
        x[k].x = fmaf(y.x, e, x[k].x); x[k].y = fmaf(y.y, e, x[k].y); x[k].z = fmaf(y.z, e, x[k].z); x[k].w = fmaf(y.w, e, x[k].w);
      }
    }
  }
  const int rr = r0 + t;
  if (!live || !ok || rr >= count) return;
  float *dst = a.parts == 1 ? a.out + (seq.first + rr / a.group) * (int64_t)a.heads * D + (int64_t)(head * a.group + rr % a.group) * D
                            : a.part + ((tile_of * a.parts + part) * K2_ROWS + t) * (D + 2);
  const float scale = a.parts > 1 ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int k = 0; k < NB; ++k) {
    float *p = dst + 32 * k + 4 * g;
    p[0] = x[k].x * scale; p[1] = x[k].y * scale; p[2] = x[k].z * scale; p[3] = x[k].w * scale;
  }
  if (a.parts > 1 && g == 0) { dst[D] = top; dst[D + 1] = sum; }
}

// ---- prompts ----------------------------------------------------------------------------------------
// 128 rows of a key head are the lanes of tensor memory, 64 tokens a step; a step's products are tcgen05.mma on fp16 halves, 22 bits of each operand:
//   S = Q_hi K_hi^T + Q_hi K_lo^T + Q_lo K_hi^T        O = P_hi V_hi + P_lo V_hi + P_hi V_lo
// (lo lo, 2^-22 of a product, is left out).  Scales are multiplied in before (d (code - 8) has 15 bits, so for Q4_0 two halves hold it exactly), a step's
// keys and 64 dims of its values times a power of two each that brings the largest near the top of fp16; P takes the values' size in exchange, so that
// steps of large values without probability do not cost others their bits.  Where the values of one step are far apart each row adds up what that may
// have cost it, and a tile in which a row has lost too much is worked out again without tensor cores (kv4_prompt_plainly).  S, P and O lie in tensor memory; a
// row's two threads (warps w and w + 4) take half of the tokens and half of the dims each, and keep the running output in registers, so that a moved maximum
// costs nothing more.  A value that is not finite would reach rows that do not see it (0 times NaN): it is zero in the product, and NaN is put into the
// blocks of the rows that see it.  By warp:
//   0 .. 7     rows of q; softmax of a step, its P, and the output of the step before
//   8 .. 14    codes into operands, two steps ahead at most (two stages each); the last asks for the tiles of the step after
//   15         issues the products: S a step ahead of the softmax
// A step takes 3.4 k cycles with heads of 64, 4.4 k of 128, of them 1.0 and 1.8 k of products; what bounds it is the instructions of warps 0 to 14 (0.5 a
// cycle and scheduler), unpacking before the softmax.  All phases by eight warps one after the other: 6.4 and 6.7 k; four warps to unpack: 195 us in place
// of 135 for 600 tokens over 2000, 32 heads of 128 over 8; two units at a time in registers: 130 in place of 127 (the code no longer fits the
// instruction cache).  That case 133 us now (tiles of 8 rows 271), 2000 of 25 heads of 64 113 (201), 5 prompts of 167 to 333 over up to 1200, 16 heads
// of 128 over 4, 62 (Q4_1 153, 123 and 69).
constexpr int K3_THREADS = 512, K3_SOFTMAX = 8, K3_CONVERT = 7;   // (warps)
constexpr float K3_LIFT = 14.0f;   // p is taken times 2^14, its sum with it
// A step's keys share a power of two, and 64 dims of its values.  Which sizes they have is a bit for each four exponents, from 2^-27 (what is stored is
// zero or 2^-24 at least) to 2^25: bit i is 2^(4i - 27) to 2^(4i - 23).  Where they are no more than two bits apart, 2^12, the last bits of 64 values and
// probabilities, 2^-3, are 2^-20 of what the smallest alone makes.
constexpr int K3_SPREAD = 2;
__device__ __forceinline__ unsigned k3_of_size(float x) { return x == 0.0f ? 0u : 1u << ((__float_as_uint(x) >> 25) - 25); }
// what brings the largest size to [2^11, 2^15); its exponent, the upper one (none: below all that can be stored)
__device__ __forceinline__ float k3_up(unsigned sizes) { return __uint_as_float((uint32_t)(127 + 38 - 4 * (31 - __clz(sizes | 1u))) << 23); }
__device__ __forceinline__ int k3_exponent(unsigned sizes) { return sizes ? 4 * (31 - __clz(sizes)) - 24 : -26; }
__host__ __device__ constexpr int k3_smem(int chunks, int tile_bytes) { return chunks * (32768 + 2 * 16384 + 2 * 16384) + 2 * 4 * tile_bytes + 1024; }
// of an operand tile: rows of 64 halves, 128-byte swizzle
__device__ __forceinline__ uint32_t k3_at(int row, int chunk) { return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4)); }
// (code - 8) d + n for two codes, as the upper and the lower half
template <bool Q41>
__device__ __forceinline__ void k3_split(uint32_t codes, uint32_t dd, float2 d, float2 n, uint32_t *hi, uint32_t *lo) {
  if (Q41) {
    const float2 c = half_pair(codes);
    const float x = fmaf(c.x, d.x, n.x), y = fmaf(c.y, d.y, n.y);
    *hi = pack_half(x, y);
    *lo = pack_half_lo(x, y, *hi);
  } else {   // exact
    const __half2 c = *reinterpret_cast<const __half2 *>(&codes), x = *reinterpret_cast<const __half2 *>(&dd), h = __hmul2_rn(c, x), l = __hfma2(c, x, __hneg2(h));
    *hi = *reinterpret_cast<const uint32_t *>(&h);
    *lo = *reinterpret_cast<const uint32_t *>(&l);
  }
}

// The rows of a tile in fp32 and without tensor cores, eight rows a warp: where a step has keys or values too far apart for halves that share a power of
// two, and a row's output is so small beside them that it counts.  64 tokens at a time become floats in shared memory (of which all else is done by now);
// scores with a token a lane, outputs with a dim a lane and sums of their own for the 64.  (5 prompts of 333 tokens over
// 1200: 1.85 ms, sixteen times as long; a row a warp, scores summed over lanes: 8.4 ms.)
template <int NC, bool Q41>
__device__ __forceinline__ void kv4_prompt_plainly(const Kv4AttnArgs &a, const Kv4Seq &seq, int b, int head, int rt, int part, float *smem) {
  constexpr int NB = 2 * NC, D = 64 * NC, PART = (Q41 ? 10 : 9) * D, ROWS = K3_ROWS * 32 / K3_THREADS, LD = D + 1;
  float *const qs = smem, *const ks = qs + K3_ROWS * D, *const vs = ks + 64 * LD;   // q times the scale; keys, a bank further on each; values
  const int tid = threadIdx.x, lane = tid & 31, count = seq.count * a.group, r0 = rt * K3_ROWS, first = tid >> 5 << 3, t0 = part * a.part_tokens;
  const int tile_shift = a.s.page == 16 ? 0 : a.s.page == 32 ? 1 : a.s.page == 64 ? 2 : 3;
  static_assert(ROWS == 8, "a warp's rows");
  auto sees_of = [&](int r) { return r < count ? min(t0 + a.part_tokens, max(0, seq.length - seq.count + r / a.group + 1)) : 0; };
  auto column_of = [&](int r) { return (int64_t)(head * a.group + r % a.group) * D; };
  const int reach = sees_of(min(count, r0 + K3_ROWS) - 1);
  for (int i = tid; i < K3_ROWS * D; i += K3_THREADS) {
    const int r = r0 + i / D;
    qs[i] = r < count ? a.q[(seq.first + r / a.group) * a.ldq + column_of(r) + i % D] * (a.scale * 1.4426950408889634f) : 0.0f;
  }
  float o[ROWS][NB], run_max[ROWS], run_sum[ROWS];
  int sees[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    sees[r] = sees_of(r0 + first + r);
    run_max[r] = -INFINITY;
    run_sum[r] = 0.0f;
#pragma unroll
    for (int k = 0; k < NB; ++k) o[r][k] = 0.0f;
  }
  for (int base = t0; base < reach; base += 64) {
    __syncthreads();   // the tokens before have been read
    unsigned there = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = base + 16 * i, id = at < reach ? a.table[(int64_t)b * a.max_pages + (at >> 4 >> tile_shift)] : -1;
      if (!kv4_page_ok(a.s, id)) continue;   // (reported by the copies)
      there |= 1u << i;
      const uint8_t *tile = a.pool + kv4_tile_at(a.s, id, head, at & (a.s.page - 1));
      for (int u = tid; u < 2 * 16 * D / 4; u += K3_THREADS) {   // four dims of a token's key or value
        const int of_v = u / (16 * D / 4), token = u / (D / 4) % 16, dim = u % (D / 4) * 4;
        const uint8_t *x = tile + of_v * PART;
        const unsigned codes = *reinterpret_cast<const uint16_t *>(x + (of_v ? kv4_v_byte(token, dim) : kv4_k_byte(token, dim)));
        const __half *sc = reinterpret_cast<const __half *>(x + 8 * D) + kv4_scale_index(token, dim / 32, D);
        const float d = __half2float(sc[0]), n = Q41 ? fmaf(8.0f, d, __half2float(sc[D / 2])) : 0.0f;
        float *dst = of_v ? vs + (16 * i + token) * D + dim : ks + (16 * i + token) * LD + dim;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float code = (float)((int)(codes >> 4 * e & 15u) - 8);
          dst[e] = Q41 ? fmaf(d, code, n) : d * code;
        }
      }
    }
    __syncthreads();
    if (base >= sees[ROWS - 1] && base >= sees_of(min(count, r0 + first + ROWS) - 1)) continue;
    float p[2][ROWS];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) p[h][r] = 0.0f;
      const float *k = ks + (32 * h + lane) * LD, *q = qs + first * D;
#pragma unroll 1
      for (int j = 0; j < D; j += 4) {
        const float k0 = k[j], k1 = k[j + 1], k2 = k[j + 2], k3 = k[j + 3];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          const float4 x = *reinterpret_cast<const float4 *>(q + r * D + j);
          p[h][r] = fmaf(x.w, k3, fmaf(x.z, k2, fmaf(x.y, k1, fmaf(x.x, k0, p[h][r]))));
        }
      }
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
        if (base + 32 * h + lane >= sees[r] || !(there >> (2 * h + lane / 16) & 1)) p[h][r] = -INFINITY;
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float top = fmaxf(run_max[r], warp_max(fmaxf(p[0][r], p[1][r]))), ref = top == -INFINITY ? 0.0f : top, corr = exp2_fast(run_max[r] - ref);
      run_max[r] = top;
      p[0][r] = exp2_fast(p[0][r] - ref);
      p[1][r] = exp2_fast(p[1][r] - ref);
      run_sum[r] = fmaf(run_sum[r], corr, warp_sum(p[0][r] + p[1][r]));
#pragma unroll
      for (int k = 0; k < NB; ++k) o[r][k] *= corr;
    }
#pragma unroll
    for (int r1 = 0; r1 < ROWS; r1 += 4) {
      float sums[4][NB];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int k = 0; k < NB; ++k) sums[r][k] = 0.0f;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll 1
        for (int at = 0; at < 32; ++at) {
          if (!(there >> (2 * h + at / 16) & 1)) continue;
          float v[NB];
#pragma unroll
          for (int k = 0; k < NB; ++k) v[k] = vs[(32 * h + at) * D + 32 * k + lane];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float w = __shfl_sync(0xffffffffu, p[h][r1 + r], at);
            if (base + 32 * h + at < sees[r1 + r])   // (0 times what a row does not see may be NaN)
#pragma unroll
              for (int k = 0; k < NB; ++k) sums[r][k] = fmaf(w, v[k], sums[r][k]);
          }
        }
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int k = 0; k < NB; ++k) o[r1 + r][k] += sums[r][k];
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = r0 + first + i;
    if (r >= count) continue;
    float *dst = a.parts == 1 ? a.out + (seq.first + r / a.group) * a.heads * D + column_of(r)
                              : a.part + (((((int64_t)b * a.s.kv_heads + head) * a.row_tiles + rt) * a.parts + part) * K3_ROWS + first + i) * (D + 2);
    const float scale = a.parts > 1 ? 1.0f : run_sum[i] == 0.0f ? 0.0f : 1.0f / run_sum[i];
#pragma unroll
    for (int k = 0; k < NB; ++k) dst[32 * k + lane] = o[i][k] * scale;
    if (a.parts > 1 && lane == 0) { dst[D] = run_max[i]; dst[D + 1] = run_sum[i]; }
  }
}
static_assert((K3_ROWS * 128 + 64 * 129 + 64 * 128) * 4 <= 2 * (32768 + 2 * 16384 + 2 * 16384) && (K3_ROWS * 64 + 64 * 65 + 64 * 64) * 4 <= 32768 + 2 * 16384 + 2 * 16384,
              "that takes no more shared memory than the operands had");

template <int NC, bool Q41>
__global__ void __launch_bounds__(K3_THREADS, 1) kv4_attention_prompt_kernel(const Kv4AttnArgs a) {
  constexpr int NB = 2 * NC, D = 64 * NC, PART = (Q41 ? 10 : 9) * D, TILE = 2 * PART, HALF = D / 2;
  constexpr uint32_t COL_P = 128, COL_O = 256, COLS = 512;   // (two blocks of scores, two of P)
  constexpr uint32_t IDESC = (1u << 4) | ((uint32_t)(K3_ROWS >> 4) << 24);   // fp32 sums, fp16 by fp16, 128 rows
  extern __shared__ unsigned char k3_raw[];
  __shared__ float red[2][2][K3_ROWS];      // [step & 1][half][row]
  __shared__ float qfactor[K3_ROWS];
  __shared__ int64_t q_at[K3_ROWS], out_at[K3_ROWS];   // where rows begin (divided once)
  // of four steps each, so that nobody need wait for their readers
  __shared__ float downs[4], ups[4][NC];      // what scores are to be multiplied with; what 64 dims of values were taken times
  __shared__ int size[4];                     // exponent of the values' largest
  __shared__ unsigned bad[4][64], any_bad[4][2];   // blocks of values that are not finite, by token; whether there are any, by half
  // of two steps: scales (of values, of an even and an odd block), minima (of keys, + 8 d)
  __shared__ float k_scale[2][64][NB], k_off[2][64][Q41 ? NB : 1];
  __shared__ uint32_t v_scale[2][64][NC], v_min[2][64][Q41 ? NC : 1];
  __shared__ __align__(8) unsigned k_sizes[4][2], v_sizes[4][NC][2];   // which sizes (k3_of_size) there are, by half of the tokens: of keys; of 64 dims of values
  __shared__ int wide[4], uneven;             // whether sizes are far apart (bit c: of the values' dims 64 c on; bit NC: of keys); whether that costs a row
  __shared__ unsigned theres[4];
  __shared__ unsigned present[2];                    // tiles of each stage
  __shared__ uint64_t bar_mem[17];
  __shared__ uint32_t tmem_slot;
  __shared__ int gave_up[2];                // [1] is never set
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = warp_index(), g = lane >> 2, t = lane & 3, quad = warp & 3, hf = warp >> 2, row = quad * 32 + lane;
  int64_t u = blockIdx.x;   // later rows see more: they start first
  const int part = (int)(u % a.parts); u /= a.parts;
  const int b = (int)(u % a.batch); u /= a.batch;
  const int head = (int)(u % a.s.kv_heads); u /= a.s.kv_heads;
  const int rt = a.row_tiles - 1 - (int)u;
  const Kv4Seq seq = kv4_seq(a, b, tid == 0 && part == 0 && rt == 0 && head == 0);
  const int count = seq.count * a.group, r0 = rt * K3_ROWS;
  if (r0 >= count) return;
  auto sees_of = [&](int r) { return r < count ? max(0, seq.length - seq.count + r / a.group + 1) : 0; };
  const int least = r0 + K3_ROWS <= count ? sees_of(r0) : 0, reach = sees_of(min(count, r0 + K3_ROWS) - 1);
  const int t0 = part * a.part_tokens, t1 = min(reach, t0 + a.part_tokens);
  if (t0 >= t1 && part > 0) return;
  const int sees = min(sees_of(r0 + row), t1), steps = t1 > t0 ? (t1 - t0 + 63) / 64 : 0;

  unsigned char *const sq = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(k3_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char *const sk = sq + NC * 32768, *const sv = sk + 2 * NC * 16384, *const raw = sv + 2 * NC * 16384;
  const uint32_t bars = smem_u32(bar_mem), q_full = bars + 112, p_full = bars + 120, o_full = bars + 128;
  auto raw_full = [&](int k) { return bars + 8u * k; };
  auto k_full = [&](int k) { return bars + 16u + 8u * k; };
  auto k_empty = [&](int k) { return bars + 32u + 8u * k; };
  auto v_full = [&](int k) { return bars + 48u + 8u * k; };
  auto v_empty = [&](int k) { return bars + 64u + 8u * k; };
  auto s_full = [&](int k) { return bars + 80u + 8u * k; };
  auto s_empty = [&](int k) { return bars + 96u + 8u * k; };
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(raw_full(i), 1);
      mbar_init(k_full(i), K3_CONVERT);
      mbar_init(k_empty(i), 1);
      mbar_init(v_full(i), K3_CONVERT);
      mbar_init(v_empty(i), 1);
      mbar_init(s_full(i), 2);   // the products, and the issuing warp for what the converters left beside K
      mbar_init(s_empty(i), K3_SOFTMAX);
    }
    mbar_init(q_full, K3_SOFTMAX);
    mbar_init(p_full, K3_SOFTMAX);
    mbar_init(o_full, 2);
    gave_up[0] = gave_up[1] = uneven = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  if (tid >= 128 && tid < 128 + K3_ROWS) {
    const int k = tid - 128, r = min(r0 + k, count - 1), token = r / a.group;
    const int64_t column = (int64_t)(head * a.group + r % a.group) * D;
    q_at[k] = (seq.first + token) * a.ldq + column;
    out_at[k] = a.parts == 1 ? (seq.first + token) * (int64_t)a.heads * D + column
                             : (((((int64_t)b * a.s.kv_heads + head) * a.row_tiles + rt) * a.parts + part) * K3_ROWS + k) * (D + 2);
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();   // not before this block has its tensor memory: the next kernel's blocks may ask for theirs and then wait for this grid
  const uint32_t tmem = tmem_slot, tlane = tmem + ((uint32_t)(quad * 32) << 16);

  const int *table = a.table + (int64_t)b * a.max_pages;
  const int64_t page_bytes = kv4_page_bytes(a.s);
  const int tile_shift = a.s.page == 16 ? 0 : a.s.page == 32 ? 1 : a.s.page == 64 ? 2 : 3;   // tiles of a page, log2
  auto page_at = [&](int step) {
    const int at = t0 + 64 * step + 16 * lane;
    return lane < 4 && at < t1 ? table[(at >> 4) >> tile_shift] : -1;
  };
  auto issue = [&](int step, int id) {   // by one warp: what can be followed is copied, the rest counts for nothing
    const int at = t0 + 64 * step + 16 * lane, stage = step & 1;
    const bool wanted = lane < 4 && at < t1, good = wanted && kv4_page_ok(a.s, id);
    if (wanted && !good) report_bad_index(a.status, 46, id);
    const unsigned there = __ballot_sync(0xffffffffu, good);
    if (lane == 0) {
      present[stage] = there;
      mbar_expect_tx(raw_full(stage), __popc(there) * TILE);   // (its arrival publishes `present`)
    }
    __syncwarp();
    if (good) bulk_load(smem_u32(raw) + (stage * 4 + lane) * TILE, a.pool + id * page_bytes + ((int64_t)(head << tile_shift) + ((at >> 4) & ((1 << tile_shift) - 1))) * TILE,
                        TILE, raw_full(stage));
  };
  int asked = 0, came = 0;   // stages asked for, stages seen (the warp that asks)
  bool ok = true;   // of the warp; one whose wait ran out goes on through the barriers that it shares, and touches nothing else
  auto wait = [&](uint32_t bar, uint32_t phase) {
    if (ok && !mbar_wait(bar, phase, &gave_up[0])) {
      ok = false;
      if (lane == 0) {
        gave_up[0] = 1;
        atomicCAS(a.status, 0, DEV_WAIT_TIMEOUT);
        a.status[1] = 50;
      }
    }
    return ok;
  };

  // rows of q, D / 8 lanes each: eight dims in the order (0, 4, 1, 5, 2, 6, 3, 7), as codes come out of a word
  auto convert_q = [&]() {
    constexpr int LANES = D / 8, ROWS = 32 / LANES;
    const int chunk = lane % LANES;
    const bool wide = (((uintptr_t)a.q | (uintptr_t)a.ldq * 4) & 15) == 0;
    const float scale2 = a.scale * 1.4426950408889634f;
#pragma unroll 1
    for (int i0 = 0; i0 < 16 / ROWS; i0 += 4) {
      float4 in[4][2];   // four rows under way
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int q_row = warp * 16 + (i0 + i) * ROWS + lane / LANES, r = r0 + q_row;
        const float *q = a.q + q_at[q_row] + 8 * chunk;
        in[i][0] = in[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < count && wide) {
          in[i][0] = reinterpret_cast<const float4 *>(q)[0];
          in[i][1] = reinterpret_cast<const float4 *>(q)[1];
        } else if (r < count) {
          in[i][0] = make_float4(q[0], q[1], q[2], q[3]);
          in[i][1] = make_float4(q[4], q[5], q[6], q[7]);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int q_row = warp * 16 + (i0 + i) * ROWS + lane / LANES;
        const float x[8] = {in[i][0].x, in[i][0].y, in[i][0].z, in[i][0].w, in[i][1].x, in[i][1].y, in[i][1].z, in[i][1].w};
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(x[j]));
#pragma unroll
        for (int j = 1; j < LANES; j <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, j));
        // What scores are multiplied with stays a power of two: then that product is exact and a row's largest score less itself is zero however large it
        // is (fused with the subtraction, from scores of 1e8 on, it was off by more than fp16 holds).  The rest of scale log2(e), in [1, 2), goes into q.
        const float up = to_top(top, 13), power = fmaxf(__uint_as_float(__float_as_uint(scale2) & 0x7f800000u), 0x1p-126f), sign_up = scale2 * (1.0f / power) * up;
        if (chunk == 0) qfactor[q_row] = top > 0.0f ? power * (1.0f / up) : 0.0f;
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float y = x[j] * sign_up, z = x[j + 4] * sign_up;
          hi[j] = pack_half(y, z);
          lo[j] = pack_half_lo(y, z, hi[j]);
        }
        unsigned char *dst = sq + chunk / 8 * 32768 + k3_at(q_row, chunk % 8);
        *reinterpret_cast<uint4 *>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4 *>(dst + 16384) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    }
    fence_proxy_async();
  };
  auto both = [](const unsigned *x) { const uint2 y = *reinterpret_cast<const uint2 *>(x); return y.x | y.y; };
  // a step's scales, a token a thread: warps 0 and 1 those of keys, 2 and 3 of values (what stands behind the last token, or is not finite, is zero)
  auto scales = [&](int step, int cw) {
    const int st = step & 1, token = (cw & 1) * 32 + lane, tk = token & 15;
    const bool in = present[st] >> (token >> 4) & 1 && t0 + 64 * step + token < t1;
    const unsigned char *tile = raw + (st * 4 + (token >> 4)) * TILE + (cw < 2 ? 0 : PART) + 8 * D;
    uint32_t d[NB], m[NB];
#pragma unroll
    for (int blk = 0; blk < NB; ++blk) {
      const int at = 2 * kv4_scale_index(tk, blk, D);
      d[blk] = *reinterpret_cast<const uint16_t *>(tile + at);
      m[blk] = Q41 ? *reinterpret_cast<const uint16_t *>(tile + D + at) : 0;
    }
    if (cw < 2) {
      unsigned sizes = 0;
#pragma unroll
      for (int blk = 0; blk < NB; ++blk) {
        const float x = half_pair(d[blk]).x, y = Q41 ? fmaf(8.0f, x, half_pair(m[blk]).x) : 0.0f, most = fmaf(8.0f, fabsf(x), fabsf(y));
        if (in && most < INFINITY) sizes |= k3_of_size(most);
        k_scale[st][token][blk] = x;
        if (Q41) k_off[st][token][blk] = y;
      }
      sizes = __reduce_or_sync(0xffffffffu, sizes);
      if (lane == 0) k_sizes[step & 3][cw] = sizes;
    } else {
      unsigned lost = 0, sizes[NC];
#pragma unroll
      for (int blk = 0; blk < NB; ++blk) {
        const uint32_t x = in ? finite_halves(d[blk]) : 0u, y = in ? finite_halves(m[blk]) : 0u;
        if (in && (x != d[blk] || y != m[blk])) lost |= 1u << blk;
        d[blk] = x;
        m[blk] = y;
        const unsigned of = k3_of_size(fmaf(Q41 ? 16.0f : 8.0f, fabsf(half_pair(x).x), fabsf(half_pair(y).x)));
        sizes[blk / 2] = blk % 2 ? sizes[blk / 2] | of : of;
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        sizes[c] = __reduce_or_sync(0xffffffffu, sizes[c]);
        if (lane == 0) v_sizes[step & 3][c][cw & 1] = sizes[c];
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        v_scale[st][token][c] = d[2 * c] | d[2 * c + 1] << 16;
        if (Q41) v_min[st][token][c] = m[2 * c] | m[2 * c + 1] << 16;
      }
      bad[step & 3][token] = lost;
      const unsigned any = __any_sync(0xffffffffu, lost);
      if (lane == 0) any_bad[step & 3][cw & 1] = any;
    }
  };
  // keys of a tile and a block
  auto convert_k = [&](int st, int unit, float up) {
    const int i = unit / (2 * NC), c = unit / 2 % NC, k = unit % 2;
    const uint4 w = *reinterpret_cast<const uint4 *>(raw + (st * 4 + i) * TILE + c * 512 + lane * 16);
#pragma unroll
    for (int h = 0; h < 2; ++h) {   // tokens g, g + 8
      const int token = 16 * i + g + 8 * h;
      const uint32_t x = h ? (k ? w.w : w.z) : (k ? w.y : w.x), codes[4] = {codes_lo(x), codes_hi(x), codes_lo(x >> 8), codes_hi(x >> 8)};
      const float d = k_scale[st][token][2 * c + k] * up, n = Q41 ? k_off[st][token][2 * c + k] * up : 0.0f;
      const uint32_t dd = pack_half(d, d);
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) k3_split<Q41>(codes[e], dd, make_float2(d, d), make_float2(n, n), &hi[e], &lo[e]);
      unsigned char *dst = sk + (st * NC + c) * 16384 + k3_at(token, 4 * k + t);
      *reinterpret_cast<uint4 *>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      *reinterpret_cast<uint4 *>(dst + 8192) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
  };
  // values of a tile, 64 dims and half of the tokens
  auto convert_v = [&](int st, int unit, const float (&ups)[NC]) {
    const int i = unit / (2 * NC), c = unit / 2 % NC, h = unit % 2;   // tokens 2t + 8 h, 2t + 8 h + 1
    const float up = NC == 1 || c == 0 ? ups[0] : ups[NC - 1];
    const uint2 w = *reinterpret_cast<const uint2 *>(raw + (st * 4 + i) * TILE + PART + c * 512 + lane * 16 + 8 * h);
#pragma unroll
    for (int j = 0; j < 2; ++j) {   // (even, odd block) in the halves of each operation
      const int token = 16 * i + 2 * t + 8 * h + j;
      const uint32_t x = j ? w.y : w.x, codes[4] = {codes_lo(x), codes_hi(x), codes_lo(x >> 8), codes_hi(x >> 8)};
      float2 d = half_pair(v_scale[st][token][c]), n = make_float2(0.f, 0.f);
      if (Q41) {
        n = half_pair(v_min[st][token][c]);
        n.x = fmaf(8.0f, d.x, n.x) * up; n.y = fmaf(8.0f, d.y, n.y) * up;
      }
      d.x *= up; d.y *= up;
      const uint32_t dd = pack_half(d.x, d.y);
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) k3_split<Q41>(codes[e], dd, d, n, &hi[e], &lo[e]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t how = k ? 0x7632 : 0x5410;
        unsigned char *dst = sv + (st * NC + c) * 16384 + k3_at(token, 4 * k + (g >> 1)) + (g & 1) * 8;
        *reinterpret_cast<uint2 *>(dst) = make_uint2(__byte_perm(hi[0], hi[1], how), __byte_perm(hi[2], hi[3], how));
        *reinterpret_cast<uint2 *>(dst + 8192) = make_uint2(__byte_perm(lo[0], lo[1], how), __byte_perm(lo[2], lo[3], how));
      }
    }
  };

  float o[HALF], run_max = -INFINITY, run_ref = -INFINITY, run_sum = 0.0f, run_down = 1.0f, lifted = 0.0f;   // (run_sum: this thread's tokens)
  float lost_bits = 0.0f;   // what o may be off because of steps in which values are far apart
#pragma unroll
  for (int e = 0; e < HALF; ++e) o[e] = 0.0f;
  auto take_outputs = [&](int step) {
#pragma unroll
    for (int e0 = 0; e0 < HALF; e0 += 16) {
      uint32_t x[16];
      tmem_ld16(tlane + COL_O + HALF * hf + e0, x);
      tmem_ld_wait();
#pragma unroll
      for (int e = 0; e < 16; ++e) o[e0 + e] = fmaf(o[e0 + e], lifted, __uint_as_float(x[e]));
    }
    // (64 tokens, each half a step of P's and of V's last bits, 2^-25, times the other's largest, 2^15 and 2^14)
    lost_bits = fmaf(lost_bits, lifted, wide[step & 3] >> (NC == 1 ? 0 : hf) & 1 ? 0x1p-3f : 0.0f);
    if (any_bad[step & 3][0] | any_bad[step & 3][1])
      for (int k = 0; k < 64; ++k) {
        const unsigned blocks = bad[step & 3][k];
        if (blocks && t0 + 64 * step + k < sees)
#pragma unroll
          for (int kk = 0; kk < NC; ++kk)
            if (blocks >> (hf * NC + kk) & 1)
#pragma unroll
              for (int e = 0; e < 32; ++e) o[32 * kk + e] = __int_as_float(0x7fffffff);
      }
  };

  if (warp >= K3_SOFTMAX && warp < K3_SOFTMAX + K3_CONVERT) {
    // ---------------- operands ----------------
    const int cw = warp - K3_SOFTMAX;
    int id_next = -1;
    if (cw == K3_CONVERT - 1) {
      for (; asked < min(steps, 2); ++asked) issue(asked, page_at(asked));
      id_next = page_at(2);
    }
    for (int step = 0; step < steps; ++step) {
      const int st = step & 1;
      const uint32_t phase = (uint32_t)(step >> 1) & 1u;
      if (wait(raw_full(st), phase)) {
        ++came;
        if (cw < 4) scales(step, cw);
      }
      asm volatile("bar.sync 5, %0;" ::"n"(32 * K3_CONVERT) : "memory");   // also: the step before has been read
      const float up_k = k3_up(both(k_sizes[step & 3]));
      float up[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) up[c] = k3_up(both(v_sizes[step & 3][c]));
      if (cw == K3_CONVERT - 1 && ok) {
        if (step > 0 && asked < steps) {
          issue(asked, id_next);
          ++asked;
          id_next = page_at(asked);
        }
        if (lane == 0) theres[step & 3] = present[st];
      }
      // units of K, then of V, dealt as one row (32 of heads of 128)
      int unit = cw;
      if (wait(k_empty(st), phase ^ 1u)) {
#pragma unroll 1
        for (; unit < 8 * NC; unit += K3_CONVERT) convert_k(st, unit, up_k);
        if (cw == K3_CONVERT - 2) {   // what the softmax has to know of the step's scales, by a warp with fewer units
          unsigned sizes = 0;
          if (lane < NC) sizes = both(v_sizes[step & 3][lane]);
          if (lane == NC) sizes = both(k_sizes[step & 3]);
          const int exponent = k3_exponent(__reduce_or_sync(0xffffffffu, lane < NC ? sizes : 0u));
          if (lane < NC) ups[step & 3][lane] = k3_up(sizes);
          if (lane == NC) {
            downs[step & 3] = inverse_power(up_k);
            size[step & 3] = exponent;
          }
          const unsigned far = __ballot_sync(0xffffffffu, sizes && 31 - __clz(sizes) - (__ffs(sizes) - 1) > K3_SPREAD);
          if (lane == 0) wide[step & 3] = (int)far;
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(k_full(st));
      }
      if (wait(v_empty(st), phase ^ 1u)) {
#pragma unroll 1
        for (; unit < 16 * NC; unit += K3_CONVERT) convert_v(st, unit - 8 * NC, up);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(v_full(st));
      }
    }
    if (!ok && cw == K3_CONVERT - 1)   // copies land before the block ends
      for (int k = came; k < asked; ++k) mbar_wait_thread(raw_full(k & 1), (uint32_t)(k >> 1) & 1u, &gave_up[1]);
  } else if (warp == K3_SOFTMAX + K3_CONVERT) {
    // ---------------- products (uniform control flow, one elected lane issues) ----------------
    const uint64_t dq = umma_desc(smem_u32(sq)), dk0 = umma_desc(smem_u32(sk));
    // V has the dims contiguous: blocks of 64 dims 16 KB apart (the leading offset), 16 tokens 2 KB
    const uint64_t dv0 = umma_desc(smem_u32(sv)) - (1ull << 16) + ((uint64_t)(16384 >> 4) << 16);
    auto scores = [&](int step) {
      const int st = step & 1;
      const uint32_t phase = (uint32_t)(step >> 1) & 1u;
      if (!wait(k_full(st), phase) || !wait(s_empty(st), phase ^ 1u)) return;
      tc_fence_after();
      const uint32_t el = elect_one(), acc = tmem + 64 * st, idesc = IDESC | (64u >> 3 << 17);
      const uint64_t dk = dk0 + (uint64_t)(st * NC * 1024);
      // The small products first: what is added to an accumulator is cut off at its last bit, so each addition to a large one costs half of that (with all
      // three of a k together the error of 5 prompts of 333 tokens was 1.4e-6).
#pragma unroll
      for (int k = 0; k < 8 * NC; ++k) {   // 16 halves are two descriptor units of 16 bytes
        const int kk = k % (4 * NC);
        const uint64_t aq = dq + (uint64_t)((kk >> 2) * 2048 + 2 * (kk & 3)), ak = dk + (uint64_t)((kk >> 2) * 1024 + 2 * (kk & 3));
        if (k < 4 * NC) {
          umma_bf16(acc, aq + 1024, ak, idesc, k > 0 ? 1u : 0u, el);   // (fp16: the kind's types are the descriptor's)
          umma_bf16(acc, aq, ak + 512, idesc, 1u, el);
        } else {
          umma_bf16(acc, aq, ak, idesc, 1u, el);
        }
      }
      umma_commit(k_empty(st), el);
      umma_commit(s_full(st), el);
      if (el) mbar_arrive(s_full(st));
      __syncwarp();
    };
    if (steps && wait(q_full, 0)) scores(0);
    for (int step = 0; step < steps && ok; ++step) {
      if (step + 1 < steps) scores(step + 1);
      const int st = step & 1;
      if (!wait(v_full(st), (uint32_t)(step >> 1) & 1u) || !wait(p_full, (uint32_t)step & 1u)) break;
      tc_fence_after();
      const int groups = (t1 - t0 - 64 * step + 15) / 16;
      const uint32_t el = elect_one(), idesc = IDESC | (1u << 16) | ((uint32_t)(D >> 3) << 17);
      const uint64_t dv = dv0 + (uint64_t)(st * NC * 1024);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int kk = k % 4;
        if (kk >= groups) continue;
        const uint32_t p = tmem + COL_P + 64 * st + 8 * kk;
        if (k < 4) {
          umma_bf16_ts(tmem + COL_O, p + 32, dv + 128 * kk, idesc, k > 0 ? 1u : 0u, el);
          umma_bf16_ts(tmem + COL_O, p, dv + 512 + 128 * kk, idesc, 1u, el);
        } else {
          umma_bf16_ts(tmem + COL_O, p, dv + 128 * kk, idesc, 1u, el);
        }
      }
      umma_commit(v_empty(st), el);
      umma_commit(o_full, el);
      if (el) mbar_arrive(o_full);
      __syncwarp();
    }
  } else {
    // ---------------- softmax ----------------
    convert_q();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_full);
    asm volatile("bar.sync 6, 256;" ::: "memory");   // rows' factors
    const float factor = qfactor[row];
    for (int step = 0; step < steps; ++step) {
      const int base = t0 + 64 * step, st = step & 1;
      uint32_t x[32];
      float top = -INFINITY, f = 0.0f;
      if (wait(s_full(st), (uint32_t)(step >> 1) & 1u)) {
        tc_fence_after();
        const unsigned there = theres[step & 3];
        f = fmaxf(factor * downs[step & 3], 1.17549435e-38f);   // (positive: it multiplies infinities)
        // a score is off by no more than 2^-3 f for the last bits of keys: as many of them as are too few matter only where scores may be millions
        if (wide[step & 3] >> NC & 1 && f > 0x1p-17f && sees > 0) uneven = 1;
        tmem_ld16(tlane + 64 * st + 32 * hf, x);
        tmem_ld16(tlane + 64 * st + 32 * hf + 16, x + 16);
        tmem_ld_wait();
        const bool hidden = base + 64 > least || base + 64 > t1 || there != 15u;   // some row does not see some token
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_empty(st));
        if (hidden) {
          keep_branch();
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (base + 32 * hf + e >= sees || !(there >> (2 * hf + e / 16) & 1)) x[e] = __float_as_uint(-INFINITY);
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) top = fmaxf(top, __uint_as_float(x[e]));
        red[st][hf][row] = top;
      }
      asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory");   // warps quad and quad + 4
      if (!ok) continue;
      // P is p times 2^size, so that beside the row's largest it has the bits that it counts for.  (From scores of some millions on, which leave no room for
      // that and give one token all of p, without; and ref is rounded upwards, for then only a part of 14 can be taken off.)
      const float most = fmaxf(red[st][0][row], red[st][1][row]) * f;
      const int exponent = fabsf(most) < 0x1p22f ? size[step & 3] : 0;
      top = fmaxf(run_max, most + (float)exponent);
      const float ref = top == -INFINITY ? 0.0f : __fsub_ru(top, K3_LIFT), less = (float)exponent - ref;
      const float corr = exp2_fast(run_ref - ref);
      run_max = top;
      run_ref = top == -INFINITY ? top : ref;
      float sum = 0.0f;
      // (this block of P was read two steps ago, whose outputs have been taken)
#pragma unroll
      for (int e0 = 0; e0 < 16; e0 += 8) {
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = exp2_fast(fmaf(__uint_as_float(x[2 * (e0 + e)]), f, less)), z = exp2_fast(fmaf(__uint_as_float(x[2 * (e0 + e) + 1]), f, less));
          sum += y + z;
          hi[e] = pack_half(y, z);
          lo[e] = pack_half_lo(y, z, hi[e]);
        }
        tmem_st8(tlane + COL_P + 64 * st + 16 * hf + e0, hi);   // token k in half k % 2 of column k / 2
        tmem_st8(tlane + COL_P + 64 * st + 32 + 16 * hf + e0, lo);
      }
      run_sum = fmaf(run_sum, corr, sum * __uint_as_float((uint32_t)(127 - exponent) << 23));
      if (step > 0) {
        if (!wait(o_full, (uint32_t)(step - 1) & 1u)) continue;
        tc_fence_after();
        take_outputs(step - 1);
      }
      const float up = ups[step & 3][NC == 1 ? 0 : hf] * __uint_as_float((uint32_t)(127 + exponent) << 23);
      lifted = corr * (up * run_down);
      run_down = inverse_power(up);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
    }
    if (steps && wait(o_full, (uint32_t)(steps - 1) & 1u)) {
      tc_fence_after();
      take_outputs(steps - 1);
    }
  }
  if (lost_bits > 0.0f)
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      float most = 0.0f;
#pragma unroll
      for (int e = 0; e < 32; ++e) most = fmaxf(most, fabsf(o[32 * k + e]));
      if (most > 0.0f && lost_bits > 0x1p-19f * most && sees > 0) uneven = 1;   // (zero: all of these dims' values are)
    }
  tc_fence_before();
  const bool failed = __syncthreads_or(!ok);
  if (uneven && !failed) kv4_prompt_plainly<NC, Q41>(a, seq, b, head, rt, part, reinterpret_cast<float *>(sq));

  // rows go out by way of shared memory (all products have been read): 32 dims of 128 rows are 16 KB
  const bool rows_warp = warp < K3_SOFTMAX;
  if (rows_warp) red[0][hf][row] = run_sum;
  unsigned char *const so = sq;
  const bool writes = !failed && !uneven;
  if (writes && rows_warp)
#pragma unroll
    for (int e = 0; e < HALF; e += 4)
      *reinterpret_cast<float4 *>(so + (hf * NC + e / 32) * 16384 + k3_at(row, e % 32 / 4)) =
          make_float4(o[e] * run_down, o[e + 1] * run_down, o[e + 2] * run_down, o[e + 3] * run_down);
  __syncthreads();
  if (warp < 4) {
    const float sum = red[0][0][row] + red[0][1][row];
    red[1][0][row] = a.parts > 1 ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
    if (a.parts > 1 && writes && r0 + row < count) {
      float *dst = a.part + out_at[row] + D;
      dst[0] = run_ref;   // (what outputs and sum are relative to)
      dst[1] = sum;
    }
  }
  __syncthreads();
  if (writes && rows_warp) {
    constexpr int LANES = D / 4, ROWS = 32 / LANES;
    const int piece = lane % LANES;
    const bool wide = a.parts == 1 && ((uintptr_t)a.out & 15) == 0;
#pragma unroll 4
    for (int i = 0; i < 16 / ROWS; ++i) {
      const int out_row = warp * 16 + i * ROWS + lane / LANES;
      if (r0 + out_row >= count) continue;
      float4 x = *reinterpret_cast<const float4 *>(so + piece / 8 * 16384 + k3_at(out_row, piece % 8));
      const float scale = red[1][0][out_row];
      x.x *= scale; x.y *= scale; x.z *= scale; x.w *= scale;
      float *dst = (a.parts == 1 ? a.out : a.part) + out_at[out_row] + 4 * piece;
      if (wide) *reinterpret_cast<float4 *>(dst) = x;
      else { dst[0] = x.x; dst[1] = x.y; dst[2] = x.z; dst[3] = x.w; }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS) : "memory");
  }
}

// ---- one row a sequence and key head ---------------------------------------------------------------
// Whole numbers: codes - 8, sixteen times, are signed bytes (a mask and an exclusive or, where fp16 needs an addition besides), the other operand is
// a fixed-point number of 31 bits in four signed bytes, each a column of its own: column 4 (block % 2) + j of the first product is digit j of q in that
// block, zero for the other block, so that one accumulator gathers two blocks for 16 tokens and each lane scales the sums of one; in the second product
// (32 tokens) it is digit j of p d, times a power of two that a group's largest p d of that block leaves room for.  Sums are exact; they start at the integer that is 1.5 * 2^23 as a float, and so need no conversion.  A score
// ends up in one lane (64 tokens: two registers a lane), so softmax and p d are not computed eight times over as by rows that are not there.
// What it is bound by: instructions, then HBM.  (256 x 25 heads x 768 tokens: 139 us with fp16 operands, 261 instructions for 16 tokens of 64 dims.)
constexpr int K1_MAGIC = 0x4b400000;
constexpr float K1_MAGIC_F = 12582912.0f;

// the same from a first sum of K1_MAGIC, which stays in registers of its own
__device__ __forceinline__ void mma_16832_first(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, int first) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(first));
}
__device__ __forceinline__ void mma_16832(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 (code - 8) of the low (high) four bits of each byte
__device__ __forceinline__ uint32_t bytes_lo(uint32_t w) { return (w << 4 & 0xf0f0f0f0u) ^ 0x80808080u; }
__device__ __forceinline__ uint32_t bytes_hi(uint32_t w) { return (w & 0xf0f0f0f0u) ^ 0x80808080u; }
// sum times a power of two w, neg = -K1_MAGIC_F * w: exact
__device__ __forceinline__ float sum_times(int c, float w, float neg) { return fmaf(__int_as_float(c), w, neg); }
// byte `digit` (as a selector of two words' such bytes) of four numbers below 2^30 in signed base 256
__device__ __forceinline__ uint32_t digits_of(float x0, float x1, float x2, float x3, uint32_t pick) {
  const uint32_t u0 = (uint32_t)__float2int_rn(x0) + 0x80808080u, u1 = (uint32_t)__float2int_rn(x1) + 0x80808080u;
  const uint32_t u2 = (uint32_t)__float2int_rn(x2) + 0x80808080u, u3 = (uint32_t)__float2int_rn(x3) + 0x80808080u;
  return __byte_perm(__byte_perm(u0, u1, pick), __byte_perm(u2, u3, pick), 0x5410) ^ 0x80808080u;
}
template <int NC, bool Q41, bool WIDE>   // WIDE: pages hold 64 tokens or more
__global__ void __launch_bounds__(K1_WARPS * 32) kv4_attention_row_kernel(const Kv4AttnArgs a) {
  constexpr int NB = 2 * NC, D = 64 * NC, PART = (Q41 ? 10 : 9) * D, TILE = 2 * PART;
  constexpr int STAGE = 4 * TILE;
  __shared__ float sm[K1_WARPS], sl[K1_WARPS];
  __shared__ uint64_t bars[K1_WARPS][2];
  __shared__ int gave_up[K1_WARPS];
  extern __shared__ __align__(128) uint8_t ring[];   // two stages a warp; behind the last group, the warps' sums
  pdl_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int share = a.warps, first_warp = warp / share * share;
  int64_t u = (int64_t)blockIdx.x * (K1_WARPS / share) + warp / share;
  const int64_t unit = u;
  const int part = (int)(u % a.parts); u /= a.parts;
  const int head = (int)(u % a.s.kv_heads);
  const int64_t b = u / a.s.kv_heads;
  Kv4Seq seq = {0, 0, 0};
  if (b < a.batch) seq = kv4_seq(a, (int)b, lane == 0 && warp == first_warp && part == 0 && head == 0);
  const int t0 = part * a.part_tokens, t1 = seq.count ? min(seq.length, t0 + a.part_tokens) : 0;
  const bool live = seq.count && (t0 < t1 || part == 0);

  float run_max = -INFINITY, run_sum = 0.0f;   // the row's; of this lane's tokens
  float off[NC];                               // Q4_1: sum of p (m + 8 d), block g / 4 of a pair, this lane's tokens
  float o[NC][2][4];                           // columns 2t, 2t + 1 (digits of block t / 2) of dims 4 g + {0 | 1} and 4 g + {2 | 3}
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    off[c] = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) o[c][i >> 2][i & 3] = 0.0f;
  }
  const uint32_t pick = (uint32_t)(g & 3) | (uint32_t)(4 + (g & 3)) << 4;
  const float w0 = t & 1 ? 65536.0f : 1.0f, w1 = 256.0f * w0, neg0 = -K1_MAGIC_F * w0;

  const int first = t0 + (warp - first_warp) * K4_GROUP, step = share * K4_GROUP;
  uint8_t *const mine = ring + warp * 2 * STAGE;
  bool ok = true;   // the copies came
  if (live && first < t1) {
    // A stage is 64 tokens.  Lanes 0 to 3 have a tile each; of pages that hold them all, lane 0 copies what there is at once.  A tile that
    // cannot be followed is left out and counts for nothing.
    const uint32_t bar = smem_u32(&bars[warp][0]), dst = smem_u32(mine);
    if (lane == 0) {
      mbar_init(bar, 1);
      mbar_init(bar + 8, 1);
      gave_up[warp] = 0;
      fence_proxy_async();
    }
    __syncwarp();
    const int *table = a.table + b * a.max_pages;
    const int64_t page_bytes = kv4_page_bytes(a.s);
    const int tile_shift = a.s.page == 16 ? 0 : a.s.page == 32 ? 1 : a.s.page == 64 ? 2 : 3;   // tiles of a page, log2
    const uint8_t *of_head = a.pool + (int64_t)(head << tile_shift) * TILE;
    auto page_at = [&](int base) {
      if (WIDE) return base < t1 ? table[base >> (4 + tile_shift)] : -1;
      return lane < 4 && base + 16 * lane < t1 ? table[((base >> 4) + lane) >> tile_shift] : -1;
    };
    auto issue = [&](int base, int id, int stage) -> unsigned {
      if (WIDE) {   // (one page; the id is every lane's)
        const bool good = kv4_page_ok(a.s, id);
        const int tiles = good ? min(4, (t1 - base + 15) >> 4) : 0;
        if (lane == 0) {
          mbar_expect_tx(bar + 8 * stage, tiles * TILE);
          if (good) bulk_load(dst + stage * STAGE, of_head + id * page_bytes + ((base >> 4) & ((1 << tile_shift) - 1)) * TILE, tiles * TILE, bar + 8 * stage);
          else report_bad_index(a.status, 46, id);
        }
        return (1u << tiles) - 1u;
      }
      const bool wanted = lane < 4 && base + 16 * lane < t1, good = wanted && kv4_page_ok(a.s, id);
      if (wanted && !good) report_bad_index(a.status, 46, id);
      const unsigned there = __ballot_sync(0xffffffffu, good);
      if (!there) {
        if (lane == 0) mbar_arrive(bar + 8 * stage);
        return 0;
      }
      if (lane == 0) mbar_expect_tx(bar + 8 * stage, __popc(there) * TILE);
      __syncwarp();
      if (good) bulk_load(dst + stage * STAGE + lane * TILE, of_head + id * page_bytes + (((base >> 4) + lane) & ((1 << tile_shift) - 1)) * TILE, TILE, bar + 8 * stage);
      return there;
    };
    unsigned there_now = issue(first, page_at(first), 0), there_next = 0;
    if (first + step < t1) there_next = issue(first + step, page_at(first + step), 1);
    int id_next = page_at(first + 2 * step);

    // q's digits: this lane's column; dims 8 t + {0, 2, 4, 6} and {1, 3, 5, 7} of a block
    uint32_t qb[NC][2][2];   // [pair][block of it][dims]
    float qsum[NC], factor;
    {
      const float *q = a.q + seq.first * a.ldq + (int64_t)head * D + 8 * t + 32 * (g >> 2);
      float x[NC][8], top = 0.0f;
      bool finite = true;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[c][j] = q[64 * c + j];
          top = fmaxf(top, fabsf(x[c][j]));
          finite &= fabsf(x[c][j]) < INFINITY;
        }
      top = warp_max(top);
      const float up = to_top(top, 29);
      factor = __all_sync(0xffffffffu, finite) ? a.scale * 1.4426950408889634f * (0.0625f / up) : NAN;   // (conversions would lose a NaN)
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[c][j] *= up;
          sum += x[c][j];
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        sum = __shfl_sync(0xffffffffu, sum, 16 * (t >> 1)) * 16.0f;
        qsum[c] = t & 1 ? 0.0f : sum;   // (two lanes have a block)
        const uint32_t d0 = digits_of(x[c][0], x[c][2], x[c][4], x[c][6], pick), d1 = digits_of(x[c][1], x[c][3], x[c][5], x[c][7], pick);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          qb[c][k][0] = (g >> 2) == k ? d0 : 0u;
          qb[c][k][1] = (g >> 2) == k ? d1 : 0u;
        }
      }
    }
    const int k_scale = 8 * D + ((g >> 1) * NB + (t >> 1)) * 8, v_scale = PART + 8 * D + (t * NB + (g >> 2)) * 8;
    int stage = 0, base = first;
    uint32_t phase = 0;
    for (; base < t1; base += step) {
      ok = mbar_wait(bar + 8 * stage, phase, &gave_up[warp]);
      if (!ok) break;
      const uint8_t *tiles = mine + stage * STAGE;
      const unsigned there = there_now;
      uint2 vd[4][NC], vm[4][NC];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          vd[i][c] = *reinterpret_cast<const uint2 *>(tiles + i * TILE + v_scale + c * 16);
          if (Q41) vm[i][c] = *reinterpret_cast<const uint2 *>(tiles + i * TILE + v_scale + D + c * 16);
        }
      // scores: tokens g and g + 8 of each tile, this lane's digits and blocks
      float x[4][2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i][0] = x[i][1] = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          int acc[4];
          const uint4 w = *reinterpret_cast<const uint4 *>(tiles + i * TILE + c * 512 + lane * 16);   // tokens g (x, y) and g + 8 (z, w); even and odd block
          const uint32_t a0[4] = {bytes_lo(w.x), bytes_lo(w.z), bytes_hi(w.x), bytes_hi(w.z)};
          const uint32_t a1[4] = {bytes_lo(w.y), bytes_lo(w.w), bytes_hi(w.y), bytes_hi(w.w)};
          mma_16832_first(acc, a0, qb[c][0][0], qb[c][0][1], K1_MAGIC);
          mma_16832(acc, a1, qb[c][1][0], qb[c][1][1]);
          const uint2 kd = *reinterpret_cast<const uint2 *>(tiles + i * TILE + k_scale + c * 16);
          const float2 d = half_pair(__byte_perm(kd.x, kd.y, g & 1 ? 0x7632 : 0x5410));
          x[i][0] = fmaf(d.x, fmaf(__int_as_float(acc[1]) - K1_MAGIC_F, w1, sum_times(acc[0], w0, neg0)), x[i][0]);
          x[i][1] = fmaf(d.y, fmaf(__int_as_float(acc[3]) - K1_MAGIC_F, w1, sum_times(acc[2], w0, neg0)), x[i][1]);
          if (Q41) {
            const uint2 km = *reinterpret_cast<const uint2 *>(tiles + i * TILE + k_scale + D + c * 16);
            const float2 m = half_pair(__byte_perm(km.x, km.y, g & 1 ? 0x7632 : 0x5410));
            x[i][0] = fmaf(fmaf(8.0f, d.x, m.x), qsum[c], x[i][0]);
            x[i][1] = fmaf(fmaf(8.0f, d.y, m.y), qsum[c], x[i][1]);
          }
        }
      }
      // summed over the four lanes, which keep a tile each
      float sc[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bool up2 = t & 2, up1 = t & 1;
        const float y0 = (up2 ? x[2][e] : x[0][e]) + __shfl_xor_sync(0xffffffffu, up2 ? x[0][e] : x[2][e], 2);
        const float y1 = (up2 ? x[3][e] : x[1][e]) + __shfl_xor_sync(0xffffffffu, up2 ? x[1][e] : x[3][e], 2);
        const float z = (up1 ? y1 : y0) + __shfl_xor_sync(0xffffffffu, up1 ? y0 : y1, 1);
        sc[e] = z * factor;
      }
      if (base + K4_GROUP > t1 || there != 15u) {
        // what stands behind the last token may be anything: it has no score, and its values' scales are none
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (base + 16 * t + g + 8 * e >= t1 || !(there >> t & 1)) sc[e] = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = base + 16 * i + 2 * t;
          const bool ok = there >> i & 1;
          const uint32_t keep0 = (ok && at < t1 ? 0xffffu : 0u) | (ok && at + 1 < t1 ? 0xffff0000u : 0u);
          const uint32_t keep1 = (ok && at + 8 < t1 ? 0xffffu : 0u) | (ok && at + 9 < t1 ? 0xffff0000u : 0u);
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            vd[i][c].x &= keep0;
            vd[i][c].y &= keep1;
            if (Q41) { vm[i][c].x &= keep0; vm[i][c].y &= keep1; }
          }
        }
      }
      const float top = fmaxf(run_max, warp_max(fmaxf(sc[0], sc[1])));
      const float ref = top == -INFINITY ? 0.0f : top;
      const float corr = exp2_fast(run_max - ref);
      run_max = top;
      sc[0] = exp2_fast(sc[0] - ref);
      sc[1] = exp2_fast(sc[1] - ref);
      run_sum = fmaf(run_sum, corr, sc[0] + sc[1]);
      float p[4][4];   // tokens 2t, 2t + 1, 2t + 8, 2t + 9 of each tile
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        p[i][0] = __shfl_sync(0xffffffffu, sc[0], 8 * t + i);
        p[i][1] = __shfl_sync(0xffffffffu, sc[0], 8 * t + 4 + i);
        p[i][2] = __shfl_sync(0xffffffffu, sc[1], 8 * t + i);
        p[i][3] = __shfl_sync(0xffffffffu, sc[1], 8 * t + 4 + i);
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        float pd[4][4], most = 0.0f, add = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 d01 = half_pair(vd[i][c].x), d23 = half_pair(vd[i][c].y);
          if (Q41) {
            const float2 m01 = half_pair(vm[i][c].x), m23 = half_pair(vm[i][c].y);
            add = fmaf(p[i][0], fmaf(8.0f, d01.x, m01.x), add);
            add = fmaf(p[i][1], fmaf(8.0f, d01.y, m01.y), add);
            add = fmaf(p[i][2], fmaf(8.0f, d23.x, m23.x), add);
            add = fmaf(p[i][3], fmaf(8.0f, d23.y, m23.y), add);
          }
          pd[i][0] = p[i][0] * d01.x; pd[i][1] = p[i][1] * d01.y; pd[i][2] = p[i][2] * d23.x; pd[i][3] = p[i][3] * d23.y;
          most = max_abs_nan(most, pd[i][0], pd[i][1]);
          most = max_abs_nan(most, pd[i][2], pd[i][3]);
        }
        most = max_abs_nan(most, __shfl_xor_sync(0xffffffffu, most, 1), 0.0f);
        most = max_abs_nan(most, __shfl_xor_sync(0xffffffffu, most, 2), 0.0f);
        const float up = to_top_of(most, 29);
        uint32_t digits[4];   // of the four tiles
#pragma unroll
        for (int i = 0; i < 4; ++i) digits[i] = digits_of(pd[i][0] * up, pd[i][1] * up, pd[i][2] * up, pd[i][3] * up, pick);
        if (Q41) off[c] = fmaf(off[c], corr, add);
        int acc[2][4];
#pragma unroll
        for (int i = 0; i < 4; i += 2) {   // 32 tokens
          uint32_t bytes[2][4];            // of the lane's four tokens: dims 4 g + {0, 1} and {2, 3} of the even block, of the odd one
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint4 w = *reinterpret_cast<const uint4 *>(tiles + (i + h) * TILE + PART + c * 512 + lane * 16);
            const uint32_t e0 = __byte_perm(w.x, w.y, 0x5140), e1 = __byte_perm(w.z, w.w, 0x5140);
            const uint32_t o0 = __byte_perm(w.x, w.y, 0x7362), o1 = __byte_perm(w.z, w.w, 0x7362);
            bytes[h][0] = __byte_perm(e0, e1, 0x5410);
            bytes[h][1] = __byte_perm(e0, e1, 0x7632);
            bytes[h][2] = __byte_perm(o0, o1, 0x5410);
            bytes[h][3] = __byte_perm(o0, o1, 0x7632);
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t b0 = (g >> 2) == k ? digits[i] : 0u, b1 = (g >> 2) == k ? digits[i + 1] : 0u;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const uint32_t av[4] = {bytes_lo(bytes[0][2 * k + n]), bytes_hi(bytes[0][2 * k + n]), bytes_lo(bytes[1][2 * k + n]), bytes_hi(bytes[1][2 * k + n])};
              if (i == 0 && k == 0) mma_16832_first(acc[n], av, b0, b1, K1_MAGIC);
              else mma_16832(acc[n], av, b0, b1);
            }
          }
        }
        // (a scale that is not finite makes its block's values NaN, as it does in the formula)
        const float down = __shfl_sync(0xffffffffu, most < INFINITY ? 0.0625f * inverse_power(up) : NAN, 16 * (t >> 1));
        const float f0 = down * w0, f1 = down * w1, n0 = -K1_MAGIC_F * f0, n1 = -K1_MAGIC_F * f1;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[c][n][e] = fmaf(o[c][n][e], corr, sum_times(acc[n][e], e & 1 ? f1 : f0, e & 1 ? n1 : n0));
      }
      __syncwarp();   // the stage has been read
      there_now = there_next;
      if (base + 2 * step < t1) {
        there_next = issue(base + 2 * step, id_next, stage);
        id_next = page_at(base + 3 * step);
      }
      phase ^= stage;
      stage ^= 1;
    }
    if (!ok) {
      if (lane == 0) {
        atomicCAS(a.status, 0, DEV_WAIT_TIMEOUT);
        a.status[1] = 47;
      }
      ring_land(stage, phase, base + step < t1, [&](int s, uint32_t p) {   // (with a flag that nobody raises)
        mbar_wait_thread(bar + 8 * s, p, &gave_up[warp]);
      });
    }
  }

  // digits and lanes together: both lanes of a block get its four dims, one writes the first two, the other the last
  run_sum = warp_sum(run_sum);
  float2 r[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    float y[2][2];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        y[n][e] = o[c][n][2 * e] + o[c][n][2 * e + 1];
        y[n][e] += __shfl_xor_sync(0xffffffffu, y[n][e], 1);
      }
    r[c] = t & 1 ? make_float2(y[1][0], y[1][1]) : make_float2(y[0][0], y[0][1]);
    if (Q41) {
      off[c] += __shfl_xor_sync(0xffffffffu, off[c], 1);
      off[c] += __shfl_xor_sync(0xffffffffu, off[c], 2);
      const float add = __shfl_sync(0xffffffffu, off[c], 16 * (t >> 1));
      r[c].x += add;
      r[c].y += add;
    }
  }
  const int at = 32 * (t >> 1) + 4 * g + 2 * (t & 1);   // of a pair of blocks
  float top = run_max, sum = run_sum;
  if (share > 1) {
    float *so = reinterpret_cast<float *>(ring);   // [warp][D], each inside the warp's own stages
    constexpr int STRIDE = 2 * STAGE / (int)sizeof(float);
#pragma unroll
    for (int c = 0; c < NC; ++c) *reinterpret_cast<float2 *>(&so[warp * STRIDE + 64 * c + at]) = r[c];
    if (lane == 0) { sm[warp] = run_max; sl[warp] = run_sum; }
    if (__syncthreads_or(!ok)) return;   // (the block is one unit's; what did not come is nobody's output)
    if (warp != first_warp) return;
    for (int w = warp + 1; w < warp + share; ++w) top = fmaxf(top, sm[w]);
    const float ref = top == -INFINITY ? 0.0f : top;
    sum = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c) r[c] = make_float2(0.0f, 0.0f);
    for (int w = warp; w < warp + share; ++w) {
      const float e = exp2_fast(sm[w] - ref);
      sum = fmaf(sl[w], e, sum);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const float2 y = *reinterpret_cast<const float2 *>(&so[w * STRIDE + 64 * c + at]);
        r[c].x = fmaf(y.x, e, r[c].x);
        r[c].y = fmaf(y.y, e, r[c].y);
      }
    }
  }
  if (!live || !ok) return;
  float *dst = a.parts == 1 ? a.out + seq.first * a.heads * D + (int64_t)head * D : a.part + unit * (D + 2);
  const float scale = a.parts > 1 ? 1.0f : sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    dst[64 * c + at] = r[c].x * scale;
    dst[64 * c + at + 1] = r[c].y * scale;
  }
  if (a.parts > 1 && lane == 0) { dst[D] = top; dst[D + 1] = sum; }
}

// The parts of a row into one, a block a row: the parts' weights first, by threads over parts, then threads over dims.  Parts behind what the row's
// tile sees were not written.
constexpr int KJ_THREADS = 128;

__global__ void __launch_bounds__(KJ_THREADS) kv4_attention_join_kernel(const Kv4AttnArgs a) {
  __shared__ float weight[KJ_PARTS], red[2][KJ_THREADS / 32];
  pdl_enter();
  const int D = a.s.dim, tile_rows = a.tile_rows, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t tile = blockIdx.x / tile_rows;
  int64_t u = tile;
  const int rt = (int)(u % a.row_tiles); u /= a.row_tiles;
  const int head = (int)(u % a.s.kv_heads);
  const int b = (int)(u / a.s.kv_heads);
  const Kv4Seq seq = kv4_seq(a, b, false);
  const int count = seq.count * a.group, row = (int)(blockIdx.x % tile_rows), rr = rt * tile_rows + row;
  if (rr >= count) return;
  const int last = min(count, rt * tile_rows + tile_rows) - 1;
  const int most = max(0, seq.length - seq.count + last / a.group + 1);
  const int parts = max(1, (most + a.part_tokens - 1) / a.part_tokens);
  const int64_t step = (int64_t)tile_rows * (D + 2);
  const float *p = a.part + tile * a.parts * step + row * (D + 2);
  float top = -INFINITY;
  for (int k = tid; k < parts; k += KJ_THREADS) {
    weight[k] = p[k * step + D];
    top = fmaxf(top, weight[k]);
  }
  top = warp_max(top);
  if (lane == 0) red[0][warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < KJ_THREADS / 32; ++w) top = fmaxf(top, red[0][w]);
  const float ref = top == -INFINITY ? 0.0f : top;
  float sum = 0.0f;
  for (int k = tid; k < parts; k += KJ_THREADS) {
    const float e = exp2_fast(weight[k] - ref);
    weight[k] = e;
    sum = fmaf(p[k * step + D + 1], e, sum);
  }
  sum = warp_sum(sum);
  if (lane == 0) red[1][warp] = sum;
  __syncthreads();
  sum = 0.0f;
#pragma unroll
  for (int w = 0; w < KJ_THREADS / 32; ++w) sum += red[1][w];
  float *out = a.out + (seq.first + rr / a.group) * (int64_t)a.heads * D + (int64_t)(head * a.group + rr % a.group) * D;
  for (int j = tid; j < D; j += KJ_THREADS) {
    float x = 0.0f;
    int k = 0;
    for (; k + 8 <= parts; k += 8) {   // eight loads under way
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = p[(k + i) * step + j];
#pragma unroll
      for (int i = 0; i < 8; ++i) x = fmaf(y[i], weight[k + i], x);
    }
    for (; k < parts; ++k) x = fmaf(p[k * step + j], weight[k], x);
    out[j] = sum == 0.0f ? 0.0f : x / sum;
  }
}

static int kv4_plan(caten_b200_ctx *ctx, const char *who, const caten_b200_kv4_desc *c, int64_t batch, int64_t rows, int64_t max_new, int64_t max_length, Kv4Plan *p) {
  Kv4Shape s;
  if (int rc = kv4_check(ctx, who, c, &s)) return rc;
  if (batch < 0 || batch > (1 << 24) || rows < 0 || rows > 0x7fffffff || max_new <= 0 || max_length < 0 || max_length > 0x3fffffff) return fail(ctx, CATEN_B200_EINVAL, "%s: bad shape", who);
  if (max_new > (1 << 24) || max_new * (c->heads / c->kv_heads) > 0x3fffffff) return fail(ctx, CATEN_B200_EUNSUPPORTED, "%s: %lld new tokens of a sequence", who, (long long)max_new);
  if (!kv4_plan_of({c->dim, c->kv_heads, c->heads / c->kv_heads}, batch, rows, max_new, max_length, p)) return fail(ctx, CATEN_B200_EUNSUPPORTED, "%s: too many rows", who);
  return 0;
}

template <int NC, bool Q41>
static int kv4_attention_launch(caten_b200_ctx *ctx, const Kv4AttnArgs &a, int64_t units) {
  if (a.tile_rows == 1) {
    const int64_t per_block = K1_WARPS / a.warps;
    const int smem = K1_WARPS * 2 * 4 * kv4_tile_bytes(a.s);
    void (*kernel)(const Kv4AttnArgs) = a.s.page >= K4_GROUP ? kv4_attention_row_kernel<NC, Q41, true> : kv4_attention_row_kernel<NC, Q41, false>;
    if (smem > 48 << 10) CB_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    CB_CUDA(ctx, launch_k(ctx, kernel, dim3((unsigned)((units * a.parts + per_block - 1) / per_block)), dim3(K1_WARPS * 32), smem, a));
    CB_LAUNCH_CHECK(ctx, "kv4_attention_row_kernel");
  } else if (a.tile_rows == K2_ROWS) {
    const int64_t per_block = K2_WARPS / a.warps;
    const int smem = K2_WARPS * 2 * K4_TILES(NC) * kv4_tile_bytes(a.s);
    if (smem > 48 << 10) CB_CUDA(ctx, cudaFuncSetAttribute(kv4_attention_few_kernel<NC, Q41>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    CB_CUDA(ctx, launch_k(ctx, kv4_attention_few_kernel<NC, Q41>, dim3((unsigned)((units * a.parts + per_block - 1) / per_block)), dim3(K2_WARPS * 32), smem, a));
    CB_LAUNCH_CHECK(ctx, "kv4_attention_few_kernel");
  } else if (a.tile_rows == K3_ROWS) {
    if constexpr (NC <= 2) {
      const int smem = k3_smem(NC, kv4_tile_bytes(a.s));
      CB_CUDA(ctx, cudaFuncSetAttribute(kv4_attention_prompt_kernel<NC, Q41>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
      CB_CUDA(ctx, launch_k(ctx, kv4_attention_prompt_kernel<NC, Q41>, dim3((unsigned)(units * a.parts)), dim3(K3_THREADS), smem, a));
      CB_LAUNCH_CHECK(ctx, "kv4_attention_prompt_kernel");
    }
  } else {
    const bool shared = a.warps == 4;
    // (no less than the sums of all warps where they are joined)
    const int smem = k4_warps(shared) / a.warps * K4_TILES(NC) * (2 * kv4_tile_bytes(a.s) + (shared ? NC * (8 * 512 + (Q41 ? 4 : 2) * 32 * 4) : 0));
    void (*kernel)(const Kv4AttnArgs) = shared ? kv4_attention_kernel<NC, Q41, true> : kv4_attention_kernel<NC, Q41, false>;
    const int64_t blocks = units / a.row_tiles * ((a.row_tiles + a.warps - 1) / a.warps) * a.parts;
    if (smem > 48 << 10) CB_CUDA(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    CB_CUDA(ctx, launch_k(ctx, kernel, dim3((unsigned)blocks), dim3(k4_warps(shared) * 32), smem, a));
    CB_LAUNCH_CHECK(ctx, "kv4_attention_kernel");
  }
  if (a.parts == 1) return 0;
  CB_CUDA(ctx, launch_k(ctx, kv4_attention_join_kernel, dim3((unsigned)(units * a.tile_rows)), dim3(KJ_THREADS), 0, a));
  CB_LAUNCH_CHECK(ctx, "kv4_attention_join_kernel");
  return 0;
}

}  // namespace cb

using namespace cb;

extern "C" {

// Arguments are checked before the context is touched.
int64_t caten_b200_kv4_attention_work(const caten_b200_kv4_desc *desc, int64_t batch, int64_t rows, int64_t max_new, int64_t max_length) {
  Kv4Plan p;
  if (kv4_plan(nullptr, "kv4_attention_work", desc, batch, rows, max_new, max_length, &p)) return -1;
  return kv4_work_bound({desc->dim, desc->kv_heads, desc->heads / desc->kv_heads}, batch, max_new, max_length);
}

int64_t caten_b200_kv4_attention_call_work(const caten_b200_kv4_desc *desc, int64_t batch, int64_t rows, int64_t max_new, int64_t max_length) {
  Kv4Plan p;
  if (kv4_plan(nullptr, "kv4_attention_call_work", desc, batch, rows, max_new, max_length, &p)) return -1;
  return std::max<int64_t>(16, kv4_plan_bytes(p, desc->dim));
}

int caten_b200_kv4_attention(caten_b200_ctx *ctx, const caten_b200_kv4_desc *desc, const float *d_q, int64_t ldq, const void *d_pool, const int32_t *d_table,
                             int64_t max_pages, const int32_t *d_lengths, const int32_t *d_starts, int64_t batch, int64_t rows, int64_t max_new,
                             int64_t max_length, float *d_out, void *d_work) {
  Kv4Plan p;
  if (int rc = kv4_plan(ctx, "kv4_attention", desc, batch, rows, max_new, max_length, &p)) return rc;
  if (max_pages <= 0 || max_pages > 0x7fffffff || max_length > max_pages * desc->page)
    return fail(ctx, CATEN_B200_EINVAL, "kv4_attention: lengths up to %lld in tables of %lld pages of %d", (long long)max_length, (long long)max_pages, desc->page);
  if (!d_starts && (rows != batch || max_new != 1)) return fail(ctx, CATEN_B200_EINVAL, "kv4_attention: without starts every sequence has one row");
  if (ldq < (int64_t)desc->heads * desc->dim) return fail(ctx, CATEN_B200_EINVAL, "kv4_attention: ldq=%lld, rows have %lld values", (long long)ldq, (long long)desc->heads * desc->dim);
  if (batch && rows && (!d_q || !d_pool || !d_table || !d_lengths || !d_out || !d_work)) return fail(ctx, CATEN_B200_EINVAL, "kv4_attention: NULL argument");
  if (((uintptr_t)d_pool | (uintptr_t)d_work) % 16) return fail(ctx, CATEN_B200_EINVAL, "kv4_attention: pool and workspace have to start on a multiple of 16 bytes");
  if (((uintptr_t)d_q | (uintptr_t)d_out | (uintptr_t)d_table | (uintptr_t)d_lengths | (uintptr_t)d_starts) % 4) return fail(ctx, CATEN_B200_EINVAL, "kv4_attention: misaligned pointer");
  if (!ctx) return fail(nullptr, CATEN_B200_EINVAL, "kv4_attention: ctx is NULL");
  cudaSetDevice(ctx->device);
  ctx->work_outside = true;
  if (!batch || !rows) return 0;
  ProfScope prof(ctx, max_new == 1 ? CATEN_B200_K_ATTN_DECODE : CATEN_B200_K_ATTN_PREFILL);
  Kv4AttnArgs a = {};
  kv4_check(ctx, "kv4_attention", desc, &a.s);
  a.q = d_q; a.ldq = ldq; a.rows = rows;
  a.pool = (const uint8_t *)d_pool;
  a.table = d_table; a.lengths = d_lengths; a.starts = d_starts;
  a.out = d_out; a.part = (float *)d_work; a.status = ctx->d_status;
  a.heads = desc->heads; a.group = desc->heads / desc->kv_heads;
  a.max_pages = (int)max_pages; a.max_new = (int)max_new; a.max_length = (int)max_length; a.batch = (int)batch;
  a.tile_rows = p.tile_rows; a.warps = p.warps; a.row_tiles = p.row_tiles; a.parts = p.parts; a.part_tokens = p.part_tokens;
  a.scale = desc->scale;
  const bool q41 = a.s.q41;
  switch (desc->dim / 64) {
    case 1: return q41 ? kv4_attention_launch<1, true>(ctx, a, p.units) : kv4_attention_launch<1, false>(ctx, a, p.units);
    case 2: return q41 ? kv4_attention_launch<2, true>(ctx, a, p.units) : kv4_attention_launch<2, false>(ctx, a, p.units);
    case 3: return q41 ? kv4_attention_launch<3, true>(ctx, a, p.units) : kv4_attention_launch<3, false>(ctx, a, p.units);
    default: return q41 ? kv4_attention_launch<4, true>(ctx, a, p.units) : kv4_attention_launch<4, false>(ctx, a, p.units);
  }
}

}  // extern "C"
