// Paged 4-bit key/value cache: page tables and slots from request lengths, rows into the cache and back.  (Attention over it:
// kv4_attention.cu.)  No counterpart in the reference, whose cache is one fp32 array a layer (external/llm/layers.lisp:25-26).
#include "common.cuh"
#include "kv4.cuh"

namespace cb {

// ---- page tables and slots -------------------------------------------------------------------------
// Some thousand integers, so the launch, the chain of dependent loads and one SM's instructions are the time.  Lengths are read once, one scan
// gives every request's pages given back, pages taken and tokens before it, and decides whether the plan can be carried out (if not, nothing
// changes).  Then warps take pages, and tokens, of all requests side by side and find the request by bisection in shared memory: a warp that walked its
// requests one after another had their chains of loads in a row.  A token's page is read from where its request took it, not from the table, so
// slots wait for nothing that this kernel writes.  Few requests are one block; many are a cluster of eight, each of which scans for itself and moves an
// eighth of the pages (1000 requests, 21000 pages moved: 22 us of one SM, most of it instructions), and their slots go to a grid of their own.
constexpr int PG_MOST = 4096;     // slots that the first kernel writes itself
constexpr int PG_BLOCKS = 8;      // of the cluster

struct PagesArgs {
  const int *have, *want;
  int *table, *free, *state, *starts, *slots;
  int requests, page, max_pages, capacity, max_tokens;
};

__device__ __forceinline__ int pages_of(int tokens, int page) { return (int)(((unsigned)tokens + (unsigned)page - 1u) / (unsigned)page); }   // tokens >= 0

// last index i of [0, n) with at[i] <= x (at ascending, at[0] = 0)
__device__ __forceinline__ int last_not_above(const int *at, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (at[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <int THREADS, int BLOCKS>
__global__ void __launch_bounds__(THREADS) kv_pages_kernel(PagesArgs a, int own_slots) {
  __shared__ int warps[3][32];
  __shared__ long long total[3];   // tokens, pages taken, pages given back
  __shared__ int bad;
  __shared__ int at_give[THREADS], at_take[THREADS], at_token[THREADS], held_pages[THREADS], wanted_pages[THREADS], had[THREADS];
  pdl_enter();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, block = BLOCKS > 1 ? blockIdx.x : 0;   // (the cluster is the grid)
  auto sync_all = [] {
    if (BLOCKS > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    else __syncthreads();
  };
  if (tid < 3) total[tid] = 0;
  if (tid == 3) bad = 0;
  const int n_free = a.state[0];
  __syncthreads();
  int have = 0, want = 0;   // of the last request looked at: with one request a thread, or fewer, read once
  {
    long long t[3] = {0, 0, 0};
    bool wrong = false;
    for (int r = tid; r < a.requests; r += THREADS) {
      have = a.have[r];
      want = a.want[r];
      if (have < 0 || want < 0 || pages_of(have, a.page) > a.max_pages || pages_of(want, a.page) > a.max_pages) { wrong = true; continue; }
      const int d = pages_of(want, a.page) - pages_of(have, a.page);
      t[0] += want > have ? want - have : 0;
      t[1] += d > 0 ? d : 0;
      t[2] += d < 0 ? -d : 0;
    }
    if (wrong) bad = 1;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      for (int o = 16; o > 0; o >>= 1) t[k] += __shfl_xor_sync(0xffffffffu, t[k], o);
      if (lane == 0 && t[k]) atomicAdd((unsigned long long *)&total[k], (unsigned long long)t[k]);
    }
  }
  __syncthreads();
  const long long missing = total[1] - total[2] - n_free;
  int why = bad;                                                                       // 1: lengths that do not fit
  if (!why && total[0] > a.max_tokens) why = 2;                                        // more tokens than slots
  if (!why && (n_free < 0 || n_free + total[2] > a.capacity)) why = 3;                 // a free list that was not this pool's
  const bool go = !why && missing <= 0;
  if (BLOCKS > 1) sync_all();   // every block has read the state
  if (tid == 0 && block == 0) {
    a.state[1] = go ? (int)total[0] : 0;
    a.state[2] = !why && missing > 0 ? (int)(missing < 0x7fffffff ? missing : 0x7fffffff) : 0;
    a.state[3] = why;
    if (go) a.state[0] = (int)(n_free + total[2] - total[1]);
  }
  if (!go) {
    for (int r = tid; block == 0 && r <= a.requests; r += THREADS) a.starts[r] = 0;
    for (int i = tid; block == 0 && own_slots && i < a.max_tokens; i += THREADS) a.slots[i] = -1;
    return;
  }
  const int top = (int)(n_free + total[2]);
  // work(i, the request that item i is of), items 0 .. count of n requests of which at[] are the first ones': a warp has items side by side, so that it
  // looks for a request once and walks on from there
  auto for_items = [&](const int *at, int n, int count, auto get, auto put) {
    const int each = (count + THREADS * BLOCKS - 1) / (THREADS * BLOCKS) * 32, nth = block * (THREADS / 32) + warp, end = min(count, (nth + 1) * each);
    int i = nth * each + lane;
    if (i >= end) return;
    for (int q = last_not_above(at, n, i); i < end; i += 4 * 32) {   // four loads under way
      int of[4], x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + 32 * e < end) {
          while (q + 1 < n && at[q + 1] <= i + 32 * e) ++q;
          of[e] = q;
          x[e] = get(i + 32 * e, q);
        }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (i + 32 * e < end) put(i + 32 * e, of[e], x[e]);
    }
  };
  // THREADS requests at a time.  Two rounds, because a page that one request gives back may be the one that another takes: the first appends the
  // pages given back to the free ones, in the order of requests and of their pages; the second takes from the end.
  for (int round = total[2] ? 0 : 1; round < 2; ++round) {
    int carry[3] = {0, 0, 0};
    for (int base = 0; base < a.requests; base += THREADS) {
      const int r = base + tid, n = min(THREADS, a.requests - base);
      if (a.requests > THREADS) {
        have = r < a.requests ? a.have[r] : 0;
        want = r < a.requests ? a.want[r] : 0;
      }
      const int held = pages_of(have, a.page), wanted = pages_of(want, a.page);
      int v[3] = {max(0, held - wanted), max(0, wanted - held), max(0, want - have)}, sum[3];
      int inc[3];
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        inc[k] = v[k];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, inc[k], o);
          if (lane >= o) inc[k] += up;
        }
      }
      __syncthreads();   // the arrays of the requests before have been read
#pragma unroll
      for (int k = 0; k < 3; ++k)
        if (lane == 31) warps[k][warp] = inc[k];
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        int w = lane < THREADS / 32 ? warps[k][lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, w, o);
          if (lane >= o) w += up;
        }
        sum[k] = __shfl_sync(0xffffffffu, w, 31);
        const int before = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
        v[k] = inc[k] - v[k] + (warp ? before : 0);
      }
      at_give[tid] = v[0];
      at_take[tid] = v[1];
      at_token[tid] = v[2];
      held_pages[tid] = held;
      wanted_pages[tid] = wanted;
      had[tid] = have;
      __syncthreads();
      if (round == 0) {
        auto cell = [&](int i, int q) { return a.table + (long long)(base + q) * a.max_pages + wanted_pages[q] + i - at_give[q]; };
        for_items(at_give, n, sum[0], [&](int i, int q) { return *cell(i, q); },
                  [&](int i, int q, int id) {
                    a.free[n_free + carry[0] + i] = id;
                    *cell(i, q) = -1;
                  });
      } else {
        if (block == 0 && r < a.requests) a.starts[r] = carry[2] + v[2];
        for_items(at_take, n, sum[1], [&](int i, int) { return a.free[top - 1 - carry[1] - i]; },
                  [&](int i, int q, int id) { a.table[(long long)(base + q) * a.max_pages + held_pages[q] + i - at_take[q]] = id; });
        if (own_slots)
          for_items(at_token, n, sum[2],
                    [&](int i, int q) {
                      const int pos = had[q] + i - at_token[q], nth = (unsigned)pos / (unsigned)a.page;
                      const int id = nth < held_pages[q] ? a.table[(long long)(base + q) * a.max_pages + nth] : a.free[top - 1 - carry[1] - at_take[q] - (nth - held_pages[q])];
                      return id >= 0 && id < a.capacity ? id * a.page + pos - nth * a.page : -1;
                    },
                    [&](int i, int, int slot) { a.slots[carry[2] + i] = slot; });
      }
#pragma unroll
      for (int k = 0; k < 3; ++k) carry[k] += sum[k];
    }
    if (round == 0) sync_all();   // pages given back are there
  }
  if (block) return;
  if (tid == 0) a.starts[a.requests] = (int)total[0];
  for (int i = (int)total[0] + tid; own_slots && i < a.max_tokens; i += THREADS) a.slots[i] = -1;
}

// The slots of a finished plan, four tokens a thread.
__global__ void __launch_bounds__(256) kv_slots_kernel(PagesArgs a) {
  pdl_enter();
  const int i0 = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (i0 >= a.max_tokens) return;
  const int added = a.state[1];
  int r = i0 < added ? last_not_above(a.starts, a.requests, i0) : a.requests;
  int slot[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    slot[e] = -1;
    if (i0 + e < added) {
      while (r + 1 < a.requests && a.starts[r + 1] <= i0 + e) ++r;   // (requests without new tokens are passed over)
      const int pos = a.have[r] + i0 + e - a.starts[r], nth = (unsigned)pos / (unsigned)a.page;
      const int id = a.table[(long long)r * a.max_pages + nth];
      if (id >= 0 && id < a.capacity) slot[e] = id * a.page + pos - nth * a.page;
    }
  }
  if (i0 + 4 <= a.max_tokens && (uintptr_t)a.slots % 16 == 0) *reinterpret_cast<int4 *>(a.slots + i0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
  else
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i0 + e < a.max_tokens) a.slots[i0 + e] = slot[e];
}

// ---- rows into the cache ---------------------------------------------------------------------------
// A block of 32 values is eight lanes' float4.  Codes are those of the GGUF formats: Q4_0  d = (value of largest magnitude) / -8,
// code = min(15, trunc(x / d + 8.5)); Q4_1  d = (max - min) / 15, code = min(15, trunc((x - min) / d + 0.5)).  Which code is nearest, and which half d
// rounds to (half a step: 2^-11; the formats hold halves), is decided exactly: in fp32, whose error in a code is below 6e-6 here, and in 64 bits for the
// few blocks in which a quotient is within 1e-5 of a border or d's last bits next to one of fp16's.  Where d or the minimum is not finite in fp16
// (a value that is not, or one beyond fp16's reach), the scale is NaN: a block is what it stands for, or NaN in all of its values.
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float min_nan(float a, float b) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }

__device__ __noinline__ uint32_t kv4_codes_exactly(float4 x, double d, double low, double offset, bool none, uint32_t without) {
  const float v[4] = {x.x, x.y, x.z, x.w};
  uint32_t codes = 0;
  for (int i = 0; i < 4; ++i) codes |= (uint32_t)min(15, max(0, (int)(((double)v[i] - low) / d + offset))) << (4 * i);
  return none ? without : codes;
}

// this lane's four values of a block that eight consecutive lanes hold -> four codes (low bits first), scale and minimum
template <bool Q41>
__device__ __forceinline__ uint32_t kv4_quantise(float4 x, __half *scale, __half *minimum) {
  constexpr float MAGIC = 12582912.0f;   // 1.5 * 2^23: added, it leaves the nearest whole number in the low bits
  const float v[4] = {x.x, x.y, x.z, x.w};
  float hi = max_nan(max_nan(v[0], v[1]), max_nan(v[2], v[3])), lo = min_nan(min_nan(v[0], v[1]), min_nan(v[2], v[3]));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
  }
  float d, base;
  bool exactly = false;
  if (Q41) {
    base = lo;
    // (hi - lo) / 15 with the difference's own rounding error (Knuth's two-sum) and the quotient's remainder taken back in
    const float r = hi - lo, back = r - hi, err = (hi - (r - back)) - (lo + back);
    const float q = r * (1.0f / 15.0f);
    d = fmaf(fmaf(-15.0f, q, r) + err, 1.0f / 15.0f, q);
  } else {
    base = 0.0f;
    const bool both = hi == -lo;   // equal magnitudes: the first one's sign (rare, and by the whole warp)
    float m = hi > -lo ? hi : lo;
    if (__any_sync(0xffffffffu, both && hi > 0.0f)) {
      int at = 32;
#pragma unroll
      for (int i = 3; i >= 0; --i)
        if (fabsf(v[i]) == hi) at = (threadIdx.x & 7) * 4 + i;
      int first = at;
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
      float mine = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (first == (int)(threadIdx.x & 7) * 4 + i) mine = v[i];
      const float sign = __shfl_sync(0xffffffffu, mine, (threadIdx.x & 24) + (first & 31) / 4);
      if (both) m = sign;
    }
    if (!(hi >= lo)) m = hi + lo;   // (NaN)
    d = m / -8.0f;
  }
  const uint32_t bits = __float_as_uint(d) & 0x7fffffffu;
  // next to a border between halves, or where halves are subnormal
  if (Q41) exactly = bits < 0x38800000u || (uint32_t)((int)(bits & 0x1fffu) - 0x1000 + 2) <= 4u;
  float inverse;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(d));
  uint32_t codes = 0;
#pragma unroll
  for (int i = 3; i >= 0; --i) {
    const float y = fminf(Q41 ? (v[i] - base) * inverse : fmaf(v[i], inverse, 8.0f), 15.25f), t = y + MAGIC;   // (up to 15.5 is 15, and so is all above)
    exactly |= !(fabsf(y - (t - MAGIC)) < 0.49999f);
    codes = codes * 16u + __float_as_uint(t);
  }
  codes -= __float_as_uint(MAGIC) * 0x1111u;
  if (exactly) {
    const double exact = Q41 ? ((double)hi - (double)lo) / 15.0 : (double)d;
    d = (float)exact;
    const bool none = __half2float(__float2half_rn(d)) == 0.0f;
    codes = kv4_codes_exactly(x, exact, (double)base, Q41 ? 0.5 : 8.5, none, Q41 ? 0u : 0x8888u);
  }
  *scale = __float2half_rn(d);
  if (Q41) *minimum = __float2half_rn(lo);
  const bool finite = fabsf(__half2float(*scale)) < INFINITY && (!Q41 || fabsf(__half2float(*minimum)) < INFINITY);
  if (!finite) *scale = __ushort_as_half((unsigned short)0x7fff);
  if (__half2float(*scale) == 0.0f) codes = Q41 ? 0u : 0x8888u;
  return codes;
}

struct RowsArgs {
  float *k, *v;              // store: read only
  uint8_t *pool;
  const int *slots;
  int *status;
  int64_t ld, tokens;
  Kv4Shape s;
  int page_shift;
  int vec;                   // rows can be read and written by 16 bytes
};

// A block has one head of sixteen rows of a call: rows that lie side by side in the cache have their codes in the same sectors, which come and go once.
// What a row costs beside its values (slot, page, address) is worked out once, by a thread a row.  (A thread for any four values, 64-bit
// divisions and all: 8191 rows of 4 x 128, stored and loaded, 47 us; now 27, bound by the instructions of both.)
constexpr int KR_THREADS = 256, KR_ROWS = 16;

struct RowsShared {
  long long tile[KR_ROWS];   // byte of the tile in the pool; -1: nowhere
  int token[KR_ROWS];        // in the tile
};
__device__ __forceinline__ void rows_begin(const RowsArgs &a, RowsShared &sh, int64_t first, int head, bool tells) {
  if (threadIdx.x < KR_ROWS) {
    const int64_t row = first + threadIdx.x;
    long long tile = -1;
    int token = 0;
    if (row < a.tokens) {
      const int slot = a.slots[row];
      const int page_id = slot >> a.page_shift, within = slot & ((1 << a.page_shift) - 1);
      if (slot >= 0 && kv4_page_ok(a.s, page_id)) {
        tile = kv4_tile_at(a.s, page_id, head, within);
        token = within & 15;
      } else if (slot != -1 && tells) {
        report_bad_index(a.status, 40, slot);
      }
    }
    sh.tile[threadIdx.x] = tile;
    sh.token[threadIdx.x] = token;
  }
  __syncthreads();
}

template <int NC, bool Q41>
__global__ void __launch_bounds__(KR_THREADS) kv4_store_kernel(RowsArgs a) {
  constexpr int D = 64 * NC, QUADS = D / 4, PART = (Q41 ? 10 : 9) * D;
  __shared__ RowsShared sh;
  pdl_enter();
  const int64_t first = (int64_t)blockIdx.x * KR_ROWS;
  const int head = blockIdx.y;
  rows_begin(a, sh, first, head, head == 0);
  constexpr int N = KR_ROWS * 2 * QUADS / KR_THREADS;
  float4 x[N];   // all of a thread's loads are under way before the first is used
#pragma unroll
  for (int it = 0; it < N; ++it) {   // (groups of eight lanes have a block each)
    const int i = it * KR_THREADS + threadIdx.x, row = i / (2 * QUADS), c = i % (2 * QUADS), dim = c % QUADS * 4;
    x[it] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (sh.tile[row] >= 0) {
      const float *src = (c < QUADS ? a.k : a.v) + (first + row) * a.ld + head * D + dim;
      if (a.vec) x[it] = __ldcs(reinterpret_cast<const float4 *>(src));
      else x[it] = make_float4(src[0], src[1], src[2], src[3]);
    }
  }
#pragma unroll
  for (int it = 0; it < N; ++it) {
    const int i = it * KR_THREADS + threadIdx.x, row = i / (2 * QUADS), c = i % (2 * QUADS), dim = c % QUADS * 4, tok = sh.token[row];
    const bool of_k = c < QUADS, ok = sh.tile[row] >= 0;
    __half d, m;
    const uint32_t codes = kv4_quantise<Q41>(x[it], &d, &m);
    const uint32_t next = __shfl_down_sync(0xffffffffu, codes, 1);
    if (!ok) continue;
    uint8_t *part = a.pool + sh.tile[row] + (of_k ? 0 : PART);
    if (of_k) {
      if (dim % 8 == 0) *reinterpret_cast<uint32_t *>(part + kv4_k_byte(tok, dim)) = codes | next << 16;
    } else {
      *reinterpret_cast<uint16_t *>(part + kv4_v_byte(tok, dim)) = (uint16_t)codes;
    }
    if (dim % 32 == 0) {
      __half *scales = reinterpret_cast<__half *>(part + 8 * D) + kv4_scale_index(tok, dim / 32, D);
      scales[0] = d;
      if (Q41) scales[D / 2] = m;
    }
  }
}

// ---- rows out of the cache -------------------------------------------------------------------------
template <int NC, bool Q41>
__global__ void __launch_bounds__(KR_THREADS) kv4_load_kernel(RowsArgs a) {
  constexpr int D = 64 * NC, QUADS = D / 4, PART = (Q41 ? 10 : 9) * D;
  __shared__ RowsShared sh;
  pdl_enter();
  const int64_t first = (int64_t)blockIdx.x * KR_ROWS;
  const int head = blockIdx.y;
  rows_begin(a, sh, first, head, head == 0);
  constexpr int N = KR_ROWS * 2 * QUADS / KR_THREADS;
  uint32_t codes[N];
  __half2 scale[N];   // d, and Q4_1's minimum
#pragma unroll
  for (int it = 0; it < N; ++it) {
    const int i = it * KR_THREADS + threadIdx.x, row = i / (2 * QUADS), c = i % (2 * QUADS), dim = c % QUADS * 4, tok = sh.token[row];
    if (sh.tile[row] < 0) continue;
    const uint8_t *part = a.pool + sh.tile[row] + (c < QUADS ? 0 : PART);
    codes[it] = *reinterpret_cast<const uint16_t *>(part + (c < QUADS ? kv4_k_byte(tok, dim) : kv4_v_byte(tok, dim)));
    const __half *scales = reinterpret_cast<const __half *>(part + 8 * D) + kv4_scale_index(tok, dim / 32, D);
    scale[it] = __halves2half2(scales[0], Q41 ? scales[D / 2] : __ushort_as_half(0));
  }
#pragma unroll
  for (int it = 0; it < N; ++it) {
    const int i = it * KR_THREADS + threadIdx.x, row = i / (2 * QUADS), c = i % (2 * QUADS), dim = c % QUADS * 4;
    if (sh.tile[row] < 0) continue;
    const float d = __low2float(scale[it]), m = __high2float(scale[it]);
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float code = __uint_as_float(0x4b000000u | (codes[it] >> (4 * e) & 15u)) - (Q41 ? 8388608.0f : 8388616.0f);   // exact
      y[e] = Q41 ? d * code + m : d * code;
    }
    float *dst = (c < QUADS ? a.k : a.v) + (first + row) * a.ld + head * D + dim;
    if (a.vec) __stcs(reinterpret_cast<float4 *>(dst), make_float4(y[0], y[1], y[2], y[3]));
    else { dst[0] = y[0]; dst[1] = y[1]; dst[2] = y[2]; dst[3] = y[3]; }
  }
}

// ---- checks ----------------------------------------------------------------------------------------
int kv4_check(caten_b200_ctx *ctx, const char *who, const caten_b200_kv4_desc *c, Kv4Shape *s) {
  if (!c) return fail(ctx, CATEN_B200_EINVAL, "%s: the description is NULL", who);
  if (c->type != CATEN_B200_Q4_0 && c->type != CATEN_B200_Q4_1) return fail(ctx, CATEN_B200_EUNSUPPORTED, "%s: cache of type %d (Q4_0 and Q4_1 are stored)", who, c->type);
  if (c->dim != 64 && c->dim != 128 && c->dim != 192 && c->dim != 256) return fail(ctx, CATEN_B200_EUNSUPPORTED, "%s: heads of %d (64, 128, 192 or 256)", who, c->dim);
  if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128) return fail(ctx, CATEN_B200_EUNSUPPORTED, "%s: pages of %d tokens (16, 32, 64 or 128)", who, c->page);
  if (c->kv_heads <= 0 || c->kv_heads > 65535 || c->heads <= 0 || c->heads > 65535 || c->heads % c->kv_heads) return fail(ctx, CATEN_B200_EINVAL, "%s: %d heads over %d", who, c->heads, c->kv_heads);
  if (c->pages <= 0 || c->pages > 0x7fffffffll / c->page) return fail(ctx, CATEN_B200_EINVAL, "%s: %lld pages of %d tokens (slots are 32-bit numbers)", who, (long long)c->pages, c->page);
  *s = {c->kv_heads, c->dim, c->type == CATEN_B200_Q4_1, c->page, c->pages};
  return 0;
}

static int rows_check(caten_b200_ctx *ctx, const char *who, const caten_b200_kv4_desc *c, const void *pool, const float *k, const float *v, int64_t ld,
                      const int32_t *slots, int64_t tokens, RowsArgs *a) {
  if (int rc = kv4_check(ctx, who, c, &a->s)) return rc;
  if (tokens < 0 || tokens > 0x7fffffff) return fail(ctx, CATEN_B200_EINVAL, "%s: %lld tokens", who, (long long)tokens);
  if (tokens && (!pool || !k || !v || !slots)) return fail(ctx, CATEN_B200_EINVAL, "%s: NULL argument", who);
  if (ld < (int64_t)c->kv_heads * c->dim) return fail(ctx, CATEN_B200_EINVAL, "%s: ld=%lld, rows have %lld values", who, (long long)ld, (long long)c->kv_heads * c->dim);
  if ((uintptr_t)pool % 16) return fail(ctx, CATEN_B200_EINVAL, "%s: the pool has to start on a multiple of 16 bytes", who);
  if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)slots) % 4) return fail(ctx, CATEN_B200_EINVAL, "%s: misaligned pointer", who);
  a->k = const_cast<float *>(k); a->v = const_cast<float *>(v);
  a->pool = (uint8_t *)const_cast<void *>(pool);
  a->slots = slots;
  a->ld = ld; a->tokens = tokens;
  a->vec = ld % 4 == 0 && ((uintptr_t)k | (uintptr_t)v) % 16 == 0;
  a->page_shift = c->page == 16 ? 4 : c->page == 32 ? 5 : c->page == 64 ? 6 : 7;
  return 0;
}

template <int NC>
static cudaError_t rows_launch_d(caten_b200_ctx *ctx, const RowsArgs &a, bool store) {
  const dim3 grid((unsigned)((a.tokens + KR_ROWS - 1) / KR_ROWS), (unsigned)a.s.kv_heads);
  void (*kernel)(RowsArgs) = store ? (a.s.q41 ? kv4_store_kernel<NC, true> : kv4_store_kernel<NC, false>) : (a.s.q41 ? kv4_load_kernel<NC, true> : kv4_load_kernel<NC, false>);
  return launch_k(ctx, kernel, grid, dim3(KR_THREADS), 0, a);
}
static int rows_launch(caten_b200_ctx *ctx, RowsArgs a, bool store) {
  a.status = ctx->d_status;
  switch (a.s.dim / 64) {
    case 1: CB_CUDA(ctx, rows_launch_d<1>(ctx, a, store)); break;
    case 2: CB_CUDA(ctx, rows_launch_d<2>(ctx, a, store)); break;
    case 3: CB_CUDA(ctx, rows_launch_d<3>(ctx, a, store)); break;
    default: CB_CUDA(ctx, rows_launch_d<4>(ctx, a, store));
  }
  CB_LAUNCH_CHECK(ctx, store ? "kv4_store_kernel" : "kv4_load_kernel");
  return 0;
}

}  // namespace cb

using namespace cb;

extern "C" {

// Arguments are checked before the context is touched.
int caten_b200_kv_pages(caten_b200_ctx *ctx, const int32_t *d_have, const int32_t *d_want, int64_t requests, int64_t page, int32_t *d_table,
                        int64_t max_pages, int32_t *d_free, int64_t pages, int32_t *d_state, int32_t *d_starts, int32_t *d_slots, int64_t max_tokens) {
  if (requests < 0 || requests > (1 << 24) || max_pages <= 0 || max_tokens < 0 || max_tokens > (1 << 30)) return fail(ctx, CATEN_B200_EINVAL, "kv_pages: bad shape");
  if (page <= 0 || pages <= 0 || page > 0x7fffffff || pages > 0x7fffffffll / page || max_pages > 0x7fffffffll / page)
    return fail(ctx, CATEN_B200_EINVAL, "kv_pages: %lld pages of %lld tokens, %lld a request (slots and positions are 32-bit numbers)", (long long)pages, (long long)page, (long long)max_pages);
  if (!d_free || !d_state || !d_starts || (requests && (!d_have || !d_want || !d_table)) || (max_tokens && !d_slots)) return fail(ctx, CATEN_B200_EINVAL, "kv_pages: NULL argument");
  if (!ctx) return fail(nullptr, CATEN_B200_EINVAL, "kv_pages: ctx is NULL");
  cudaSetDevice(ctx->device);
  ctx->work_outside = true;
  ProfScope prof(ctx, CATEN_B200_K_PREP);
  PagesArgs a = {d_have, d_want, d_table, d_free, d_state, d_starts, d_slots, (int)requests, (int)page, (int)max_pages, (int)pages, (int)max_tokens};
  const int own_slots = max_tokens <= PG_MOST;
  if (requests <= 128 && own_slots) {
    CB_CUDA(ctx, launch_k(ctx, kv_pages_kernel<128, 1>, dim3(1), dim3(128), 0, a, own_slots));
  } else {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(PG_BLOCKS);
    cfg.blockDim = dim3(1024);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = PG_BLOCKS;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = take_pdl(ctx) ? 2 : 1;
    CB_CUDA(ctx, cudaLaunchKernelEx(&cfg, kv_pages_kernel<1024, PG_BLOCKS>, a, own_slots));
  }
  CB_LAUNCH_CHECK(ctx, "kv_pages_kernel");
  if (own_slots) return 0;
  CB_CUDA(ctx, launch_k(ctx, kv_slots_kernel, dim3((unsigned)((max_tokens + 1023) / 1024)), dim3(256), 0, a));
  CB_LAUNCH_CHECK(ctx, "kv_slots_kernel");
  return 0;
}

int64_t caten_b200_kv4_nbytes(const caten_b200_kv4_desc *desc) {
  Kv4Shape s;
  if (kv4_check(nullptr, "kv4_nbytes", desc, &s)) return -1;
  return kv4_page_bytes(s) * s.pages;
}

int caten_b200_kv4_store(caten_b200_ctx *ctx, const caten_b200_kv4_desc *desc, void *d_pool, const float *d_k, const float *d_v, int64_t ld,
                         const int32_t *d_slots, int64_t tokens) {
  RowsArgs a = {};
  if (int rc = rows_check(ctx, "kv4_store", desc, d_pool, d_k, d_v, ld, d_slots, tokens, &a)) return rc;
  if (!ctx) return fail(nullptr, CATEN_B200_EINVAL, "kv4_store: ctx is NULL");
  cudaSetDevice(ctx->device);
  ctx->work_outside = true;
  if (tokens == 0) return 0;
  ProfScope prof(ctx, CATEN_B200_K_PREP);
  return rows_launch(ctx, a, true);
}

int caten_b200_kv4_load(caten_b200_ctx *ctx, const caten_b200_kv4_desc *desc, const void *d_pool, const int32_t *d_slots, int64_t tokens, float *d_k,
                        float *d_v, int64_t ld) {
  RowsArgs a = {};
  if (int rc = rows_check(ctx, "kv4_load", desc, d_pool, d_k, d_v, ld, d_slots, tokens, &a)) return rc;
  if (!ctx) return fail(nullptr, CATEN_B200_EINVAL, "kv4_load: ctx is NULL");
  cudaSetDevice(ctx->device);
  ctx->work_outside = true;
  if (tokens == 0) return 0;
  ProfScope prof(ctx, CATEN_B200_K_PREP);
  return rows_launch(ctx, a, false);
}

}  // extern "C"
