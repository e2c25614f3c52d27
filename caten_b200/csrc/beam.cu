// Beam search: selection over beams and vocabulary, and the reordering of states behind it.  No counterpart in the reference, whose
// generate loop is greedy (apps/gpt2/gpt2.lisp:97-113).
//
// Selection.  Candidate (beam b, token v) has the value score_b + x_bv - lse_b, lse_b = max + log(sum exp(x - max)); the first `keep` by value,
// equal ones by b * V + v.  Within a beam that order is the order of the logits, so a pass over the logits needs no lse: each block reads a chunk
// of a row once into registers and leaves its maximum, its sum of exponentials (fp32) and its `keep` largest logits; a second kernel joins the
// chunks' sums, turns the few logits left into values and picks among them; where the sums' errors could decide between beams it makes those rows' sums
// in 64 bits, by a second pass over them, and picks again.  Both pick by a bound first: `keep` values
// are not behind the `keep`-th of disjoint groups' largest, and with a few dozen candidates left each counts those before it, which is its place.
// Bound by instructions and the barriers of the ranking: 64 x 8 beams over 50257 logits 34 us, 26 of them the chunks (79 MB at 3 TB/s; a quarter has
// ended), 8 the join; one group of 4 beams 8.7 us, two dependent launches.  Rows summed again (of random logits, 16 kept of 8 beams: in one request of
// some hundreds) take 13 us each, most of it exp in 64 bits on one SM.
#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "kv4.cuh"

namespace cb {

constexpr int BS_THREADS = 256;
constexpr int BS_KEEP = 32;     // a warp's lanes
constexpr int BS_FEW = 64;      // threads of a block that may have candidates (of at most 32 logits each) without a closer look

typedef unsigned long long u64;

// larger float <=> larger key; equal floats: the lower index is the larger key.  0: no candidate (-inf, NaN).
__device__ __forceinline__ u64 beam_key(float x, int index) {
  const uint32_t b = __float_as_uint(x + 0.0f);   // (-0 is 0)
  const uint32_t k = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return x > -INFINITY ? (u64)k << 32 | (uint32_t)~index : 0ull;
}
__device__ __forceinline__ float beam_key_value(u64 key) {
  const uint32_t k = (uint32_t)(key >> 32);
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ int beam_key_index(u64 key) { return (int)~(uint32_t)key; }

// the lanes' keys in descending order (Batcher's bitonic network)
__device__ __forceinline__ u64 warp_sort(u64 key) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const u64 other = __shfl_xor_sync(0xffffffffu, key, j);
      const bool larger = ((lane & j) == 0) == ((lane & k) == 0);
      key = larger == (other > key) ? other : key;
    }
  return key;
}

__device__ __forceinline__ float warp_sort_floats(float x) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const float other = __shfl_xor_sync(0xffffffffu, x, j);
      x = ((lane & j) == 0) == ((lane & k) == 0) ? fmaxf(x, other) : fminf(x, other);
    }
  return x;
}

// The `keep`-th largest of the block's keys (one a thread, 0: none; all others different), 1 if there are fewer.  A key's rank is the number of
// larger ones, found in each warp's descending list by bisection.  Called by the whole block; `lists` and `answer` are its scratch.
__device__ u64 block_kth_key(u64 key, int keep, u64 (*lists)[32], u64 *answer) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  key = warp_sort(key);
  lists[warp][lane] = key;
  if (threadIdx.x == 0) *answer = 1;
  __syncthreads();
  if (lane < keep && key) {
    int rank = 0;
#pragma unroll 1
    for (int w = 0; w < BS_THREADS / 32; ++w) {
      int lo = 0;
#pragma unroll
      for (int step = 16; step > 0; step >>= 1)
        if (lists[w][lo + step - 1] > key) lo += step;
      rank += lo + (lists[w][lo] > key ? 1 : 0);
    }
    if (rank == keep - 1) *answer = key;
  }
  __syncthreads();
  return *answer;
}

// What a block leaves of its chunk: `keep` keys (descending, 0 behind the last), then maximum and sum.
__host__ __device__ __forceinline__ int64_t beam_part_words(int keep) { return keep + 1; }

template <int VECS>
__global__ void __launch_bounds__(BS_THREADS) beam_chunk_kernel(const float *__restrict__ x, const uint8_t *__restrict__ ended, int64_t V, int keep, u64 *__restrict__ parts) {
  constexpr int CHUNK = BS_THREADS * VECS * 4;
  __shared__ float group_top[32];
  __shared__ double sums[BS_THREADS / 32];
  __shared__ u64 lists[BS_THREADS / 32][32], answer;
  __shared__ u64 found[BS_FEW * VECS * 4];
  __shared__ float kth_top;
  __shared__ int count;
  pdl_enter();
  const int64_t row = blockIdx.y;
  if (ended && ended[row]) return;   // its one candidate needs no logits
  const float *p = x + row * V;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // chunks start on 16-byte boundaries of memory, wherever the row does
  const int64_t e0 = (int64_t)blockIdx.x * CHUNK - (int64_t)(((uintptr_t)p >> 2) & 3);
  const int index0 = (int)e0 + tid * 4;
  float v[VECS][4];
  if (e0 >= 0 && e0 + CHUNK <= V) {
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const float4 q = __ldcs(reinterpret_cast<const float4 *>(p + e0) + i * BS_THREADS + tid);
      v[i][0] = q.x; v[i][1] = q.y; v[i][2] = q.z; v[i][3] = q.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int64_t e = e0 + (i * BS_THREADS + tid) * 4;
      if (e >= 0 && e + 4 <= V) {
        const float4 q = __ldcs(reinterpret_cast<const float4 *>(p + e));
        v[i][0] = q.x; v[i][1] = q.y; v[i][2] = q.z; v[i][3] = q.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i][j] = e + j >= 0 && e + j < V ? p[e + j] : -INFINITY;
      }
    }
  }
  if (tid == 0) count = 0;
  // the largest of each thread, of each eight threads, and of those 32 in order the first and the `keep`-th
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < VECS; ++i) top = fmaxf(top, fmaxf(fmaxf(v[i][0], v[i][1]), fmaxf(v[i][2], v[i][3])));
  float gt = top;
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) gt = fmaxf(gt, __shfl_xor_sync(0xffffffffu, gt, o));
  if (lane % 8 == 0) group_top[tid / 8] = gt;
  __syncthreads();
  float m = group_top[lane];
  if (warp == 0) {   // (the others go on; the bound is needed behind the next barrier)
    const float sorted = warp_sort_floats(m);
    if (lane == keep - 1) kth_top = sorted;
    m = __shfl_sync(0xffffffffu, sorted, 0);
  } else {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  }
  // sum of exponentials; a maximum of -inf (nothing left) makes it 0, a NaN or +inf makes it NaN
  const float base = m == -INFINITY ? 0.0f : m;
  float q[VECS];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    float e[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e[j]) : "f"((v[i][j] - base) * 1.4426950408889634f));
    q[i] = (e[0] + e[1]) + (e[2] + e[3]);
#pragma unroll
    for (int k = 1; k < VECS; k <<= 1)   // (in pairs: five roundings for 32 logits)
      if ((i & (2 * k - 1)) == 2 * k - 1) q[i] += q[i - k];
  }
  double sum = q[VECS - 1];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sums[warp] = sum;
  __syncthreads();
  const float least = kth_top;
  const bool may = top >= least && top > -INFINITY;
  const int threads = __syncthreads_count(may);
  // Many threads at the bound: equal logits (a mask's value), or masks that empty whole groups.  Then by keys, which are all different.
  u64 bound = 1;
  bool look = may;
  if (threads > BS_FEW) {
    u64 best = 0;
#pragma unroll
    for (int i = VECS - 1; i >= 0; --i)
#pragma unroll
      for (int j = 3; j >= 0; --j)
        if (v[i][j] == top) best = beam_key(v[i][j], index0 + i * BS_THREADS * 4 + j);   // (the lowest index of equal ones)
    bound = block_kth_key(best, keep, lists, &answer);
    look = best >= bound;   // (`keep` threads, or fewer than that in all)
  }
  if (look) {
    const float floor_value = bound == 1 ? least : beam_key_value(bound);
#pragma unroll
    for (int i = 0; i < VECS; ++i)
      if (fmaxf(fmaxf(v[i][0], v[i][1]), fmaxf(v[i][2], v[i][3])) >= floor_value)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (v[i][j] >= floor_value) {
            const u64 key = beam_key(v[i][j], index0 + i * BS_THREADS * 4 + j);
            if (key >= bound) found[atomicAdd(&count, 1)] = key;
          }
  }
  __syncthreads();
  const int n = count;
  u64 *part = parts + (row * gridDim.x + blockIdx.x) * beam_part_words(keep);
  for (int i = tid; i < n; i += BS_THREADS) {
    const u64 key = found[i];
    int place = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) place += found[j] > key;
    if (place < keep) part[place] = key;
  }
  for (int i = n + tid; i < keep; i += BS_THREADS) part[i] = 0;
  if (tid == 0) {
    sum = sums[0];
#pragma unroll
    for (int w = 1; w < BS_THREADS / 32; ++w) sum += sums[w];
    part[keep] = (u64)__float_as_uint(base) << 32 | __float_as_uint(m < INFINITY ? (float)sum : NAN);
  }
}

// ---- the chunks' lists into one --------------------------------------------------------------------
// order-preserving image of a 64-bit value; 0: none
__device__ __forceinline__ u64 order_of(double x) {
  const u64 b = (u64)__double_as_longlong(x + 0.0);
  return !(x > -INFINITY) ? 0ull : (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double value_of(u64 k) { return __longlong_as_double((long long)((k >> 63) ? (k & 0x7fffffffffffffffull) : ~k)); }

constexpr int BJ_THREADS = 1024;
constexpr int BJ_HEADS = 256;    // threads that look at the lists' first entries
constexpr int BJ_LANES = 16;     // threads that find one candidate's place
constexpr int BJ_BEAMS = 32;
constexpr int BJ_LISTS = 4096;   // of a request: beams x chunks
constexpr int BJ_FOUND = BS_KEEP * BS_KEEP;
constexpr int BJ_QUEUE = 64;

// A candidate: the order-preserving images of its value and, for equal values, of its beam (lower), its logit and its token (lower): larger ones come
// first.  (Beside a score of -1e30, or the lowest value as a mask, all of a beam's values are one number; what its logits say still counts.)
struct __align__(16) Cand {
  u64 value, tie;
  __device__ __forceinline__ bool operator>(const Cand &o) const { return value > o.value || (value == o.value && tie > o.tie); }
  __device__ __forceinline__ int beam() const { return BJ_BEAMS - 1 - (int)(tie >> 52); }
  __device__ __forceinline__ int64_t token() const { return 0xfffff - (int64_t)(tie & 0xfffff); }
};
__device__ __forceinline__ u64 cand_tie(int beam, u64 key) { return (u64)(BJ_BEAMS - 1 - beam) << 52 | (key >> 32) << 20 | (u64)(0xfffff - beam_key_index(key)); }

struct JoinArgs {
  const u64 *parts;
  const float *x, *scores;
  const uint8_t *ended;
  float *out_scores;
  int *out_parents;
  int64_t *out_tokens;
  uint8_t *out_ended;
  int64_t V, eos;
  int chunks, beams, keep;
  float close;
};
struct JoinShared {
  __align__(128) Cand found[BJ_FOUND];
  Cand sorted[BJ_FOUND], bound;
  double base[BJ_BEAMS], tops[BJ_BEAMS];   // a candidate's value: base + (x - top)
  double sums[BJ_THREADS / 32];
  uint8_t over[BJ_BEAMS];
  int queue[BJ_QUEUE];
  int count, queued;
  unsigned close_beams;

  // Candidates of different beams whose values, by the chunks' sums, are no farther apart than this may be in either order: by what the sums may be off,
  // and what the additions of a value in 64 bits round off.
  __device__ __forceinline__ double close_to(const JoinArgs &a, double value) const { return a.close + fabs(value) * 0x1p-50; }
  __device__ __forceinline__ Cand cand_of(const JoinArgs &a, int i, int j, u64 key) const {   // entry j of list i
    const int b = i / a.chunks;
    if (over[b])   // its one candidate stands first in its first list
      return {i == b * a.chunks && j == 0 && a.eos >= 0 ? order_of(base[b]) : 0ull, cand_tie(b, (u64)~(uint32_t)a.eos)};
    return {key ? order_of(base[b] + ((double)beam_key_value(key) - tops[b])) : 0ull, cand_tie(b, key)};
  }
  // a found candidate's value by what base[] is now
  __device__ __forceinline__ u64 value_at(const JoinArgs &a, const Cand &c) const {
    const int b = c.beam();
    return order_of(over[b] ? base[b] : base[b] + ((double)beam_key_value(c.tie >> 20 << 32) - tops[b]));
  }
  __device__ __forceinline__ void write(const JoinArgs &a, int place, bool there, const Cand &c) const {
    const int64_t at = (int64_t)blockIdx.x * a.keep + place;
    const int parent = there ? c.beam() : min(place, a.beams - 1);
    const int64_t token = there ? c.token() : a.eos >= 0 ? a.eos : 0;
    a.out_scores[at] = there ? (float)value_of(c.value) : -INFINITY;
    a.out_parents[at] = parent;
    a.out_tokens[at] = token;
    if (a.out_ended) a.out_ended[at] = over[parent] || (a.eos >= 0 && token == a.eos);
  }
};

// Sums of the given beams' rows in 64 bits, each in an order that depends on V alone (equal rows have equal sums), and the places of the n candidates
// found anew; n < 0: too many were close to look at, so all lists give their best, one after another.  Rarely needed, and a function of its own:
// inside the kernel it cost every call 0.4 us of registers and of instructions to fetch.
__device__ __noinline__ void beam_join_exactly(const JoinArgs &a, JoinShared &sh) {
  const int n = sh.queued > BJ_QUEUE || sh.count > BJ_FOUND ? -1 : sh.count;
  const unsigned beams = n < 0 ? ~0u : sh.close_beams;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int b = 0; b < a.beams; ++b) {
    if (!(beams >> b & 1) || sh.over[b]) continue;
    const int64_t row = (int64_t)blockIdx.x * a.beams + b;
    const float *x = a.x + row * a.V;
    const double top = sh.tops[b];
    double s = 0.0;
#pragma unroll 8
    for (int64_t i = tid; i < a.V; i += BJ_THREADS) s += exp((double)x[i] - top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) sh.sums[warp] = s;
    __syncthreads();
    if (warp == 0) {
      s = sh.sums[lane];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) sh.base[b] = (double)a.scores[row] - log(s);
    }
    __syncthreads();
  }
  if (n >= 0) {
    for (int i = tid; i < n; i += BJ_THREADS) sh.found[i].value = sh.value_at(a, sh.found[i]);
    __syncthreads();
    for (int i = tid; i < n; i += BJ_THREADS) {
      const Cand c = sh.found[i];
      int place = 0;
      for (int j = 0; j < n; ++j) place += sh.found[j] > c;
      if (place < a.keep) sh.write(a, place, true, c);
    }
    return;
  }
  Cand *warps = sh.found;                                                  // their best
  uint8_t *next = reinterpret_cast<uint8_t *>(sh.found + BJ_THREADS / 32);   // of each list, of which a thread has several
  const int lists = a.beams * a.chunks;
  const u64 *mine = a.parts + (int64_t)blockIdx.x * lists * beam_part_words(a.keep);
  for (int i = tid; i < lists; i += BJ_THREADS) next[i] = 0;
  for (int place = 0; place < a.keep; ++place) {
    Cand best = {0ull, 0ull};
    int of = 0;
    for (int i = tid; i < lists; i += BJ_THREADS) {
      if (next[i] == a.keep) continue;
      const Cand c = sh.cand_of(a, i, next[i], mine[i * beam_part_words(a.keep) + next[i]]);
      if (c.value && c > best) { best = c; of = i; }
    }
    Cand most = best;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const Cand other = {__shfl_xor_sync(0xffffffffu, most.value, o), __shfl_xor_sync(0xffffffffu, most.tie, o)};
      if (other > most) most = other;
    }
    if (lane == 0) warps[warp] = most;
    __syncthreads();
    for (int w = 0; w < BJ_THREADS / 32; ++w)
      if (warps[w] > most) most = warps[w];
    __syncthreads();
    if (!most.value) {
      if (tid == 0) sh.write(a, place, false, most);
    } else if (best.value == most.value && best.tie == most.tie) {   // (one thread's)
      sh.write(a, place, true, best);
      ++next[of];
    }
  }
}

__global__ void __launch_bounds__(BJ_THREADS) beam_join_kernel(const __grid_constant__ JoinArgs a) {
  __shared__ JoinShared sh;
  pdl_enter();
  const int64_t batch = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int keep = a.keep, chunks = a.chunks;
  const int64_t words = beam_part_words(keep);
  const int lists = a.beams * chunks;
  const u64 *mine = a.parts + batch * lists * words;
  if (tid == 0) { sh.bound = {1, 0}; sh.count = 0; sh.queued = 0; sh.close_beams = 0; }   // (that bound: every candidate)
  const u64 head = tid < min(lists, BJ_HEADS) ? mine[(int64_t)tid * words] : 0ull;     // (of an ended hypothesis: whatever is there, unused)
  for (int b = warp; b < a.beams; b += BJ_THREADS / 32) {
    const int64_t row = batch * a.beams + b;
    const float score = a.scores[row];
    const bool end = a.ended && a.ended[row];
    double log_sum = 0.0, top = 0.0;
    if (!end) {
      const u64 *part = mine + (int64_t)b * chunks * words + keep;
      const u64 first = lane < chunks ? part[lane * words] : 0ull;
      float m = (uint32_t)first != 0u ? __uint_as_float((uint32_t)(first >> 32)) : -INFINITY;   // (sum 0: nothing in that chunk)
      for (int c = lane + 32; c < chunks; c += 32)
        if ((uint32_t)part[c * words] != 0u) m = fmaxf(m, __uint_as_float((uint32_t)(part[c * words] >> 32)));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      double s = 0.0;
      for (int c = lane; c < chunks; c += 32) {
        const u64 w = c == lane ? first : part[c * words];
        if ((uint32_t)w != 0u) s += (double)__uint_as_float((uint32_t)w) * exp((double)__uint_as_float((uint32_t)(w >> 32)) - (double)m);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      log_sum = log(s);   // (nothing left in the row: -inf, but then there is no key either)
      top = (double)m;
    }
    if (lane == 0) {
      sh.base[b] = (double)score - log_sum;
      sh.tops[b] = top;
      sh.over[b] = end;
    }
  }
  __syncthreads();
  auto entry = [&](int i, int j) { return sh.cand_of(a, i, j, mine[(int64_t)i * words + j]); };
  // for each i of the n found: then(candidate, how many are before it), by one of the threads that count them
  auto for_places = [&](int n, auto then) {
    for (int i0 = 0; i0 < n; i0 += BJ_THREADS / BJ_LANES) {
      const int i = i0 + tid / BJ_LANES;
      const Cand c = sh.found[min(i, n - 1)];
      int place = 0;
#pragma unroll 4
      for (int j = tid % BJ_LANES; j < n; j += BJ_LANES) place += sh.found[j] > c;
#pragma unroll
      for (int o = 1; o < BJ_LANES; o <<= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
      if (i < n && tid % BJ_LANES == 0) then(c, place);
    }
  };
  // The keep-th of the lists' first entries: `keep` candidates are not behind it, and at most `keep` lists have any that are not.  Where a thread
  // has several lists, the threads' best give a first bound, and the few first entries that it leaves the second.  The last bound is lowered by
  // what a value may be off, so that whatever could change places with one that is taken is found too.
  Cand best = tid < min(lists, BJ_HEADS) ? sh.cand_of(a, tid, 0, head) : Cand{0ull, 0ull};
  if (tid < BJ_HEADS) {
    for (int i = tid + BJ_HEADS; i < lists; i += BJ_HEADS) {
      const Cand c = entry(i, 0);
      if (c > best) best = c;
    }
    sh.found[tid] = best;
  }
  __syncthreads();
  auto lowered = [&](const Cand &c) { return Cand{max(1ull, order_of(value_of(c.value) - sh.close_to(a, value_of(c.value)))), 0ull}; };
  for_places(min(lists, BJ_HEADS), [&](const Cand &c, int place) {
    if (c.value && place == keep - 1) sh.bound = lists > BJ_HEADS ? c : lowered(c);
  });
  __syncthreads();
  if (lists > BJ_HEADS) {
    const Cand first = sh.bound;
    for (int i = tid; i < lists; i += BJ_THREADS) {
      const Cand c = entry(i, 0);
      if (c.value && !(first > c)) sh.found[atomicAdd(&sh.count, 1)] = c;   // (of at most `keep` threads, 16 lists each)
    }
    __syncthreads();
    const int n = sh.count;
    for_places(n, [&](const Cand &c, int place) {
      if (place == keep - 1) sh.bound = lowered(c);
    });
    __syncthreads();
    if (tid == 0) sh.count = 0;
  }
  const u64 least = sh.bound.value;
  auto enqueue = [&](int i) {
    const int at = atomicAdd(&sh.queued, 1);
    if (at < BJ_QUEUE) sh.queue[at] = i;
  };
  if (lists <= BJ_HEADS) {
    if (best.value >= least) enqueue(tid);
  } else {
    for (int i = tid; i < lists; i += BJ_THREADS)
      if (entry(i, 0).value >= least) enqueue(i);
  }
  __syncthreads();
  for (int i = tid; i < min(sh.queued, BJ_QUEUE) * keep; i += BJ_THREADS) {
    const Cand c = entry(sh.queue[i / keep], i % keep);
    if (c.value >= least) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < BJ_FOUND) sh.found[at] = c;
    }
  }
  __syncthreads();
  const int n = min(sh.count, BJ_FOUND);
  for_places(n, [&](const Cand &c, int place) {
    if (place < keep) sh.write(a, place, true, c);
    sh.sorted[place] = c;
  });
  if (tid >= n && tid < keep) sh.write(a, tid, false, Cand{0ull, 0ull});
  __syncthreads();
  // Where two candidates of different beams are close, and one is taken, so are two neighbours, which are taken or close to the last that is.
  bool close = false;
  if (tid + 1 < n) {
    const Cand c = sh.sorted[tid], next = sh.sorted[tid + 1];
    const double value = value_of(next.value);
    close = c.beam() != next.beam() && value_of(sh.sorted[min(tid, keep - 1)].value) - value <= sh.close_to(a, value);
  }
  if (!__syncthreads_or(close || sh.queued > BJ_QUEUE || sh.count > BJ_FOUND)) return;   // (or so many are equal that some were not looked at)
  if (tid / BJ_LANES < min(n, keep)) {   // each that was taken, and whatever of other beams is close to it
    const Cand c = sh.sorted[tid / BJ_LANES];
    const double value = value_of(c.value), apart = sh.close_to(a, value);
    const u64 from = order_of(value - apart), to = order_of(value + apart);
    unsigned beams = 0;
    for (int j = tid % BJ_LANES; j < n; j += BJ_LANES) {
      const u64 v = sh.found[j].value;
      if (v >= from && v <= to) beams |= 1u << sh.found[j].beam();
    }
    if (beams & ~(1u << c.beam())) atomicOr(&sh.close_beams, beams | 1u << c.beam());
  }
  __syncthreads();
  beam_join_exactly(a, sh);
}

// Chunks of 8192 logits, or of 2048 where the larger ones would not give every SM a block.
constexpr int64_t BS_VOCAB = (1 << 20) - 8192;
static_assert(BS_KEEP * BJ_LANES <= BJ_THREADS, "a pass for those taken");
static_assert(BS_VOCAB <= 0xfffff, "a candidate has 20 bits for its token");
static_assert(BJ_BEAMS * ((BS_VOCAB + 3 + 8191) / 8192) <= BJ_LISTS && BS_KEEP * (BJ_LISTS / BJ_HEADS) <= BJ_FOUND, "lists of a request");
static int beam_vecs(int64_t batch, int64_t beams, int64_t V) {
  return batch * beams * ((V + 3 + 8191) / 8192) >= 148 || beams * ((V + 3 + 2047) / 2048) > BJ_LISTS ? 8 : 2;
}
// How far apart two rows' log sums may be in fp32 and equal in truth: a sum's relative error is, in units of 2^-24, that of the exponents, 2.23 of each (two
// roundings and the constant's), of which the sum of p (max - x) is the entropy less log(sum) and at most log(V); 4 of ex2.approx; 5 of the additions
// in a thread (warps, blocks and chunks join in 64 bits); 1 of the chunk's sum.
static float beam_close(int64_t V) { return (float)(2.0 * (11.0 + 2.25 * std::log((double)V)) * 0x1p-24); }
static int64_t beam_chunks(int64_t batch, int64_t beams, int64_t V) {
  const int64_t chunk = beam_vecs(batch, beams, V) * BS_THREADS * 4;
  return (V + 3 + chunk - 1) / chunk;
}

static int beam_check(caten_b200_ctx *ctx, const char *who, int64_t batch, int64_t beams, int64_t V, int64_t keep) {
  if (batch < 0 || beams <= 0 || V <= 0 || keep <= 0) return fail(ctx, CATEN_B200_EINVAL, "%s: bad shape", who);
  if (beams > BJ_BEAMS || keep > BS_KEEP) return fail(ctx, CATEN_B200_EUNSUPPORTED, "%s: %lld beams, %lld kept (at most %d)", who, (long long)beams, (long long)keep, BS_KEEP);
  if (V > BS_VOCAB) return fail(ctx, CATEN_B200_EUNSUPPORTED, "%s: V=%lld", who, (long long)V);
  if (batch > 65535 || batch * beams > 65535) return fail(ctx, CATEN_B200_EUNSUPPORTED, "%s: %lld rows", who, (long long)(batch * beams));
  return 0;
}

// ---- reordering ------------------------------------------------------------------------------------
// Row i of a group becomes what row parent(i) was, in place: a thread takes the same 16 (or 4) bytes of all the group's rows that change into
// registers before it writes any of them, so nothing is read after it was overwritten, whatever the parents are.  Rows that stay
// are neither read for themselves nor written.  Bound by HBM: 24 layers of 16 x 4 beams, 4.2 GB, 543 to 576 us (7.3 to 7.7 TB/s: a row that several
// children take comes once).  Pages, 16 x 8 beams of 24 of 82 KB, 251 MB: 54 us (4.7 TB/s, HBM 40 % busy): a block's four dependent loads (parents, lengths,
// table, page), for a word of 16 bytes a thread.
constexpr int RO_STATES = 128;   // of a launch
constexpr int RO_MOST = 1024;    // of a call
struct ReorderArgs {
  void *state[RO_STATES];
  const int *parents;
  int *status;
  int64_t planes, stride, words;   // words of a plane that move; stride between planes, in words
  int beams;
};

template <typename T, int BEAMS>
__global__ void __launch_bounds__(256) beam_reorder_kernel(const __grid_constant__ ReorderArgs a) {
  pdl_enter();
  const int *parents = a.parents + (int64_t)blockIdx.y * a.beams;
  int from[BEAMS];
  bool moves = false;
#pragma unroll
  for (int i = 0; i < BEAMS; ++i) {
    from[i] = i;
    if (i < a.beams) {
      const int p = parents[i];
      if (p >= 0 && p < a.beams) from[i] = p;
      else if (blockIdx.x == 0 && threadIdx.x == 0) report_bad_index(a.status, 42, p);
    }
    moves |= from[i] != i;
  }
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (!moves || at >= a.planes * a.words) return;
  T *base = (T *)a.state[blockIdx.z] + (int64_t)blockIdx.y * a.beams * a.planes * a.stride + at / a.words * a.stride + at % a.words;
  const int64_t row = a.planes * a.stride;
  T v[BEAMS];
#pragma unroll
  for (int i = 0; i < BEAMS; ++i)
    if (from[i] != i) v[i] = base[from[i] * row];
#pragma unroll
  for (int i = 0; i < BEAMS; ++i)
    if (from[i] != i) base[i * row] = v[i];
}

struct PagesReorderArgs {
  uint8_t *pool;
  const int *table, *lengths, *parents;
  int *status;
  int64_t page_words, pages;
  int max_pages, page, beams;
};

template <int BEAMS>
__global__ void __launch_bounds__(256) beam_reorder_pages_kernel(PagesReorderArgs a) {
  pdl_enter();
  const int64_t group = blockIdx.z;
  const int j = blockIdx.y;
  const int64_t first = group * a.beams;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const bool tells = at == 0;
  int src[BEAMS], dst[BEAMS];
  bool moves = false;
#pragma unroll
  for (int i = 0; i < BEAMS; ++i) {
    dst[i] = -1;
    src[i] = 0;
    if (i < a.beams) {
      const int p = a.parents[first + i];
      if (p < 0 || p >= a.beams) {
        if (tells) report_bad_index(a.status, 42, p);
      } else if (p != i && (int64_t)j * a.page < a.lengths[first + i]) {
        const int to = a.table[(first + i) * a.max_pages + j], from = a.table[(first + p) * a.max_pages + j];
        if (to < 0 || to >= a.pages || from < 0 || from >= a.pages) {
          if (tells) report_bad_index(a.status, 43, to < 0 || to >= a.pages ? to : from);
        } else {
          dst[i] = to;
          src[i] = from;
          moves = true;
        }
      }
    }
  }
  if (!moves || at >= a.page_words) return;
  uint4 *pool = reinterpret_cast<uint4 *>(a.pool) + at;
  uint4 v[BEAMS];
#pragma unroll
  for (int i = 0; i < BEAMS; ++i)
    if (dst[i] >= 0) v[i] = pool[(int64_t)src[i] * a.page_words];
#pragma unroll
  for (int i = 0; i < BEAMS; ++i)
    if (dst[i] >= 0) pool[(int64_t)dst[i] * a.page_words] = v[i];
}

template <typename T>
static cudaError_t reorder_launch(caten_b200_ctx *ctx, dim3 grid, const ReorderArgs &a) {
  if (a.beams <= 4) return launch_k(ctx, beam_reorder_kernel<T, 4>, grid, dim3(256), 0, a);
  if (a.beams <= 8) return launch_k(ctx, beam_reorder_kernel<T, 8>, grid, dim3(256), 0, a);
  if (a.beams <= 16) return launch_k(ctx, beam_reorder_kernel<T, 16>, grid, dim3(256), 0, a);
  return launch_k(ctx, beam_reorder_kernel<T, 32>, grid, dim3(256), 0, a);
}

}  // namespace cb

using namespace cb;

extern "C" {

// Arguments are checked before the context is touched.
int64_t caten_b200_beam_select_work(int64_t batch, int64_t beams, int64_t V, int64_t keep) {
  if (beam_check(nullptr, "beam_select_work", batch, beams, V, keep)) return -1;
  // Enough for every call of sizes up to these: fewer rows, or a smaller V, may go in chunks of 2048, but only as long as the larger ones, of which
  // each is four at most, would be fewer than 148.
  const int64_t rows = batch * beams, parts = std::max(rows * ((V + 3 + 8191) / 8192), std::min<int64_t>(rows * ((V + 3 + 2047) / 2048), 4 * 147));
  return (parts * beam_part_words((int)keep) + 1) * (int64_t)sizeof(u64);
}

int caten_b200_beam_select(caten_b200_ctx *ctx, const float *d_logits, const float *d_scores, const uint8_t *d_ended, int64_t batch, int64_t beams, int64_t V,
                           int64_t eos, int64_t keep, float *d_out_scores, int32_t *d_out_parents, int64_t *d_out_tokens, uint8_t *d_out_ended, void *d_work) {
  if (int rc = beam_check(ctx, "beam_select", batch, beams, V, keep)) return rc;
  if (eos >= V) return fail(ctx, CATEN_B200_EINVAL, "beam_select: eos=%lld of %lld ids", (long long)eos, (long long)V);
  if (eos < 0 && d_ended) return fail(ctx, CATEN_B200_EINVAL, "beam_select: ended hypotheses need an eos id");
  if (batch && (!d_logits || !d_scores || !d_out_scores || !d_out_parents || !d_out_tokens || !d_work)) return fail(ctx, CATEN_B200_EINVAL, "beam_select: NULL argument");
  if (((uintptr_t)d_logits | (uintptr_t)d_scores | (uintptr_t)d_out_scores | (uintptr_t)d_out_parents) % 4 || ((uintptr_t)d_out_tokens | (uintptr_t)d_work) % 8)
    return fail(ctx, CATEN_B200_EINVAL, "beam_select: misaligned pointer");
  if (!ctx) return fail(nullptr, CATEN_B200_EINVAL, "beam_select: ctx is NULL");
  cudaSetDevice(ctx->device);
  ctx->work_outside = true;
  if (batch == 0) return 0;
  ProfScope prof(ctx, CATEN_B200_K_ARGMAX);
  const int64_t chunks = beam_chunks(batch, beams, V);
  const dim3 grid((unsigned)chunks, (unsigned)(batch * beams));
  CB_CUDA(ctx, launch_k(ctx, beam_vecs(batch, beams, V) == 8 ? beam_chunk_kernel<8> : beam_chunk_kernel<2>, grid, dim3(BS_THREADS), 0, d_logits, d_ended, V, (int)keep, (u64 *)d_work));
  CB_LAUNCH_CHECK(ctx, "beam_chunk_kernel");
  const JoinArgs join = {(const u64 *)d_work, d_logits, d_scores, d_ended, d_out_scores, d_out_parents, d_out_tokens, d_out_ended, V, eos, (int)chunks, (int)beams, (int)keep, beam_close(V)};
  CB_CUDA(ctx, launch_k(ctx, beam_join_kernel, dim3((unsigned)batch), dim3(BJ_THREADS), 0, join));
  CB_LAUNCH_CHECK(ctx, "beam_join_kernel");
  return 0;
}

int caten_b200_beam_reorder(caten_b200_ctx *ctx, void *const *h_states, int64_t count, const int32_t *d_parents, int64_t groups, int64_t beams, int64_t planes,
                            int64_t plane_stride, int64_t nbytes) {
  if (count < 0 || groups < 0 || groups > 65535 || beams <= 0 || planes <= 0 || plane_stride < 0 || nbytes < 0 || nbytes > plane_stride)
    return fail(ctx, CATEN_B200_EINVAL, "beam_reorder: bad shape");
  if (count > RO_MOST) return fail(ctx, CATEN_B200_EUNSUPPORTED, "beam_reorder: %lld states (at most %d)", (long long)count, RO_MOST);
  if (beams > BJ_BEAMS) return fail(ctx, CATEN_B200_EUNSUPPORTED, "beam_reorder: %lld beams (at most %d)", (long long)beams, BJ_BEAMS);
  if (plane_stride % 4 || nbytes % 4) return fail(ctx, CATEN_B200_EUNSUPPORTED, "beam_reorder: planes of %lld bytes, %lld of them moved (multiples of 4)", (long long)plane_stride, (long long)nbytes);
  if (count && groups && nbytes && (!h_states || !d_parents)) return fail(ctx, CATEN_B200_EINVAL, "beam_reorder: NULL argument");
  uintptr_t bits = (uintptr_t)(plane_stride | nbytes), sorted[RO_MOST];
  const __int128 state_bytes = (__int128)groups * beams * planes * plane_stride;   // (the last plane's unmoved end counted in)
  if (groups && nbytes) {
    for (int64_t i = 0; i < count; ++i) {
      sorted[i] = (uintptr_t)h_states[i];
      if (!sorted[i] || sorted[i] % 4) return fail(ctx, CATEN_B200_EINVAL, "beam_reorder: state %lld is NULL or misaligned", (long long)i);
      bits |= sorted[i];
    }
    std::sort(sorted, sorted + count);
    for (int64_t i = 1; i < count; ++i)
      if ((__int128)(sorted[i] - sorted[i - 1]) < state_bytes) return fail(ctx, CATEN_B200_EINVAL, "beam_reorder: states overlap");
  }
  const int width = bits % 16 ? 4 : 16;
  const int64_t words = nbytes / width;
  if (planes > 0x3fffffffffll || words > 0x3fffffffffll || (words && planes > 0x7fffff0000ll / words)) return fail(ctx, CATEN_B200_EUNSUPPORTED, "beam_reorder: %lld planes of %lld bytes", (long long)planes, (long long)nbytes);
  if (!ctx) return fail(nullptr, CATEN_B200_EINVAL, "beam_reorder: ctx is NULL");
  cudaSetDevice(ctx->device);
  ctx->work_outside = true;
  if (!groups || !nbytes) return 0;
  ProfScope prof(ctx, CATEN_B200_K_PREP);
  for (int64_t first = 0; first < count; first += RO_STATES) {
    ReorderArgs a;
    const int64_t n = count - first < RO_STATES ? count - first : RO_STATES;
    for (int64_t i = 0; i < n; ++i) a.state[i] = h_states[first + i];
    a.parents = d_parents; a.status = ctx->d_status;
    a.planes = planes; a.stride = plane_stride / width; a.words = words; a.beams = (int)beams;
    // (a group of one only has its parents checked)
    const dim3 grid(beams == 1 ? 1u : (unsigned)((planes * words + 255) / 256), (unsigned)groups, beams == 1 ? 1u : (unsigned)n);
    CB_CUDA(ctx, width == 16 ? reorder_launch<uint4>(ctx, grid, a) : reorder_launch<uint32_t>(ctx, grid, a));
    CB_LAUNCH_CHECK(ctx, "beam_reorder_kernel");
    if (beams == 1) break;
  }
  return 0;
}

int caten_b200_beam_reorder_pages(caten_b200_ctx *ctx, void *d_pool, int64_t pages, int64_t page_nbytes, const int32_t *d_table, int64_t max_pages,
                                  const int32_t *d_lengths, int64_t page, const int32_t *d_parents, int64_t groups, int64_t beams) {
  if (pages <= 0 || pages > 0x7fffffff || page_nbytes <= 0 || max_pages <= 0 || max_pages > 65535 || page <= 0 || page > 0x7fffffff / max_pages || groups < 0 || groups > 65535 || beams <= 0)
    return fail(ctx, CATEN_B200_EINVAL, "beam_reorder_pages: bad shape");
  if (beams > BJ_BEAMS) return fail(ctx, CATEN_B200_EUNSUPPORTED, "beam_reorder_pages: %lld beams (at most %d)", (long long)beams, BJ_BEAMS);
  if (page_nbytes % 16 || page_nbytes / 16 > 0x7fffffffll * 256) return fail(ctx, CATEN_B200_EUNSUPPORTED, "beam_reorder_pages: pages of %lld bytes (a multiple of 16)", (long long)page_nbytes);
  if (groups && (!d_pool || !d_table || !d_lengths || !d_parents)) return fail(ctx, CATEN_B200_EINVAL, "beam_reorder_pages: NULL argument");
  if ((uintptr_t)d_pool % 16) return fail(ctx, CATEN_B200_EINVAL, "beam_reorder_pages: the pool has to start on a multiple of 16 bytes");
  if (!ctx) return fail(nullptr, CATEN_B200_EINVAL, "beam_reorder_pages: ctx is NULL");
  cudaSetDevice(ctx->device);
  ctx->work_outside = true;
  if (!groups) return 0;
  ProfScope prof(ctx, CATEN_B200_K_PREP);
  const PagesReorderArgs a = {(uint8_t *)d_pool, d_table, d_lengths, d_parents, ctx->d_status, page_nbytes / 16, pages, (int)max_pages, (int)page, (int)beams};
  const dim3 grid(beams == 1 ? 1u : (unsigned)((a.page_words + 255) / 256), beams == 1 ? 1u : (unsigned)max_pages, (unsigned)groups);
  void (*kernel)(PagesReorderArgs) = beams <= 4 ? beam_reorder_pages_kernel<4> : beams <= 8 ? beam_reorder_pages_kernel<8> : beams <= 16 ? beam_reorder_pages_kernel<16> : beam_reorder_pages_kernel<32>;
  CB_CUDA(ctx, launch_k(ctx, kernel, grid, dim3(256), 0, a));
  CB_LAUNCH_CHECK(ctx, "beam_reorder_pages_kernel");
  return 0;
}

}  // extern "C"
