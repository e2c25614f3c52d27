// Beam search: selection over beams and vocabulary, and the reordering of states behind it.  No counterpart in the reference, whose
// generate loop is greedy (apps/gpt2/gpt2.lisp:97-113).
//
// Selection.  Candidate (beam b, token v) has the value score_b + x_bv - lse_b, lse_b = max + log(sum exp(x - max)); the first `keep` by value,
// equal ones by b * V + v.  Within a beam that order is the order of the logits, so a pass over the logits needs no lse: each block reads a chunk
// of a row once into registers and leaves its maximum, its sum of exponentials and its `keep` largest logits; a second kernel joins the
// chunks' sums in 64 bits, turns the few logits left into values and merges them.
#include <algorithm>

#include "common.cuh"
#include "kv4.cuh"

namespace cb {

constexpr int BS_THREADS = 256, BS_VECS = 8, BS_CHUNK = BS_THREADS * BS_VECS * 4;   // a thread holds 32 logits
constexpr int BS_KEEP = 32;   // a warp's lanes

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
// the 32 largest of two descending lists, descending
__device__ __forceinline__ u64 warp_merge(u64 a, u64 b) {
  const int lane = threadIdx.x & 31;
  const u64 r = __shfl_sync(0xffffffffu, b, 31 - lane);
  u64 key = a > r ? a : r;
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) {
    const u64 other = __shfl_xor_sync(0xffffffffu, key, j);
    key = ((lane & j) == 0) == (other > key) ? other : key;
  }
  return key;
}

// What a block leaves of its chunk: `keep` keys (descending, 0 behind the last), then maximum and sum.
__host__ __device__ __forceinline__ int64_t beam_part_words(int keep) { return keep + 1; }

__global__ void __launch_bounds__(BS_THREADS) beam_chunk_kernel(const float *__restrict__ x, const uint8_t *__restrict__ ended, int64_t V, int keep, u64 *__restrict__ parts) {
  __shared__ float red[BS_THREADS / 32];
  __shared__ u64 lists[BS_THREADS / 32][32];
  __shared__ u64 found[BS_KEEP * BS_VECS * 4];
  __shared__ u64 threshold;
  __shared__ int count;
  pdl_enter();
  const int64_t row = blockIdx.y;
  if (ended && ended[row]) return;   // its one candidate needs no logits
  const float *p = x + row * V;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // chunks start on 16-byte boundaries of memory, wherever the row does
  const int64_t e0 = (int64_t)blockIdx.x * BS_CHUNK - (int64_t)(((uintptr_t)p >> 2) & 3);
  float v[BS_VECS][4];
#pragma unroll
  for (int i = 0; i < BS_VECS; ++i) {
    const int64_t e = e0 + (i * BS_THREADS + tid) * 4;
    if (e >= 0 && e + 4 <= V) {
      const float4 q = __ldcs(reinterpret_cast<const float4 *>(p + e));
      v[i][0] = q.x; v[i][1] = q.y; v[i][2] = q.z; v[i][3] = q.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[i][j] = e + j >= 0 && e + j < V ? p[e + j] : -INFINITY;
    }
  }
  // the thread's largest, the block's
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < BS_VECS; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) top = fmaxf(top, v[i][j]);
  u64 best = 0;
#pragma unroll
  for (int i = BS_VECS - 1; i >= 0; --i)
#pragma unroll
    for (int j = 3; j >= 0; --j)
      if (v[i][j] == top) best = beam_key(v[i][j], (int)(e0 + (i * BS_THREADS + tid) * 4 + j));   // (the lowest index of equal ones)
  float m = top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) red[warp] = m;
  lists[warp][lane] = warp_sort(best);
  if (tid == 0) { threshold = 1; count = 0; }
  __syncthreads();
  m = red[0];
#pragma unroll
  for (int w = 1; w < BS_THREADS / 32; ++w) m = fmaxf(m, red[w]);
  // the keep-th largest of the threads' largest: nothing below it is among the chunk's `keep` largest.  A key's rank is the number of
  // larger ones, found in each warp's descending list by bisection.
  if (lane < keep) {
    const u64 mine = lists[warp][lane];
    int rank = 0;
#pragma unroll
    for (int w = 0; w < BS_THREADS / 32; ++w) {
      int lo = 0;
#pragma unroll
      for (int step = 16; step > 0; step >>= 1)
        if (lists[w][lo + step - 1] > mine) lo += step;
      rank += lo + (lists[w][lo] > mine ? 1 : 0);
    }
    if (mine && rank == keep - 1) threshold = mine;
  }
  // sum of exponentials; a maximum of -inf (nothing left) makes it 0, a NaN or +inf makes it NaN
  // (x - max) log2 e with the constant in two parts: rounded to one, it would shift every sum by 1e-8 of the distance
  const float base = m == -INFINITY ? 0.0f : m;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < BS_VECS; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float d = v[i][j] - base;
      float e;
      asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(d, 1.44269502162933349609375f, d * 1.925963033500e-8f)));
      s[j] += m < INFINITY ? e : NAN;
    }
  float sum = (s[0] + s[1]) + (s[2] + s[3]);
  sum = warp_sum(sum);
  __syncthreads();   // threshold, and red has been read
  if (lane == 0) red[warp] = sum;
  const u64 least = threshold;
  if (best >= least) {
    const float floor_value = beam_key_value(least);
#pragma unroll
    for (int i = 0; i < BS_VECS; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (least == 1 || v[i][j] >= floor_value) {
          const u64 key = beam_key(v[i][j], (int)(e0 + (i * BS_THREADS + tid) * 4 + j));
          if (key >= least) found[atomicAdd(&count, 1)] = key;   // (at most `keep` threads, or fewer, get here: at most 32 keys each)
        }
  }
  __syncthreads();
  if (warp) return;
  const int n = count;
  u64 list = warp_sort(lane < n ? found[lane] : 0ull);
  for (int i = 32; i < n; i += 32) list = warp_merge(list, warp_sort(i + lane < n ? found[i + lane] : 0ull));
  u64 *part = parts + (row * gridDim.x + blockIdx.x) * beam_part_words(keep);
  if (lane < keep) part[lane] = list;
  sum = red[0];
#pragma unroll
  for (int w = 1; w < BS_THREADS / 32; ++w) sum += red[w];
  if (lane == 0) part[keep] = (u64)__float_as_uint(base) << 32 | __float_as_uint(sum);
}

// ---- the chunks' lists into one --------------------------------------------------------------------
struct Cand {
  u64 value;      // order-preserving image of the 64-bit value; 0: none
  uint32_t index; // beam * V + token, complemented
  __device__ __forceinline__ bool operator>(const Cand &o) const { return value > o.value || (value == o.value && index > o.index); }
};
__device__ __forceinline__ u64 order_of(double x) {
  const u64 b = (u64)__double_as_longlong(x + 0.0);
  return !(x > -INFINITY) ? 0ull : (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}
__device__ __forceinline__ double value_of(u64 k) { return __longlong_as_double((long long)((k >> 63) ? (k & 0x7fffffffffffffffull) : ~k)); }
__device__ __forceinline__ Cand cand_shfl_xor(const Cand &c, int j) { return {__shfl_xor_sync(0xffffffffu, c.value, j), __shfl_xor_sync(0xffffffffu, c.index, j)}; }
__device__ __forceinline__ Cand cand_merge(const Cand &a, const Cand &b) {
  const int lane = threadIdx.x & 31;
  const Cand r = {__shfl_sync(0xffffffffu, b.value, 31 - lane), __shfl_sync(0xffffffffu, b.index, 31 - lane)};
  Cand c = a > r ? a : r;
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) {
    const Cand o = cand_shfl_xor(c, j);
    c = ((lane & j) == 0) == (o > c) ? o : c;
  }
  return c;
}

constexpr int BJ_THREADS = 256;
constexpr int BJ_BEAMS = 32;

__global__ void __launch_bounds__(BJ_THREADS) beam_join_kernel(const u64 *__restrict__ parts, int chunks, const float *__restrict__ scores, const uint8_t *__restrict__ ended,
                                                               int beams, int64_t V, int64_t eos, int keep, float *__restrict__ out_scores, int *__restrict__ out_parents,
                                                               int64_t *__restrict__ out_tokens, uint8_t *__restrict__ out_ended) {
  __shared__ double base[BJ_BEAMS], tops[BJ_BEAMS];   // a candidate's value: base + (x - top)
  __shared__ uint8_t over[BJ_BEAMS];
  __shared__ Cand lists[BJ_THREADS / 32][32];
  pdl_enter();
  const int64_t batch = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t words = beam_part_words(keep);
  for (int b = warp; b < beams; b += BJ_THREADS / 32) {
    const int64_t row = batch * beams + b;
    const float score = scores[row];
    const bool end = ended && ended[row];
    double log_sum = 0.0, top = 0.0;
    if (!end) {
      const u64 *part = parts + row * chunks * words + keep;
      float m = -INFINITY;
      bool none = true;
      double s = 0.0;
      for (int c = lane; c < chunks; c += 32) {
        const u64 w = part[c * words];
        const float pm = __uint_as_float((uint32_t)(w >> 32)), ps = __uint_as_float((uint32_t)w);
        if (ps == 0.0f) continue;   // nothing in that chunk
        if (none || pm > m) { s = none ? (double)ps : s * exp((double)m - (double)pm) + (double)ps; m = pm; }
        else s += (double)ps * exp((double)pm - (double)m);
        none = false;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const float om = __shfl_xor_sync(0xffffffffu, m, o);
        const double os = __shfl_xor_sync(0xffffffffu, s, o);
        const float both = fmaxf(m, om);
        const double a = m == -INFINITY ? 0.0 : s * exp((double)m - (double)both), c = om == -INFINITY ? 0.0 : os * exp((double)om - (double)both);
        s = a + c;
        m = both;
      }
      log_sum = log(s);   // (nothing left in the row: -inf, but then there is no key either)
      top = (double)m;
    }
    if (lane == 0) {
      base[b] = (double)score - log_sum;
      tops[b] = top;
      over[b] = end;
    }
  }
  __syncthreads();
  Cand best = {0ull, 0u};
  const int total = beams * chunks;
  for (int i = warp; i < total; i += BJ_THREADS / 32) {
    const int b = i / chunks, c = i % chunks;
    const int64_t row = batch * beams + b;
    Cand mine = {0ull, 0u};
    if (over[b]) {
      if (c == 0 && lane == 0 && eos >= 0 && eos < V) {
        mine.value = order_of(base[b]);
        mine.index = ~(uint32_t)(b * V + eos);
      }
    } else {
      const u64 key = lane < keep ? parts[(row * chunks + c) * words + lane] : 0ull;
      if (key) {
        mine.value = order_of(base[b] + ((double)beam_key_value(key) - tops[b]));
        mine.index = ~(uint32_t)(b * V + beam_key_index(key));
      }
    }
    if (!mine.value) mine.index = 0;
    // (a list whose first is behind this warp's last so far adds nothing)
    const u64 head = __shfl_sync(0xffffffffu, mine.value, 0), tail = __shfl_sync(0xffffffffu, best.value, keep - 1);
    if (head && head >= tail) best = cand_merge(best, mine);
  }
  lists[warp][lane] = best;
  __syncthreads();
  if (warp) return;
#pragma unroll 1
  for (int w = 1; w < BJ_THREADS / 32; ++w) {
    const Cand other = lists[w][lane];
    if (__shfl_sync(0xffffffffu, other.value, 0)) best = cand_merge(best, other);
  }
  if (lane < keep) {
    const int64_t at = batch * keep + lane;
    const bool there = best.value != 0;
    const uint32_t index = ~best.index;
    const int parent = there ? (int)(index / (uint64_t)V) : min(lane, beams - 1);
    const int64_t token = there ? (int64_t)(index % (uint64_t)V) : eos >= 0 ? eos : 0;
    out_scores[at] = there ? (float)value_of(best.value) : -INFINITY;
    out_parents[at] = parent;
    out_tokens[at] = token;
    if (out_ended) out_ended[at] = over[parent] || (eos >= 0 && token == eos);
  }
}

static int64_t beam_chunks(int64_t V) { return (V + 3 + BS_CHUNK - 1) / BS_CHUNK; }

static int beam_check(caten_b200_ctx *ctx, const char *who, int64_t batch, int64_t beams, int64_t V, int64_t keep) {
  if (batch < 0 || beams <= 0 || V <= 0 || keep <= 0) return fail(ctx, CATEN_B200_EINVAL, "%s: bad shape", who);
  if (beams > BJ_BEAMS || keep > BS_KEEP) return fail(ctx, CATEN_B200_EUNSUPPORTED, "%s: %lld beams, %lld kept (at most %d)", who, (long long)beams, (long long)keep, BS_KEEP);
  if (V > 0x7fffffffll / BJ_BEAMS) return fail(ctx, CATEN_B200_EUNSUPPORTED, "%s: V=%lld", who, (long long)V);
  if (batch > 65535 || batch * beams > 65535) return fail(ctx, CATEN_B200_EUNSUPPORTED, "%s: %lld rows", who, (long long)(batch * beams));
  return 0;
}

// ---- reordering ------------------------------------------------------------------------------------
// Row i of a group becomes what row parent(i) was, in place: a thread takes the same 16 (or 4) bytes of all the group's rows that change into
// registers before it writes any of them, so nothing is read after it was overwritten, whatever the parents are.  Rows that stay
// are neither read for themselves nor written.
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
  return (batch * beams * beam_chunks(V) * beam_part_words((int)keep) + 1) * (int64_t)sizeof(u64);
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
  const int64_t chunks = beam_chunks(V);
  CB_CUDA(ctx, launch_k(ctx, beam_chunk_kernel, dim3((unsigned)chunks, (unsigned)(batch * beams)), dim3(BS_THREADS), 0, d_logits, d_ended, V, (int)keep, (u64 *)d_work));
  CB_LAUNCH_CHECK(ctx, "beam_chunk_kernel");
  CB_CUDA(ctx, launch_k(ctx, beam_join_kernel, dim3((unsigned)batch), dim3(BJ_THREADS), 0, (const u64 *)d_work, (int)chunks, d_scores, d_ended, (int)beams, V, eos, (int)keep,
                        d_out_scores, d_out_parents, d_out_tokens, d_out_ended));
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
  if (!groups || !nbytes || beams == 1) return 0;
  ProfScope prof(ctx, CATEN_B200_K_PREP);
  for (int64_t first = 0; first < count; first += RO_STATES) {
    ReorderArgs a;
    const int64_t n = count - first < RO_STATES ? count - first : RO_STATES;
    for (int64_t i = 0; i < n; ++i) a.state[i] = h_states[first + i];
    a.parents = d_parents; a.status = ctx->d_status;
    a.planes = planes; a.stride = plane_stride / width; a.words = words; a.beams = (int)beams;
    const dim3 grid((unsigned)((planes * words + 255) / 256), (unsigned)groups, (unsigned)n);
    CB_CUDA(ctx, width == 16 ? reorder_launch<uint4>(ctx, grid, a) : reorder_launch<uint32_t>(ctx, grid, a));
    CB_LAUNCH_CHECK(ctx, "beam_reorder_kernel");
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
  if (!groups || beams == 1) return 0;
  ProfScope prof(ctx, CATEN_B200_K_PREP);
  const PagesReorderArgs a = {(uint8_t *)d_pool, d_table, d_lengths, d_parents, ctx->d_status, page_nbytes / 16, pages, (int)max_pages, (int)page, (int)beams};
  const dim3 grid((unsigned)((a.page_words + 255) / 256), (unsigned)max_pages, (unsigned)groups);
  void (*kernel)(PagesReorderArgs) = beams <= 4 ? beam_reorder_pages_kernel<4> : beams <= 8 ? beam_reorder_pages_kernel<8> : beams <= 16 ? beam_reorder_pages_kernel<16> : beam_reorder_pages_kernel<32>;
  CB_CUDA(ctx, launch_k(ctx, kernel, grid, dim3(256), 0, a));
  CB_LAUNCH_CHECK(ctx, "beam_reorder_pages_kernel");
  return 0;
}

}  // extern "C"
