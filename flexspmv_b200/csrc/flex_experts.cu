// Routed expert layers: the router (softmax over the experts, the k largest, the plan in expert order), its gradient, and the weighted
// reduce of the experts' results into the tokens' rows, with its gradient.  The matrix products between them: flex_grouped.cu.
//
// A plan is what flexspmv_sort_rows makes of an unsorted Reducer, for (token, choice) pairs and the experts as rows: the pairs in
// a stable order by expert, `offsets` (where an expert's pairs begin), `slots` (pair -> place in that order) and `rows` (place -> token).
#include <cuda_runtime.h>

#include <type_traits>

#include "flex_common.cuh"
#include "flex_expert_types.cuh"
#include "flex_umma.cuh"

namespace flex {

int device_sm_count();

// ---- router --------------------------------------------------------------------------------------------------------

// 2^x by the special-function unit (relative error 2^-22, results below 2^-126 are 0).
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f;
// e^(v - top).  The difference first: top log2 e as one rounded number would put an error of 2^-24 |top| into the power.  The product's rounding
// is left, d * 6e-8 of the power for a difference of d: for sums of powers, where it counts e^-d, and for results of 16 bits.
__device__ __forceinline__ float exp_below(float v, float top) { return exp2_fast((v - top) * kLog2e); }
// For results of 32 bits: to 3 units of the result whatever the difference, whose own rounding is made up for (Knuth's exact sum of two numbers).
__device__ __forceinline__ float exp_below_exact(float v, float top) {
  const float d = v - top, w = d - v, lost = (v - (d - w)) - (top + w), e = expf(d);
  return fmaf(e, fminf(lost, 1e-5f), e);           // less than 4e-6 wherever e is not 0, no number where d is infinite
}

// What a choice goes by: a number that is larger for a larger logit and, among equal ones, for a lower expert.  The order of a sign and
// magnitude number x is 0x8000... +- its magnitude (so that -0 and 0 are equal); NaN's is 0.  kNone: the key of -infinity and below, never chosen.
// The expert makes all keys of a row different, NaN's too, and none of them 0.
// A 16-bit logit and the expert fit 32 bits, so that one instruction finds the largest of a warp; a 32-bit one takes 64.
template <class T>
struct Choice {
  using Key = uint32_t;
  static constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  static constexpr Key kNone = (0x8000u - kInf) << 16 | 0xffffu;
  static __device__ __forceinline__ int expert(Key k) { return (int)(0xffffu - (k & 0xffffu)); }
  static __device__ __forceinline__ float logit(Key k) {
    const uint32_t order = k >> 16, u = order & 0x8000u ? order & 0x7fffu : 0x10000u - order;      // 0x8000 | (0x8000 - order)
    if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)u));
    else return __uint_as_float(u << 16);
  }
  static __device__ __forceinline__ Key warp_max(Key k) { return __reduce_max_sync(0xffffffffu, k); }
  // The orders of two logits in one word.  Sign bits spread over their halves by a byte permutation (0xbb99).
  static __device__ __forceinline__ uint32_t spread(uint32_t two) {
    uint32_t r;
    asm("prmt.b32 %0, %1, 0, 0xbb99;" : "=r"(r) : "r"(two));
    return r;
  }
  static __device__ __forceinline__ uint32_t orders(uint32_t two) {
    const uint32_t negative = spread(two), nan = spread((two & 0x7fff7fffu) + (0x7fffu - kInf) * 0x00010001u);
    return ((two ^ ((negative & 0x7fff7fffu) ^ 0x80008000u)) + (negative & 0x00010001u)) & ~nan;
  }
};
template <>
struct Choice<float> {
  using Key = unsigned long long;
  static constexpr Key kNone = (Key)0x00800000u << 32 | 0xffffu;
  static __device__ __forceinline__ Key make(float v, int e) {
    const uint32_t u = __float_as_uint(v), order = u & 0x80000000u ? 0u - u : u | 0x80000000u;       // 0x80000000 - magnitude
    return (Key)(v != v ? 0u : order) << 32 | (0xffffu - (uint32_t)e);
  }
  static __device__ __forceinline__ int expert(Key k) { return (int)(0xffffu - (uint32_t)k); }
  static __device__ __forceinline__ float logit(Key k) {
    const uint32_t order = (uint32_t)(k >> 32);
    return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : 0u - order);
  }
  static __device__ __forceinline__ Key warp_max(Key k) {
    const uint32_t high = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
    return (Key)high << 32 | __reduce_max_sync(0xffffffffu, high == (uint32_t)(k >> 32) ? (uint32_t)k : 0u);
  }
};

// Largest first, by odd-even merging (Batcher): exchanges whose places are known when it is compiled.  The rounds are a recursion, since as loops
// the compiler left those of 16 keys of 64 bits in place and the keys in local memory (us, 8192 tokens of 500 experts in 32 bits 35.5 / 25.8, of 1024
// in 16 bits 76.5 / 32.8).
template <int P, int Q, class K, int V>
__device__ __forceinline__ void sort_down_from(K (&k)[V]) {
#pragma unroll
  for (int j = Q % P; j + Q < V; j += 2 * Q)
#pragma unroll
    for (int i = 0; i < Q; ++i)
      if (i + j + Q < V && (i + j) / (2 * P) == (i + j + Q) / (2 * P)) {
        const K x = k[i + j], y = k[i + j + Q];
        k[i + j] = x > y ? x : y;
        k[i + j + Q] = x > y ? y : x;
      }
  if constexpr (Q > 1) sort_down_from<P, Q / 2>(k);
  else if constexpr (2 * P < V) sort_down_from<2 * P, 2 * P>(k);
}

template <class K, int V>
__device__ __forceinline__ void sort_down(K (&k)[V]) {
  if constexpr (V > 1) sort_down_from<1, 1>(k);
}

// A row's part of lane l: V experts, W neighbouring ones at a time.  What lies beyond the experts is -infinity.
template <class T, int V, int W>
struct LanePart {
  Pack<T, W> piece[V / W];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < V; ++i) piece[i / W].set(i % W, -INFINITY);
  }
  __device__ __forceinline__ void load(const T* row, int experts, int lane) {
#pragma unroll
    for (int i = 0; i < V / W; ++i) {
      const int e = (i * 32 + lane) * W;
      if (e < experts) piece[i].load(row + e);
    }
  }
};

// One token by one warp.  Each lane sorts its experts once and leaves them in shared memory (`list`, V + 1 keys a lane); then k rounds of a
// maximum over the lanes' first ones, the winner's lane taking up its next (equal logits: the lowest expert, as the plain form's stable
// sort has it).  Lane j ends with choice j.  The softmax is over the true logits, largest subtracted, sums in 32 bits.
// Bound by instructions: 660 a token of 256 experts where every round moved the sorted keys up in registers and every logit was made a key
// and a power on its own.
template <class T, int V, int W>
__device__ __forceinline__ void choose_token(const LanePart<T, V, W>& part, int k, bool renormalize, int lane, typename Choice<T>::Key* list, int& my_id,
                                             float& my_weight) {
  using C = Choice<T>;
  using Key = typename C::Key;
  Key key[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const uint32_t e = (uint32_t)((i / W * 32 + lane) * W + i % W);
    if constexpr (std::is_same<T, float>::value) {
      key[i] = C::make(part.piece[i / W].get(i % W), (int)e);
    } else if constexpr (W > 1) {
      if (i % 2 == 0) {
        const uint32_t order = C::orders(part.piece[i / W].word(i % W / 2));
        key[i] = order << 16 | (0xffffu - e);
        key[i + 1] = (order & 0xffff0000u) | (0xfffeu - e);
      }
    } else {
      key[i] = C::orders(part.piece[i].bits()) << 16 | (0xffffu - e);
    }
  }
  sort_down(key);
#pragma unroll
  for (int i = 1; i < V; ++i) list[i] = key[i];
  Key first = key[0], mine_key = 0;
  const Key* next = list + 1;
#pragma unroll 4
  for (int j = 0; j < k; ++j) {
    const Key most = C::warp_max(first);
    if (lane == j) mine_key = most;
    if (first == most) first = *next++;          // one lane's: all 32 V keys differ, and as k <= experts <= 32 V a round always finds one before the zeros
  }
  if (mine_key <= C::kNone) mine_key = 0;
  const Key top_key = __shfl_sync(0xffffffffu, mine_key, 0);
  my_id = mine_key ? C::expert(mine_key) : -1;
  const float top = top_key ? C::logit(top_key) : 0.f;
  const float mine = mine_key ? exp_below_exact(C::logit(mine_key), top) : 0.f;
  float sum = 0.f;
  if (renormalize) {
    sum = mine;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) sum += exp_below(part.piece[i / W].get(i % W), top);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  my_weight = mine_key ? __fdividef(mine, sum) : 0.f;          // to 2 units
}

struct RouteArgs {
  const void* logits;
  long long tokens, stride;
  int experts, k, renormalize;
  long long chunk;                 // tokens of a CTA
  float* weights;
  int *ids, *offsets, *rows, *slots;
  unsigned* counts;                // [CTAs][experts, a multiple of four]
};

// Choices of this CTA's tokens, a run of them for each warp.  `seen` (shared, [warps][experts]) counts each warp's pairs of an expert, in
// their order and without atomics: a token's experts are different ones.  In the end slots[pair] is the pair's number among the CTA's pairs of its
// expert, and total[e] (shared) how many there are.
template <class T, int V, int W, int THREADS>
__device__ __forceinline__ void choose_chunk(const RouteArgs& a, unsigned* seen, unsigned* total) {
  using Key = typename Choice<T>::Key;
  Key* const lists = reinterpret_cast<Key*>(seen + (a.experts * (THREADS / 32) + 1) / 2 * 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Key* const list = lists + threadIdx.x * (V + 1);
  list[V] = 0;
  for (int i = threadIdx.x; i < a.experts * (THREADS / 32); i += THREADS) seen[i] = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const long long first = a.chunk * blockIdx.x, last = first + a.chunk < a.tokens ? first + a.chunk : a.tokens;
  const long long each = (a.chunk + THREADS / 32 - 1) / (THREADS / 32);
  const long long from = first + warp * each, to = from + each < last ? from + each : last;
  const T* const logits = static_cast<const T*>(a.logits);
  unsigned* const mine = seen + warp * a.experts;
  LanePart<T, V, W> next;
  next.clear();
  if (from < to) next.load(logits + from * a.stride, a.experts, lane);
  for (long long t = from; t < to; ++t) {
    const LanePart<T, V, W> part = next;
    if (t + 1 < to) next.load(logits + (t + 1) * a.stride, a.experts, lane);
    int id;
    float weight;
    choose_token<T, V, W>(part, a.k, a.renormalize != 0, lane, list, id, weight);
    if (lane < a.k) {
      a.weights[t * a.k + lane] = weight;
      a.ids[t * a.k + lane] = id;
      int number = -1;
      if (id >= 0) number = (int)mine[id]++;
      a.slots[t * a.k + lane] = number;
    }
    __syncwarp();
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += THREADS) {
    unsigned sum = 0;
#pragma unroll 8
    for (int w = 0; w < THREADS / 32; ++w) {
      const unsigned n = seen[w * a.experts + e];
      seen[w * a.experts + e] = sum;
      sum += n;
    }
    total[e] = sum;
  }
  __syncthreads();
  for (long long p = from * a.k + lane; p < to * a.k; p += 32) {
    const int id = a.ids[p];
    if (id >= 0) a.slots[p] += (int)mine[id];
  }
}

// total[e] becomes the sum of those before it; returns the sum of all.  With `offsets`, they are also written there.
template <int THREADS>
__device__ __forceinline__ unsigned sums_before(unsigned* total, int experts, int* offsets) {
  constexpr int kWarps = THREADS / 32;
  __shared__ unsigned warp_sum[32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned done = 0;
  for (int base = 0; base < experts; base += THREADS) {
    const int e = base + tid;
    const unsigned n = e < experts ? total[e] : 0u;
    unsigned s = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned up = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += up;
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = s;
    __syncthreads();
    const unsigned mine = lane < kWarps ? warp_sum[lane] : 0u;
    const unsigned prior = __reduce_add_sync(0xffffffffu, lane < warp ? mine : 0u), all = __reduce_add_sync(0xffffffffu, mine);
    if (e < experts) {
      total[e] = done + prior + s - n;
      if (offsets) offsets[e] = (int)(done + prior + s - n);
    }
    done += all;
  }
  if (offsets && tid == 0) offsets[experts] = (int)done;
  __syncthreads();
  return done;
}

// Small batches: everything in one CTA and one launch.
template <class T, int V, int W, int THREADS>
__global__ void __launch_bounds__(THREADS) route_small_kernel(RouteArgs a) {
  extern __shared__ __align__(16) unsigned route_sm[];
  unsigned* const total = route_sm;
  choose_chunk<T, V, W, THREADS>(a, total + (a.experts + 1) / 2 * 2, total);
  const unsigned used = sums_before<THREADS>(total, a.experts, a.offsets);
  const int pairs = (int)a.tokens * a.k;
  for (int p = threadIdx.x; p < pairs; p += THREADS) {
    const int id = a.ids[p];
    if (id >= 0) {
      const int place = a.slots[p] + (int)total[id];
      a.slots[p] = place;
      a.rows[place] = p / a.k;
    }
    if (p >= (int)used) a.rows[p] = -1;
  }
}

template <class T, int V, int W, int THREADS>
__global__ void __launch_bounds__(THREADS) route_choose_kernel(RouteArgs a) {
  extern __shared__ __align__(16) unsigned route_sm[];
  unsigned* const total = route_sm;
  choose_chunk<T, V, W, THREADS>(a, total + (a.experts + 1) / 2 * 2, total);
  const int wide = (a.experts + 3) / 4 * 4;              // the place kernel reads four at a time
  for (int i = threadIdx.x; i < wide; i += THREADS) a.counts[(size_t)blockIdx.x * wide + i] = i < a.experts ? total[i] : 0u;
}

// Every CTA adds up the counts of all CTAs by itself (they lie in L2): a launch fewer than a scan between the two would take.
constexpr int kPlaceThreads = 1024;
__global__ void __launch_bounds__(kPlaceThreads) route_place_kernel(RouteArgs a) {
  extern __shared__ unsigned route_sm[];
  unsigned *total = route_sm, *before = total + a.experts;
  for (int i = threadIdx.x; i < a.experts; i += kPlaceThreads) total[i] = before[i] = 0;
  __syncthreads();
  pdl_wait();
  const long long from = a.chunk * blockIdx.x * a.k, end = from + a.chunk * a.k, pairs = a.tokens * a.k, to = end < pairs ? end : pairs;
  int id[2], number[2];                    // this thread's first pairs, under way while the counts are added up
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const long long p = from + threadIdx.x + u * kPlaceThreads;
    id[u] = p < to ? a.ids[p] : -1;
    number[u] = p < to ? a.slots[p] : -1;
  }
  // as many threads on four experts as there are; each adds every parts-th CTA's counts
  const int fours = (a.experts + 3) / 4, parts = kPlaceThreads / fours;
  for (int i = threadIdx.x; i < fours * parts; i += kPlaceThreads) {
    const int e = i % fours * 4, part = i / fours;
    unsigned all[4] = {}, prior[4] = {};
#pragma unroll 8
    for (unsigned b = part; b < gridDim.x; b += parts) {
      const uint4 n = *reinterpret_cast<const uint4*>(a.counts + (size_t)b * fours * 4 + e);
      const unsigned c[4] = {n.x, n.y, n.z, n.w};
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        all[x] += c[x];
        prior[x] += b < blockIdx.x ? c[x] : 0u;
      }
    }
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (e + x < a.experts) {
        atomicAdd(&total[e + x], all[x]);
        if (prior[x]) atomicAdd(&before[e + x], prior[x]);
      }
  }
  __syncthreads();
  const unsigned used = sums_before<kPlaceThreads>(total, a.experts, blockIdx.x == 0 ? a.offsets : nullptr);
  for (int e = threadIdx.x; e < a.experts; e += kPlaceThreads) before[e] += total[e];
  __syncthreads();
  const auto put = [&](long long p, int i, int n) {
    if (i >= 0) {
      const int place = n + (int)before[i];
      a.slots[p] = place;
      a.rows[place] = (int)((unsigned)p / (unsigned)a.k);
    }
    if (p >= (long long)used) a.rows[p] = -1;
  };
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const long long p = from + threadIdx.x + u * kPlaceThreads;
    if (p < to) put(p, id[u], number[u]);
  }
  for (long long p = from + threadIdx.x + 2 * kPlaceThreads; p < to; p += kPlaceThreads) put(p, a.ids[p], a.slots[p]);
}

// Gradient of the chosen weights with respect to the logits.  p_i = w_0 exp(l_i - l_{e_0}): the largest weight and its logit stand for the
// softmax's maximum and sum, so that one pass over the row is enough.  A warp takes a token: first the row as if nothing were chosen,
// -p_i sum_j g_j w_j (renormalized: zeros), then the chosen ones' w_j (g_j - sum g w) over it.
template <class T, int W>
__global__ void __launch_bounds__(256) route_backward_kernel(const float* __restrict__ dweights, const T* __restrict__ logits, const float* __restrict__ weights,
                                                             const int* __restrict__ ids, T* __restrict__ dlogits, long long tokens, long long stride,
                                                             int experts, int k, int renormalize) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  for (long long t = (long long)blockIdx.x * 8 + warp; t < tokens; t += (long long)gridDim.x * 8) {
    int id = lane < k ? ids[t * k + lane] : -1;
    if (id >= experts) id = -1;              // a plan of other logits: not an expert of these
    const float w = id >= 0 ? weights[t * k + lane] : 0.f, g = id >= 0 ? dweights[t * k + lane] : 0.f;
    const T* row = logits + t * stride;
    Pack<T, W> v;
    if (!renormalize && lane * W < experts) v.load(row + lane * W);          // under way while the sum is made
    float mean = w * g;
#pragma unroll
    for (int o = 16; o; o >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, o);
    const int top_id = __shfl_sync(0xffffffffu, id, 0);
    const float top_w = __shfl_sync(0xffffffffu, w, 0);
    T* out = dlogits + t * experts;
    if (renormalize || top_id < 0) {
      Pack<T, W> none;
      none.zero();
      for (int e = lane * W; e < experts; e += 32 * W) none.store(out + e);
    } else {
      const float top = to_float(row[top_id]), scale = -top_w * mean;
      for (int e = lane * W; e < experts; e += 32 * W) {
        if (e >= 32 * W) v.load(row + e);
        Pack<T, W> r;
        // A result of 32 bits: 10 units at most, 8 below the largest.  us, 32 771 tokens of 64 experts: none by the exact power 7.5, those that are
        // further below 8.4, all 9.6.
        bool far = false;
        if constexpr (sizeof(T) == 4)
#pragma unroll
          for (int x = 0; x < W; ++x) far |= v.get(x) < top - 8.f;
        if (far)
#pragma unroll
          for (int x = 0; x < W; ++x) r.set(x, scale * exp_below_exact(v.get(x), top));
        else
#pragma unroll
          for (int x = 0; x < W; ++x) r.set(x, scale * exp_below(v.get(x), top));
        r.store(out + e);
      }
    }
    __syncwarp();
    if (id >= 0) out[id] = from_float<T>(w * (g - mean));
  }
}

// ---- balance -------------------------------------------------------------------------------------------------------

// The largest of a warp's values; NaN only where all are.
__device__ __forceinline__ float warp_largest(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
// The softmax of a row whose part is in this warp's lanes: powers in e, their base and the factor that makes probabilities of them.  A row of -infinity
// alone has none: its powers are 0.  `more`: other values that are added up over the lanes, in the same steps; it gets the powers first.
template <class T, int V, int W, int N, class F>
__device__ __forceinline__ bool softmax_of(const LanePart<T, V, W>& part, float (&e)[V], float& base, float& factor, float (&more)[N], const F& before) {
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) top = fmaxf(top, part.piece[i / W].get(i % W));
  top = warp_largest(top);
  const bool there = top > -INFINITY;
  base = there ? top : 0.f;
  // 32-bit logits far below the largest: as in the router's gradient
  bool far = false;
  if constexpr (std::is_same<T, float>::value)
#pragma unroll
    for (int i = 0; i < V; ++i) far |= part.piece[i / W].get(i % W) < base - 8.f;
  if (far) {
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = exp_below_exact(part.piece[i / W].get(i % W), base);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = exp_below(part.piece[i / W].get(i % W), base);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) sum += e[i];
  before();
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
    for (int n = 0; n < N; ++n) more[n] += __shfl_xor_sync(0xffffffffu, more[n], o);
  }
  factor = there ? __frcp_rn(sum) : 1.f;
  return there;
}

struct BalanceArgs {
  const void* logits;
  const int* offsets;
  long long tokens, stride;
  int experts;
  float* parts;                    // [clusters][experts]: sums of the probabilities of a cluster's tokens
  int* part_tokens;                // [clusters]: its rows that are not all -infinity
  float *loss, *mean;
  int *counts, *there;
};

// loss = experts / (pairs tokens) sum_e counts[e] total[e], counts from the plan's offsets; total in shared memory.
template <int THREADS>
__device__ __forceinline__ void balance_end(const BalanceArgs& a, const float* total, int tokens) {
  __shared__ float warp_sum[THREADS / 32];
  const float inverse = __frcp_rn((float)(tokens > 0 ? tokens : 1));
  float sum = 0.f;
  for (int e = threadIdx.x; e < a.experts; e += THREADS) {
    const int count = a.offsets[e + 1] - a.offsets[e];
    const float mean = total[e] * inverse;
    a.counts[e] = count;
    a.mean[e] = mean;
    sum = fmaf((float)count, mean, sum);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (threadIdx.x % 32 == 0) warp_sum[threadIdx.x / 32] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    float all = 0.f;
    for (int w = 0; w < THREADS / 32; ++w) all += warp_sum[w];
    const int pairs = a.offsets[a.experts] - a.offsets[0];
    *a.loss = all * (float)a.experts / (float)(pairs > 0 ? pairs : 1);
    *a.there = tokens;
  }
}

// A warp takes every so-many-th token and keeps its lanes' experts' sums in registers; the warps' and two CTAs' sums meet in shared memory, the clusters' in a second
// launch, each in a fixed order.  Bound by memory with many tokens (the logits are read once), by the launch with few (SMALL: one CTA does it all).
// us, 32 771 tokens of 256 experts in 16 bits: 13.5; with 16 warps an SM 15.9, two tokens a warp at a time 14.3, single CTAs 14.4, clusters of four, not all of which
// are on the chip at once, 19.8.
constexpr int kBalanceCtas = 2;
template <class T, int V, int W, int THREADS, bool SMALL>
__global__ void __launch_bounds__(THREADS) balance_kernel(BalanceArgs a) {
  extern __shared__ __align__(16) float balance_sm[];          // [warps][experts]
  __shared__ int seen[THREADS / 32];
  constexpr int kWarps = THREADS / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long step = (long long)gridDim.x * kWarps;
  const T* const logits = static_cast<const T*>(a.logits);
  pdl_wait();
  pdl_launch_dependents();
  float acc[V];
#pragma unroll
  for (int i = 0; i < V; ++i) acc[i] = 0.f;
  int there = 0;
  LanePart<T, V, W> next;
  next.clear();
  long long t = (long long)blockIdx.x * kWarps + warp;
  if (t < a.tokens) next.load(logits + t * a.stride, a.experts, lane);
  for (; t < a.tokens; t += step) {
    const LanePart<T, V, W> part = next;
    if (t + step < a.tokens) next.load(logits + (t + step) * a.stride, a.experts, lane);
    float e[V], base, factor, none[1] = {0.f};
    there += softmax_of<T, V, W>(part, e, base, factor, none, [] {});
#pragma unroll
    for (int i = 0; i < V; ++i) acc[i] = fmaf(e[i], factor, acc[i]);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = (i / W * 32 + lane) * W + i % W;
    if (e < a.experts) balance_sm[warp * a.experts + e] = acc[i];
  }
  if (lane == 0) seen[warp] = there;
  __syncthreads();
  int tokens = 0;
  for (int w = 0; w < kWarps; ++w) tokens += seen[w];
  for (int e = threadIdx.x; e < a.experts; e += THREADS) {
    float sum = 0.f;
#pragma unroll 8
    for (int w = 0; w < kWarps; ++w) sum += balance_sm[w * a.experts + e];
    balance_sm[e] = sum;                   // column e is this thread's alone
  }
  if (SMALL) {
    __syncthreads();
    balance_end<THREADS>(a, balance_sm, tokens);
    return;
  }
  __shared__ int cta_tokens;
  if (threadIdx.x == 0) cta_tokens = tokens;
  cluster_sync();
  const int share = (int)cluster_rank(), cluster = blockIdx.x / kBalanceCtas;
  for (int e = threadIdx.x * kBalanceCtas + share; e < a.experts; e += THREADS * kBalanceCtas) {
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < kBalanceCtas; ++c) sum += cluster_load(cluster_smem(&balance_sm[e], c));
    a.parts[(size_t)cluster * a.experts + e] = sum;
  }
  if (share == 0 && threadIdx.x == 0) {
    int all = 0;
    for (int c = 0; c < kBalanceCtas; ++c) all += __float_as_int(cluster_load(cluster_smem(&cta_tokens, c)));
    a.part_tokens[cluster] = all;
  }
  cluster_sync();                          // no CTA leaves while its sums may be read
}

__global__ void __launch_bounds__(1024) balance_end_kernel(BalanceArgs a, int clusters) {
  __shared__ float total[FLEXSPMV_MAX_EXPERTS], group_sum[1024];
  __shared__ int tokens;
  const int tid = threadIdx.x, wide = (a.experts + 31) / 32 * 32, groups = 1024 / wide, group = tid / wide, e = tid % wide;
  pdl_wait();
  if (tid < 32) {
    int n = 0;
    for (int p = tid; p < clusters; p += 32) n += a.part_tokens[p];
    n = __reduce_add_sync(0xffffffffu, n);
    if (tid == 0) tokens = n;
  }
  float sum = 0.f;
  if (e < a.experts && group < groups)
#pragma unroll 8
    for (int p = group; p < clusters; p += groups) sum += a.parts[(size_t)p * a.experts + e];
  group_sum[tid] = sum;
  __syncthreads();
  if (tid < a.experts) {
    for (int g = 1; g < groups; ++g) sum += group_sum[g * wide + tid];
    total[tid] = sum;
  }
  __syncthreads();
  balance_end<1024>(a, total, tokens);
}

struct BalanceGradArgs {
  const float* dloss;
  const void* logits;
  const int *counts, *there;
  const float *dweights, *weights;     // of the router, or null
  const int* ids;
  void* dlogits;
  long long tokens, stride;
  int experts, k, renormalize;
};

// dlogits = dloss experts / (pairs tokens) p (counts - sum p counts), and with dweights the router's gradient on top, in one pass over the logits: first
// every value as if it were not chosen, then the chosen ones' over it.  A warp takes a token; the counts stay in its registers.
template <class T, int V, int W>
__global__ void __launch_bounds__(256) balance_backward_kernel(BalanceGradArgs a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  float count[V];
  int pairs = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = (i / W * 32 + lane) * W + i % W, n = e < a.experts ? a.counts[e] : 0;
    count[i] = (float)n;
    pairs += n;
  }
  pairs = __reduce_add_sync(0xffffffffu, pairs);
  const int there = *a.there;
  const float scale = *a.dloss * (float)a.experts / ((float)(pairs > 0 ? pairs : 1) * (float)(there > 0 ? there : 1));
  const T* const logits = static_cast<const T*>(a.logits);
  // one token at a time: with two (us, 32 771 tokens of 256 experts) 20.4 for 15.0
  const long long step = (long long)gridDim.x * 8;
  LanePart<T, V, W> next;
  struct Choice { int id; float w, g; } next_choice;          // a lane's choice of a token
  const auto load = [&](long long t) {
    next_choice = {-1, 0.f, 0.f};
    next.load(logits + t * a.stride, a.experts, lane);
    if (a.dweights && lane < a.k) {
      const long long p = t * a.k + lane;
      next_choice = {a.ids[p], a.weights[p], a.dweights[p]};
    }
  };
  next.clear();
  long long t = (long long)blockIdx.x * 8 + warp;
  if (t < a.tokens) load(t);
  for (; t < a.tokens; t += step) {
    const LanePart<T, V, W> part = next;
    Choice c = next_choice;
    float chosen = 0.f;
    if ((unsigned)c.id >= (unsigned)a.experts) c = {-1, 0.f, 0.f};          // not an expert of these logits: no choice
    else chosen = to_float(logits[t * a.stride + c.id]);
    if (t + step < a.tokens) load(t + step);
    float e[V], base, factor, sums[2] = {c.w * c.g, 0.f};
    softmax_of<T, V, W>(part, e, base, factor, sums, [&] {
#pragma unroll
      for (int i = 0; i < V; ++i) sums[1] = fmaf(e[i], count[i], sums[1]);
    });
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] *= factor;
    const float mean = sums[0], expected = sums[1] * factor, common = a.renormalize ? 0.f : mean;
    T* const out = static_cast<T*>(a.dlogits) + t * a.experts;
#pragma unroll
    for (int i = 0; i < V / W; ++i) {
      const int first = (i * 32 + lane) * W;
      Pack<T, W> r;
#pragma unroll
      for (int x = 0; x < W; ++x) r.set(x, e[i * W + x] * (scale * (count[i * W + x] - expected) - common));
      if (first < a.experts) r.store(out + first);
    }
    __syncwarp();
    if (c.id >= 0) {
      const float p = exp_below_exact(chosen, base) * factor, n = (float)a.counts[c.id];
      out[c.id] = from_float<T>(fmaf(p, scale * (n - expected) - common, a.renormalize ? c.w * (c.g - mean) : c.w * c.g));
    }
    __syncwarp();
  }
}

// ---- combine -------------------------------------------------------------------------------------------------------

// out[t] = sum_j w[t, j] z[slots[t, j]]: a thread takes W neighbouring columns at U places, 256 threads apart, and has the loads of K choices of
// each in flight: four loads, whatever the choices (two choices of 8192 columns: 4.1 TB/s with U = 1, 4.4 with U = 2).
// Bound by memory; the choices are added in their order, in 32 bits, rounded once.
template <class T, int W, int K, int U>
__global__ void __launch_bounds__(256) combine_kernel(const T* __restrict__ z, const int* __restrict__ slots, const float* __restrict__ weights,
                                                      T* __restrict__ out, long long tokens, long long num_slots, int k, int width, long long stride) {
  pdl_wait();
  const int pieces = width / W;
  const long long work = tokens * pieces;
  for (long long i = (long long)blockIdx.x * 256 * U + threadIdx.x; i < work; i += (long long)gridDim.x * 256 * U) {
    float acc[U][W];
    long long t[U];
    int c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long at = i + u * 256;
      t[u] = at >> 32 ? at / pieces : (unsigned)at / (unsigned)pieces;        // a division of 64 bits is some 70 instructions
      c[u] = (int)(at - t[u] * pieces) * W;
#pragma unroll
      for (int x = 0; x < W; ++x) acc[u][x] = 0.f;
    }
    for (int j0 = 0; j0 < k; j0 += K) {
      Pack<T, W> v[U][K];
      float w[U][K];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < K; ++j) {
          const bool there = j0 + j < k && i + u * 256 < work;
          const int s = there ? slots[t[u] * k + j0 + j] : -1;
          const bool on = (unsigned)s < (unsigned long long)num_slots;
          w[u][j] = !on ? 0.f : weights ? weights[t[u] * k + j0 + j] : 1.f;
          if (on) v[u][j].load(z + s * stride + c[u]);
          else v[u][j].zero();
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
          for (int x = 0; x < W; ++x) acc[u][x] = fmaf(w[u][j], v[u][j].get(x), acc[u][x]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u * 256 >= work) continue;
      Pack<T, W> r;
#pragma unroll
      for (int x = 0; x < W; ++x) r.set(x, acc[u][x]);
      r.store(out + t[u] * width + c[u]);
    }
  }
}

// dz[slots[t, j]] = w[t, j] dout[t];  dw[t, j] = <dout[t], z[slots[t, j]]>.  A CTA takes a token: dout's row is read once for kGroup choices,
// z's rows once, dz's written once.  Rows of dz that no pair has (from the last offset on) are zeros.
constexpr int kGradGroup = 8;
template <class T, int W, int THREADS>
__global__ void __launch_bounds__(THREADS) combine_backward_kernel(const T* __restrict__ dout, const T* __restrict__ z, const int* __restrict__ slots,
                                                                        const float* __restrict__ weights, const int* __restrict__ last_offset,
                                                                        T* __restrict__ dz, float* __restrict__ dweights, long long tokens,
                                                                        long long num_slots, int k, int width, long long dout_stride, long long z_stride) {
  __shared__ float part[THREADS / 32][kGradGroup];
  const int tid = threadIdx.x;
  pdl_wait();
  for (long long t = blockIdx.x; t < tokens; t += gridDim.x) {
    const T* d = dout + t * dout_stride;
    for (int j0 = 0; j0 < k; j0 += kGradGroup) {
      float acc[kGradGroup];
#pragma unroll
      for (int j = 0; j < kGradGroup; ++j) acc[j] = 0.f;
      for (int c = tid * W; c < width; c += THREADS * W) {
        Pack<T, W> g;
        g.load(d + c);
#pragma unroll
        for (int j = 0; j < kGradGroup; ++j) {
          if (j0 + j >= k) continue;
          const int s = slots[t * k + j0 + j];
          if ((unsigned)s >= (unsigned long long)num_slots) continue;
          const float w = weights ? weights[t * k + j0 + j] : 1.f;
          Pack<T, W> v, r;
          v.load(z + s * z_stride + c);
#pragma unroll
          for (int x = 0; x < W; ++x) {
            acc[j] = fmaf(g.get(x), v.get(x), acc[j]);
            r.set(x, w * g.get(x));
          }
          r.store(dz + (long long)s * width + c);
        }
      }
#pragma unroll
      for (int j = 0; j < kGradGroup; ++j)
#pragma unroll
        for (int o = 16; o; o >>= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
      if ((tid & 31) == 0)
#pragma unroll
        for (int j = 0; j < kGradGroup; ++j) part[tid >> 5][j] = acc[j];
      __syncthreads();
      if (tid < kGradGroup && j0 + tid < k) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < THREADS / 32; ++w) s += part[w][tid];
        dweights[t * k + j0 + tid] = s;
      }
      __syncthreads();
    }
  }
  const long long used = *last_offset < 0 ? 0 : *last_offset;
  Pack<T, W> none;
  none.zero();
  const long long pieces = width / W, empty = used < num_slots ? (num_slots - used) * pieces : 0;
  for (long long i = (long long)blockIdx.x * THREADS + tid; i < empty; i += (long long)gridDim.x * THREADS) none.store(dz + used * width + i * W);
}

// ---- host ----------------------------------------------------------------------------------------------------------

// CTAs of the router: one for each 32 tokens up to one an SM, so that the sums over all CTAs' counts stay short.
static int route_ctas(long long tokens) {
  const long long want = (tokens + 31) / 32;
  const int sms = device_sm_count();
  return (int)(want < 1 ? 1 : want > sms ? sms : want);
}
constexpr long long kRouteSmall = 64;      // tokens up to which one CTA does it all

// THREADS: as many as leave `seen` (a word for each warp and expert) within 64 KB of shared memory, beside it up to 106 KB for the lists.
template <class T, int V, int W, int THREADS, bool SMALL>
static int route_kernel(const RouteArgs& a, int ctas, cudaStream_t st) {
  constexpr auto kernel = SMALL ? route_small_kernel<T, V, W, THREADS> : route_choose_kernel<T, V, W, THREADS>;
  const int smem = ((a.experts + 1) / 2 * 2 + (a.experts * (THREADS / 32) + 1) / 2 * 2) * 4 + THREADS * (V + 1) * (int)sizeof(typename Choice<T>::Key);
  if (int e = allow_smem<kernel>(smem)) return e;
  return launch_pdl(kernel, ctas, THREADS, smem, st, a);
}

template <class T, int V, int W, int THREADS>
static int route_launch(const RouteArgs& args, cudaStream_t st) {
  RouteArgs a = args;
  if (a.tokens <= kRouteSmall) {
    a.chunk = a.tokens;
    return a.tokens <= 8 ? route_kernel<T, V, W, 256, true>(a, 1, st) : route_kernel<T, V, W, THREADS, true>(a, 1, st);
  }
  const int ctas = route_ctas(a.tokens);
  a.chunk = (a.tokens + ctas - 1) / ctas;
  if (int e = route_kernel<T, V, W, THREADS, false>(a, ctas, st)) return e;
  return launch_pdl(route_place_kernel, ctas, kPlaceThreads, (size_t)a.experts * 8, st, a);
}

template <class T, int V, int THREADS>
static int route_width(const RouteArgs& a, cudaStream_t st) {
  constexpr int kFull = 16 / (int)sizeof(T), W = V < kFull ? 1 : V % kFull == 0 ? kFull : 4;          // 16 bytes, or 8
  // wide loads where every row allows them
  const bool wide = a.experts % W == 0 && a.stride % W == 0 && aligned16(a.logits);
  return wide ? route_launch<T, V, W, THREADS>(a, st) : route_launch<T, V, 1, THREADS>(a, st);
}

template <class T>
static int route_typed(const RouteArgs& a, cudaStream_t st) {
  if (a.experts <= 32) return route_width<T, 1, 1024>(a, st);
  if (a.experts <= 64) return route_width<T, 2, 1024>(a, st);
  if (a.experts <= 128) return route_width<T, 4, 1024>(a, st);
  if (a.experts <= 256) return route_width<T, 8, 1024>(a, st);
  // us, 32 771 tokens in 32 bits: 384 experts by 12 keys a lane 47.3, 388 by 16 60.0
  if (a.experts <= 384) return route_width<T, 12, 1024>(a, st);
  if (a.experts <= 512) return route_width<T, 16, 512>(a, st);
  return route_width<T, 32, 256>(a, st);
}

// Clusters of the balance loss: a few tokens a warp, up to one CTA an SM.
// Tokens up to which one CTA does it all, half as many where it has half the threads; us, one / two launches: 48 tokens of 64 experts 3.0 / 5.8, 128 5.1 / 5.3, 200
// 7.0 / 5.4; 128 of 256 5.2 / 6.6, 200 6.8 / 6.8; 128 of 384 5.7 / 6.2, 200 7.8 / 6.1; 64 of 1024 9.0 / 9.1, 128 14.5 / 9.5.
constexpr long long kBalanceSmall = 128;
static int balance_clusters(long long tokens) {
  const long long want = (tokens + 63) / 64;
  const int most = device_sm_count() / kBalanceCtas;
  return (int)(want < 1 ? 1 : want > most ? most : want);
}

template <class T, int V, int W>
static int balance_launch(const BalanceArgs& a, cudaStream_t st) {
  constexpr int kThreads = V <= 8 ? 1024 : V <= 16 ? 512 : 256;          // 32 KB for the warps' sums at the most
  const size_t smem = (size_t)a.experts * (kThreads / 32) * 4;
  constexpr int kFew = V <= 12 ? 512 : 256;
  if (a.tokens <= kBalanceSmall * kFew / 512) {
    return launch_pdl(balance_kernel<T, V, W, kFew, true>, 1, kFew, (size_t)a.experts * (kFew / 32) * 4, st, a);
  }
  const int clusters = balance_clusters(a.tokens);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(clusters * kBalanceCtas)); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kBalanceCtas; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = pdl_enabled() ? 2 : 1;
  if (int e = (int)cudaLaunchKernelEx(&cfg, balance_kernel<T, V, W, kThreads, false>, a)) return e;
  return launch_pdl(balance_end_kernel, 1, 1024, 0, st, a, clusters);
}
template <class T, int V, int W>
static int balance_launch(const BalanceGradArgs& a, cudaStream_t st) {
  const long long want = (a.tokens + 7) / 8;
  return launch_pdl(balance_backward_kernel<T, V, W>, (unsigned)(want < device_sm_count() * 8ll ? want : device_sm_count() * 8ll), 256, 0, st, a);
}

template <class T, int V, class A>
static int balance_width(const A& a, bool aligned, cudaStream_t st) {
  constexpr int kFull = 16 / (int)sizeof(T), W = V < kFull ? 1 : V % kFull == 0 ? kFull : 4;
  return aligned && a.experts % W == 0 && a.stride % W == 0 ? balance_launch<T, V, W>(a, st) : balance_launch<T, V, 1>(a, st);
}

// `aligned`: the logits and their gradient begin on 16 bytes.
template <class A>
static int balance_call(const A& a, int type, bool aligned, cudaStream_t st) {
  const auto go = [&](auto zero) {
    using T = decltype(zero);
    if (a.experts <= 32) return balance_width<T, 1>(a, aligned, st);
    if (a.experts <= 64) return balance_width<T, 2>(a, aligned, st);
    if (a.experts <= 128) return balance_width<T, 4>(a, aligned, st);
    if (a.experts <= 256) return balance_width<T, 8>(a, aligned, st);
    if (a.experts <= 384) return balance_width<T, 12>(a, aligned, st);
    if (a.experts <= 512) return balance_width<T, 16>(a, aligned, st);
    return balance_width<T, 32>(a, aligned, st);
  };
  switch (type) {
    case FLEXSPMV_TYPE_F32: return go(0.f);
    case FLEXSPMV_TYPE_BF16: return go(__nv_bfloat16());
    default: return go(__half());
  }
}

static int grid_of(long long ctas, int most) { return (int)(ctas < 1 ? 1 : ctas > most ? most : ctas); }

template <class T, int W, int K, int U>
static int combine_launch(const flexspmv_expert_desc& d, const void* const* in, void* const* out, cudaStream_t st) {
  const long long work = d.tokens * (d.n / W);
  return launch_pdl(combine_kernel<T, W, K, U>, grid_of((work + 256 * U - 1) / (256 * U), 1 << 20), 256, 0, st, static_cast<const T*>(in[0]),
                    static_cast<const int*>(in[1]), static_cast<const float*>(in[2]), static_cast<T*>(out[0]), (long long)d.tokens, (long long)d.slots, d.choices,
                    d.n, (long long)d.in_stride);
}
template <class T, int W>
static int combine_typed(const flexspmv_expert_desc& d, const void* const* in, void* const* out, cudaStream_t st) {
  // several places a thread only where there are threads enough without
  const bool many = d.tokens * (d.n / W) >= (long long)device_sm_count() * 2048 * 4;
  if (many && d.choices == 1) return combine_launch<T, W, 1, 4>(d, in, out, st);
  if (many && d.choices == 2) return combine_launch<T, W, 2, 2>(d, in, out, st);
  return combine_launch<T, W, 4, 1>(d, in, out, st);
}

template <class T, int W, int THREADS>
static int combine_backward_launch(const flexspmv_expert_desc& d, const void* const* in, void* const* out, cudaStream_t st) {
  return launch_pdl(combine_backward_kernel<T, W, THREADS>, grid_of(d.tokens, 1 << 20), THREADS, 0, st, static_cast<const T*>(in[0]), static_cast<const T*>(in[1]),
                    static_cast<const int*>(in[2]), static_cast<const float*>(in[3]), static_cast<const int*>(in[4]) + d.experts,
                    static_cast<T*>(out[0]), static_cast<float*>(out[1]), (long long)d.tokens, (long long)d.slots, d.choices, d.n,
                    (long long)d.in_stride, (long long)d.in2_stride);
}
template <class T, int W>
static int combine_backward_typed(const flexspmv_expert_desc& d, const void* const* in, void* const* out, cudaStream_t st) {
  // few tokens with long rows: four times the threads on each (256 tokens, 8 choices of 4096 columns 12.3 us with 128 threads, 6.4 with 512)
  if (d.tokens < device_sm_count() * 8ll && d.n / W >= 512) return combine_backward_launch<T, W, 512>(d, in, out, st);
  return combine_backward_launch<T, W, 128>(d, in, out, st);
}

}  // namespace flex

extern "C" {

int flexspmv_expert_route_bytes(const flexspmv_expert_desc* d, size_t* bytes) {
  if (!d || !bytes || d->tokens < 0 || d->experts < 1) return FLEXSPMV_ERR_BAD_ARG;
  if (d->experts > FLEXSPMV_MAX_EXPERTS) return FLEXSPMV_ERR_TOO_LARGE;
  *bytes = (size_t)flex::route_ctas(d->tokens) * ((d->experts + 3) / 4 * 16);
  return 0;
}

static int check_route(const flexspmv_expert_desc* d) {
  if (!d || d->tokens < 0 || d->experts < 1 || d->choices < 1 || d->choices > d->experts || d->in_stride < d->experts) return FLEXSPMV_ERR_BAD_ARG;
  if (d->type != FLEXSPMV_TYPE_F32 && d->type != FLEXSPMV_TYPE_BF16 && d->type != FLEXSPMV_TYPE_F16) return FLEXSPMV_ERR_BAD_ARG;
  if (d->experts > FLEXSPMV_MAX_EXPERTS || d->choices > FLEXSPMV_MAX_CHOICES || d->tokens > 0x7fffffffLL / d->choices) return FLEXSPMV_ERR_TOO_LARGE;
  return 0;
}

int flexspmv_expert_route(const flexspmv_expert_desc* d, const void* const* in, void* const* out, void* ws, size_t ws_bytes, void* stream) {
  if (int e = check_route(d)) return e;
  if (!in || !out || (!in[0] && d->tokens) || !out[2]) return FLEXSPMV_ERR_BAD_ARG;
  if (d->tokens && (!out[0] || !out[1] || !out[3] || !out[4])) return FLEXSPMV_ERR_BAD_ARG;
  size_t need = 0;
  flexspmv_expert_route_bytes(d, &need);
  if (!ws || ws_bytes < need) return FLEXSPMV_ERR_WORKSPACE;
  if (!flex::aligned16(ws) || !flex::aligned_to(flex::type_bytes(d->type), in[0]) || !flex::aligned_to(4, out[0], out[1], out[2], out[3], out[4]))
    return FLEXSPMV_ERR_ALIGN;
  const long long pairs = 4 * d->tokens * d->choices;
  if (!flex::apart({{out[0], pairs}, {out[1], pairs}, {out[2], 4ll * d->experts + 4}, {out[3], pairs}, {out[4], pairs}, {ws, (long long)need}},
                   {flex::rows_at(in[0], d->tokens, d->experts, d->in_stride, d->type)}))
    return FLEXSPMV_ERR_BAD_ARG;
  flex::RouteArgs a = {in[0], d->tokens, d->in_stride, d->experts, d->choices, d->flags & FLEXSPMV_EXPERT_RENORMALIZE, 0,
                       static_cast<float*>(out[0]), static_cast<int*>(out[1]), static_cast<int*>(out[2]), static_cast<int*>(out[3]),
                       static_cast<int*>(out[4]), static_cast<unsigned*>(ws)};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (d->type) {
    case FLEXSPMV_TYPE_F32: return flex::route_typed<float>(a, st);
    case FLEXSPMV_TYPE_BF16: return flex::route_typed<__nv_bfloat16>(a, st);
    default: return flex::route_typed<__half>(a, st);
  }
}

int flexspmv_expert_route_backward(const flexspmv_expert_desc* d, const void* const* in, void* const* out, void* stream) {
  if (int e = check_route(d)) return e;
  if (!in || !out) return FLEXSPMV_ERR_BAD_ARG;
  if (d->tokens == 0) return 0;
  if (!in[0] || !in[1] || !in[2] || !in[3] || !out[0]) return FLEXSPMV_ERR_BAD_ARG;
  if (!flex::aligned_to(flex::type_bytes(d->type), in[1], out[0]) || !flex::aligned_to(4, in[0], in[2], in[3])) return FLEXSPMV_ERR_ALIGN;
  const long long pairs = 4 * d->tokens * d->choices;
  if (!flex::apart({{out[0], d->tokens * d->experts * flex::type_bytes(d->type)}},
                   {{in[0], pairs}, flex::rows_at(in[1], d->tokens, d->experts, d->in_stride, d->type), {in[2], pairs}, {in[3], pairs}}))
    return FLEXSPMV_ERR_BAD_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int grid = flex::grid_of((d->tokens + 7) / 8, flex::device_sm_count() * 8);
  auto go = [&](auto zero) {
    using T = decltype(zero);
    constexpr int W = 16 / (int)sizeof(T);
    const bool wide = d->experts % W == 0 && d->in_stride % W == 0 && flex::aligned16(in[1]) && flex::aligned16(out[0]);
    return flex::launch_pdl(wide ? flex::route_backward_kernel<T, W> : flex::route_backward_kernel<T, 1>, grid, 256, 0, st, static_cast<const float*>(in[0]), static_cast<const T*>(in[1]),
                            static_cast<const float*>(in[2]), static_cast<const int*>(in[3]), static_cast<T*>(out[0]), (long long)d->tokens,
                            (long long)d->in_stride, d->experts, d->choices, d->flags & FLEXSPMV_EXPERT_RENORMALIZE);
  };
  switch (d->type) {
    case FLEXSPMV_TYPE_F32: return go(0.f);
    case FLEXSPMV_TYPE_BF16: return go(__nv_bfloat16());
    default: return go(__half());
  }
}

// Checks that the balance loss and its gradient share.
static int check_balance(const flexspmv_expert_desc* d) {
  if (!d || d->tokens < 0 || d->experts < 1 || d->in_stride < d->experts || !flex::known_type(d->type)) return FLEXSPMV_ERR_BAD_ARG;
  if (d->experts > FLEXSPMV_MAX_EXPERTS || d->tokens > 0x7fffffffLL) return FLEXSPMV_ERR_TOO_LARGE;
  return 0;
}

int flexspmv_balance_loss_bytes(const flexspmv_expert_desc* d, size_t* bytes) {
  if (!d || !bytes || d->tokens < 0 || d->experts < 1) return FLEXSPMV_ERR_BAD_ARG;
  if (d->experts > FLEXSPMV_MAX_EXPERTS) return FLEXSPMV_ERR_TOO_LARGE;
  *bytes = (size_t)flex::balance_clusters(d->tokens) * (d->experts + 1) * 4;
  return 0;
}

int flexspmv_balance_loss(const flexspmv_expert_desc* d, const void* const* in, void* const* out, void* ws, size_t ws_bytes, void* stream) {
  if (int e = check_balance(d)) return e;
  if (!in || !out || (d->tokens && !in[0]) || !in[1] || !out[0] || !out[1] || !out[2] || !out[3]) return FLEXSPMV_ERR_BAD_ARG;
  size_t need = 0;
  flexspmv_balance_loss_bytes(d, &need);
  if (!ws || ws_bytes < need) return FLEXSPMV_ERR_WORKSPACE;
  if (!flex::aligned16(ws) || !flex::aligned_to(flex::type_bytes(d->type), in[0]) || !flex::aligned_to(4, in[1], out[0], out[1], out[2], out[3]))
    return FLEXSPMV_ERR_ALIGN;
  const long long each = 4ll * d->experts;
  if (!flex::apart({{out[0], 4}, {out[1], each}, {out[2], each}, {out[3], 4}, {ws, (long long)need}},
                   {flex::rows_at(in[0], d->tokens, d->experts, d->in_stride, d->type), {in[1], each + 4}}))
    return FLEXSPMV_ERR_BAD_ARG;
  float* const parts = static_cast<float*>(ws);
  const flex::BalanceArgs a = {in[0], static_cast<const int*>(in[1]), d->tokens, d->in_stride, d->experts, parts,
                               reinterpret_cast<int*>(parts + (size_t)flex::balance_clusters(d->tokens) * d->experts), static_cast<float*>(out[0]),
                               static_cast<float*>(out[2]), static_cast<int*>(out[1]), static_cast<int*>(out[3])};
  return flex::balance_call(a, d->type, flex::aligned16(in[0]), static_cast<cudaStream_t>(stream));
}

int flexspmv_balance_loss_backward(const flexspmv_expert_desc* d, const void* const* in, void* const* out, void* stream) {
  if (int e = check_balance(d)) return e;
  if (!in || !out) return FLEXSPMV_ERR_BAD_ARG;
  if (d->tokens == 0) return 0;
  if (!in[0] || !in[1] || !in[2] || !in[3] || !out[0] || (in[4] && (!in[5] || !in[6]))) return FLEXSPMV_ERR_BAD_ARG;
  if (in[4] && (d->choices < 1 || d->choices > d->experts)) return FLEXSPMV_ERR_BAD_ARG;
  if (in[4] && d->choices > FLEXSPMV_MAX_CHOICES) return FLEXSPMV_ERR_TOO_LARGE;
  if (!flex::aligned_to(flex::type_bytes(d->type), in[1], out[0]) || !flex::aligned_to(4, in[0], in[2], in[3], in[4], in[5], in[6])) return FLEXSPMV_ERR_ALIGN;
  const long long pairs = in[4] ? 4 * d->tokens * d->choices : 0;
  if (!flex::apart({{out[0], d->tokens * d->experts * flex::type_bytes(d->type)}},
                   {{in[0], 4}, flex::rows_at(in[1], d->tokens, d->experts, d->in_stride, d->type), {in[2], 4ll * d->experts}, {in[3], 4}, {in[4], pairs},
                    {in[5], pairs}, {in[6], pairs}}))
    return FLEXSPMV_ERR_BAD_ARG;
  const flex::BalanceGradArgs a = {static_cast<const float*>(in[0]), in[1], static_cast<const int*>(in[2]), static_cast<const int*>(in[3]),
                                   static_cast<const float*>(in[4]), static_cast<const float*>(in[5]), static_cast<const int*>(in[6]), out[0], d->tokens,
                                   d->in_stride, d->experts, d->choices, d->flags & FLEXSPMV_EXPERT_RENORMALIZE};
  return flex::balance_call(a, d->type, flex::aligned16(in[1]) && flex::aligned16(out[0]), static_cast<cudaStream_t>(stream));
}

// Checks that combine and its gradient share.
static int check_combine(const flexspmv_expert_desc* d) {
  if (!d || d->tokens < 0 || d->slots < 0 || d->choices < 1 || d->n < 1 || d->in_stride < d->n) return FLEXSPMV_ERR_BAD_ARG;
  if (d->type != FLEXSPMV_TYPE_BF16 && d->type != FLEXSPMV_TYPE_F16) return FLEXSPMV_ERR_BAD_ARG;
  if (d->slots > 0x7fffffffLL || d->tokens > 0x7fffffffLL || d->choices > FLEXSPMV_MAX_CHOICES) return FLEXSPMV_ERR_TOO_LARGE;
  return 0;
}

int flexspmv_expert_combine(const flexspmv_expert_desc* d, const void* const* in, void* const* out, void* stream) {
  if (int e = check_combine(d)) return e;
  if (!in || !out) return FLEXSPMV_ERR_BAD_ARG;
  if (d->tokens == 0) return 0;
  if ((d->slots && !in[0]) || !in[1] || !out[0]) return FLEXSPMV_ERR_BAD_ARG;
  if (!flex::aligned_to(2, in[0], out[0]) || !flex::aligned_to(4, in[1], in[2])) return FLEXSPMV_ERR_ALIGN;
  const long long pairs = 4 * d->tokens * d->choices;
  if (!flex::apart({{out[0], 2 * d->tokens * d->n}}, {flex::rows_at(in[0], d->slots, d->n, d->in_stride, d->type), {in[1], pairs}, {in[2], pairs}}))
    return FLEXSPMV_ERR_BAD_ARG;
  // 16-byte accesses where every row allows them
  const bool wide = d->n % 8 == 0 && d->in_stride % 8 == 0 && flex::aligned16(in[0]) && flex::aligned16(out[0]);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d->type == FLEXSPMV_TYPE_BF16)
    return (wide ? flex::combine_typed<__nv_bfloat16, 8> : flex::combine_typed<__nv_bfloat16, 1>)(*d, in, out, st);
  return (wide ? flex::combine_typed<__half, 8> : flex::combine_typed<__half, 1>)(*d, in, out, st);
}

int flexspmv_expert_combine_backward(const flexspmv_expert_desc* d, const void* const* in, void* const* out, void* stream) {
  if (int e = check_combine(d)) return e;
  if (!in || !out || d->experts < 1 || d->in2_stride < d->n) return FLEXSPMV_ERR_BAD_ARG;
  if (!in[4] || (d->tokens && (!in[0] || !in[2] || !out[1])) || (d->slots && (!in[1] || !out[0]))) return FLEXSPMV_ERR_BAD_ARG;
  if (!flex::aligned_to(2, in[0], in[1], out[0]) || !flex::aligned_to(4, in[2], in[3], in[4], out[1])) return FLEXSPMV_ERR_ALIGN;
  const long long pairs = 4 * d->tokens * d->choices;
  if (!flex::apart({{out[0], 2 * d->slots * d->n}, {out[1], pairs}},
                   {flex::rows_at(in[0], d->tokens, d->n, d->in_stride, d->type), flex::rows_at(in[1], d->slots, d->n, d->in2_stride, d->type), {in[2], pairs},
                    {in[3], pairs}, {in[4], 4ll * d->experts + 4}}))
    return FLEXSPMV_ERR_BAD_ARG;
  const bool wide = d->n % 8 == 0 && d->in_stride % 8 == 0 && d->in2_stride % 8 == 0 && flex::aligned16(in[0]) && flex::aligned16(in[1]) &&
                    flex::aligned16(out[0]);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d->type == FLEXSPMV_TYPE_BF16)
    return (wide ? flex::combine_backward_typed<__nv_bfloat16, 8> : flex::combine_backward_typed<__nv_bfloat16, 1>)(*d, in, out, st);
  return (wide ? flex::combine_backward_typed<__half, 8> : flex::combine_backward_typed<__half, 1>)(*d, in, out, st);
}

}  // extern "C"
