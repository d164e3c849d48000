// Routed expert layers: the router (softmax over the experts, the k largest, the plan in expert order), its gradient, and the weighted
// reduce of the experts' results into the tokens' rows, with its gradient.  The matrix products between them: flex_grouped.cu.
//
// A plan is what flexspmv_sort_rows makes of an unsorted Reducer, for (token, choice) pairs and the experts as rows: the pairs in
// a stable order by expert, `offsets` (where an expert's pairs begin), `slots` (pair -> place in that order) and `rows` (place -> token).
#include <cuda_runtime.h>

#include <type_traits>

#include "flex_common.cuh"
#include "flex_expert_types.cuh"

namespace flex {

int device_sm_count();

// ---- router --------------------------------------------------------------------------------------------------------

// A float as an unsigned number of the same order; NaN and -infinity are 0, which is never chosen.
__device__ __forceinline__ unsigned choice_key(float v) {
  const unsigned u = __float_as_uint(v + 0.f);         // -0 and 0 are equal
  const unsigned key = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return (v != v || v == -INFINITY) ? 0u : key;
}

// One token by one warp; lane l holds the experts l, l + 32, ...: V of them.  The k largest by k rounds of a maximum over the warp (equal
// logits: the lowest expert, as the plain form's stable sort has it), each after the chosen one's key has been taken out.
// Lane j ends with choice j.  The softmax is over the true logits, largest subtracted, sums in 32 bits.
template <class T, int V>
__device__ __forceinline__ void choose_token(const T* row, int experts, int k, bool renormalize, int lane, int& my_id, float& my_weight) {
  float v[V];
  unsigned key[V];
  unsigned best = 0;
  int best_at = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = i * 32 + lane;
    v[i] = e < experts ? to_float(row[e]) : -INFINITY;
    key[i] = choice_key(v[i]);
    if (key[i] > best) { best = key[i]; best_at = i; }
  }
  my_id = -1;
  float my_logit = -INFINITY, top = -INFINITY;
  for (int j = 0; j < k; ++j) {
    const unsigned most = __reduce_max_sync(0xffffffffu, best);
    if (most == 0) break;
    const int at = __reduce_min_sync(0xffffffffu, best == most ? best_at * 32 + lane : 0x7fffffff);
    const float logit = __uint_as_float((most & 0x80000000u) ? (most & 0x7fffffffu) : ~most);
    if (j == 0) top = logit;
    if (lane == j) { my_id = at; my_logit = logit; }
    if ((at & 31) == lane) {
      best = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (i == (at >> 5)) key[i] = 0;
        if (key[i] > best) { best = key[i]; best_at = i; }
      }
    }
  }
  const float mine = my_id >= 0 ? expf(my_logit - top) : 0.f;
  float sum = 0.f;
  if (renormalize) {
    sum = mine;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) sum += (v[i] == -INFINITY) ? 0.f : expf(v[i] - top);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  my_weight = my_id >= 0 ? mine / sum : 0.f;
}

constexpr int kRouteThreads = 256, kRouteWarps = kRouteThreads / 32;

struct RouteArgs {
  const void* logits;
  long long tokens, stride;
  int experts, k, renormalize;
  long long chunk;                 // tokens of a CTA
  float* weights;
  int *ids, *offsets, *rows, *slots;
  unsigned* counts;                // [CTAs][experts]
};

// Choices of this CTA's tokens; `hist` (shared, zeroed, experts entries) gets their number for each expert.
template <class T, int V>
__device__ __forceinline__ void choose_chunk(const RouteArgs& a, unsigned* hist) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long from = a.chunk * blockIdx.x, to = from + a.chunk < a.tokens ? from + a.chunk : a.tokens;
  for (long long t = from + warp; t < to; t += kRouteWarps) {
    int id;
    float weight;
    choose_token<T, V>(static_cast<const T*>(a.logits) + t * a.stride, a.experts, a.k, a.renormalize != 0, lane, id, weight);
    if (lane < a.k) {
      a.weights[t * a.k + lane] = weight;
      a.ids[t * a.k + lane] = id;
      if (id >= 0) atomicAdd(&hist[id], 1u);
    }
  }
}

// Places this CTA's pairs: `start` (shared, [warps][experts]) holds for each warp and expert the place of the warp's first pair of it.  A warp
// takes 32 pairs at a time in their order, so that the order by expert is stable and no atomic decides it.
__device__ __forceinline__ void warp_pairs(const RouteArgs& a, long long& from, long long& to) {
  const long long first = a.chunk * blockIdx.x, last = first + a.chunk < a.tokens ? first + a.chunk : a.tokens;
  const long long pairs = last > first ? (last - first) * a.k : 0;
  const long long each = (pairs + kRouteWarps * 32 - 1) / (kRouteWarps * 32) * 32;
  from = first * a.k + min(each * (threadIdx.x >> 5), pairs);
  to = first * a.k + min(each * (threadIdx.x >> 5) + each, pairs);
}

__device__ __forceinline__ void place_chunk(const RouteArgs& a, unsigned* start) {
  const int lane = threadIdx.x & 31;
  unsigned* mine = start + (threadIdx.x >> 5) * a.experts;
  long long from, to;
  warp_pairs(a, from, to);
  for (long long p = from; p < to; p += 32) {
    const long long pair = p + lane;
    const int id = pair < to ? a.ids[pair] : -1;
    const unsigned same = __match_any_sync(0xffffffffu, id);
    unsigned place = 0;
    if (id >= 0) place = mine[id] + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (id >= 0 && (same >> lane) == 1u) mine[id] = place + 1u;          // the last of its kind
    __syncwarp();
    if (pair < to) {
      a.slots[pair] = id >= 0 ? (int)place : -1;
      if (id >= 0) a.rows[place] = (int)(pair / a.k);
    }
  }
}

// In: `total` and `before` (shared, experts entries): an expert's pairs altogether, and those of the CTAs before this one.  Out: `start` as
// place_chunk wants it.  Needs the CTA's ids visible to it.
__device__ __forceinline__ unsigned plan_chunk(const RouteArgs& a, unsigned* total, const unsigned* before, unsigned* start) {
  __shared__ unsigned warp_sum[kRouteWarps + 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int i = tid; i < a.experts * kRouteWarps; i += kRouteThreads) start[i] = 0;
  __syncthreads();
  {
    long long from, to;
    warp_pairs(a, from, to);
    unsigned* mine = start + warp * a.experts;
    for (long long p = from + lane; p < to; p += 32) {
      const int id = a.ids[p];
      if (id >= 0) atomicAdd(&mine[id], 1u);
    }
  }
  // exclusive sums of the totals, kRouteThreads at a time
  unsigned done = 0;
  for (int base = 0; base < a.experts; base += kRouteThreads) {
    const int e = base + tid;
    const unsigned n = e < a.experts ? total[e] : 0u;
    unsigned s = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned up = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += up;
    }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = s;
    __syncthreads();
    unsigned all = 0, prior = 0;
#pragma unroll
    for (int w = 0; w < kRouteWarps; ++w) {
      if (w < warp) prior += warp_sum[w];
      all += warp_sum[w];
    }
    if (e < a.experts) {
      const unsigned off = done + prior + s - n;
      if (blockIdx.x == 0) a.offsets[e] = (int)off;
      unsigned at = off + before[e];
      for (int w = 0; w < kRouteWarps; ++w) {
        const unsigned c = start[w * a.experts + e];
        start[w * a.experts + e] = at;
        at += c;
      }
    }
    done += all;
  }
  if (blockIdx.x == 0 && tid == 0) a.offsets[a.experts] = (int)done;
  __syncthreads();
  return done;
}

// Small batches: everything in one CTA and one launch.
template <class T, int V>
__global__ void __launch_bounds__(kRouteThreads) route_small_kernel(RouteArgs a) {
  extern __shared__ unsigned route_sm[];
  unsigned *total = route_sm, *before = total + a.experts, *start = before + a.experts;
  for (int i = threadIdx.x; i < a.experts; i += kRouteThreads) total[i] = before[i] = 0;
  __syncthreads();
  pdl_wait();
  choose_chunk<T, V>(a, total);
  __syncthreads();
  const unsigned used = plan_chunk(a, total, before, start);
  place_chunk(a, start);
  for (long long i = used + threadIdx.x; i < a.tokens * a.k; i += kRouteThreads) a.rows[i] = -1;
}

template <class T, int V>
__global__ void __launch_bounds__(kRouteThreads) route_choose_kernel(RouteArgs a) {
  extern __shared__ unsigned route_sm[];
  for (int i = threadIdx.x; i < a.experts; i += kRouteThreads) route_sm[i] = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  choose_chunk<T, V>(a, route_sm);
  __syncthreads();
  for (int i = threadIdx.x; i < a.experts; i += kRouteThreads) a.counts[(size_t)blockIdx.x * a.experts + i] = route_sm[i];
}

// Every CTA adds up the counts of all CTAs by itself (they lie in L2): a launch fewer than a scan between the two would take.
__global__ void __launch_bounds__(kRouteThreads) route_place_kernel(RouteArgs a) {
  extern __shared__ unsigned route_sm[];
  unsigned *total = route_sm, *before = total + a.experts, *start = before + a.experts;
  pdl_wait();
  for (int e = threadIdx.x; e < a.experts; e += kRouteThreads) {
    unsigned all = 0, prior = 0;
#pragma unroll 8
    for (unsigned b = 0; b < gridDim.x; ++b) {
      const unsigned n = a.counts[(size_t)b * a.experts + e];
      all += n;
      prior += b < blockIdx.x ? n : 0u;
    }
    total[e] = all;
    before[e] = prior;
  }
  __syncthreads();
  const unsigned used = plan_chunk(a, total, before, start);
  place_chunk(a, start);
  for (long long i = used + (long long)blockIdx.x * kRouteThreads + threadIdx.x; i < a.tokens * a.k; i += (long long)gridDim.x * kRouteThreads)
    a.rows[i] = -1;
}

// Gradient of the chosen weights with respect to the logits.  p_i = w_0 exp(l_i - l_{e_0}): the largest weight and its logit stand for the
// softmax's maximum and sum, so that one pass over the row is enough.  A warp takes a token.
template <class T>
__global__ void __launch_bounds__(256) route_backward_kernel(const float* __restrict__ dweights, const T* __restrict__ logits, const float* __restrict__ weights,
                                                             const int* __restrict__ ids, T* __restrict__ dlogits, long long tokens, long long stride,
                                                             int experts, int k, int renormalize) {
  extern __shared__ float route_grad_sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* grad = route_grad_sm + warp * experts;
  for (int e = lane; e < experts; e += 32) grad[e] = 0.f;
  pdl_wait();
  for (long long t = (long long)blockIdx.x * 8 + warp; t < tokens; t += (long long)gridDim.x * 8) {
    const int id = lane < k ? ids[t * k + lane] : -1;
    const float w = id >= 0 ? weights[t * k + lane] : 0.f, g = id >= 0 ? dweights[t * k + lane] : 0.f;
    float mean = w * g;
#pragma unroll
    for (int o = 16; o; o >>= 1) mean += __shfl_xor_sync(0xffffffffu, mean, o);
    const int top_id = __shfl_sync(0xffffffffu, id, 0);
    const float top_w = __shfl_sync(0xffffffffu, w, 0);
    __syncwarp();
    if (id >= 0) grad[id] = renormalize ? w * (g - mean) : g;
    __syncwarp();
    T* out = dlogits + t * experts;
    if (renormalize || top_id < 0) {
      for (int e = lane; e < experts; e += 32) out[e] = from_float<T>(grad[e]);
    } else {
      const T* row = logits + t * stride;
      const float top = to_float(row[top_id]);
      for (int e = lane; e < experts; e += 32) {
        const float v = to_float(row[e]);
        out[e] = from_float<T>(v == -INFINITY ? 0.f : top_w * expf(v - top) * (grad[e] - mean));
      }
    }
    __syncwarp();
    if (id >= 0) grad[id] = 0.f;
  }
}

// ---- combine -------------------------------------------------------------------------------------------------------

// out[t] = sum_j w[t, j] z[slots[t, j]]: a thread takes W neighbouring columns of one token and has the loads of four choices in flight.
// Bound by memory; the choices are added in their order, in 32 bits, rounded once.
template <class T, int W>
__global__ void __launch_bounds__(256) combine_kernel(const T* __restrict__ z, const int* __restrict__ slots, const float* __restrict__ weights,
                                                      T* __restrict__ out, long long tokens, long long num_slots, int k, int width, long long stride) {
  pdl_wait();
  const int pieces = width / W;
  const long long work = tokens * pieces;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < work; i += (long long)gridDim.x * 256) {
    const long long t = i / pieces;
    const int c = (int)(i - t * pieces) * W;
    float acc[W];
#pragma unroll
    for (int x = 0; x < W; ++x) acc[x] = 0.f;
    for (int j0 = 0; j0 < k; j0 += 4) {
      Pack<T, W> v[4];
      float w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int s = j0 + j < k ? slots[t * k + j0 + j] : -1;
        const bool on = (unsigned)s < (unsigned long long)num_slots;
        w[j] = !on ? 0.f : weights ? weights[t * k + j0 + j] : 1.f;
        if (on) v[j].load(z + s * stride + c);
        else v[j].zero();
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int x = 0; x < W; ++x) acc[x] = fmaf(w[j], v[j].get(x), acc[x]);
    }
    Pack<T, W> r;
#pragma unroll
    for (int x = 0; x < W; ++x) r.set(x, acc[x]);
    r.store(out + t * width + c);
  }
}

// dz[slots[t, j]] = w[t, j] dout[t];  dw[t, j] = <dout[t], z[slots[t, j]]>.  A CTA takes a token: dout's row is read once for kGroup choices,
// z's rows once, dz's written once.  Rows of dz that no pair has (from the last offset on) are zeros.
constexpr int kGradThreads = 128, kGradGroup = 8;
template <class T, int W>
__global__ void __launch_bounds__(kGradThreads) combine_backward_kernel(const T* __restrict__ dout, const T* __restrict__ z, const int* __restrict__ slots,
                                                                        const float* __restrict__ weights, const int* __restrict__ last_offset,
                                                                        T* __restrict__ dz, float* __restrict__ dweights, long long tokens,
                                                                        long long num_slots, int k, int width, long long dout_stride, long long z_stride) {
  __shared__ float part[kGradThreads / 32][kGradGroup];
  const int tid = threadIdx.x;
  pdl_wait();
  for (long long t = blockIdx.x; t < tokens; t += gridDim.x) {
    const T* d = dout + t * dout_stride;
    for (int j0 = 0; j0 < k; j0 += kGradGroup) {
      float acc[kGradGroup];
#pragma unroll
      for (int j = 0; j < kGradGroup; ++j) acc[j] = 0.f;
      for (int c = tid * W; c < width; c += kGradThreads * W) {
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
        for (int w = 0; w < kGradThreads / 32; ++w) s += part[w][tid];
        dweights[t * k + j0 + tid] = s;
      }
      __syncthreads();
    }
  }
  const long long used = *last_offset < 0 ? 0 : *last_offset;
  Pack<T, W> none;
  none.zero();
  const long long pieces = width / W, empty = used < num_slots ? (num_slots - used) * pieces : 0;
  for (long long i = (long long)blockIdx.x * kGradThreads + tid; i < empty; i += (long long)gridDim.x * kGradThreads) none.store(dz + used * width + i * W);
}

// ---- host ----------------------------------------------------------------------------------------------------------

// CTAs of the router: one for each 32 tokens up to one an SM, so that the sums over all CTAs' counts stay short.
static int route_ctas(long long tokens) {
  const long long want = (tokens + 31) / 32;
  const int sms = device_sm_count();
  return (int)(want < 1 ? 1 : want > sms ? sms : want);
}
constexpr long long kRouteSmall = 64;      // tokens up to which one CTA does it all

template <class T, int V>
static int route_launch(const RouteArgs& args, cudaStream_t st) {
  RouteArgs a = args;
  const size_t lists = (size_t)a.experts * 4 * (2 + kRouteWarps);
  if (a.tokens <= kRouteSmall) {
    a.chunk = a.tokens;
    return launch_pdl(route_small_kernel<T, V>, 1, kRouteThreads, lists, st, a);
  }
  const int ctas = route_ctas(a.tokens);
  a.chunk = (a.tokens + ctas - 1) / ctas;
  if (int e = launch_pdl(route_choose_kernel<T, V>, ctas, kRouteThreads, (size_t)a.experts * 4, st, a)) return e;
  return launch_pdl(route_place_kernel, ctas, kRouteThreads, lists, st, a);
}

template <class T>
static int route_typed(const RouteArgs& a, cudaStream_t st) {
  if (a.experts <= 32) return route_launch<T, 1>(a, st);
  if (a.experts <= 64) return route_launch<T, 2>(a, st);
  if (a.experts <= 128) return route_launch<T, 4>(a, st);
  if (a.experts <= 256) return route_launch<T, 8>(a, st);
  if (a.experts <= 512) return route_launch<T, 16>(a, st);
  return route_launch<T, 32>(a, st);
}

static int grid_of(long long ctas, int most) { return (int)(ctas < 1 ? 1 : ctas > most ? most : ctas); }

template <class T, int W>
static int combine_typed(const flexspmv_expert_desc& d, const void* z, const void* slots, const void* weights, void* out, cudaStream_t st) {
  const long long work = d.tokens * (d.n / W);
  return launch_pdl(combine_kernel<T, W>, grid_of((work + 255) / 256, 1 << 20), 256, 0, st, static_cast<const T*>(z), static_cast<const int*>(slots),
                    static_cast<const float*>(weights), static_cast<T*>(out), (long long)d.tokens, (long long)d.slots, d.choices, d.n,
                    (long long)d.in_stride);
}

template <class T, int W>
static int combine_backward_typed(const flexspmv_expert_desc& d, const void* const* in, void* const* out, cudaStream_t st) {
  return launch_pdl(combine_backward_kernel<T, W>, grid_of(d.tokens, 1 << 20), kGradThreads, 0, st, static_cast<const T*>(in[0]), static_cast<const T*>(in[1]),
                    static_cast<const int*>(in[2]), static_cast<const float*>(in[3]), static_cast<const int*>(in[4]) + d.experts,
                    static_cast<T*>(out[0]), static_cast<float*>(out[1]), (long long)d.tokens, (long long)d.slots, d.choices, d.n,
                    (long long)d.in_stride, (long long)d.in2_stride);
}

}  // namespace flex

extern "C" {

int flexspmv_expert_route_bytes(const flexspmv_expert_desc* d, size_t* bytes) {
  if (!d || !bytes || d->tokens < 0 || d->experts < 1) return FLEXSPMV_ERR_BAD_ARG;
  if (d->experts > FLEXSPMV_MAX_EXPERTS) return FLEXSPMV_ERR_TOO_LARGE;
  *bytes = (size_t)flex::route_ctas(d->tokens) * d->experts * 4;
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int grid = flex::grid_of((d->tokens + 7) / 8, flex::device_sm_count() * 8);
  const size_t smem = (size_t)8 * d->experts * 4;
  auto go = [&](auto zero) {
    using T = decltype(zero);
    return flex::launch_pdl(flex::route_backward_kernel<T>, grid, 256, smem, st, static_cast<const float*>(in[0]), static_cast<const T*>(in[1]),
                            static_cast<const float*>(in[2]), static_cast<const int*>(in[3]), static_cast<T*>(out[0]), (long long)d->tokens,
                            (long long)d->in_stride, d->experts, d->choices, d->flags & FLEXSPMV_EXPERT_RENORMALIZE);
  };
  switch (d->type) {
    case FLEXSPMV_TYPE_F32: return go(0.f);
    case FLEXSPMV_TYPE_BF16: return go(__nv_bfloat16());
    default: return go(__half());
  }
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
  // 16-byte accesses where every row allows them
  const bool wide = d->n % 8 == 0 && d->in_stride % 8 == 0 && flex::aligned16(in[0]) && flex::aligned16(out[0]);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d->type == FLEXSPMV_TYPE_BF16)
    return (wide ? flex::combine_typed<__nv_bfloat16, 8> : flex::combine_typed<__nv_bfloat16, 1>)(*d, in[0], in[1], in[2], out[0], st);
  return (wide ? flex::combine_typed<__half, 8> : flex::combine_typed<__half, 1>)(*d, in[0], in[1], in[2], out[0], st);
}

int flexspmv_expert_combine_backward(const flexspmv_expert_desc* d, const void* const* in, void* const* out, void* stream) {
  if (int e = check_combine(d)) return e;
  if (!in || !out || d->experts < 1 || d->in2_stride < d->n) return FLEXSPMV_ERR_BAD_ARG;
  if (!in[4] || (d->tokens && (!in[0] || !in[2] || !out[1])) || (d->slots && (!in[1] || !out[0]))) return FLEXSPMV_ERR_BAD_ARG;
  const bool wide = d->n % 8 == 0 && d->in_stride % 8 == 0 && d->in2_stride % 8 == 0 && flex::aligned16(in[0]) && flex::aligned16(in[1]) &&
                    flex::aligned16(out[0]);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d->type == FLEXSPMV_TYPE_BF16)
    return (wide ? flex::combine_backward_typed<__nv_bfloat16, 8> : flex::combine_backward_typed<__nv_bfloat16, 1>)(*d, in, out, st);
  return (wide ? flex::combine_backward_typed<__half, 8> : flex::combine_backward_typed<__half, 1>)(*d, in, out, st);
}

}  // extern "C"
