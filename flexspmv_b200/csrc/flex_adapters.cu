// Low-rank adapters of many requests beside a shared projection: y[t] = W x[t] + scale[a] B[a] (A[a] x[t]), a = ids[t].
// Here: the plan of a batch and the first product, low[t] = scale A x[t].  The rest is the shared product's epilogue (flex_grouped.cu).
#include <cuda_runtime.h>

#include <atomic>

#include "flex_adapters.cuh"
#include "flex_common.cuh"
#include "flex_expert_types.cuh"
#include "flex_umma.cuh"

namespace flex {

int device_sm_count();

// ---- plan ----------------------------------------------------------------------------------------------------------

struct AdapterTile {
  int adapter, from, count, unused;          // places from .. from + count of `rows`, all of one adapter
};

// Where a plan's parts lie, in ints; it begins with the number of tiles, the tokens and the adapters that it is of.  Groups: for the shared product of many tokens, runs of one adapter that are long enough for tiles of
// their own, and what lies between them.
constexpr int kLowTile = 16;
// Tokens up to which they are one group, whose tiles go round the SMs better than those of many short groups; us, one / several: 900 tokens of rank 64 in 60 runs (2048 x 2048,
// float16) 36 / 47, 1000 of rank 32 in 40 (4096 x 4096) 57 / 64, 1031 of rank 8 in 40 (1000 x 1416) 19.5 / 20.1, but 600 of rank 128 with one adapter (2000 x 2000) 37 / 23, 1400 of rank 64 in
// 20 runs (5000 x 1024) 67 / 53, 2000 in runs of 400 (4096 x 4096) 83 / 77.
constexpr long long kOneGroup = 1536;
constexpr long long kLowTiles = 4096;        // tokens up to which the first product may be in tiles
// ... and is: an adapter is read again for every 16 tokens.  us, both products (2048 x 2048, runs of 10 to 100 tokens), tiles / the grouped kernel: rank 16, 100 tokens
// 13.6 / 21.3, 600 24.6 / 27.6, 1500 33.3 / 31.1, 2000 38.1 / 43.5, 4000 57.5 / 52.3; rank 64, 300 26.9 / 29.1, 500 28.9 / 32.7, 600 36.5 / 38.6, 2000 65.6 / 59.5; rank 128, 250
// 60.8 / 52.7, 600 59.8 / 51.9.
static bool low_in_tiles(long long tokens, int rank) { return tokens <= kLowTiles && tokens * rank <= 32768; }
// us, runs of 100 and 200 tokens: from 64 on 54.7 and 41.2 (3000 tokens, 2048 x 2048, ranks 32 and 64), from 128 on 50.3 and 41.0, from 256 on 50.2 and 54.9.
constexpr int kLongRun = 128;
struct AdapterPlan {
  long long ids, rows, tiles, offsets, groups, group_adapters, runs, ints;
  int most_tiles, most_groups, long_run;
};
static AdapterPlan adapter_plan_of(long long tokens, int adapters) {
  AdapterPlan p;
  p.most_tiles = tokens <= kLowTiles ? (int)(tokens / kLowTile + (tokens < adapters ? tokens : adapters)) : 0;
  p.tiles = 8;
  p.offsets = p.tiles + 4ll * p.most_tiles;
  p.ids = p.offsets + adapters + 1;
  p.rows = p.ids + tokens;
  // at most some 1000 groups, which the product keeps in shared memory
  p.long_run = (int)(tokens / 500 > kLongRun ? tokens / 500 : kLongRun);
  p.most_groups = tokens <= kOneGroup ? 1 : (int)(2 * (tokens / p.long_run) + 1);
  p.groups = p.rows + tokens;
  p.group_adapters = p.groups + p.most_groups + 1;
  p.runs = p.group_adapters + p.most_groups;
  p.ints = p.runs + (tokens <= kOneGroup ? 0 : tokens);
  p.ints = (p.ints + 3) / 4 * 4;
  return p;
}

struct AdapterPlanArgs {
  const int* ids;
  int* plan;
  AdapterPlan at;
  long long tokens;
  int adapters;
  int* status;
};

// Sums of `n` over the CTA's threads before each; `all` becomes the whole sum.
template <int THREADS>
__device__ __forceinline__ int sums_before_thread(int n, int* warp_sums, int& all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int s = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += up;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = s;
  __syncthreads();
  const int mine = lane < THREADS / 32 ? warp_sums[lane] : 0;
  all = __reduce_add_sync(0xffffffffu, mine);
  return s - n + __reduce_add_sync(0xffffffffu, lane < warp ? mine : 0);
}

// One CTA: a stable counting sort of the tokens by adapter, and each adapter's tiles.  A warp takes a run of the tokens, 32 at a time, and counts them in a row of
// its own (shared, [warps][adapters]); lanes of one adapter agree by a match, so that there is no atomic.
constexpr int kPlanThreads = 1024;
__global__ void __launch_bounds__(kPlanThreads) adapter_plan_kernel(AdapterPlanArgs a) {
  extern __shared__ int plan_sm[];
  constexpr int kWarps = kPlanThreads / 32;
  int* const counts = plan_sm;                           // [warps][adapters]
  int* const first = counts + kWarps * a.adapters;       // an adapter's first place
  int* const first_tile = first + a.adapters;
  int* const count = first_tile + a.adapters;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int i = tid; i < kWarps * a.adapters; i += kPlanThreads) counts[i] = 0;
  pdl_wait();
  __syncthreads();
  const long long each = ((a.tokens + kWarps - 1) / kWarps + 31) / 32 * 32, from = warp * each, to = from + each < a.tokens ? from + each : a.tokens;
  int* const mine = counts + warp * a.adapters;
  for (long long t0 = from; t0 < to; t0 += 32) {
    const long long t = t0 + lane;
    int id = t < to ? a.ids[t] : -1;
    if (id < -1 || id >= a.adapters) {
      if (a.status) *a.status = FLEXSPMV_ERR_BAD_CSR;
      id = -1;
    }
    if (t < to) a.plan[a.at.ids + t] = id;
    const unsigned same = __match_any_sync(0xffffffffu, id);
    if (id >= 0 && lane == __ffs(same) - 1) mine[id] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int i = tid; i < a.adapters; i += kPlanThreads) {
    int sum = 0;
    for (int w = 0; w < kWarps; ++w) {
      const int n = counts[w * a.adapters + i];
      counts[w * a.adapters + i] = sum;
      sum += n;
    }
    first[i] = sum;
  }
  __syncthreads();
  if (warp == 0) {
    int places = 0, tiles = 0;
    for (int i0 = 0; i0 < a.adapters; i0 += 32) {
      const int i = i0 + lane, n = i < a.adapters ? first[i] : 0, m = (n + kLowTile - 1) / kLowTile;
      int s = n, u = m;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, s, o), up_tiles = __shfl_up_sync(0xffffffffu, u, o);
        if (lane >= o) {
          s += up;
          u += up_tiles;
        }
      }
      if (i < a.adapters) {
        first[i] = places + s - n;
        first_tile[i] = tiles + u - m;
        count[i] = n;
        a.plan[a.at.offsets + i] = places + s - n;
      }
      places += __shfl_sync(0xffffffffu, s, 31);
      tiles += __shfl_sync(0xffffffffu, u, 31);
    }
    if (lane == 0) {
      a.plan[a.at.offsets + a.adapters] = places;
      a.plan[0] = a.at.most_tiles ? tiles : 0;
      a.plan[1] = (int)a.tokens;
      a.plan[2] = a.adapters;
    }
  }
  __syncthreads();
  if (a.at.most_tiles)
    for (int i = warp; i < a.adapters; i += kWarps) {
      AdapterTile* const out = reinterpret_cast<AdapterTile*>(a.plan + 8) + first_tile[i];
      for (int j = lane; j * kLowTile < count[i]; j += 32)
        out[j] = {i, first[i] + j * kLowTile, count[i] - j * kLowTile < kLowTile ? count[i] - j * kLowTile : kLowTile, 0};
    }
  for (long long t0 = from; t0 < to; t0 += 32) {
    const long long t = t0 + lane;
    const int id = t < to ? a.plan[a.at.ids + t] : -1;
    const unsigned same = __match_any_sync(0xffffffffu, id);
    if (id >= 0) a.plan[a.at.rows + first[id] + mine[id] + __popc(same & ((1u << lane) - 1))] = (int)t;
    __syncwarp();
    if (id >= 0 && lane == __ffs(same) - 1) mine[id] += __popc(same);
    __syncwarp();
  }
  // the groups
  int* const groups = a.plan + a.at.groups;
  int* const group_adapters = a.plan + a.at.group_adapters;
  const int tokens = (int)a.tokens;
  int found = 0;
  if (a.at.most_groups == 1) {
    if (tid == 0) {
      groups[0] = 0;
      group_adapters[0] = kGroupMixed;
    }
    found = 1;
  } else {
    __shared__ int warp_sums[kWarps];
    const int* const ids = a.plan + a.at.ids;
    int* const runs = a.plan + a.at.runs;
    int starts = 0;
    for (int t0 = 0; t0 < tokens; t0 += kPlanThreads) {
      const int t = t0 + tid;
      const bool begins = t < tokens && (t == 0 || ids[t] != ids[t - 1]);
      int all;
      const int before = sums_before_thread<kPlanThreads>(begins, warp_sums, all);
      if (begins) runs[starts + before] = t;
      starts += all;
    }
    __syncthreads();
    const auto is_long = [&](int r) { return (r + 1 < starts ? runs[r + 1] : tokens) - runs[r] >= a.at.long_run; };
    for (int r0 = 0; r0 < starts; r0 += kPlanThreads) {
      const int r = r0 + tid;
      const bool own = r < starts && is_long(r), begins = r < starts && (r == 0 || own || is_long(r - 1));
      int all;
      const int before = sums_before_thread<kPlanThreads>(begins, warp_sums, all);
      if (begins && found + before < a.at.most_groups) {
        groups[found + before] = runs[r];
        const int id = ids[runs[r]];
        group_adapters[found + before] = !own ? kGroupMixed : id >= 0 ? id : kGroupBare;
      }
      found += all;
    }
  }
  for (int i = found + tid; i <= a.at.most_groups; i += kPlanThreads) {
    groups[i] = tokens;
    if (i < a.at.most_groups) group_adapters[i] = kGroupBare;
  }
}

// ---- the first product ---------------------------------------------------------------------------------------------

struct LowArgs {
  const void *x, *down;
  const float* scale;
  const int *rows, *plan;
  const AdapterTile* tiles;
  void* low;
  float* wide;
  unsigned char* flags;
  long long stride;
  int tokens, adapters, rank, k, width, wide_width;
  int* status;
};

// low[t] = scale A x[t] of few tokens: a cluster of four CTAs takes a tile of up to 16 tokens of one adapter and 8 NB values of the rank (blockIdx.y), their warps every 32nd 32
// of the sum, so that a long one is a few rounds of loads; the warps' and the CTAs' sums meet in shared memory in their order.  Bound by the latency of reading the
// adapter, not by arithmetic, so the warp's own matrix instruction is enough and its operands come from global memory as they are: as the sum's index may be permuted, a
// lane's share of two instructions is 16 contiguous bytes of a row, and eight rows of 64 bytes are one load of the warp.  Many tokens: grouped_kernel.
// 256 threads leave room on their SM for a CTA of the product that begins meanwhile (NB = 2).
constexpr int kLowThreads = 256, kLowCtas = 4;
template <class T, int NB>
__global__ void __launch_bounds__(kLowThreads) adapter_low_kernel(LowArgs a) {
  constexpr int kAhead = NB == 2 ? 4 : 2;          // loads of so many steps under way
  constexpr int kWarps = kLowThreads / 32, kStep = 32 * kWarps * kLowCtas, kRanks = 8 * NB, kValues = 16 * kRanks;
  __shared__ float part[kWarps][16][kRanks + 1], sums[kValues];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = lane & 3, g = lane >> 2, r0 = blockIdx.y * kRanks, share = (int)cluster_rank();
  pdl_wait();
  pdl_launch_dependents();
  const int4 head = *reinterpret_cast<const int4*>(a.plan);
  const AdapterTile tile = a.tiles[blockIdx.x];     // on its way with the head; the plan has room for all that are launched
  // The whole cluster.  A plan of other tokens or adapters, or none yet: the next launch says so.
  if ((int)blockIdx.x >= head.x || head.y != a.tokens || head.z != a.adapters) return;
  if ((unsigned)tile.adapter >= (unsigned)a.adapters || tile.count < 1 || tile.count > kLowTile || tile.from < 0 || tile.from > a.tokens - tile.count) {
    if (threadIdx.x == 0 && a.status) *a.status = FLEXSPMV_ERR_BAD_CSR;
    return;
  }
  // rows and ranks that are not there: the first one's, whose results are left out
  const T *x[2], *down[NB];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int p = i * 8 + g, row = a.rows[tile.from + (p < tile.count ? p : 0)];
    const bool there = (unsigned)row < (unsigned)a.tokens;
    if (!there && a.status) *a.status = FLEXSPMV_ERR_BAD_CSR;
    x[i] = static_cast<const T*>(a.x) + (there ? row : 0) * a.stride;
  }
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int r = r0 + j * 8 + g;
    down[j] = static_cast<const T*>(a.down) + ((size_t)tile.adapter * a.rank + (r < a.rank ? r : r0)) * a.k;
  }
  float acc[NB][4];
#pragma unroll
  for (int i = 0; i < 4 * NB; ++i) acc[i / 4][i % 4] = 0.f;
  const bool high = tile.count > 8;          // else the upper rows' loads are left out
  for (int k0 = (share * kWarps + warp) * 32; k0 < a.k; k0 += kStep * kAhead) {
    uint4 v[kAhead][2], w[kAhead][NB];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int k = k0 + u * kStep + q * 8;
      v[u][0] = v[u][1] = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < NB; ++j) w[u][j] = v[u][0];
      if (k < a.k) {
#pragma unroll
        for (int j = 0; j < NB; ++j) w[u][j] = *reinterpret_cast<const uint4*>(down[j] + k);
        v[u][0] = *reinterpret_cast<const uint4*>(x[0] + k);
        if (high) v[u][1] = *reinterpret_cast<const uint4*>(x[1] + k);
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        warp_mma<T>(acc[j], v[u][0].x, v[u][1].x, v[u][0].y, v[u][1].y, w[u][j].x, w[u][j].y);
        warp_mma<T>(acc[j], v[u][0].z, v[u][1].z, v[u][0].w, v[u][1].w, w[u][j].z, w[u][j].w);
      }
  }
#pragma unroll
  for (int j = 0; j < NB; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[warp][g + i / 2 * 8][j * 8 + q * 2 + i % 2] = acc[j][i];
  __syncthreads();
#pragma unroll
  for (int i = threadIdx.x; i < kValues; i += kLowThreads) {
    float h = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) h += part[w][i / kRanks][i % kRanks];
    sums[i] = h;
  }
  cluster_sync();
  // each CTA some of the tokens; 16 of the rank at a time, with zeros: the second product takes as many
  static_assert(kValues / kLowCtas % 32 == 0, "whole warps");
  for (int i = threadIdx.x; i < kValues / kLowCtas; i += kLowThreads) {
    const int p = i / kRanks * kLowCtas + share, j = i % kRanks, r = r0 + j;
    const int to = p < tile.count ? a.rows[tile.from + p] : -1;
    float h = 0.f;
    if (p < tile.count && r < a.rank) {
#pragma unroll
      for (int c = 0; c < kLowCtas; ++c) h += cluster_load(cluster_smem(&sums[p * kRanks + j], c));
      if (a.scale) h *= a.scale[tile.adapter];
    }
    bool wide = false;
    if constexpr (kHasWide<T>) {             // the 32 that a flag is of (ranks up to 16: 16) are a warp's (a half's)
      const unsigned mine = kRanks >= 32 ? 0xffffffffu : 0xffffu << (lane & 16);
      const unsigned above = __ballot_sync(0xffffffffu, !(fabsf(h) <= kWideAbove)), some = __ballot_sync(0xffffffffu, h != 0.f),
                     large = __ballot_sync(0xffffffffu, fabsf(h) >= kWideBelow);
      wide = (above & mine) || ((some & mine) && !(large & mine));
    }
    if ((unsigned)to >= (unsigned)a.tokens || r >= ((a.rank + 15) & ~15)) continue;
    if constexpr (kHasWide<T>) {
      if (j % 32 == 0) a.flags[(long long)(r / 32) * a.tokens + to] = wide;
      if (wide) {
        a.wide[(long long)to * a.wide_width + r] = h;
        h = 0.f;
      }
    }
    T* const row = static_cast<T*>(a.low) + (long long)to * a.width;
    float part[kLowParts<T>];
    low_parts<T>(h, part);
#pragma unroll
    for (int x = 0; x < kLowParts<T>; ++x) row[low_at<T>(r, a.rank, x)] = from_float<T>(part[x]);
  }
  cluster_sync();                          // no CTA leaves while its sums may be read
}

// The SMs divide their memory as for the kernel that follows: else a CTA of that one waits until an SM is empty.
template <auto KERNEL>
static int shared_memory_first() {
  static std::atomic<bool> done[64];
  int device = 0;
  if (cudaError_t e = cudaGetDevice(&device); e != cudaSuccess) return (int)e;
  const bool known = device >= 0 && device < 64;
  if (known && done[device].load(std::memory_order_relaxed)) return 0;
  if (cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared); e != cudaSuccess)
    return (int)e;
  if (known) done[device].store(true, std::memory_order_relaxed);
  return 0;
}

template <class T, int NB>
static int low_launch(const LowArgs& a, const AdapterPlan& p, cudaStream_t st) {
  if (int e = shared_memory_first<adapter_low_kernel<T, NB>>()) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.most_tiles, (unsigned)((a.rank + 8 * NB - 1) / (8 * NB)), kLowCtas); cfg.blockDim = dim3(kLowThreads); cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = kLowCtas;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, adapter_low_kernel<T, NB>, a);
}
template <class T>
static int low_product(const LowArgs& a, const AdapterPlan& p, cudaStream_t st) {
  if (a.rank <= 16) return low_launch<T, 2>(a, p, st);
  if (a.rank <= 32) return low_launch<T, 4>(a, p, st);
  return low_launch<T, 8>(a, p, st);
}

// `product`: n, k and the rank count too.
static int check_adapters(const flexspmv_adapter_desc* d, bool product) {
  if (!d || d->tokens < 0 || d->adapters < 1) return FLEXSPMV_ERR_BAD_ARG;
  if (product && (d->rank < 1 || d->n < 1 || d->k < 1 || d->x_stride < d->k || (d->type != FLEXSPMV_TYPE_BF16 && d->type != FLEXSPMV_TYPE_F16)))
    return FLEXSPMV_ERR_BAD_ARG;
  if (d->tokens > 0x7fff0000LL || d->adapters > FLEXSPMV_MAX_ADAPTERS) return FLEXSPMV_ERR_TOO_LARGE;
  if (product) {
    // places and tiles are counted in 32 bits
    if (d->rank > FLEXSPMV_MAX_RANK || (d->n / 128 + 1.0) * (d->tokens / 32 + 2.0) > 2e9) return FLEXSPMV_ERR_TOO_LARGE;
    if (d->rank % 8 || d->n % 8 || d->k % 8 || d->x_stride % 8) return FLEXSPMV_ERR_ALIGN;
  }
  return 0;
}

}  // namespace flex

extern "C" {

int flexspmv_adapter_plan_bytes(const flexspmv_adapter_desc* d, size_t* bytes) {
  if (!bytes) return FLEXSPMV_ERR_BAD_ARG;
  if (int e = flex::check_adapters(d, false)) return e;
  *bytes = (size_t)flex::adapter_plan_of(d->tokens, d->adapters).ints * 4;
  return 0;
}

int flexspmv_adapter_plan(const flexspmv_adapter_desc* d, const int32_t* ids, void* plan, size_t plan_bytes, int32_t* status, void* stream) {
  using namespace flex;
  if (int e = check_adapters(d, false)) return e;
  if (d->tokens && !ids) return FLEXSPMV_ERR_BAD_ARG;
  const AdapterPlan p = adapter_plan_of(d->tokens, d->adapters);
  if (!plan || plan_bytes < (size_t)p.ints * 4) return FLEXSPMV_ERR_WORKSPACE;
  if (!aligned16(plan) || !aligned_to(4, ids, status)) return FLEXSPMV_ERR_ALIGN;
  if (!apart({{plan, p.ints * 4}}, {{ids, 4 * d->tokens}})) return FLEXSPMV_ERR_BAD_ARG;
  const AdapterPlanArgs a = {ids, static_cast<int*>(plan), p, d->tokens, d->adapters, status};
  const int smem = (kPlanThreads / 32 + 3) * d->adapters * 4;
  if (int e = allow_smem<adapter_plan_kernel>(smem)) return e;
  return launch_pdl(adapter_plan_kernel, 1, kPlanThreads, (size_t)smem, static_cast<cudaStream_t>(stream), a);
}

int flexspmv_adapted_project_bytes(const flexspmv_adapter_desc* d, size_t* bytes) {
  if (!bytes) return FLEXSPMV_ERR_BAD_ARG;
  if (int e = flex::check_adapters(d, true)) return e;
  *bytes = (size_t)flex::low_places(d->tokens, d->rank, d->type).bytes;
  return 0;
}

int flexspmv_adapted_project(const flexspmv_adapter_desc* d, const void* const* in, void* const* out, void* ws, size_t ws_bytes, int32_t* status, void* stream) {
  using namespace flex;
  if (int e = check_adapters(d, true)) return e;
  if (!in || !out) return FLEXSPMV_ERR_BAD_ARG;
  if (d->tokens == 0) return 0;
  if (!in[0] || !in[1] || !in[2] || !in[3] || !in[5] || !out[0]) return FLEXSPMV_ERR_BAD_ARG;
  const LowPlaces low = low_places(d->tokens, d->rank, d->type);
  const size_t need = (size_t)low.bytes;
  if (!ws || ws_bytes < need) return FLEXSPMV_ERR_WORKSPACE;
  if (!aligned16(in[0]) || !aligned16(in[1]) || !aligned16(in[2]) || !aligned16(in[3]) || !aligned16(in[5]) || !aligned16(out[0]) || !aligned16(ws) ||
      !aligned_to(4, in[4], status))
    return FLEXSPMV_ERR_ALIGN;
  const AdapterPlan p = adapter_plan_of(d->tokens, d->adapters);
  const long long all = (long long)d->adapters * d->rank;
  if (!apart({{out[0], 2 * d->tokens * d->n}, {ws, (long long)need}},
             {rows_at(in[0], d->tokens, d->k, d->x_stride, d->type), {in[1], 2ll * d->n * d->k}, {in[2], 2 * all * d->k}, {in[3], 2 * all * d->n},
              {in[4], 4ll * d->adapters}, {in[5], p.ints * 4}}))
    return FLEXSPMV_ERR_BAD_ARG;
  const int* const plan = static_cast<const int*>(in[5]);
  const LowArgs a = {in[0], in[2], static_cast<const float*>(in[4]), plan + p.rows, plan, reinterpret_cast<const AdapterTile*>(plan + p.tiles), ws,
                     reinterpret_cast<float*>(static_cast<char*>(ws) + low.wide), static_cast<unsigned char*>(ws) + low.flags, d->x_stride, (int)d->tokens,
                     d->adapters, d->rank, d->k, low.width, low.wide_width, status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int e;
  if (!low_in_tiles(d->tokens, d->rank)) e = low_product_of_many(d, in[0], in[2], a.scale, plan + p.offsets, a.rows, ws, status, st);
  else e = d->type == FLEXSPMV_TYPE_BF16 ? low_product<__nv_bfloat16>(a, p, st) : low_product<__half>(a, p, st);
  if (e) return e;
  return adapted_product(d, in[0], in[1], in[3], ws, plan, p.most_groups, plan + p.groups, plan + p.group_adapters, plan + p.ids, out[0], status, st);
}

}  // extern "C"
