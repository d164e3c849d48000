// Low-rank adapters of many requests beside a shared projection: y[t] = W x[t] + scale[a] B[a] (A[a] x[t]), a = ids[t].
// Here: the plan of a batch and the first product, low[t] = scale A x[t].  The rest is the shared product's epilogue (flex_grouped.cu).
#include <cuda_runtime.h>

#include "flex_adapters.cuh"
#include "flex_common.cuh"
#include "flex_expert_types.cuh"

namespace flex {

int device_sm_count();

// ---- plan ----------------------------------------------------------------------------------------------------------

struct AdapterTile {
  int adapter, from, count, unused;          // places from .. from + count of `rows`, all of one adapter
};

// Where a plan's parts lie, in ints: [0] the number of tiles, [4, 5] the offsets of one group of all tokens.
struct AdapterPlan {
  long long ids, rows, tiles, ints;
  int most_tiles, tile;
};
static AdapterPlan adapter_plan_of(long long tokens, int adapters) {
  AdapterPlan p;
  // few tokens: tiles of one instruction's rows, as many as can be for the sake of their latency; else of four, which read an adapter a quarter as often
  p.tile = tokens <= 1024 ? 16 : 64;
  p.most_tiles = (int)(tokens / p.tile + (tokens < adapters ? tokens : adapters));
  p.tiles = 8;
  p.ids = p.tiles + 4ll * p.most_tiles;
  p.rows = p.ids + tokens;
  p.ints = (p.rows + tokens + 3) / 4 * 4;
  return p;
}

struct AdapterPlanArgs {
  const int* ids;
  int* plan;
  long long tokens, at_ids, at_rows;
  int adapters, tile;
  int* status;
};

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
    if (t < to) a.plan[a.at_ids + t] = id;
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
      const int i = i0 + lane, n = i < a.adapters ? first[i] : 0, m = (n + a.tile - 1) / a.tile;
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
      }
      places += __shfl_sync(0xffffffffu, s, 31);
      tiles += __shfl_sync(0xffffffffu, u, 31);
    }
    if (lane == 0) {
      a.plan[0] = tiles;
      a.plan[4] = 0;
      a.plan[5] = (int)a.tokens;
    }
  }
  __syncthreads();
  for (int i = warp; i < a.adapters; i += kWarps) {
    AdapterTile* const out = reinterpret_cast<AdapterTile*>(a.plan + 8) + first_tile[i];
    for (int j = lane; j * a.tile < count[i]; j += 32)
      out[j] = {i, first[i] + j * a.tile, count[i] - j * a.tile < a.tile ? count[i] - j * a.tile : a.tile, 0};
  }
  for (long long t0 = from; t0 < to; t0 += 32) {
    const long long t = t0 + lane;
    const int id = t < to ? a.plan[a.at_ids + t] : -1;
    const unsigned same = __match_any_sync(0xffffffffu, id);
    if (id >= 0) a.plan[a.at_rows + first[id] + mine[id] + __popc(same & ((1u << lane) - 1))] = (int)t;
    __syncwarp();
    if (id >= 0 && lane == __ffs(same) - 1) mine[id] += __popc(same);
    __syncwarp();
  }
}

// ---- the first product ---------------------------------------------------------------------------------------------

struct LowArgs {
  const void *x, *down;
  const float* scale;
  const int *rows, *count;
  const AdapterTile* tiles;
  void* low;
  long long stride;
  int rank, k, width;
};

// low[t] = scale A x[t]: a CTA takes a tile of up to 16 MB tokens of one adapter and 8 NB values of the rank (blockIdx.y), its eight warps every eighth 32 of the
// sum, and their sums meet in shared memory in the warps' order.  Bound by reading x and the adapters, not by arithmetic, so the warps' own matrix instruction is
// enough and its operands come from global memory as they are: as the sum's index may be permuted, a lane's share of two instructions is 16 contiguous
// bytes of a row, and eight rows of 64 bytes are one load of the warp.
template <class T, int MB, int NB>
__global__ void __launch_bounds__(256) adapter_low_kernel(LowArgs a) {
  __shared__ float joined[16 * MB][8 * NB + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = lane & 3, g = lane >> 2, r0 = blockIdx.y * 8 * NB;
  pdl_wait();
  pdl_launch_dependents();
  if ((int)blockIdx.x >= *a.count) return;
  const AdapterTile tile = a.tiles[blockIdx.x];
  const T* x[MB][2];
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int p = m * 16 + i * 8 + g;
      x[m][i] = p < tile.count ? static_cast<const T*>(a.x) + (long long)a.rows[tile.from + p] * a.stride : nullptr;
    }
  const T* const down = static_cast<const T*>(a.down) + ((size_t)tile.adapter * a.rank + r0 + g) * a.k;
  const int blocks = (tile.count + 15) / 16;
  float acc[MB][NB][4];
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[m][j][i] = 0.f;
  const uint4 none = make_uint4(0, 0, 0, 0);
#pragma unroll MB == 1 ? 4 : 1
  for (int k0 = warp * 32; k0 < a.k; k0 += 256) {
    const int k = k0 + q * 8;
    uint4 v[MB][2], w[NB];
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int i = 0; i < 2; ++i) v[m][i] = x[m][i] && k < a.k ? *reinterpret_cast<const uint4*>(x[m][i] + k) : none;
#pragma unroll
    for (int j = 0; j < NB; ++j) w[j] = r0 + j * 8 + g < a.rank && k < a.k ? *reinterpret_cast<const uint4*>(down + (size_t)j * 8 * a.k + k) : none;
#pragma unroll
    for (int m = 0; m < MB; ++m) {
      if (m >= blocks) break;
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        warp_mma<T>(acc[m][j], v[m][0].x, v[m][1].x, v[m][0].y, v[m][1].y, w[j].x, w[j].y);
        warp_mma<T>(acc[m][j], v[m][0].z, v[m][1].z, v[m][0].w, v[m][1].w, w[j].z, w[j].w);
      }
    }
  }
  for (int turn = 0; turn < 8; ++turn) {
    if (warp == turn)
#pragma unroll
      for (int m = 0; m < MB; ++m)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float& s = joined[m * 16 + g + i / 2 * 8][j * 8 + q * 2 + i % 2];
            s = turn ? s + acc[m][j][i] : acc[m][j][i];
          }
    __syncthreads();
  }
  const float scale = a.scale ? a.scale[tile.adapter] : 1.f;
  for (int i = threadIdx.x; i < tile.count * NB; i += 256) {
    const int p = i / NB, j = i % NB * 8;
    if (r0 + j >= a.rank) continue;
    Pack<T, 8> high, rest;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const float h = joined[p][j + u] * scale;
      high.set(u, h);
      const float r = h - high.get(u);
      rest.set(u, fabsf(high.get(u)) <= 3.4e38f ? r : 0.f);          // of what is not finite: none
    }
    T* const row = static_cast<T*>(a.low) + (long long)a.rows[tile.from + p] * a.width;
    high.store(row + low_high(r0 + j, a.rank));
    rest.store(row + low_rest(r0 + j, a.rank));
  }
}

template <class T>
static int low_product(const LowArgs& a, const AdapterPlan& p, cudaStream_t st) {
  const auto go = [&](auto kernel, int ranks) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.most_tiles, (unsigned)((a.rank + ranks - 1) / ranks)); cfg.blockDim = dim3(256); cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = pdl_enabled() ? 1 : 0;
    return (int)cudaLaunchKernelEx(&cfg, kernel, a);
  };
  if (p.tile == 16) return go(adapter_low_kernel<T, 1, 2>, 16);
  if (a.rank <= 16) return go(adapter_low_kernel<T, 4, 2>, 16);
  if (a.rank <= 32) return go(adapter_low_kernel<T, 4, 4>, 32);
  return go(adapter_low_kernel<T, 4, 8>, 64);
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
  const AdapterPlanArgs a = {ids, static_cast<int*>(plan), d->tokens, p.ids, p.rows, d->adapters, p.tile, status};
  const int smem = (kPlanThreads / 32 + 3) * d->adapters * 4;
  if (int e = allow_smem<adapter_plan_kernel>(smem)) return e;
  return launch_pdl(adapter_plan_kernel, 1, kPlanThreads, (size_t)smem, static_cast<cudaStream_t>(stream), a);
}

int flexspmv_adapted_project_bytes(const flexspmv_adapter_desc* d, size_t* bytes) {
  if (!bytes) return FLEXSPMV_ERR_BAD_ARG;
  if (int e = flex::check_adapters(d, true)) return e;
  *bytes = (size_t)d->tokens * flex::low_width(d->rank) * 2;
  return 0;
}

int flexspmv_adapted_project(const flexspmv_adapter_desc* d, const void* const* in, void* const* out, void* ws, size_t ws_bytes, int32_t* status, void* stream) {
  using namespace flex;
  if (int e = check_adapters(d, true)) return e;
  if (!in || !out) return FLEXSPMV_ERR_BAD_ARG;
  if (d->tokens == 0) return 0;
  if (!in[0] || !in[1] || !in[2] || !in[3] || !in[5] || !out[0]) return FLEXSPMV_ERR_BAD_ARG;
  const int width = low_width(d->rank);
  const size_t need = (size_t)d->tokens * width * 2;
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
  const LowArgs a = {in[0], in[2], static_cast<const float*>(in[4]), plan + p.rows, plan, reinterpret_cast<const AdapterTile*>(plan + p.tiles), ws, d->x_stride,
                     d->rank, d->k, width};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int e = d->type == FLEXSPMV_TYPE_BF16 ? low_product<__nv_bfloat16>(a, p, st) : low_product<__half>(a, p, st)) return e;
  return adapted_product(d, in[0], in[1], in[3], ws, width, plan + 4, plan + p.ids, out[0], status, st);
}

}  // extern "C"
