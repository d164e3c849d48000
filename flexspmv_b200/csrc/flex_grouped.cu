// Matrix products grouped by expert over ragged groups of rows:
//   forward  y[i] = W[e] x[rows[i]]        dx  dx[i] = W[e]^T dy[i]        dw  dW[e] = sum_i dy[i] x[rows[i]]^T
#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "flex_common.cuh"
#include "flex_expert_types.cuh"
#include "flex_umma.cuh"

namespace flex {

int device_sm_count();

enum GroupedMode { kGroupedForward, kGroupedDx, kGroupedDw };

struct GroupedArgs {
  const void *a, *b;             // forward: x, weight; dx: dy, weight; dw: dy, x
  const int *offsets, *rows;     // rows: of x, in the places' order; null: place i is x's row i
  void* out;
  long long tokens, slots, a_stride, b_stride;
  int experts, n, k;
  int* status;
};

__device__ __forceinline__ void raise(int* status, int code) {
  if (status) *status = code;
}

// The places of an expert, kept inside [0, slots] whatever offsets holds.
__device__ __forceinline__ void group_of(const GroupedArgs& a, int e, int& from, int& to) {
  const int f = a.offsets[e], t = a.offsets[e + 1];
  from = f < 0 ? 0 : f > a.slots ? (int)a.slots : f;
  to = t < from ? from : t > a.slots ? (int)a.slots : t;
  if (f != from || t != to) raise(a.status, FLEXSPMV_ERR_BAD_CSR);
}

// dw with a list of rows: x's rows in the places' order, in the workspace.
__global__ void __launch_bounds__(256) take_rows_kernel(const uint4* __restrict__ x, const int* __restrict__ rows, const int* __restrict__ offsets, uint4* __restrict__ out,
                                                        long long tokens, long long slots, long long stride, int experts, int pieces, int* status) {
  pdl_wait();
  pdl_launch_dependents();
  const long long from = offsets[0] < 0 ? 0 : offsets[0], to = offsets[experts] < slots ? offsets[experts] : slots;
  const long long work = (to - from) * pieces;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < work; i += (long long)gridDim.x * 256) {
    const long long p = from + i / pieces;
    const int c = (int)(i % pieces), r = rows[p];
    const bool in = r >= 0 && r < tokens;
    if (!in) raise(status, FLEXSPMV_ERR_BAD_CSR);
    out[p * pieces + c] = in ? x[r * stride + c] : make_uint4(0, 0, 0, 0);
  }
}

// One CTA an SM walks over tiles of 128 rows by NT columns of the accumulator; the accumulator's rows are a matrix side, so that
//   forward, dx   128 values of y (dx) by up to NT places: the weights are the first operand, and a group's last tile is as narrow as its
//                 rows need (a multiple of 16), down to one place
//   dw            128 of n by 256 of k, summed over the expert's places
// PAIR = 2: two CTAs on two neighbouring SMs take a tile of 256 rows, 128 each; each copies half of the columns' operand for both, which
// halves what those columns cost the L2 (from 48 KB to 32 KB an SM for 64 of the sum).
// HALVES = 2: a tile has twice the rows, half of them in each accumulator; the columns' operand is copied once for both.
// SPLIT: few tiles.  A cluster of up to eight CTAs takes one tile, each its share of the sum; the parts meet in shared memory, where every CTA
// adds up some of the columns in the CTAs' order.  No workspace, no atomics.
// GATHER (forward): x's rows by a list.  Four more warps copy them, 16 bytes a thread, to where a tile copy would have put them; as fast as contiguous
// rows up to some thousand rows, 2 - 4 % slower for 32 768 of 2048.  (Tile copies that gather four rows each took 72 cycles an instruction: 2.2 ms
// there instead of 0.43.)  dw's rows are other ones in every step: gathered like this they take 0.57 ms of the 32 768; a copy of them in the
// workspace and contiguous tile copies 0.44.
// Warps 0-7 store finished accumulators, warp 8 issues the tile copies, warp 9 the matrix instructions; two accumulators in tensor memory,
// so that one is stored while the next is computed (HALVES = 2: while the other half of the next tile begins).  The sum goes 64 values (128 bytes of a row) a stage.
constexpr int kStoreWarps = 8, kCopyWarp = kStoreWarps, kMathWarp = kStoreWarps + 1, kGroupedThreads = (kStoreWarps + 2) * 32;
constexpr int kGatherWarps = 4;
constexpr int grouped_threads(bool gather) { return kGroupedThreads + (gather ? kGatherWarps * 32 : 0); }
constexpr int kTileBytesA = 128 * 128;
constexpr uint64_t kWaitLimitNs = 1000000000ull;
// The tensor cores cut a sum's low bits at every addition, always towards zero: a relative error of 4e-9 to 6e-9 a row where all products have one sign
// (1e-9 of random ones).  PARTS (dw): sums are added up, correctly rounded, from parts of so many steps that the result does not show it.  Of 32 bits:
// always, from 512 rows each.  Of 16, whose half unit is 2.4e-4 of a float16 and 2e-3 of a bfloat16 at the least: from 4096 (2e-5), where there are more rows
// than keep a whole sum below 0.4 of that.  A kernel of its own, since the sums' registers cost all others 2 - 10 %.
constexpr int kPartSteps32 = 8, kPartSteps16 = 64;
template <class T> constexpr int kWholeRows = std::is_same<T, __half>::value ? 16384 : 131072;

template <int MODE, int NT, int PAIR, int HALVES, int OUT_BYTES>
struct GroupedCfg {
  static constexpr int kBytesA = HALVES * kTileBytesA, kBytesB = NT / PAIR * 128;
  static constexpr int kStageBytes = kBytesA + kBytesB;
  static constexpr int kStages = (OUT_BYTES == 4 ? 180224 : 196608) / kStageBytes;
  static constexpr int kTmemCols = 2 * NT < 32 ? 32 : 2 * NT;
  static constexpr int kStoreBytes = kStoreWarps * 1024 * OUT_BYTES;        // 32 x 32 results a warp
};

struct GroupedTable {            // of an expert: its first place, its places, its first tile; and of one past the last: the number of tiles
  int from, count, first;
};

struct GroupedBars {
  uint64_t full[9], empty[9], gathered[9], acc_full[2], acc_empty[2];
  uint32_t tmem;
  int abort;
};

struct GroupedTile {
  int e, m0, n0, from, count, cols;     // dw: m0 of n, n0 of k; else m0 of the features, places from .. from + count; cols: the accumulator's
  int half, halves_end;                 // the halves of its rows that are this cluster's: half .. halves_end - 1
};

// How many places a tile of a group of `count` takes: the group in equal parts, in 16s (a pair: in 32s).
template <int NT, int PAIR>
__device__ __forceinline__ int tile_places(int count) {
  constexpr int kStep = 16 * PAIR;
  const int tiles = (count + NT - 1) / NT;
  return ((count + tiles - 1) / tiles + kStep - 1) & ~(kStep - 1);
}

template <int MODE, int NT, int PAIR, int HALVES>
__device__ __forceinline__ GroupedTile tile_at(const GroupedArgs& a, const GroupedTable* table, int t) {
  GroupedTile r;
  const int m = MODE == kGroupedDx ? a.k : a.n;
  constexpr int kRows = 128 * PAIR * HALVES;
  const int m_tiles = (m + kRows - 1) / kRows;
  constexpr int kStep = 16 * PAIR;
  if (MODE == kGroupedDw) {
    const int n_tiles = (a.k + NT - 1) / NT, each = m_tiles * n_tiles;
    r.e = t / each;
    const int i = t - r.e * each;
    r.m0 = i / n_tiles * kRows;
    r.n0 = i % n_tiles * NT;
    r.from = table[r.e].from;
    r.count = table[r.e].count;
    const int left = a.k - r.n0;
    r.cols = left < NT ? (left + kStep - 1) & ~(kStep - 1) : NT;
    return r;
  }
  int lo = 0, hi = a.experts;             // the last expert whose first tile is at or before t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (table[mid].first <= t) lo = mid;
    else hi = mid;
  }
  r.e = lo;
  const int i = t - table[lo].first, size = tile_places<NT, PAIR>(table[lo].count), part = i / m_tiles * size;
  r.m0 = i % m_tiles * kRows;
  r.n0 = 0;
  r.from = table[lo].from + part;
  r.count = table[lo].count - part < size ? table[lo].count - part : size;
  r.cols = (r.count + kStep - 1) & ~(kStep - 1);
  return r;
}

template <class T, class TO, int MODE, int NT, int PAIR, int HALVES, bool SPLIT, bool GATHER, bool PARTS>
__global__ void __launch_bounds__(grouped_threads(GATHER), 1) grouped_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                                                                     const __grid_constant__ CUtensorMap row_a, const __grid_constant__ CUtensorMap row_b,
                                                                     const __grid_constant__ CUtensorMap map_out,
                                                                     GroupedArgs a) {
  using Cfg = GroupedCfg<MODE, NT, PAIR, HALVES, (int)sizeof(TO)>;
  constexpr int kThreads = grouped_threads(GATHER);
  extern __shared__ __align__(1024) unsigned char grouped_sm[];
  unsigned char* const base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(grouped_sm) + 1023) & ~(uintptr_t)1023);
  unsigned char* const store = base + Cfg::kStages * Cfg::kStageBytes;
  GroupedBars& bars = *reinterpret_cast<GroupedBars*>(store + Cfg::kStoreBytes);
  GroupedTable* const table = reinterpret_cast<GroupedTable*>(&bars + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = PAIR == 2 ? (int)cluster_rank() : 0;
  const int split = SPLIT ? (int)cluster_size() : 1, share = SPLIT ? (int)cluster_rank() : 0;
  constexpr bool kA_mn = MODE != kGroupedForward, kB_mn = MODE == kGroupedDw;
  constexpr int kPartSteps = sizeof(TO) == 4 ? kPartSteps32 : kPartSteps16;

  if (tid == 0) {
    for (int i = 0; i < Cfg::kStages; ++i) {
      mbar_init(&bars.full[i], GATHER && PAIR == 2 ? 2 : 1);          // the copies, and the other CTA's gathered rows
      mbar_init(&bars.empty[i], 1);
      mbar_init(&bars.gathered[i], kGatherWarps * 32);
    }
    for (int i = 0; i < 2; ++i) { mbar_init(&bars.acc_full[i], 1); mbar_init(&bars.acc_empty[i], kStoreWarps * PAIR); }
    bars.abort = 0;
    mbar_fence_init();
    tma_prefetch_map(&map_a);
    tma_prefetch_map(&map_b);
    if (MODE == kGroupedDw) tma_prefetch_map(&map_out);
  }
  if (warp == kMathWarp) tmem_alloc<PAIR, Cfg::kTmemCols>(&bars.tmem);
  pdl_wait();
  for (int e = tid; e < a.experts; e += kThreads) {
    int from, to;
    group_of(a, e, from, to);
    table[e].from = from;
    table[e].count = to - from;
  }
  __syncthreads();
  const int m_rows = MODE == kGroupedDx ? a.k : a.n;
  const int m_tiles = (m_rows + 128 * PAIR * HALVES - 1) / (128 * PAIR * HALVES);
  if (warp == 0) {                         // exclusive sums of the experts' tiles
    int done = 0;
    for (int e0 = 0; e0 <= a.experts; e0 += 32) {
      const int e = e0 + lane;
      const int n = e < a.experts ? (table[e].count + NT - 1) / NT * m_tiles : 0;
      int s = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += up;
      }
      if (e <= a.experts) table[e].first = done + s - n;
      done += __shfl_sync(0xffffffffu, s, 31);
    }
  }
  tmem_fence_before();
  __syncthreads();
  if (PAIR == 2) cluster_sync();           // the other CTA's barriers are set up
  tmem_fence_after();
  const uint32_t tmem = bars.tmem;
  const int tiles = MODE == kGroupedDw ? a.experts * m_tiles * ((a.k + NT - 1) / NT) : table[a.experts].first;
  const int first = blockIdx.x / (PAIR * split);
  const int stride = gridDim.x / PAIR;
  volatile int* const abort = &bars.abort;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort) return false;
    if (mbar_wait_bounded(bar, parity, kWaitLimitNs)) return true;
    *abort = 1;
    raise(a.status, FLEXSPMV_ERR_TIMEOUT);
    return false;
  };
  // for a whole warp: all of its lanes go on, or none
  auto wait_warp = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
  auto stopped = [&] { return __any_sync(0xffffffffu, *abort) != 0; };
  auto steps_of = [&](const GroupedTile& t) {
    return ((MODE == kGroupedForward ? a.k : MODE == kGroupedDx ? a.n : t.count) + 63) / 64;
  };
  // This cluster's tile of round u.  Where the last round has tiles for half or a quarter of the clusters at most, each is divided in two or four: HALVES = 2
  // in two by rows, else by places.  us, whole / divided: 4102 rows of 16 experts of 1024 x 2048 26.8 / 25.1, dx 22.8 / 22.3, with a list of rows
  // 27.7 / 27.1; 5003 rows of 40 experts of 1000 x 1416 with a list 37.1 / 36.1; 1024 rows of 8 experts of 2048 x 2048 14.4 / 14.5.
  const int rounds = SPLIT ? 0 : tiles / stride, rest = SPLIT ? tiles : tiles - rounds * stride;
  constexpr int kMostHalvings = HALVES == 2 ? 1 : SPLIT || MODE == kGroupedDw || NT == 64 ? 0 : 2;
  const int halvings = kMostHalvings >= 2 && rest * 4 <= stride ? 2 : kMostHalvings >= 1 && rest * 2 <= stride ? 1 : 0;
  auto tile_of = [&](int u, GroupedTile& t) {
    const int by = u == rounds ? halvings : 0;
    if (u > rounds || (u == rounds && first >= rest << by)) return false;
    t = tile_at<MODE, NT, PAIR, HALVES>(a, table, u * stride + (first >> by));
    t.half = 0;
    t.halves_end = HALVES == 2 && t.m0 + 128 * PAIR < m_rows ? 2 : 1;
    if (by > 0) {
      const int part = first & ((1 << by) - 1);
      if (HALVES == 2) {
        t.half = part;
        if (part == 0) t.halves_end = 1;
      } else {
        constexpr int kStep = 16 * PAIR;
        const int size = ((t.cols / kStep + (1 << by) - 1) >> by) * kStep, left = t.count - part * size;
        t.from += part * size;
        t.count = left < size ? left : size;
        t.cols = left <= 0 ? 0 : (t.count + kStep - 1) & ~(kStep - 1);
      }
    }
    return true;
  };
  auto nothing_of = [&](const GroupedTile& t) { return HALVES == 2 ? t.half >= t.halves_end : kMostHalvings > 0 && t.cols == 0; };
  // this CTA's steps of a tile
  auto step_from = [&](int steps) { return SPLIT ? steps * share / split : 0; };
  auto step_to = [&](int steps) { return SPLIT ? steps * (share + 1) / split : steps; };

  if (warp == kCopyWarp) {
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    if (elect_one()) {
      GroupedTile t;
      for (int u = 0; !*abort && tile_of(u, t); ++u) {
        const int steps = steps_of(t), from = step_from(steps), to = step_to(steps), half = t.cols / PAIR;
        if (nothing_of(t)) continue;
        const int pieces = GATHER ? 0 : MODE == kGroupedDw ? (half + 63) / 64 : (half + 31) / 32;          // of the columns' operand
        const int m0 = t.m0 + rank * 128, halves = t.halves_end - t.half;
        for (int s = from; s < to; ++s) {
          if (!wait(&bars.empty[stage], phase ^ 1)) break;
          unsigned char* const sa = base + stage * Cfg::kStageBytes;
          unsigned char* const sb = sa + Cfg::kBytesA;
          const uint32_t bar = PAIR == 2 ? cluster_smem(&bars.full[stage], 0) : smem_u32(&bars.full[stage]);
          if (MODE == kGroupedDw) {
            // A step's last rows may be the next group's.  The maps count rows by two dimensions of one stride, y + z, and y ends at 64: with the
            // step's last valid row at y = 63, what follows it is out of range and zero.
            const int valid = t.count - s * 64 < 64 ? t.count - s * 64 : 64, place = t.from + s * 64, z = place + valid - 64;
            const int rows = z >= 0 ? 64 : (valid + 15) & ~15, n0 = t.n0 + rank * half;          // rows: how many are copied
            if (rank == 0) mbar_expect_tx(&bars.full[stage], PAIR * (2 * halves + pieces) * rows * 128);
            if (z >= 0) {
              for (int h = t.half; h < t.halves_end; ++h) {
                tma_3d<PAIR>(sa + h * kTileBytesA, &map_a, m0 + h * 128 * PAIR, 64 - valid, z, bar);
                tma_3d<PAIR>(sa + h * kTileBytesA + 8192, &map_a, m0 + h * 128 * PAIR + 64, 64 - valid, z, bar);
              }
              for (int g = 0; g < pieces; ++g) tma_3d<PAIR>(sb + g * 8192, &map_b, n0 + g * 64, 64 - valid, z, bar);
            } else {                       // a group that ends in the first 64 rows: row by row, rows out of range for the rest
              for (int r = 0; r < rows; ++r) {
                const int y = r < valid ? place + r : (int)a.slots;
                for (int h = t.half; h < t.halves_end; ++h) {
                  tma_2d<PAIR>(sa + h * kTileBytesA + r * 128, &row_a, m0 + h * 128 * PAIR, y, bar);
                  tma_2d<PAIR>(sa + h * kTileBytesA + 8192 + r * 128, &row_a, m0 + h * 128 * PAIR + 64, y, bar);
                }
                for (int g = 0; g < pieces; ++g) tma_2d<PAIR>(sb + g * 8192 + r * 128, &row_b, n0 + g * 64, y, bar);
              }
            }
          } else {
            if (rank == 0) mbar_expect_tx(&bars.full[stage], PAIR * (halves * kTileBytesA + pieces * 4096));
            for (int h = t.half; h < t.halves_end; ++h) {
              unsigned char* const half_a = sa + h * kTileBytesA;
              const int row = m0 + h * 128 * PAIR;
              if (MODE == kGroupedForward) {
                tma_3d<PAIR>(half_a, &map_a, s * 64, row, t.e, bar);
              } else {
                tma_3d<PAIR>(half_a, &map_a, row, s * 64, t.e, bar);
                tma_3d<PAIR>(half_a + 8192, &map_a, row + 64, s * 64, t.e, bar);
              }
            }
            for (int g = 0; g < pieces; ++g) tma_2d<PAIR>(sb + g * 4096, &map_b, s * 64, t.from + rank * half + g * 32, bar);
          }
          ++issued;
          if (++stage == Cfg::kStages) { stage = 0; phase ^= 1; }
        }
      }
      if (*abort && rank == 0) {           // copies in flight land before the CTA leaves
        for (int i = 0; i < Cfg::kStages && i < issued; ++i) {
          if (stage == 0) { stage = Cfg::kStages; phase ^= 1; }
          --stage;
          mbar_wait_bounded(&bars.full[stage], phase, kWaitLimitNs);
        }
      }
    }
    __syncwarp();
  } else if (warp == kMathWarp) {
    if (rank == 0 && elect_one()) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0, phases = 0;         // phases: HALVES = 2, a bit for each accumulator
      const auto copied = [&](int stage, uint32_t phase) {
        if (!wait(&bars.full[stage], phase)) return false;
        if (GATHER) {
          if (!wait(&bars.gathered[stage], phase)) return false;
          fence_proxy_async_smem();        // here, where nothing is under way, for the threads that copied
        }
        tmem_fence_after();
        return true;
      };
      GroupedTile t;
      for (int u = 0; !*abort && tile_of(u, t); ++u) {
        const int steps = steps_of(t), from = step_from(steps), to = step_to(steps);
        if (from == to || nothing_of(t)) continue;
        const uint32_t instr = umma_instr(std::is_same<T, __nv_bfloat16>::value, kA_mn, kB_mn, 128 * PAIR, t.cols);
        // step s of the tile: half h of its rows, from a stage into accumulator `acc`
        const auto multiply = [&](int s, int stage, int h, int acc, bool begins) {
          const uint32_t sa = smem_u32(base + stage * Cfg::kStageBytes) + h * kTileBytesA, sb = smem_u32(base + stage * Cfg::kStageBytes) + Cfg::kBytesA;
          const uint64_t da = kA_mn ? umma_desc(sa, 8192, 1024) : umma_desc(sa, 16, 1024);
          const uint64_t db = kB_mn ? umma_desc(sb, 8192, 1024) : umma_desc(sb, 16, 1024);
          const int inner = MODE == kGroupedDw && t.count - s * 64 < 64 ? (t.count - s * 64 + 15) / 16 : 4;
          for (int x = 0; x < inner; ++x)  // the descriptors' addresses are in 16 bytes
            umma<PAIR>(tmem + acc * NT, da + x * (kA_mn ? 128 : 2), db + x * (kB_mn ? 128 : 2), instr, !begins || x > 0);
        };
        if constexpr (HALVES == 2) {
          // Both accumulators belong to the tile, one to each half.  The first half of its first steps goes ahead while the last tile's second half
          // is still being stored; their stages are free once the second half has followed.
          const int h = t.half, lead = to - from < Cfg::kStages ? to - from : Cfg::kStages;
          const bool both = t.halves_end - h == 2;
          if (!wait(&bars.acc_empty[h], (phases >> h & 1) ^ 1)) break;
          tmem_fence_after();
          int ahead = stage;
          uint32_t ahead_phase = phase;
          bool good = true;
          for (int s = from; s < from + lead && good; ++s) {
            good = copied(ahead, ahead_phase);
            if (good) multiply(s, ahead, h, h, s == from);
            if (++ahead == Cfg::kStages) { ahead = 0; ahead_phase ^= 1; }
          }
          if (!good) break;
          if (both) {
            if (!wait(&bars.acc_empty[1], (phases >> 1) ^ 1)) break;
            tmem_fence_after();
          }
          for (int s = from; s < to; ++s) {
            if (s >= from + lead) {
              if (!copied(stage, phase)) break;
              multiply(s, stage, h, h, false);
            }
            if (s + 1 == to) umma_commit<PAIR>(&bars.acc_full[h]);
            if (both) multiply(s, stage, 1, 1, s == from);
            umma_commit<PAIR>(&bars.empty[stage]);
            if (++stage == Cfg::kStages) { stage = 0; phase ^= 1; }
          }
          if (both) umma_commit<PAIR>(&bars.acc_full[1]);
          phases ^= both ? 3u : 1u << h;
          continue;
        }
        for (int s = from; s < to; ++s) {
          const bool begins = s == from || (PARTS && (s - from) % kPartSteps == 0);
          const bool ends = s + 1 == to || (PARTS && (s + 1 - from) % kPartSteps == 0);
          if (begins) {
            if (!wait(&bars.acc_empty[acc], acc_phase ^ 1)) break;
            tmem_fence_after();
          }
          if (!copied(stage, phase)) break;
          multiply(s, stage, 0, acc, begins);
          umma_commit<PAIR>(&bars.empty[stage]);
          if (ends) {
            umma_commit<PAIR>(&bars.acc_full[acc]);
            if (++acc == 2) { acc = 0; acc_phase ^= 1; }
          }
          if (++stage == Cfg::kStages) { stage = 0; phase ^= 1; }
        }
      }
    }
    if (GATHER && rank == 1 && elect_one()) {
      // Tells the first CTA of rows that are gathered here.  Not the gathering warps themselves: a fence, and an arrival at the cluster's scope,
      // wait for all that their thread has under way (1.0 to 1.8 us a step).
      int stage = 0;
      uint32_t phase = 0;
      GroupedTile t;
      for (int u = 0; !*abort && tile_of(u, t); ++u) {
        if (nothing_of(t)) continue;
        const int steps = steps_of(t);
        for (int s = step_from(steps); s < step_to(steps); ++s) {
          if (!wait(&bars.gathered[stage], phase)) break;
          fence_proxy_async_smem();
          mbar_arrive_cluster_shared(cluster_smem(&bars.full[stage], 0));
          if (++stage == Cfg::kStages) { stage = 0; phase ^= 1; }
        }
      }
    }
    __syncwarp();
  } else if (GATHER && warp > kMathWarp) {
    // 8 pieces of 16 bytes a row, 16 rows a pass
    constexpr int kPasses = NT / PAIR / 16;
    const int l = tid - kGroupedThreads, piece = l & 7, row0 = l >> 3;
    const char* const x = static_cast<const char*>(a.a);
    const long long row_bytes = a.a_stride * 2;
    const int x_rows = (int)a.tokens, x_columns = a.k;
    int stage = 0;
    uint32_t phase = 0;
    GroupedTile t;
    for (int u = 0; !stopped() && tile_of(u, t); ++u) {
      if (nothing_of(t)) continue;
      const int steps = steps_of(t), from = step_from(steps), to = step_to(steps), half = t.cols / PAIR;
      int row[kPasses];                    // of x; -1: beyond the group, or not a row of x: zeros
#pragma unroll
      for (int j = 0; j < kPasses; ++j) {
        const int r = row0 + j * 16, p = rank * half + r;
        row[j] = r < half && p < t.count ? a.rows[t.from + p] : -1;
      }
#pragma unroll
      for (int j = 0; j < kPasses; ++j) {
        const int r = row0 + j * 16, p = rank * half + r;
        if ((unsigned)row[j] >= (unsigned)x_rows) {
          if (r < half && p < t.count) raise(a.status, FLEXSPMV_ERR_BAD_CSR);
          row[j] = -1;
        }
      }
      for (int s = from; s < to; ++s) {
        if (!wait_warp(&bars.empty[stage], phase ^ 1)) break;
        const uint32_t sb = smem_u32(base + stage * Cfg::kStageBytes + Cfg::kBytesA);
        const int c = s * 64 + piece * 8;
        const bool inside = c < x_columns;
        const char* const x_piece = x + c * 2;
#pragma unroll
        for (int j = 0; j < kPasses; ++j) {
          const int r = row0 + j * 16;
          if (r >= half) continue;
          const bool copied = inside && row[j] >= 0;
          copy16(sb + r * 128 + ((piece ^ (r & 7)) << 4), copied ? x_piece + row[j] * row_bytes : x, copied ? 16 : 0);
        }
        copy16_arrive(&bars.gathered[stage]);
        if (++stage == Cfg::kStages) { stage = 0; phase ^= 1; }
      }
    }
    copy16_wait_all();
  } else {
    int acc = 0;
    uint32_t acc_phase = 0, second_phase = 0;
    TO* const out = static_cast<TO*>(a.out);
    unsigned char* const mine = store + warp * (Cfg::kStoreBytes / kStoreWarps);
    const int quarter = warp & 3, part = warp >> 2;     // of the accumulator's rows, of its columns
    GroupedTile t;
    for (int u = 0; !stopped() && tile_of(u / HALVES, t); ++u) {           // tiles, or their halves
      const int half = u % HALVES;
      if (nothing_of(t) || half < t.half || half >= t.halves_end) continue;
      if (HALVES == 2) acc = half;
      const uint32_t full_phase = half ? second_phase : acc_phase;
      const int m = t.m0 + half * 128 * PAIR + rank * 128 + quarter * 32;          // this warp's first row of the accumulator
      const int steps = steps_of(t), from = step_from(steps), to = step_to(steps);
      const auto free_accumulator = [&] {  // once this warp's last of it is in registers
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (PAIR == 2) mbar_arrive_cluster_relaxed(cluster_smem(&bars.acc_empty[acc], 0));
          else mbar_arrive(&bars.acc_empty[acc]);
        }
      };
      // this warp's four times 32 columns, added up from the parts
      float sum[PARTS ? NT / 64 : 1][32];
      if (PARTS) {
#pragma unroll
        for (int g = 0; g < NT / 64; ++g)
#pragma unroll
          for (int x = 0; x < 32; ++x) sum[PARTS ? g : 0][x] = 0.f;
        bool there = true;
        for (int s = from; s < to && there; s += kPartSteps) {
          there = wait_warp(&bars.acc_full[acc], acc_phase);
          if (!there) break;
          tmem_fence_after();
          const uint32_t d = tmem + acc * NT + ((uint32_t)(quarter * 32) << 16) + part * 32;
#pragma unroll
          for (int g = 0; g < NT / 64; ++g)
            if (part * 32 + g * 64 < t.cols) {
              uint32_t v[32];
              tmem_load32(d + g * 64, v);
#pragma unroll
              for (int x = 0; x < 32; ++x) sum[PARTS ? g : 0][x] += __uint_as_float(v[x]);
            }
          free_accumulator();
          if (++acc == 2) { acc = 0; acc_phase ^= 1; }
        }
        if (!there) break;
      }
      if (SPLIT && PARTS) {
        float* const sums = reinterpret_cast<float*>(base);
#pragma unroll
        for (int g = 0; g < NT / 64; ++g)
          if (part * 32 + g * 64 < t.cols)
#pragma unroll
            for (int x = 0; x < 32; ++x) sums[(part * 32 + g * 64 + x) * 128 + quarter * 32 + lane] = sum[PARTS ? g : 0][x];
        break;
      }
      if (SPLIT) {
        // this CTA's part of the sum, 128 rows a column, over the stages: all that was copied there has been used
        float* const sums = reinterpret_cast<float*>(base);
        const bool any = from < to;
        if (any && !wait_warp(&bars.acc_full[0], 0)) break;
        tmem_fence_after();
        for (int c0 = part * 32; c0 < t.cols; c0 += 64) {
          uint32_t v[32];
          if (any) tmem_load32(tmem + ((uint32_t)(quarter * 32) << 16) + c0, v);
#pragma unroll
          for (int x = 0; x < 32; ++x) sums[(c0 + x) * 128 + quarter * 32 + lane] = any ? __uint_as_float(v[x]) : 0.f;
        }
        break;
      }
      if (MODE == kGroupedDw && t.count == 0) {
        constexpr int kW = 16 / (int)sizeof(TO);
        const int pieces = t.cols / kW;
        for (int x = part * 32 + lane; x < 32 * pieces; x += 64) {
          const int r = m + x / pieces, c = t.n0 + x % pieces * kW;
          if (r < a.n && c < a.k) *reinterpret_cast<uint4*>(out + ((size_t)t.e * a.n + r) * a.k + c) = make_uint4(0, 0, 0, 0);
        }
        continue;
      }
      // dw: 32 columns from c0 on, of row m + lane, to shared memory and from there as a tile, which leaves out what the matrix does not have
      const auto store_rows = [&](int c0, const auto& value) {
        constexpr int kW = 16 / (int)sizeof(TO), kPieces = 32 / kW;         // values of a 16-byte piece, pieces of a row
        if (lane == 0) tma_stores_read();
        __syncwarp();
#pragma unroll
        for (int p = 0; p < kPieces; ++p) {
          Pack<TO, kW> q;
#pragma unroll
          for (int x = 0; x < kW; ++x) q.set(x, value(p * kW + x));
          reinterpret_cast<uint4*>(mine)[lane * kPieces + (p ^ (kPieces == 8 ? lane & 7 : (lane >> 1) & 3))] = q.raw[0];          // the map's swizzle
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && m < a.n && t.n0 + c0 < a.k) tma_store_3d(&map_out, mine, t.n0 + c0, m, t.e);
      };
      if constexpr (PARTS) {
#pragma unroll
        for (int g = 0; g < NT / 64; ++g)
          if (part * 32 + g * 64 < t.cols) store_rows(part * 32 + g * 64, [&](int x) { return sum[g][x]; });
        continue;
      }
      if (!wait_warp(&bars.acc_full[acc], full_phase)) break;
      tmem_fence_after();
      const uint32_t d = tmem + acc * NT + ((uint32_t)(quarter * 32) << 16);
      for (int c0 = part * 32;; c0 += 64) {
        uint32_t v[32], low[16], high[16];
        const bool there = c0 < t.cols, last = c0 + 64 >= t.cols;
        if (there) {
          if (MODE == kGroupedDw) {
            tmem_load32(d + c0, v);
          } else {
            tmem_load_blocks(d + c0, low);
            tmem_load_blocks(d + (16u << 16) + c0, high);
            tmem_wait_loads();
          }
        }
        if (last) free_accumulator();
        if (!there) break;
        if (MODE == kGroupedDw) {
          store_rows(c0, [&](int x) { return __uint_as_float(v[x]); });
        } else {
          // blocks of 8 features by 8 places, turned on their way into rows of 32 features a place (16-byte pieces, exchanged so that neither
          // way meets in a bank)
          if constexpr (sizeof(TO) == 2) {
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              const auto pair = [&](const uint32_t (&w)[16], int i) {
                return two_of<TO>(__uint_as_float(w[b * 4 + i]), __uint_as_float(w[b * 4 + i + 1]));
              };
              const int p = b * 8 + (lane & 7);
              store_blocks_turned(mine + p * 64 + (((lane >> 3) ^ (p >> 1)) & 3) * 16, pair(low, 0), pair(low, 2), pair(high, 0), pair(high, 2));
            }
          }
          __syncwarp();
          const int width = MODE == kGroupedDx ? a.k : a.n;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int p = x * 8 + (lane >> 2), c = m + (lane & 3) * 8;
            if (c0 + p < t.count && c < width)
              *reinterpret_cast<uint4*>(out + (size_t)(t.from + c0 + p) * width + c) = reinterpret_cast<const uint4*>(mine)[p * 4 + (((lane & 3) ^ (p >> 1)) & 3)];
          }
          __syncwarp();
        }
        if (last) break;
      }
      if (HALVES == 2) {
        if (half) second_phase ^= 1;
        else acc_phase ^= 1;
      } else if (++acc == 2) {
        acc = 0;
        acc_phase ^= 1;
      }
    }
    if (MODE == kGroupedDw && lane == 0) tma_stores_done();
    if (MODE != kGroupedDw) {     // places of no expert: before the first group and after the last
      const int width = (MODE == kGroupedDx ? a.k : a.n) / 8;
      const long long head = table[0].from, tail = table[a.experts - 1].from + table[a.experts - 1].count, none = head + a.slots - tail;
      for (long long x = blockIdx.x; x < none; x += gridDim.x) {
        uint4* const row = reinterpret_cast<uint4*>(out + (size_t)(x < head ? x : tail + x - head) * width * 8);
        for (int c = tid; c < width; c += kStoreWarps * 32) row[c] = make_uint4(0, 0, 0, 0);
      }
    }
  }
  if (SPLIT) {
    // every CTA stores some of the tile's columns, eight neighbouring rows (dw: columns) at a time
    cluster_sync();
    if (first < tiles && !*abort) {
      const GroupedTile t = tile_at<MODE, NT, PAIR, HALVES>(a, table, first);
      const int eights = (t.cols + 7) / 8, c_from = eights * share / split * 8, c_to = eights * (share + 1) / split * 8;
      const uint32_t sums = smem_u32(base);
      TO* const out = static_cast<TO*>(a.out);
      constexpr bool kDw = MODE == kGroupedDw;
      const int items = (c_to - c_from) * 16;            // of eight values
      for (int i = tid; i < items; i += kThreads) {
        // forward, dx: 16 items a column; dw: 128 items for eight columns
        const int c = kDw ? c_from + i / 128 * 8 : c_from + i / 16, r = kDw ? i % 128 : i % 16 * 8;
        float sum[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) sum[x] = 0.f;
        for (int p = 0; p < split; ++p) {
          const uint32_t from = cluster_address(sums, p) + (uint32_t)(c * 128 + r) * 4;
          float v[8];
          if (kDw) {
#pragma unroll
            for (int x = 0; x < 8; ++x) v[x] = cluster_load(from + x * 512);
          } else {
            cluster_load4(from, v);
            cluster_load4(from + 16, v + 4);
          }
#pragma unroll
          for (int x = 0; x < 8; ++x) sum[x] += v[x];
        }
        Pack<TO, 8> q;
#pragma unroll
        for (int x = 0; x < 8; ++x) q.set(x, sum[x]);
        if (kDw) {
          if (t.m0 + r < a.n && t.n0 + c < a.k) q.store(out + ((size_t)t.e * a.n + t.m0 + r) * a.k + t.n0 + c);
        } else {
          const int width = MODE == kGroupedDx ? a.k : a.n;
          if (c < t.count && t.m0 + r < width) q.store(out + (size_t)(t.from + c) * width + t.m0 + r);
        }
      }
    }
  }
  tmem_fence_before();
  __syncthreads();
  if (PAIR == 2 || SPLIT) cluster_sync();  // no CTA leaves while another one's instructions may reach its memory
  tmem_fence_after();
  if (warp == kMathWarp) tmem_free<PAIR, Cfg::kTmemCols>(tmem);
}

// How many clusters of `ctas` of this kernel a device holds at once; what the runtime says is kept for a kernel, a device and a size.
template <auto KERNEL, int THREADS>
static int clusters_at_once(int ctas, int smem) {
  static std::atomic<int> known[64][4];
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 0;
  std::atomic<int>& slot = known[device][ctas >= 8 ? 3 : ctas >= 4 ? 2 : ctas >= 2 ? 1 : 0];
  int n = slot.load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ctas; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, KERNEL, &cfg) != cudaSuccess || n < 0) { cudaGetLastError(); n = 0; }
    slot.store(n + 1, std::memory_order_relaxed);
    return n;
  }
  return n - 1;
}

template <int MODE, int NT, int PAIR, int HALVES, int OUT_BYTES>
static int grouped_smem(int experts) {
  using Cfg = GroupedCfg<MODE, NT, PAIR, HALVES, OUT_BYTES>;
  return 1024 + Cfg::kStages * Cfg::kStageBytes + Cfg::kStoreBytes + (int)sizeof(GroupedBars) + (experts + 1) * (int)sizeof(GroupedTable);
}

// `split`: CTAs that share a tile, `grid` of them altogether; 1: whole tiles.
template <class T, class TO, int MODE, int NT, int PAIR, int HALVES, bool SPLIT, bool GATHER, bool PARTS>
static int grouped_launch_as(const GroupedArgs& a, int grid, int split, cudaStream_t st) {
  constexpr CUtensorMapDataType kIn = std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap ma, mb, row_a, row_b, out;
  if (MODE == kGroupedDw) {
    const uint64_t rows = a.slots ? a.slots : 1;
    const uint64_t da[3] = {(uint64_t)a.n, 64, rows}, sa[2] = {(uint64_t)a.a_stride, (uint64_t)a.a_stride};
    const uint64_t db[3] = {(uint64_t)a.k, 64, rows}, sb[2] = {(uint64_t)a.b_stride, (uint64_t)a.b_stride};
    const uint64_t ra[2] = {(uint64_t)a.n, rows}, rb[2] = {(uint64_t)a.k, rows};
    const uint32_t box[3] = {64, 64, 1}, one[2] = {64, 1};
    const void *pa = a.slots ? a.a : a.out, *pb = a.slots ? a.b : a.out;          // without rows nothing is copied
    if (int e = make_map(&ma, pa, kIn, 3, da, sa, box)) return e;
    if (int e = make_map(&row_a, pa, kIn, 2, ra, sa, one)) return e;
    if (int e = make_map(&mb, pb, kIn, 3, db, sb, box)) return e;
    if (int e = make_map(&row_b, pb, kIn, 2, rb, sb, one)) return e;
    const uint64_t dims[3] = {(uint64_t)a.k, (uint64_t)a.n, (uint64_t)a.experts}, strides[2] = {(uint64_t)a.k, (uint64_t)a.k * a.n};
    const uint32_t block[3] = {32, 32, 1};
    constexpr bool kWide = sizeof(TO) == 4;
    if (int e = make_map(&out, a.out, kWide ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : kIn, 3, dims, strides, block,
                         kWide ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B))
      return e;
  } else {
    const uint64_t dw[3] = {(uint64_t)a.k, (uint64_t)a.n, (uint64_t)a.experts}, sw[2] = {(uint64_t)a.k, (uint64_t)a.k * a.n};
    const uint32_t wide[3] = {64, 128, 1}, high[3] = {64, 64, 1};
    if (int e = make_map(&ma, a.b, kIn, 3, dw, sw, MODE == kGroupedForward ? wide : high)) return e;
    const uint64_t dx[2] = {(uint64_t)(MODE == kGroupedForward ? a.k : a.n), (uint64_t)a.slots}, sx[1] = {(uint64_t)a.a_stride};
    const uint32_t box[2] = {64, 32};
    mb = ma;
    if (!GATHER)
      if (int e = make_map(&mb, a.a, kIn, 2, dx, sx, box)) return e;
    row_a = out = ma;
    row_b = mb;
  }
  const int smem = grouped_smem<MODE, NT, PAIR, HALVES, (int)sizeof(TO)>(a.experts);
  constexpr auto kernel = grouped_kernel<T, TO, MODE, NT, PAIR, HALVES, SPLIT, GATHER, PARTS>;
  if (int e = allow_smem<kernel>(smem)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid); cfg.blockDim = dim3((unsigned)grouped_threads(GATHER)); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = PAIR * split; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, kernel, ma, mb, row_a, row_b, out, a);
}

template <class T, class TO, int MODE, int NT, int PAIR, bool GATHER, bool PARTS = false>
static int grouped_tiles(const GroupedArgs& a, cudaStream_t st) {
  const int sms = device_sm_count();
  // tiles of 128 rows, no more than these whatever the groups are
  const long long m_tiles = ((MODE == kGroupedDx ? a.k : a.n) + 127) / 128;
  const long long most = m_tiles * (MODE == kGroupedDw ? (long long)a.experts * ((a.k + NT - 1) / NT)
                                                                : (a.slots < a.experts ? a.slots : a.experts) + a.slots / NT);
  const long long steps = (MODE == kGroupedForward ? a.k : MODE == kGroupedDx ? a.n : a.slots / a.experts) / 64;
  // What dividing saves is most of a tile's steps, 0.3 us each (a narrow tile's 0.13); what it costs is the parts' meeting, about 5 us (1.5).
  // us, whole / divided: 8 rows, one expert of 2048 x 4096 17.4 / 9.4; dw of 8192 rows, 1024 x 1024 43.8 / 22; but 4096 rows, two experts of
  // 512 x 512 (8 steps) 9.8 / 12.6.
  constexpr auto divided = grouped_kernel<T, TO, MODE, NT, 1, 1, true, GATHER, PARTS>;
  const int smem = grouped_smem<MODE, NT, 1, 1, (int)sizeof(TO)>(a.experts);
  for (int split = 8; split > 1; split /= 2) {
    if (most * split > sms || steps - steps / split < (NT > 64 ? 20 : 12)) continue;
    if (int e = allow_smem<divided>(smem)) return e;
    if (most <= clusters_at_once<divided, grouped_threads(GATHER)>(split, smem)) return grouped_launch_as<T, TO, MODE, NT, 1, 1, true, GATHER, PARTS>(a, (int)most * split, split, st);
  }
  // Tiles of both accumulators (HALVES = 2): a quarter less between L2 and the SMs for a tile's step, a stage less under way, and the end of a tile's
  // sum that only half of it is behind.  It pays where the sums are long and the tiles go round the pairs, most with gathered rows, which are gathered
  // half as often.  us, one / both: 32 768 rows, 32 experts of 4096 x 2048, with a list 437 / 419, without 411 / 413, dw 418 / 410, dx 411 / 419;
  // 10 599 rows, 8 experts of 1488 x 2792 87.6 / 75.7; 8192 x 8192 x 8192 737 / 688; but 8192 rows of 328 85 / 89, 4102 rows of 2048 28 / 30.
  if constexpr (NT > 64 && !PARTS && MODE != kGroupedDx) {
    const long long columns = MODE == kGroupedDw ? (long long)a.experts * ((a.k + NT - 1) / NT) : a.slots / NT + a.experts / 2;          // of tiles, about
    const int long_sum = MODE == kGroupedDw ? 16 : GATHER ? 32 : 40, half_rounds = MODE == kGroupedDw ? 20 : 3;
    if (steps >= long_sum && columns * ((a.n + 511) / 512) * 2 >= half_rounds * (sms / 2))
      return grouped_launch_as<T, TO, MODE, NT, 2, 2, false, GATHER, false>(a, sms / 2 * 2, 1, st);
  }
  return grouped_launch_as<T, TO, MODE, NT, PAIR, 1, false, GATHER, PARTS>(a, sms / PAIR * PAIR, 1, st);
}

template <class T, class TO, int MODE, bool GATHER>
static int grouped_launch(const GroupedArgs& a, cudaStream_t st) {
  if constexpr (MODE == kGroupedDw) {
    // us, whole / in parts: 200 000 rows of 2048 x 2048 in float16 1160 / 1195, 600 000 of 512 x 512 512 / 540, 102 400 in 32 such groups 591 / 597
    if constexpr (sizeof(TO) == 2)
      if (a.slots <= kWholeRows<T>) return grouped_tiles<T, TO, MODE, 256, 2, GATHER, false>(a, st);
    return grouped_tiles<T, TO, MODE, 256, 2, GATHER, true>(a, st);
  } else {
    // Tiles of 64 places and single CTAs for up to 32 places an expert on average: more of the weights on their way at once.  us, 64 / 256 places:
    // 16 an expert, 64 experts of 1408 x 2048 59.8 / 66.8; 32 experts of 2048 x 2048, 32 an expert 47.0 / 49.7, 48 51.0 / 50.5, 128 72.1 / 54.9.
    // And where as narrow tiles all of them run at once: a part of the sum is a quarter as much to add up, a gathered step a quarter of the rows.
    // us, narrow / wide: 753 rows, 4 experts of 104 x 1512 8.9 / 15.1; 256 rows of 2048 x 2048 10.5 / 14.3, of a list 11.0 / 16.0; 512 rows of 1024 x 1024
    // 7.3 / 8.1; but 100 rows of 4096 x 4096 13.0 / 12.3.
    const long long narrow = ((MODE == kGroupedDx ? a.k : a.n) + 127) / 128 * ((a.slots < a.experts ? a.slots : a.experts) + a.slots / 64);
    if (a.slots <= 32ll * a.experts || narrow <= device_sm_count()) return grouped_tiles<T, TO, MODE, 64, 1, GATHER>(a, st);
    return grouped_tiles<T, TO, MODE, 256, 2, GATHER>(a, st);
  }
}

static int check_grouped(const flexspmv_expert_desc* d, int which) {
  if (!d || d->tokens < 0 || d->slots < 0 || d->experts < 1 || d->n < 1 || d->k < 1) return FLEXSPMV_ERR_BAD_ARG;
  if (d->type != FLEXSPMV_TYPE_BF16 && d->type != FLEXSPMV_TYPE_F16) return FLEXSPMV_ERR_BAD_ARG;
  if (which == kGroupedDw && d->out_type != FLEXSPMV_TYPE_F32 && d->out_type != d->type) return FLEXSPMV_ERR_BAD_ARG;
  if (d->in_stride < (which == kGroupedForward ? d->k : d->n) || (which == kGroupedDw && d->in2_stride < d->k)) return FLEXSPMV_ERR_BAD_ARG;
  if (d->experts > FLEXSPMV_MAX_EXPERTS || d->slots > 0x7fffffffLL || d->tokens > 0x7fffffffLL) return FLEXSPMV_ERR_TOO_LARGE;
  // places and tiles are counted in 32 bits
  const double sides = (d->n / 128 + 1.0) * (d->k / 128 + 1.0);
  if (d->slots > 0x7fff0000LL || sides * (d->slots / 32 + 2.0 * d->experts) > 2e9) return FLEXSPMV_ERR_TOO_LARGE;
  if (d->n % 8 || d->k % 8 || d->in_stride % 8 || (which == kGroupedDw && d->in2_stride % 8)) return FLEXSPMV_ERR_ALIGN;
  return 0;
}

static bool grouped_apart(const flexspmv_expert_desc* d, int mode, const void* const* in, const int* rows, void* out, void* ws) {
  const bool dw = mode == kGroupedDw, forward = mode == kGroupedForward;
  const long long matrices = (long long)d->experts * d->n * d->k, x_rows = rows ? d->tokens : d->slots;
  const Region results[2] = {{out, dw ? matrices * type_bytes(d->out_type) : 2 * d->slots * (forward ? d->n : d->k)}, {ws, 2 * d->slots * d->k}};
  Region inputs[4] = {rows_at(in[0], forward ? x_rows : d->slots, forward ? d->k : d->n, d->in_stride, d->type), {in[1], 2 * matrices},
                      {in[2], 4ll * d->experts + 4}, {rows, 4 * d->slots}};
  if (dw) inputs[1] = rows_at(in[1], x_rows, d->k, d->in2_stride, d->type);
  return apart(results, inputs);
}

// in: forward x, weight, offsets, rows; dx dy, weight, offsets; dw dy, x, offsets, rows
template <int MODE>
static int grouped_call(const flexspmv_expert_desc* d, const void* const* in, void* const* out, void* ws, size_t ws_bytes, int32_t* status, void* stream) {
  if (int e = check_grouped(d, MODE)) return e;
  constexpr bool kDw = MODE == kGroupedDw, kDx = MODE == kGroupedDx;
  if (!in || !out) return FLEXSPMV_ERR_BAD_ARG;
  if (d->slots == 0 && !kDw) return 0;
  const int* const rows = kDx ? nullptr : static_cast<const int*>(in[3]);
  if (!in[2] || !out[0]) return FLEXSPMV_ERR_BAD_ARG;
  if (d->slots && (!in[0] || !in[1] || (!kDx && d->tokens < (rows ? 1 : d->slots)))) return FLEXSPMV_ERR_BAD_ARG;
  if (!aligned16(in[0]) || !aligned16(in[1]) || !aligned16(out[0]) || !aligned_to(4, in[2], rows, status)) return FLEXSPMV_ERR_ALIGN;
  GroupedArgs a = {in[0], in[1], static_cast<const int*>(in[2]), rows, out[0], d->tokens, d->slots, d->in_stride, d->in2_stride, d->experts,
                   d->n, d->k, status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool copied = kDw && rows && d->slots;
  if (copied) {
    if (!ws || ws_bytes < (size_t)d->slots * d->k * 2) return FLEXSPMV_ERR_WORKSPACE;
    if (!aligned16(ws)) return FLEXSPMV_ERR_ALIGN;
  }
  if (!grouped_apart(d, MODE, in, rows, out[0], copied ? ws : nullptr)) return FLEXSPMV_ERR_BAD_ARG;
  if (copied) {
    const int pieces = d->k / 8;
    const long long ctas = ((long long)d->slots * pieces + 1023) / 1024, most = device_sm_count() * 8ll;
    if (int e = launch_pdl(take_rows_kernel, (unsigned)(ctas < most ? ctas : most), 256, 0, st, static_cast<const uint4*>(in[1]), rows, a.offsets,
                           static_cast<uint4*>(ws), (long long)d->tokens, (long long)d->slots, (long long)d->in2_stride / 8, d->experts, pieces, status))
      return e;
    a.b = ws;
    a.b_stride = d->k;
  }
  const auto go = [&](auto zero) {
    using T = decltype(zero);
    if constexpr (kDw) {
      return d->out_type == FLEXSPMV_TYPE_F32 ? grouped_launch<T, float, MODE, false>(a, st) : grouped_launch<T, T, MODE, false>(a, st);
    } else if constexpr (kDx) {
      return grouped_launch<T, T, MODE, false>(a, st);
    } else {
      return rows ? grouped_launch<T, T, MODE, true>(a, st) : grouped_launch<T, T, MODE, false>(a, st);
    }
  };
  return d->type == FLEXSPMV_TYPE_BF16 ? go(__nv_bfloat16()) : go(__half());
}

}  // namespace flex

extern "C" {

int flexspmv_grouped_matmul(const flexspmv_expert_desc* d, const void* const* in, void* const* out, int32_t* status, void* stream) {
  return flex::grouped_call<flex::kGroupedForward>(d, in, out, nullptr, 0, status, stream);
}
int flexspmv_grouped_matmul_dx(const flexspmv_expert_desc* d, const void* const* in, void* const* out, int32_t* status, void* stream) {
  return flex::grouped_call<flex::kGroupedDx>(d, in, out, nullptr, 0, status, stream);
}
int flexspmv_grouped_matmul_dw_bytes(const flexspmv_expert_desc* d, size_t* bytes) {
  if (!bytes) return FLEXSPMV_ERR_BAD_ARG;
  if (int e = flex::check_grouped(d, flex::kGroupedDw)) return e;
  *bytes = (size_t)d->slots * d->k * 2;
  return 0;
}
int flexspmv_grouped_matmul_dw(const flexspmv_expert_desc* d, const void* const* in, void* const* out, void* ws, size_t ws_bytes, int32_t* status,
                               void* stream) {
  return flex::grouped_call<flex::kGroupedDw>(d, in, out, ws, ws_bytes, status, stream);
}

}  // extern "C"
