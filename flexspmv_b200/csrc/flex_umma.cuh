// Tensor-memory-accelerator copies of tiles and the tcgen05 matrix instructions: what the grouped products are built from.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "flex_common.cuh"

namespace flex {

// ---- pairs of CTAs -----------------------------------------------------------------------------------------------
// With PAIR = 2 two CTAs of a cluster work on one tile: each copies its half of both operands, the first of them issues the matrix
// instructions for both, and the barriers that it waits on are its own.  No copy is multicast.
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address, for the whole cluster, of CTA `rank`'s copy of a shared variable.
__device__ __forceinline__ uint32_t cluster_address(uint32_t own, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(own), "r"(rank));
  return r;
}
__device__ __forceinline__ uint32_t cluster_smem(const void* p, uint32_t rank) { return cluster_address(smem_u32(p), rank); }
__device__ __forceinline__ float cluster_load(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_load4(uint32_t addr, float* v) {
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(addr) : "memory");
}
// Orders what this thread knows of its CTA's shared memory before the arrival, and nothing else (an arrival that releases at the cluster's scope
// waits for all memory accesses).
__device__ __forceinline__ void mbar_arrive_cluster_shared(uint32_t bar) {
  asm volatile("fence.release.sync_restrict::shared::cta.cluster;\n\tmbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Without ordering of this thread's memory accesses: a release at the cluster's scope waits for all of a warp's stores to global memory (it took
// half of the time of a launch that stores much).  For a barrier that frees tensor memory whose loads are complete.
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// ---- copies of 16 bytes -----------------------------------------------------------------------------------------
// `bytes`: 16, or 0 for zeros (the source is not read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(__cvta_generic_to_global(src)), "r"(bytes));
}
// The barrier (which counts threads) is arrived on when this thread's copies so far have landed; the thread does not wait.
__device__ __forceinline__ void copy16_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void copy16_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// ---- tile copies -----------------------------------------------------------------------------------------------
// `bar`: a cluster address; PAIR = 2: of either CTA of the pair.
template <int PAIR>
__device__ __forceinline__ void tma_2d(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if constexpr (PAIR == 2)
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(
                     smem_u32(dst)),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
                 : "memory");
}
template <int PAIR>
__device__ __forceinline__ void tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  if constexpr (PAIR == 2)
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                     smem_u32(dst)),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                     smem_u32(dst)),
                 "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}
// From shared memory; what lies beyond the tensor is left out.  The source may be written again after tma_stores_read, and is needed till then.
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x),
               "r"(y), "r"(z), "r"(smem_u32(src))
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void tma_stores_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void tma_stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void tma_prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// ---- tensor memory ---------------------------------------------------------------------------------------------
// One warp of the CTA; PAIR = 2: of each of the two.
template <int PAIR, int COLS>
__device__ __forceinline__ void tmem_alloc(uint32_t* slot) {
  if constexpr (PAIR == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "n"(COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "n"(COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
}
template <int PAIR, int COLS>
__device__ __forceinline__ void tmem_free(uint32_t base) {
  if constexpr (PAIR == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "n"(COLS));
  else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "n"(COLS));
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 32 columns of this warp's 32 lanes: lane l gets its row's 32 values.
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
      "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
        "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]),
        "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]),
        "=r"(v[31])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// 32 columns of 16 lanes from `addr` on: for each 8 columns, lane l gets of row l / 4 the columns 2 (l % 4) and the next one, then the same of
// row l / 4 + 8.
__device__ __forceinline__ void tmem_load_blocks(uint32_t addr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
        "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Four 8 x 8 blocks of 16-bit values, two of a row in each lane's register (rows l / 4, columns 2 (l % 4) and the next), stored turned:
// lane 8 i + j has the address of column j of block i.
__device__ __forceinline__ void store_blocks_turned(void* row, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(smem_u32(row)), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// ---- matrix instructions ---------------------------------------------------------------------------------------
// Shared-memory descriptors of operands in rows of 128 bytes with the 128-byte swizzle that the tile copies write.
//   along the sum (K-major): rows are the tile's rows, 64 values of the inner length each; groups of 8 rows are 1024 bytes apart.
//   across it (MN-major): rows are the inner length, 64 of the tile's rows (or columns) each; `group` bytes to the next 64 of them.
__device__ __forceinline__ uint64_t umma_desc(uint32_t addr, uint32_t lead_bytes, uint32_t stride_bytes) {
  return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)((lead_bytes >> 4) & 0x3fffu) << 16) | ((uint64_t)((stride_bytes >> 4) & 0x3fffu) << 32) |
         (1ull << 46) | (2ull << 61);
}
// 16-bit inputs of one type, 32-bit sums.
__device__ __forceinline__ uint32_t umma_instr(bool bf16, bool a_mn, bool b_mn, int m, int n) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}
template <int PAIR>
__device__ __forceinline__ void umma(uint32_t d, uint64_t a, uint64_t b, uint32_t instr, bool add) {
  if constexpr (PAIR == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(instr), "r"((uint32_t)add)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(instr), "r"((uint32_t)add)
        : "memory");
}
// The barrier is arrived on when the matrix instructions issued so far are done (PAIR = 2: that of both CTAs).
template <int PAIR>
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
  if constexpr (PAIR == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                 "h"((uint16_t)3)
                 : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// ---- host: tensor maps -----------------------------------------------------------------------------------------
// Rows of 128 bytes, swizzled, or of 64; dims and box innermost first, strides in values, of the second dimension on.
using TensorMapEncode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                     const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline TensorMapEncode tensor_map_encode() {
  static const TensorMapEncode fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<TensorMapEncode>(p);
  }();
  return fn;
}
inline int make_map(CUtensorMap* map, const void* base, CUtensorMapDataType type, int rank, const uint64_t* dims, const uint64_t* strides, const uint32_t* box,
                    CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
  const TensorMapEncode encode = tensor_map_encode();
  if (!encode) return (int)cudaErrorNotSupported;
  cuuint64_t d[3], s[2];
  cuuint32_t b[3], one[3] = {1, 1, 1};
  for (int i = 0; i < rank; ++i) { d[i] = dims[i]; b[i] = box[i]; }
  for (int i = 0; i + 1 < rank; ++i) s[i] = strides[i] * (type == CU_TENSOR_MAP_DATA_TYPE_FLOAT32 ? 4 : 2);
  const CUresult r = encode(map, type, (cuuint32_t)rank, const_cast<void*>(base), d, s, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : FLEXSPMV_ERR_BAD_ARG;
}

}  // namespace flex
