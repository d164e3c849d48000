// Low-rank adapters beside a shared projection: what the adapters' first product and the shared product with its epilogue have in common.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "flex_expert_types.cuh"

namespace flex {

// A place's vector scale A x is kept as two 16-bit values each, the rounded one and the rest (2^-17 of it, a float16 2^-22; a value beyond the type's largest
// is infinite), in rows that the matrix instructions take as they are.  Up to 32 values: 32 high ones, 32 rests; else by 64.
__host__ __device__ constexpr int low_width(int rank) { return rank <= 32 ? 64 : (rank + 63) / 64 * 128; }
__host__ __device__ constexpr int low_high(int k, int rank) { return rank <= 32 ? k : k / 64 * 128 + k % 64; }
__host__ __device__ constexpr int low_rest(int k, int rank) { return low_high(k, rank) + (rank <= 32 ? 32 : 64); }

// What of a value is left by its rounding to T; of what is not finite once rounded, nothing.
template <class T>
__device__ __forceinline__ float low_rest_of(float v) {
  const float high = to_float(from_float<T>(v));
  return fabsf(high) <= 3.4e38f ? v - high : 0.f;
}

// The warp's matrix instruction: d (16 x 8, 32-bit) += a (16 x 16) b (16 x 8).
template <class T>
__device__ __forceinline__ void warp_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// low[rows[i]] = scale[e] down[e] x[rows[i]] (flex_grouped.cu) for the places offsets[e] <= i < offsets[e + 1].
int low_product_of_many(const flexspmv_adapter_desc* d, const void* x, const void* down, const float* scale, const int* offsets, const int* rows, void* low,
                        int low_width, int* status, cudaStream_t st);
// y = weight x + up low (flex_grouped.cu).  The kernel before it on the stream has been launched for it (see ADAPT there).  groups: offsets of groups of
// tokens, group_adapters: the adapter that all tokens of a group have, or one of these.
enum { kGroupMixed = -1, kGroupBare = -2 };
int adapted_product(const flexspmv_adapter_desc* d, const void* x, const void* weight, const void* up, const void* low, int low_width, int num_groups,
                    const int* groups, const int* group_adapters, const int* ids, void* out, int* status, cudaStream_t st);

}  // namespace flex
