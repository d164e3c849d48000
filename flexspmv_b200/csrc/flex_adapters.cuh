// Low-rank adapters beside a shared projection: what the adapters' first product and the shared product with its epilogue have in common.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "flex_expert_types.cuh"

namespace flex {

// A place's vector scale A x, a sum of 32 bits, is kept as 16-bit values that add up to it, which the matrix instructions take as they are: three bfloat16
// have all 24 of its bits; two float16 22 of them, which is 2^-11 of what y's own rounding takes.  (Two bfloat16, 17 bits, made 1.1 of 1000 values of y another
// one than the 32-bit vector does.)  us, two / three: 8192 tokens of rank 64 (4096 x 4096, 12 runs) 223 / 227, 2000 in 5 runs 80.5 / 82, 300 of rank 16 in
// short runs 42 / 46, 48 of rank 16 14.6 / 14.7.
// In a row: ranks up to 16: a part behind the other, 16 values each; up to 32: 32 each; else 64 of the vector at a time, their parts behind one another.  Rows
// are whole steps of 64 values.
template <class T> constexpr int kLowParts = std::is_same<T, __nv_bfloat16>::value ? 3 : 2;
__host__ __device__ constexpr int low_width(int rank, int parts) {
  return rank <= 16 ? 64 : rank <= 32 ? (parts * 32 + 63) / 64 * 64 : (rank + 63) / 64 * 64 * parts;
}
template <class T>
__host__ __device__ constexpr int low_at(int k, int rank, int part) {
  return rank <= 16 ? part * 16 + k : rank <= 32 ? part * 32 + k : (k / 64 * kLowParts<T> + part) * 64 + k % 64;
}
// The parts of a value.  A bfloat16's are cut, not rounded, so that none is beyond the type's largest; of what is not finite the first has all.
template <class T>
__device__ __forceinline__ void low_parts(float v, float (&part)[kLowParts<T>]) {
  const bool finite = fabsf(v) <= 3.402823466e38f;
  float left = v;
#pragma unroll
  for (int p = 0; p < kLowParts<T>; ++p) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) part[p] = __uint_as_float(__float_as_uint(left) & 0xffff0000u);
    else part[p] = to_float(from_float<T>(left));
    left = finite && fabsf(part[p]) <= 3.402823466e38f ? left - part[p] : 0.f;
  }
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
// tokens, group_adapters: the adapter that all tokens of a group have, or one of these.  plan: its second and third int say of how many tokens and adapters
// all of this is; of others: nothing is written, and the status says so.
enum { kGroupMixed = -1, kGroupBare = -2 };
int adapted_product(const flexspmv_adapter_desc* d, const void* x, const void* weight, const void* up, const void* low, int low_width, const int* plan, int num_groups,
                    const int* groups, const int* group_adapters, const int* ids, void* out, int* status, cudaStream_t st);

}  // namespace flex
