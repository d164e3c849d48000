// Low-rank adapters beside a shared projection: what the adapters' first product and the shared product with its epilogue have in common.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "flex_expert_types.cuh"

namespace flex {

// A place's vector scale A x, a sum of 32 bits, is kept as 16-bit values that add up to it, which the matrix instructions take as they are: three bfloat16
// have all 24 of its bits; two float16 22 of them, which is 2^-11 of what y's own rounding takes.  (Two bfloat16, 17 bits, made 1.1 of 1000 values of y another
// one than the 32-bit vector does.)  us, two / three: 8192 tokens of rank 64 (4096 x 4096, 12 runs) 223 / 227, 300 of rank 16 in short runs 36.4 / 37.4, 48 of
// rank 16 14.6 / 15.2.
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
    left = finite ? left - part[p] : 0.f;
  }
}
// Float16 parts go from 65504 down to steps of 2^-24.  A vector's 32 neighbouring values that leave this range, by one that is larger (or not finite) or by all of them
// being so small that the steps show, are kept as they are, in 32 bits, and their parts are zeros; a flag says so.  The flagged ones' products are added on the
// result's way out (low_rank_wide), which costs the others the flags' loads (us, none flagged, without flags / with: one token 8.6 / 9.0, 8192 of rank 64 234 / 238; all
// flagged 451, by ordinary arithmetic 2800).
// kWideBelow: the largest of the 32 has 2^-17 of itself in those steps' halves then, a 32nd of y's own rounding.
template <class T> constexpr bool kHasWide = std::is_same<T, __half>::value;
constexpr float kWideAbove = 65504.f, kWideBelow = 0x1p-8f;
// Where the vectors' workspace has what: the parts, then (float16) the values of flagged ones and the flags.
struct LowPlaces {
  long long wide, flags, bytes;          // bytes from its beginning
  int width, wide_width;                 // values of a row
};
inline LowPlaces low_places(long long tokens, int rank, int type) {
  const bool has_wide = type != FLEXSPMV_TYPE_BF16;
  const int parts = type == FLEXSPMV_TYPE_BF16 ? kLowParts<__nv_bfloat16> : kLowParts<__half>;
  LowPlaces p;
  p.width = low_width(rank, parts);
  p.wide_width = (rank + 31) / 32 * 32;
  p.wide = tokens * p.width * 2;
  p.flags = p.wide + (has_wide ? tokens * p.wide_width * 4 : 0);
  p.bytes = p.flags + (has_wide ? (tokens * (p.wide_width / 32) + 15) / 16 * 16 : 0);
  return p;
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

// The same of 32-bit values whose last 13 bits are zeros, 8 of them: d (16 x 8) += a (16 x 8) b (8 x 8).
__device__ __forceinline__ void warp_mma_wide(float (&d)[4], float a0, float a1, float a2, float a3, float b0, float b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(__float_as_uint(a0)), "r"(__float_as_uint(a1)), "r"(__float_as_uint(a2)), "r"(__float_as_uint(a3)), "r"(__float_as_uint(b0)),
                 "r"(__float_as_uint(b1)));
}

// The vectors of the places offsets[e] <= i < offsets[e + 1], scale[e] down[e] x[rows[i]], into the workspace (flex_grouped.cu).
int low_product_of_many(const flexspmv_adapter_desc* d, const void* x, const void* down, const float* scale, const int* offsets, const int* rows, void* ws,
                        int* status, cudaStream_t st);
// y = weight x + up low (flex_grouped.cu), with the vectors of the workspace.  The kernel before it on the stream has been launched for it (see ADAPT there).  groups:
// offsets of groups of tokens, group_adapters: the adapter that all tokens of a group have, or one of these.  plan: its second and third int say of how many tokens
// and adapters all of this is; of others: nothing is written, and the status says so.
enum { kGroupMixed = -1, kGroupBare = -2 };
int adapted_product(const flexspmv_adapter_desc* d, const void* x, const void* weight, const void* up, const void* ws, const int* plan, int num_groups,
                    const int* groups, const int* group_adapters, const int* ids, void* out, int* status, cudaStream_t st);

}  // namespace flex
