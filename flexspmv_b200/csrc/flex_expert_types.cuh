// Value types of the expert operators: 16- and 32-bit floats, W of them in one access.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "../../include/flexspmv.h"

namespace flex {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// Two values in a word, the first one low.
template <class T> __device__ __forceinline__ uint32_t two_of(float a, float b) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __half2 r = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}

// W values: in pieces of 16 bytes or one of 8, where they are that many, else a value on its own.
template <class T, int W>
struct Pack {
  union { uint4 raw[(sizeof(T) * W + 15) / 16]; uint2 half; T v[W]; };
  __device__ __forceinline__ Pack() {}
  static constexpr bool kWide = sizeof(T) * W % 16 == 0, kHalf = sizeof(T) * W == 8;
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kWide) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) * W / 16; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
    } else if constexpr (kHalf) {
      half = *reinterpret_cast<const uint2*>(p);
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] = p[i];
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kWide) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) * W / 16; ++i) reinterpret_cast<uint4*>(p)[i] = raw[i];
    } else if constexpr (kHalf) {
      *reinterpret_cast<uint2*>(p) = half;
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) p[i] = v[i];
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = from_float<T>(0.f);
  }
  // 16-bit values as they are: two of them, or the only one.
  __device__ __forceinline__ uint32_t word(int i) const { return i % 4 == 0 ? raw[i / 4].x : i % 4 == 1 ? raw[i / 4].y : i % 4 == 2 ? raw[i / 4].z : raw[i / 4].w; }
  __device__ __forceinline__ uint32_t bits() const { return *reinterpret_cast<const unsigned short*>(&v[0]); }
  // The bits of all values, those of 16 bits by two.
  __device__ __forceinline__ uint32_t all_bits() const {
    if constexpr (kWide) {
      uint32_t r = 0;
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) * W / 16; ++i) r |= raw[i].x | raw[i].y | raw[i].z | raw[i].w;
      return r;
    } else {
      uint32_t r = 0;
#pragma unroll
      for (int i = 0; i < W; ++i)
        if constexpr (sizeof(T) == 4) r |= *reinterpret_cast<const uint32_t*>(&v[i]);
        else r |= *reinterpret_cast<const unsigned short*>(&v[i]);
      return r;
    }
  }
  __device__ __forceinline__ float get(int i) const { return to_float(v[i]); }
  __device__ __forceinline__ void set(int i, float x) { v[i] = from_float<T>(x); }
};

// Lets a kernel have this much dynamic shared memory; the runtime is asked once for a kernel, a device and a size above 48 KB.
template <auto KERNEL>
int allow_smem(int bytes) {
  static std::atomic<int> allowed[64];
  int device = 0;
  if (bytes <= 48 * 1024) return 0;
  if (cudaError_t e = cudaGetDevice(&device); e != cudaSuccess) return (int)e;
  const bool known = device >= 0 && device < 64;
  if (known && allowed[device].load(std::memory_order_relaxed) >= bytes) return 0;
  if (cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); e != cudaSuccess) return (int)e;
  if (known) allowed[device].store(bytes, std::memory_order_relaxed);
  return 0;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// Whether every array begins on a value of so many bytes; null ones do.
template <class... P>
bool aligned_to(int bytes, P... p) { return (((reinterpret_cast<uintptr_t>(p) & (uintptr_t)(bytes - 1)) | ...) == 0); }
inline bool known_type(int t) { return t == FLEXSPMV_TYPE_F32 || t == FLEXSPMV_TYPE_BF16 || t == FLEXSPMV_TYPE_F16; }
inline int type_bytes(int t) { return t == FLEXSPMV_TYPE_F32 ? 4 : 2; }

// Where an array lies: rows of `row` bytes, `stride` bytes apart (one row: contiguous).
struct Region {
  const void* at;
  long long row, rows = 1, stride = 1;
};
inline Region rows_at(const void* at, long long rows, long long n, long long stride, int type) {
  return {at, n * type_bytes(type), rows, stride * type_bytes(type)};
}
// Whether the first row of `out`, which is all of it, shares a byte with `in`; between the rows of `in` it may lie.
inline bool meets(const Region& out, const Region& in) {
  if (!out.at || !in.at || out.row <= 0 || in.row <= 0) return false;
  const long long o = (long long)(reinterpret_cast<uintptr_t>(out.at) - reinterpret_cast<uintptr_t>(in.at));
  const long long i = o < in.row ? 0 : (o - in.row) / in.stride + 1;          // the first row that ends after out begins
  return i < in.rows && i * in.stride < o + out.row;
}
// What a launch writes lies apart from all that it reads, and from what else it writes.
template <int OUTS, int INS>
bool apart(const Region (&outs)[OUTS], const Region (&ins)[INS]) {
  for (int o = 0; o < OUTS; ++o) {
    for (const Region& in : ins)
      if (meets(outs[o], in)) return false;
    for (int p = 0; p < o; ++p)
      if (meets(outs[o], outs[p])) return false;
  }
  return true;
}

}  // namespace flex
