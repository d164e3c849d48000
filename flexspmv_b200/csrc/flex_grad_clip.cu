// The norm over many gradient tensors, and the tensors scaled to a largest norm.
//
//   norm = sqrt(sum of all squares);  out = grad * min(1, max_norm / (norm + 1e-6))
//
// Two launches for up to kMost tensors, which travel in the kernels' parameters: no table is copied to the device.  Bound by memory:
// the gradients are read twice (the scale needs the whole sum) and the result written once.  The tensors are cut into pieces that go round the
// CTAs in order; the second launch takes them in the opposite order, so that what the first read last is still in L2.
// A thread adds the squares of a piece in 32 bits and the pieces in 64, the CTAs' sums are added in one fixed order: no atomics, the same
// bits every time.
#include <cuda_runtime.h>

#include "flex_common.cuh"
#include "flex_expert_types.cuh"

namespace flex {

int device_sm_count();

constexpr int kClipThreads = 256, kClipCtasPerSm = 4;
constexpr float kClipEps = 1e-6f;
constexpr int kMost = 1000;                 // 28 KB of parameters; a launch may have 32 764 bytes

struct ClipTensor {
  const void* in;
  void* out;
  long long length;
};
template <int N>
struct ClipArgs {
  ClipTensor tensor[N];
  int first[N + 1];              // first piece of each tensor: pieces of tensor i are first[i] .. first[i + 1]
  unsigned char types[N];        // in: bits 0-1, out: bits 2-3
  int count, piece;              // tensors, elements of a piece
  double* partial;               // a sum for each CTA of every first launch
  int partial_at, partials;      // this launch's place among them, and how many there are
  float max_norm;
  float* norm;
  int write;
};

template <class T, int W>
__device__ __forceinline__ float square_sum(const T* p, int n) {
  float acc[W];
#pragma unroll
  for (int i = 0; i < W; ++i) acc[i] = 0.f;
  const int full = n / W;
  int i = threadIdx.x;
  for (; i + 3 * kClipThreads < full; i += 4 * kClipThreads) {
    Pack<T, W> v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u].load(p + (size_t)(i + u * kClipThreads) * W);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int x = 0; x < W; ++x) acc[x] = fmaf(v[u].get(x), v[u].get(x), acc[x]);
  }
  for (; i < full; i += kClipThreads) {
    Pack<T, W> v;
    v.load(p + (size_t)i * W);
#pragma unroll
    for (int x = 0; x < W; ++x) acc[x] = fmaf(v.get(x), v.get(x), acc[x]);
  }
  for (int j = full * W + threadIdx.x; j < n; j += kClipThreads) acc[0] = fmaf(to_float(p[j]), to_float(p[j]), acc[0]);
  float s = 0.f;
#pragma unroll
  for (int x = 0; x < W; ++x) s += acc[x];
  return s;
}

template <class T>
__device__ __forceinline__ float square_sum_of(const void* in, long long at, int n) {
  const T* p = static_cast<const T*>(in) + at;
  // a tensor that does not start on 16 bytes is read a value at a time
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 ? square_sum<T, 16 / (int)sizeof(T)>(p, n) : square_sum<T, 1>(p, n);
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kClipThreads / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0;
#pragma unroll
  for (int w = 0; w < kClipThreads / 32; ++w) s += part[w];
  return s;
}

template <int N>
__global__ void __launch_bounds__(kClipThreads, kClipCtasPerSm) clip_norm_kernel(const __grid_constant__ ClipArgs<N> a) {
  pdl_wait();
  pdl_launch_dependents();
  double sum = 0;
  int t = 0;
  for (int c = blockIdx.x; c < a.first[a.count]; c += gridDim.x) {
    while (a.first[t + 1] <= c) ++t;
    const long long at = (long long)(c - a.first[t]) * a.piece, left = a.tensor[t].length - at;
    const int n = (int)(left < a.piece ? left : a.piece);
    const int type = a.types[t] & 3;
    float s;
    if (type == FLEXSPMV_TYPE_F32) s = square_sum_of<float>(a.tensor[t].in, at, n);
    else if (type == FLEXSPMV_TYPE_BF16) s = square_sum_of<__nv_bfloat16>(a.tensor[t].in, at, n);
    else s = square_sum_of<__half>(a.tensor[t].in, at, n);
    sum += (double)s;
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) a.partial[a.partial_at + blockIdx.x] = sum;
}

// kW values at a time (the number that fills 16 bytes of the narrower side).
template <class TI, class TO>
__device__ __forceinline__ void scale_piece(const TI* in, TO* out, int n, float scale) {
  constexpr int kW = 16 / (int)(sizeof(TI) < sizeof(TO) ? sizeof(TI) : sizeof(TO));
  int done = 0;
  if (((reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(out)) & 15u) == 0) {
    const int full = n / kW;
    int i = threadIdx.x;
    for (; i + 3 * kClipThreads < full; i += 4 * kClipThreads) {
      Pack<TI, kW> v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u].load(in + (size_t)(i + u * kClipThreads) * kW);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        Pack<TO, kW> r;
#pragma unroll
        for (int x = 0; x < kW; ++x) r.set(x, v[u].get(x) * scale);
        r.store(out + (size_t)(i + u * kClipThreads) * kW);
      }
    }
    for (; i < full; i += kClipThreads) {
      Pack<TI, kW> v;
      Pack<TO, kW> r;
      v.load(in + (size_t)i * kW);
#pragma unroll
      for (int x = 0; x < kW; ++x) r.set(x, v.get(x) * scale);
      r.store(out + (size_t)i * kW);
    }
    done = full * kW;
  }
  for (int j = done + threadIdx.x; j < n; j += kClipThreads) out[j] = from_float<TO>(to_float(in[j]) * scale);
}

template <class TI>
__device__ __forceinline__ void scale_piece_to(const TI* in, void* out, int type, long long at, int n, float scale) {
  if (type == FLEXSPMV_TYPE_F32) scale_piece(in, static_cast<float*>(out) + at, n, scale);
  else if (type == FLEXSPMV_TYPE_BF16) scale_piece(in, static_cast<__nv_bfloat16*>(out) + at, n, scale);
  else scale_piece(in, static_cast<__half*>(out) + at, n, scale);
}

template <int N>
__global__ void __launch_bounds__(kClipThreads, kClipCtasPerSm) clip_scale_kernel(const __grid_constant__ ClipArgs<N> a) {
  pdl_wait();
  pdl_launch_dependents();
  double sum = 0;
  for (int i = threadIdx.x; i < a.partials; i += kClipThreads) sum += a.partial[i];
  const float norm = (float)sqrt(block_sum(sum));
  if (a.partial_at == 0 && blockIdx.x == 0 && threadIdx.x == 0) *a.norm = norm;
  if (!a.write) return;
  const float ratio = a.max_norm / (norm + kClipEps);
  const float scale = ratio > 1.f ? 1.f : ratio;           // a NaN stays one
  int t = a.count - 1;
  const int all = a.first[a.count];
  for (int c = all - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
    while (a.first[t] > c) --t;
    const int type = a.types[t] & 3, out_type = a.types[t] >> 2;
    if (scale == 1.f && a.tensor[t].in == a.tensor[t].out && type == out_type) continue;       // nothing to change
    const long long at = (long long)(c - a.first[t]) * a.piece, left = a.tensor[t].length - at;
    const int n = (int)(left < a.piece ? left : a.piece);
    if (type == FLEXSPMV_TYPE_F32) scale_piece_to(static_cast<const float*>(a.tensor[t].in) + at, a.tensor[t].out, out_type, at, n, scale);
    else if (type == FLEXSPMV_TYPE_BF16) scale_piece_to(static_cast<const __nv_bfloat16*>(a.tensor[t].in) + at, a.tensor[t].out, out_type, at, n, scale);
    else scale_piece_to(static_cast<const __half*>(a.tensor[t].in) + at, a.tensor[t].out, out_type, at, n, scale);
  }
}

static int clip_ctas() { return device_sm_count() * kClipCtasPerSm; }

template <int N>
static int clip_launches(int count, const void* const* grads, void* const* outs, const int64_t* lengths, const int32_t* types, const int32_t* out_types,
                         long long total, float max_norm, float* norm, double* partial, cudaStream_t st) {
  static_assert(sizeof(ClipArgs<N>) <= 32764, "kernel parameters");
  // pieces of 4096 elements, larger where every CTA would have many
  const int ctas = clip_ctas();
  long long piece = (total / ((long long)ctas * 8) + 4095) / 4096 * 4096;
  piece = piece < 4096 ? 4096 : piece > 65536 ? 65536 : piece;
  const int parts = (count + N - 1) / N > 0 ? (count + N - 1) / N : 1;
  for (int pass = 0; pass < 2; ++pass) {
    // the second launches run from the last part to the first, as each runs from its last piece to its first
    for (int i = 0; i < parts; ++i) {
      const int part = pass ? parts - 1 - i : i, from = part * N, n = count - from < N ? count - from : N;
      ClipArgs<N> a;
      long long pieces = 0;
      for (int j = 0; j < n; ++j) {
        a.tensor[j] = {grads[from + j], outs ? outs[from + j] : nullptr, lengths[from + j]};
        a.types[j] = (unsigned char)(types[from + j] | ((outs ? out_types[from + j] : 0) << 2));
        a.first[j] = (int)pieces;
        pieces += (lengths[from + j] + piece - 1) / piece;
        if (pieces > 0x3fffffffLL) return FLEXSPMV_ERR_TOO_LARGE;
      }
      a.first[n] = (int)pieces;
      a.count = n;
      a.piece = (int)piece;
      a.partial = partial;
      a.partial_at = part * ctas;
      a.partials = parts * ctas;
      a.max_norm = max_norm;
      a.norm = norm;
      a.write = outs != nullptr;
      if (pass == 0) {
        if (int e = launch_pdl(clip_norm_kernel<N>, ctas, kClipThreads, 0, st, a)) return e;
      } else if (a.write || part == 0) {
        if (int e = launch_pdl(clip_scale_kernel<N>, a.write ? ctas : 1, kClipThreads, 0, st, a)) return e;
      }
    }
  }
  return 0;
}

}  // namespace flex

extern "C" {

int flexspmv_clip_gradients_bytes(int32_t count, size_t* bytes) {
  if (!bytes || count < 0) return FLEXSPMV_ERR_BAD_ARG;
  *bytes = (size_t)((count + flex::kMost - 1) / flex::kMost + 1) * flex::clip_ctas() * sizeof(double);
  return 0;
}

int flexspmv_clip_gradients(int32_t count, const void* const* grads, const int32_t* types, const int64_t* lengths, void* const* outs,
                            const int32_t* out_types, float max_norm, float* norm, void* ws, size_t ws_bytes, void* stream) {
  if (count < 0 || !norm || (count && (!grads || !types || !lengths)) || (outs && !out_types)) return FLEXSPMV_ERR_BAD_ARG;
  long long total = 0;
  for (int i = 0; i < count; ++i) {
    if (lengths[i] < 0 || (lengths[i] && (!grads[i] || (outs && !outs[i]))) || !flex::known_type(types[i]) || (outs && !flex::known_type(out_types[i])))
      return FLEXSPMV_ERR_BAD_ARG;
    const uintptr_t off = (reinterpret_cast<uintptr_t>(grads[i]) & (uintptr_t)(flex::type_bytes(types[i]) - 1)) |
                          (outs ? reinterpret_cast<uintptr_t>(outs[i]) & (uintptr_t)(flex::type_bytes(out_types[i]) - 1) : 0);
    if (off) return FLEXSPMV_ERR_ALIGN;
    if (outs && lengths[i] && outs[i] == grads[i] && out_types[i] != types[i]) return FLEXSPMV_ERR_BAD_ARG;      // in place: one type
    total += lengths[i];
  }
  size_t need = 0;
  flexspmv_clip_gradients_bytes(count, &need);
  if (!ws || ws_bytes < need) return FLEXSPMV_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(ws) & 7u) return FLEXSPMV_ERR_ALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // a launch copies its parameters, so lists that fit 100 entries take the smaller ones
  if (count <= 100) return flex::clip_launches<100>(count, grads, outs, lengths, types, out_types, total, max_norm, norm, static_cast<double*>(ws), st);
  if (count <= 300) return flex::clip_launches<300>(count, grads, outs, lengths, types, out_types, total, max_norm, norm, static_cast<double*>(ws), st);
  return flex::clip_launches<flex::kMost>(count, grads, outs, lengths, types, out_types, total, max_norm, norm, static_cast<double*>(ws), st);
}

}  // extern "C"
