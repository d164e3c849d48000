// The norm over many gradient tensors, and the tensors scaled to a largest norm.
//
//   norm = sqrt(sum of all squares);  out = grad * min(1, max_norm / (norm + 1e-6))
//
// A plan cuts the tensors into pieces and writes a record of each into the workspace, once for tensors that stay where they are.  The pieces
// go round the CTAs in order; the second of the two launches takes them in the opposite order, so that what the first read last is still in
// L2.  Bound by memory: the gradients are read twice (the scale needs the whole sum) and the result written once.
// A thread adds the squares of a piece in 32 bits (where those leave its range, once more in 64) and the pieces in 64, the CTAs' sums are
// added in one fixed order: no atomics, the same bits every time.
#include <cuda_runtime.h>
#include <stdlib.h>

#include <algorithm>

#include "flex_common.cuh"
#include "flex_expert_types.cuh"

namespace flex {

int device_sm_count();

constexpr int kClipThreads = 256, kClipCtasPerSm = 6;
constexpr float kClipEps = 1e-6f;

struct ClipPiece {
  const void* in;
  void* out;
  int length, types;             // types: the input's in bits 0-1, the output's in bits 2-3
};

// The tensors of one planning launch travel in its parameters.
constexpr int kPlanTensors = 256;
struct ClipTensors {
  const void* in[kPlanTensors];
  void* out[kPlanTensors];
  long long length[kPlanTensors];
  long long first[kPlanTensors];         // number of the tensor's first piece
  unsigned char types[kPlanTensors];
  ClipPiece* piece;
  int size;                      // elements of a piece
};
__global__ void __launch_bounds__(256) clip_plan_kernel(const __grid_constant__ ClipTensors t) {
  const int i = blockIdx.x;
  const long long length = t.length[i], pieces = (length + t.size - 1) / t.size;
  const int types = t.types[i], in_bytes = (types & 3) == FLEXSPMV_TYPE_F32 ? 4 : 2, out_bytes = types >> 2 == FLEXSPMV_TYPE_F32 ? 4 : 2;
  pdl_wait();
  for (long long p = threadIdx.x; p < pieces; p += 256) {
    const long long at = p * t.size, left = length - at;
    ClipPiece r;
    r.in = static_cast<const char*>(t.in[i]) + at * in_bytes;
    r.out = t.out[i] ? static_cast<char*>(t.out[i]) + at * out_bytes : nullptr;
    r.length = (int)(left < t.size ? left : t.size);
    r.types = types;
    t.piece[t.first[i] + p] = r;
  }
}

// `bits`: those of all values together, by which a sum of nothing but zeros is known.
template <class T, int W>
__device__ __forceinline__ float square_sum(const T* p, int n, uint32_t& bits) {
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
    for (int u = 0; u < 4; ++u) {
      bits |= v[u].all_bits();
#pragma unroll
      for (int x = 0; x < W; ++x) acc[x] = fmaf(v[u].get(x), v[u].get(x), acc[x]);
    }
  }
  for (; i < full; i += kClipThreads) {
    Pack<T, W> v;
    v.load(p + (size_t)i * W);
    bits |= v.all_bits();
#pragma unroll
    for (int x = 0; x < W; ++x) acc[x] = fmaf(v.get(x), v.get(x), acc[x]);
  }
  for (int j = full * W + threadIdx.x; j < n; j += kClipThreads) {
    Pack<T, 1> v;
    v.load(p + j);
    bits |= v.all_bits();
    acc[0] = fmaf(v.get(0), v.get(0), acc[0]);
  }
  float s = 0.f;
#pragma unroll
  for (int x = 0; x < W; ++x) s += acc[x];
  return s;
}

// The same values' squares in 64 bits.
template <class T, int W>
__device__ __forceinline__ double square_sum_wide(const T* p, int n) {
  double s = 0;
  const int full = n / W * W;
  for (int i = threadIdx.x * W; i < full; i += kClipThreads * W)
#pragma unroll 1
    for (int x = 0; x < W; ++x) {
      const double d = (double)to_float(p[i + x]);
      s = fma(d, d, s);
    }
  for (int j = full + threadIdx.x; j < n; j += kClipThreads) s = fma((double)to_float(p[j]), (double)to_float(p[j]), s);
  return s;
}

template <class T, int W>
__device__ __forceinline__ double square_sum_as(const T* p, int n) {
  uint32_t bits = 0;
  const float s = square_sum<T, W>(p, n, bits);
  // Squares leave the 32 bits' range from 1.8e19 on (sums of them earlier) and below 1e-19; float16's do not.  A sum inside these bounds has lost
  // nothing: at most 65536 / 256 squares below 2^-126, each by less than 2^-149.
  if (std::is_same<T, __half>::value || (s >= 0x1p-100f && s <= 0x1.fffffep127f)) return (double)s;
  if ((bits & (sizeof(T) == 2 ? 0x7fff7fffu : 0x7fffffffu)) == 0) return 0;
  return square_sum_wide<T, W>(p, n);
}

template <class T>
__device__ __forceinline__ double square_sum_of(const void* in, int n) {
  const T* p = static_cast<const T*>(in);
  // a tensor that does not start on 16 bytes is read a value at a time
  return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 ? square_sum_as<T, 16 / (int)sizeof(T)>(p, n) : square_sum_as<T, 1>(p, n);
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

__global__ void __launch_bounds__(kClipThreads, kClipCtasPerSm) clip_norm_kernel(const ClipPiece* __restrict__ piece, int pieces, double* __restrict__ partial) {
  pdl_wait();
  pdl_launch_dependents();
  double sum = 0;
  ClipPiece next;
  if ((int)blockIdx.x < pieces) next = piece[blockIdx.x];
  for (int c = blockIdx.x; c < pieces; c += gridDim.x) {
    const ClipPiece p = next;
    if (c + (int)gridDim.x < pieces) next = piece[c + gridDim.x];
    const int type = p.types & 3;
    if (type == FLEXSPMV_TYPE_F32) sum += square_sum_of<float>(p.in, p.length);
    else if (type == FLEXSPMV_TYPE_BF16) sum += square_sum_of<__nv_bfloat16>(p.in, p.length);
    else sum += square_sum_of<__half>(p.in, p.length);
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// kW values at a time: 16 bytes of the wider side, so that a warp's stores are whole lines (8 values of bfloat16 into 32 bits as two stores of 16
// bytes each, 32 bytes apart, took 580 us for 400 M values).
template <class TI, class TO>
__device__ __forceinline__ void scale_piece(const TI* in, TO* out, int n, float scale) {
  constexpr int kW = 16 / (int)(sizeof(TI) < sizeof(TO) ? sizeof(TO) : sizeof(TI));
  int done = 0;
  if (((reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(out)) & 15u) == 0) {
    const int full = n / kW;
    int i = threadIdx.x;
    constexpr int kU = 8;
    for (; i + (kU - 1) * kClipThreads < full; i += kU * kClipThreads) {
      Pack<TI, kW> v[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u) v[u].load(in + (size_t)(i + u * kClipThreads) * kW);
#pragma unroll
      for (int u = 0; u < kU; ++u) {
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
__device__ __forceinline__ void scale_piece_to(const void* in, void* out, int type, int n, float scale) {
  const TI* from = static_cast<const TI*>(in);
  if (type == FLEXSPMV_TYPE_F32) scale_piece(from, static_cast<float*>(out), n, scale);
  else if (type == FLEXSPMV_TYPE_BF16) scale_piece(from, static_cast<__nv_bfloat16*>(out), n, scale);
  else scale_piece(from, static_cast<__half*>(out), n, scale);
}

__global__ void __launch_bounds__(kClipThreads, kClipCtasPerSm) clip_scale_kernel(const ClipPiece* __restrict__ piece, int pieces, const double* __restrict__ partial,
                                                                                  int partials, float max_norm, float* __restrict__ norm_out, int write) {
  pdl_wait();
  pdl_launch_dependents();
  const int first = pieces - 1 - (int)blockIdx.x;
  ClipPiece next;
  if (first >= 0) next = piece[first];
  double sum = 0;
  for (int i = threadIdx.x; i < partials; i += kClipThreads) sum += partial[i];
  const float norm = (float)sqrt(block_sum(sum));
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
  if (!write) return;
  const float ratio = max_norm / (norm + kClipEps);
  const float scale = ratio > 1.f ? 1.f : ratio;           // a NaN stays one
  for (int c = first; c >= 0; c -= gridDim.x) {
    const ClipPiece p = next;
    if (c >= (int)gridDim.x) next = piece[c - gridDim.x];
    const int type = p.types & 3, out_type = p.types >> 2;
    if (!p.out || (scale == 1.f && p.in == p.out && type == out_type)) continue;       // a plan for the norm alone; nothing to change
    if (type == FLEXSPMV_TYPE_F32) scale_piece_to<float>(p.in, p.out, out_type, p.length, scale);
    else if (type == FLEXSPMV_TYPE_BF16) scale_piece_to<__nv_bfloat16>(p.in, p.out, out_type, p.length, scale);
    else scale_piece_to<__half>(p.in, p.out, out_type, p.length, scale);
  }
}

// Pieces are scaled in any order: what is written may meet nothing else, other tensors' results as little as other tensors.  Only a tensor and its
// own result may be the same.
static int clip_apart(int count, const void* const* grads, const int32_t* types, const int64_t* lengths, void* const* outs, const int32_t* out_types,
                      const void* ws, size_t ws_bytes) {
  struct Span { uintptr_t from, to; };
  Span* const written = static_cast<Span*>(malloc(((size_t)(outs ? count : 0) + 1) * sizeof(Span)));
  if (!written) return FLEXSPMV_ERR_WORKSPACE;
  const auto span = [](const void* p, size_t bytes) { return Span{reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + bytes}; };
  int n = 0;
  written[n++] = span(ws, ws_bytes);
  for (int i = 0; outs && i < count; ++i)
    if (lengths[i]) written[n++] = span(outs[i], (size_t)lengths[i] * type_bytes(out_types[i]));
  std::sort(written, written + n, [](const Span& a, const Span& b) { return a.from < b.from; });
  bool good = true;
  for (int i = 1; i < n; ++i) good &= written[i - 1].to <= written[i].from;
  for (int i = 0; good && i < count; ++i) {
    if (!lengths[i] || (outs && outs[i] == grads[i])) continue;
    const Span in = span(grads[i], (size_t)lengths[i] * type_bytes(types[i]));
    const Span* const after = std::lower_bound(written, written + n, in.to, [](const Span& a, uintptr_t at) { return a.from < at; });
    good = after == written || after[-1].to <= in.from;
  }
  free(written);
  return good ? 0 : FLEXSPMV_ERR_BAD_ARG;
}

static int clip_ctas() { return device_sm_count() * kClipCtasPerSm; }

// Pieces of 4096 elements, larger ones where every CTA would have many.
struct ClipSizes {
  long long size, pieces;
  size_t piece_at, bytes;              // the workspace: a sum for each CTA, then the pieces
};
static int clip_sizes(int count, const int64_t* lengths, ClipSizes& z) {
  long long total = 0;
  for (int i = 0; i < count; ++i) {
    if (lengths[i] < 0) return FLEXSPMV_ERR_BAD_ARG;
    total += lengths[i];
  }
  z.size = (total / ((long long)clip_ctas() * 8) + 4095) / 4096 * 4096;
  z.size = z.size < 4096 ? 4096 : z.size > 65536 ? 65536 : z.size;
  z.pieces = 0;
  for (int i = 0; i < count; ++i) z.pieces += (lengths[i] + z.size - 1) / z.size;
  if (z.pieces > 0x3fffffffLL) return FLEXSPMV_ERR_TOO_LARGE;
  z.piece_at = (size_t)clip_ctas() * sizeof(double);
  z.bytes = z.piece_at + (size_t)z.pieces * sizeof(ClipPiece);
  return 0;
}

}  // namespace flex

extern "C" {

int flexspmv_clip_gradients_bytes(int32_t count, const int64_t* lengths, size_t* bytes, int32_t* pieces) {
  if (!bytes || !pieces || count < 0 || (count && !lengths)) return FLEXSPMV_ERR_BAD_ARG;
  flex::ClipSizes z;
  if (int e = flex::clip_sizes(count, lengths, z)) return e;
  *bytes = z.bytes;
  *pieces = (int32_t)z.pieces;
  return 0;
}

int flexspmv_clip_gradients_plan(int32_t count, const void* const* grads, const int32_t* types, const int64_t* lengths, void* const* outs,
                                 const int32_t* out_types, void* ws, size_t ws_bytes, void* stream) {
  if (count < 0 || (count && (!grads || !types || !lengths)) || (outs && !out_types)) return FLEXSPMV_ERR_BAD_ARG;
  flex::ClipSizes z;
  if (int e = flex::clip_sizes(count, lengths, z)) return e;
  for (int i = 0; i < count; ++i) {
    if ((lengths[i] && (!grads[i] || (outs && !outs[i]))) || !flex::known_type(types[i]) || (outs && !flex::known_type(out_types[i])))
      return FLEXSPMV_ERR_BAD_ARG;
    const uintptr_t off = (reinterpret_cast<uintptr_t>(grads[i]) & (uintptr_t)(flex::type_bytes(types[i]) - 1)) |
                          (outs ? reinterpret_cast<uintptr_t>(outs[i]) & (uintptr_t)(flex::type_bytes(out_types[i]) - 1) : 0);
    if (off) return FLEXSPMV_ERR_ALIGN;
    if (outs && lengths[i] && outs[i] == grads[i] && out_types[i] != types[i]) return FLEXSPMV_ERR_BAD_ARG;      // in place: one type
  }
  if (!ws || ws_bytes < z.bytes) return FLEXSPMV_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(ws) & 15u) return FLEXSPMV_ERR_ALIGN;
  if (int e = flex::clip_apart(count, grads, types, lengths, outs, out_types, ws, z.bytes)) return e;
  flex::ClipTensors t;
  t.piece = reinterpret_cast<flex::ClipPiece*>(static_cast<char*>(ws) + z.piece_at);
  t.size = (int)z.size;
  long long first = 0;
  for (int from = 0; from < count; from += flex::kPlanTensors) {
    const int n = count - from < flex::kPlanTensors ? count - from : flex::kPlanTensors;
    for (int i = 0; i < n; ++i) {
      t.in[i] = grads[from + i];
      t.out[i] = outs ? outs[from + i] : nullptr;
      t.length[i] = lengths[from + i];
      t.first[i] = first;
      t.types[i] = (unsigned char)(types[from + i] | ((outs ? out_types[from + i] : types[from + i]) << 2));
      first += (lengths[from + i] + z.size - 1) / z.size;
    }
    if (int e = flex::launch_pdl(flex::clip_plan_kernel, n, 256, 0, static_cast<cudaStream_t>(stream), t)) return e;
  }
  return 0;
}

int flexspmv_clip_gradients(int32_t pieces, int32_t write, float max_norm, float* norm, void* ws, size_t ws_bytes, void* stream) {
  const int most = flex::clip_ctas();
  if (pieces < 0 || !norm) return FLEXSPMV_ERR_BAD_ARG;
  if (!ws || ws_bytes < (size_t)most * sizeof(double) + (size_t)pieces * sizeof(flex::ClipPiece)) return FLEXSPMV_ERR_WORKSPACE;
  if (!flex::aligned16(ws) || !flex::aligned_to(4, norm)) return FLEXSPMV_ERR_ALIGN;
  double* const partial = static_cast<double*>(ws);
  const flex::ClipPiece* const piece = reinterpret_cast<const flex::ClipPiece*>(static_cast<char*>(ws) + (size_t)most * sizeof(double));
  const int ctas = pieces < 1 ? 1 : pieces < most ? pieces : most;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int e = flex::launch_pdl(flex::clip_norm_kernel, ctas, flex::kClipThreads, 0, st, piece, pieces, partial)) return e;
  return flex::launch_pdl(flex::clip_scale_kernel, write ? ctas : 1, flex::kClipThreads, 0, st, piece, pieces, static_cast<const double*>(partial), ctas, max_norm, norm, write);
}

}  // extern "C"
