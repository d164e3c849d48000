// Matrix products grouped by expert over ragged groups of rows:
//   forward  y[i] = W[e] x[rows[i]]        dx  dx[i] = W[e]^T dy[i]        dw  dW[e] = sum_i dy[i] x[rows[i]]^T
#include <cuda_runtime.h>

#include "flex_common.cuh"
#include "flex_expert_types.cuh"

namespace flex {

int device_sm_count();

struct GroupedArgs {
  const void *a, *b;             // forward: x, weight; dx: dy, weight; dw: dy, x
  const int *offsets, *rows;
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

__device__ __forceinline__ long long row_of(const GroupedArgs& a, int place) {
  if (!a.rows) return place;
  const int r = a.rows[place];
  if (r < 0 || r >= a.tokens) { raise(a.status, FLEXSPMV_ERR_BAD_CSR); return 0; }
  return r;
}

// 64 x 64 outputs by 256 threads, 16 of the inner length at a time through shared memory.
template <class T, class TO, int MODE>
__global__ void __launch_bounds__(256) grouped_simple_kernel(GroupedArgs a) {
  __shared__ float sa[16][65], sb[16][65];
  const int e = blockIdx.z, tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  int from, to;
  group_of(a, e, from, to);
  const T *pa = static_cast<const T*>(a.a), *pb = static_cast<const T*>(a.b);
  const int cols = MODE == FLEXSPMV_GROUPED_FORWARD ? a.n : a.k;
  const int inner = MODE == FLEXSPMV_GROUPED_FORWARD ? a.k : MODE == FLEXSPMV_GROUPED_DX ? a.n : to - from;
  const int m_end = MODE == FLEXSPMV_GROUPED_DW ? a.n : to - from;
  const int c0 = blockIdx.x * 64;
  for (int m0 = blockIdx.y * 64; m0 < m_end; m0 += gridDim.y * 64) {
    float acc[4][4] = {};
    for (int k0 = 0; k0 < inner; k0 += 16) {
      for (int i = tid; i < 1024; i += 256) {
        const int kk = i & 15, r = i >> 4, k = k0 + kk;
        float va = 0.f, vb = 0.f;
        if (k < inner) {
          if (m0 + r < m_end) {
            if (MODE == FLEXSPMV_GROUPED_FORWARD) va = to_float(pa[row_of(a, from + m0 + r) * a.a_stride + k]);
            else if (MODE == FLEXSPMV_GROUPED_DX) va = to_float(pa[(long long)(from + m0 + r) * a.a_stride + k]);
            else va = to_float(pa[(long long)(from + k) * a.a_stride + m0 + r]);
          }
          if (c0 + r < cols) {
            if (MODE == FLEXSPMV_GROUPED_FORWARD) vb = to_float(pb[((long long)e * a.n + c0 + r) * a.k + k]);
            else if (MODE == FLEXSPMV_GROUPED_DX) vb = to_float(pb[((long long)e * a.n + k) * a.k + c0 + r]);
            else vb = to_float(pb[row_of(a, from + k) * a.b_stride + c0 + r]);
          }
        }
        sa[kk][r] = va;
        sb[kk][r] = vb;
      }
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < 16; ++kk)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[kk][ty + 16 * i], sb[kk][tx + 16 * j], acc[i][j]);
      __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
      for (int j = 0; j < 4; ++j) {
        const int m = m0 + ty + 16 * i, c = c0 + tx + 16 * j;
        if (m >= m_end || c >= cols) continue;
        const long long at = MODE == FLEXSPMV_GROUPED_DW ? ((long long)e * a.n + m) * a.k + c : (long long)(from + m) * cols + c;
        static_cast<TO*>(a.out)[at] = from_float<TO>(acc[i][j]);
      }
  }
  // rows in no expert's places
  if (MODE != FLEXSPMV_GROUPED_DW && (e == 0 || e == a.experts - 1)) {
    const long long lo = e == 0 ? 0 : to, hi = e == 0 ? from : a.slots;
    for (int part = 0; part < (a.experts == 1 ? 2 : 1); ++part) {
      const long long l = part ? to : lo, h = part ? a.slots : hi;
      for (long long m = l + blockIdx.y; m < h; m += gridDim.y)
        for (int c = c0 + tid; c < cols && c < c0 + 64; c += 256) static_cast<TO*>(a.out)[m * cols + c] = from_float<TO>(0.f);
    }
  }
}

template <class T, class TO, int MODE>
static int grouped_launch(const GroupedArgs& a, cudaStream_t st) {
  const int cols = MODE == FLEXSPMV_GROUPED_FORWARD ? a.n : a.k;
  const int m = MODE == FLEXSPMV_GROUPED_DW ? (a.n + 63) / 64 : 16;
  grouped_simple_kernel<T, TO, MODE><<<dim3((cols + 63) / 64, m, a.experts), 256, 0, st>>>(a);
  return (int)cudaGetLastError();
}

static int check_grouped(const flexspmv_expert_desc* d, int which) {
  if (!d || d->tokens < 0 || d->slots < 0 || d->experts < 1 || d->n < 1 || d->k < 1) return FLEXSPMV_ERR_BAD_ARG;
  if (d->type != FLEXSPMV_TYPE_BF16 && d->type != FLEXSPMV_TYPE_F16) return FLEXSPMV_ERR_BAD_ARG;
  if (which == FLEXSPMV_GROUPED_DW && d->out_type != FLEXSPMV_TYPE_F32 && d->out_type != d->type) return FLEXSPMV_ERR_BAD_ARG;
  if (d->in_stride < (which == FLEXSPMV_GROUPED_FORWARD ? d->k : d->n) || (which == FLEXSPMV_GROUPED_DW && d->in2_stride < d->k)) return FLEXSPMV_ERR_BAD_ARG;
  if (d->experts > FLEXSPMV_MAX_EXPERTS || d->slots > 0x7fffffffLL || d->tokens > 0x7fffffffLL) return FLEXSPMV_ERR_TOO_LARGE;
  if (d->n % 8 || d->k % 8 || d->in_stride % 8 || (which == FLEXSPMV_GROUPED_DW && d->in2_stride % 8)) return FLEXSPMV_ERR_ALIGN;
  return 0;
}

}  // namespace flex

extern "C" {

int flexspmv_grouped_matmul_bytes(const flexspmv_expert_desc* d, int32_t which, size_t* bytes) {
  if (!bytes || which < FLEXSPMV_GROUPED_FORWARD || which > FLEXSPMV_GROUPED_DW) return FLEXSPMV_ERR_BAD_ARG;
  if (int e = flex::check_grouped(d, which)) return e;
  *bytes = 0;
  return 0;
}

int flexspmv_grouped_matmul(const flexspmv_expert_desc* d, const void* const* in, void* const* out, void* ws, size_t ws_bytes, int32_t* status,
                            void* stream) {
  if (int e = flex::check_grouped(d, FLEXSPMV_GROUPED_FORWARD)) return e;
  if (!in || !out) return FLEXSPMV_ERR_BAD_ARG;
  if (d->slots == 0) return 0;
  if (!in[0] || !in[1] || !in[2] || !out[0] || d->tokens < (in[3] ? 1 : d->slots)) return FLEXSPMV_ERR_BAD_ARG;
  if (!flex::aligned16(in[0]) || !flex::aligned16(in[1]) || !flex::aligned16(out[0])) return FLEXSPMV_ERR_ALIGN;
  flex::GroupedArgs a = {in[0], in[1], static_cast<const int*>(in[2]), static_cast<const int*>(in[3]), out[0], d->tokens, d->slots, d->in_stride, 0,
                         d->experts, d->n, d->k, status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d->type == FLEXSPMV_TYPE_BF16) return flex::grouped_launch<__nv_bfloat16, __nv_bfloat16, FLEXSPMV_GROUPED_FORWARD>(a, st);
  return flex::grouped_launch<__half, __half, FLEXSPMV_GROUPED_FORWARD>(a, st);
}

int flexspmv_grouped_matmul_dx(const flexspmv_expert_desc* d, const void* const* in, void* const* out, void* ws, size_t ws_bytes, int32_t* status,
                               void* stream) {
  if (int e = flex::check_grouped(d, FLEXSPMV_GROUPED_DX)) return e;
  if (!in || !out) return FLEXSPMV_ERR_BAD_ARG;
  if (d->slots == 0) return 0;
  if (!in[0] || !in[1] || !in[2] || !out[0]) return FLEXSPMV_ERR_BAD_ARG;
  if (!flex::aligned16(in[0]) || !flex::aligned16(in[1]) || !flex::aligned16(out[0])) return FLEXSPMV_ERR_ALIGN;
  flex::GroupedArgs a = {in[0], in[1], static_cast<const int*>(in[2]), nullptr, out[0], d->slots, d->slots, d->in_stride, 0, d->experts, d->n, d->k, status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d->type == FLEXSPMV_TYPE_BF16) return flex::grouped_launch<__nv_bfloat16, __nv_bfloat16, FLEXSPMV_GROUPED_DX>(a, st);
  return flex::grouped_launch<__half, __half, FLEXSPMV_GROUPED_DX>(a, st);
}

int flexspmv_grouped_matmul_dw(const flexspmv_expert_desc* d, const void* const* in, void* const* out, void* ws, size_t ws_bytes, int32_t* status,
                               void* stream) {
  if (int e = flex::check_grouped(d, FLEXSPMV_GROUPED_DW)) return e;
  if (!in || !out || !in[2] || !out[0]) return FLEXSPMV_ERR_BAD_ARG;
  if (d->slots && (!in[0] || !in[1] || d->tokens < (in[3] ? 1 : d->slots))) return FLEXSPMV_ERR_BAD_ARG;
  if (!flex::aligned16(in[0]) || !flex::aligned16(in[1]) || !flex::aligned16(out[0])) return FLEXSPMV_ERR_ALIGN;
  flex::GroupedArgs a = {in[0], in[1], static_cast<const int*>(in[2]), static_cast<const int*>(in[3]), out[0], d->tokens, d->slots, d->in_stride,
                         d->in2_stride, d->experts, d->n, d->k, status};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = d->out_type == FLEXSPMV_TYPE_F32;
  if (d->type == FLEXSPMV_TYPE_BF16)
    return wide ? flex::grouped_launch<__nv_bfloat16, float, FLEXSPMV_GROUPED_DW>(a, st)
                : flex::grouped_launch<__nv_bfloat16, __nv_bfloat16, FLEXSPMV_GROUPED_DW>(a, st);
  return wide ? flex::grouped_launch<__half, float, FLEXSPMV_GROUPED_DW>(a, st) : flex::grouped_launch<__half, __half, FLEXSPMV_GROUPED_DW>(a, st);
}

}  // extern "C"
