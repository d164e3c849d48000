// What stands around a layer on the residual stream: layer norm with the sum (and the dropout) in front of it, its gradients, and dropout.
#include <cuda_runtime.h>

#include <type_traits>

#include "flex_common.cuh"
#include "flex_expert_types.cuh"

namespace flex {

int device_sm_count();

// ---- random numbers ------------------------------------------------------------------------------------------------

// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers, as easy as 1, 2, 3; 2011).  Four words for four neighbouring columns of
// a row: counter (column / 4, row, offset), key = seed, so that a value's word goes by its place alone, whatever the launch, the strides or the type,
// and the backward pass makes it again.
struct Random {
  uint32_t offset1, first, second;     // the counter's last word, and what every first round makes of the one before it
  uint32_t key0[10], key1[10];         // of the rounds; made once a thread
  __device__ __forceinline__ Random(const unsigned long long* seed, bool used) {
    unsigned long long k = 0, o = 0;
    if (used) {
      k = seed[0];
      o = seed[1];
    }
#pragma unroll
    for (int i = 0; i < 10; ++i) {
      key0[i] = (uint32_t)k + i * 0x9E3779B9u;
      key1[i] = (uint32_t)(k >> 32) + i * 0xBB67AE85u;
    }
    const unsigned long long b = (o & 0xffffffffull) * 0xCD9E8D57u;
    first = (uint32_t)(b >> 32) ^ key0[0];
    second = (uint32_t)b;
    offset1 = (uint32_t)(o >> 32) ^ key1[0];
  }
  __device__ __forceinline__ void words(uint32_t group, uint32_t row, uint32_t (&w)[4]) const {
    const unsigned long long begin = (unsigned long long)group * 0xD2511F53u;
    uint32_t c0 = first ^ row, c1 = second, c2 = (uint32_t)(begin >> 32) ^ offset1, c3 = (uint32_t)begin;
#pragma unroll
    for (int i = 1; i < 10; ++i) {
      const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
      c0 = (uint32_t)(b >> 32) ^ c1 ^ key0[i];
      c1 = (uint32_t)b;
      c2 = (uint32_t)(a >> 32) ^ c3 ^ key1[i];
      c3 = (uint32_t)a;
    }
    w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
  }
  // C values from column c (a multiple of four) on: t plus what is kept of them, scaled.
  template <int C>
  __device__ __forceinline__ void drop(float (&v)[C], const float (&t)[C], int c, uint32_t row, uint32_t below, float scale) const {
    static_assert(C % 4 == 0, "whole groups");
#pragma unroll
    for (int g = 0; g < C / 4; ++g) {
      uint32_t w[4];
      words((uint32_t)(c / 4 + g), row, w);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[g * 4 + j] = fmaf(w[j] < below ? 0.f : v[g * 4 + j], scale, t[g * 4 + j]);
    }
  }
  template <int C>
  __device__ __forceinline__ void drop(float (&v)[C], int c, uint32_t row, uint32_t below, float scale) const {
    float none[C];
#pragma unroll
    for (int j = 0; j < C; ++j) none[j] = 0.f;
    drop(v, none, c, row, below, scale);
  }
};

// ---- rows ----------------------------------------------------------------------------------------------------------

// C neighbouring values of a row as they are, in one access (WIDE: all of them exist or none) or one by one.
template <class T, int C, bool WIDE>
struct Values {
  static constexpr bool kPairs = WIDE && sizeof(T) == 2;
  Pack<T, C> q;
  __device__ __forceinline__ void load(const T* row, int c, int width) {
    if constexpr (WIDE) {
      if (c < width) q.load(row + c);
      else q.zero();
    } else {
#pragma unroll
      for (int j = 0; j < C; ++j) q.v[j] = c + j < width ? row[c + j] : from_float<T>(0.f);
    }
  }
  __device__ __forceinline__ void get(float (&v)[C]) const {
#pragma unroll
    for (int j = 0; j < C; ++j) v[j] = q.get(j);
  }
};
template <class T, int C, bool WIDE>
__device__ __forceinline__ void load_values(const T* row, int c, int width, float (&v)[C]) {
  Values<T, C, WIDE> q;
  q.load(row, c, width);
  q.get(v);
}
template <class T, int C, bool WIDE>
__device__ __forceinline__ void store_values(T* row, int c, int width, const float (&v)[C]) {
  if constexpr (WIDE && sizeof(T) == 2) {          // rounded by two: an instruction, and none to put them together
    static_assert(C == 8, "16 bytes");
    if (c < width) *reinterpret_cast<uint4*>(row + c) = make_uint4(two_of<T>(v[0], v[1]), two_of<T>(v[2], v[3]), two_of<T>(v[4], v[5]), two_of<T>(v[6], v[7]));
  } else if constexpr (WIDE) {
    Pack<T, C> q;
#pragma unroll
    for (int j = 0; j < C; ++j) q.set(j, v[j]);
    if (c < width) q.store(row + c);
  } else {
#pragma unroll
    for (int j = 0; j < C; ++j)
      if (c + j < width) row[c + j] = from_float<T>(v[j]);
  }
}
// Weights are 32-bit or of the rows' type; none: `value`.
template <class T, int C, bool WIDE>
__device__ __forceinline__ void load_params(const void* p, bool wide_type, int c, int width, float value, float (&v)[C]) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < C; ++j) v[j] = value;
  } else if (std::is_same<T, float>::value || wide_type) {
    load_values<float, C, WIDE>(static_cast<const float*>(p), c, width, v);
  } else {
    load_values<T, C, WIDE>(static_cast<const T*>(p), c, width, v);
  }
}

// Sums over the TPR threads of a row, the same bits in all of them.  `buf` alternates between two halves, so that a barrier lies between a half's reading
// and its next writing.
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*buf)[N][32], int& turn) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int o = 16; o; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
  if constexpr (TPR > 32) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) buf[turn][n][warp] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = lane < TPR / 32 ? buf[turn][n][lane] : 0.f;
#pragma unroll
      for (int o = 16; o; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
    }
    turn ^= 1;
  }
}

struct NormArgs {
  const void *x, *residual, *weight, *bias;
  const unsigned long long* seed;      // null: nothing is dropped
  void *y, *sum;
  float *mean, *rstd;
  long long rows, x_stride, residual_stride;
  int width, wide_params;
  float eps, scale;
  uint32_t below;
};

constexpr int row_threads(int tpr) { return tpr == 32 ? 256 : tpr; }
// CTAs an SM that the registers leave room for: 64 a thread.
constexpr int norm_ctas(int, int tpr) { return 1024 / row_threads(tpr); }

// y = (s - mean) rstd weight + bias, s = residual + dropout(x).  Bound by memory: TPR threads hold a row in registers, L values each, so that every
// array is read or written once; the variance is the mean square of the differences, from the registers too.  Statistics and sums in 32 bits; s is
// normalised as it is there and rounded only where it is stored.
template <class T, int C, bool WIDE, int L, int TPR>
__global__ void __launch_bounds__(row_threads(TPR), norm_ctas(L, TPR)) layer_norm_kernel(NormArgs a) {
  constexpr int V = L / C, kRows = row_threads(TPR) / TPR;
  __shared__ float buf[2][1][32];
  const int at = threadIdx.x % TPR;
  int turn = 0;
  pdl_wait();
  const Random random(a.seed, a.seed != nullptr);
  const float inverse = 1.f / (float)a.width;
  for (long long r = (long long)blockIdx.x * kRows + threadIdx.x / TPR; r < a.rows; r += (long long)gridDim.x * kRows) {
    float s[V][C];
    Values<T, C, WIDE> x[V], t[V];
    const T* const row = static_cast<const T*>(a.x) + r * a.x_stride;
#pragma unroll
    for (int i = 0; i < V; ++i) x[i].load(row, (i * TPR + at) * C, a.width);
    if (a.residual) {
      const T* const residual = static_cast<const T*>(a.residual) + r * a.residual_stride;
#pragma unroll
      for (int i = 0; i < V; ++i) t[i].load(residual, (i * TPR + at) * C, a.width);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) t[i].q.zero();
    }
    float total[1] = {0.f};
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (i * TPR + at) * C;
      float added[C];
      x[i].get(s[i]);
      t[i].get(added);
      if (a.seed) {
        random.drop(s[i], added, c, (uint32_t)r, a.below, a.scale);
      } else {
#pragma unroll
        for (int j = 0; j < C; ++j) s[i][j] += added[j];
      }
      if (a.sum) store_values<T, C, WIDE>(static_cast<T*>(a.sum) + r * a.width, c, a.width, s[i]);
#pragma unroll
      for (int j = 0; j < C; ++j) total[0] += s[i][j];          // beyond the width: zeros
    }
    row_sums<TPR>(total, buf, turn);
    const float mean = total[0] * inverse;
    total[0] = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if ((i * TPR + at) * C < a.width)
#pragma unroll
        for (int j = 0; j < C; ++j) {
          s[i][j] -= mean;
          if (WIDE || (i * TPR + at) * C + j < a.width) total[0] = fmaf(s[i][j], s[i][j], total[0]);
        }
    row_sums<TPR>(total, buf, turn);
    const float rstd = 1.f / sqrtf(fmaf(total[0], inverse, a.eps));
    if (at == 0) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float w[C], b[C];
      const int c = (i * TPR + at) * C;
      load_params<T, C, WIDE>(a.weight, a.wide_params, c, a.width, 1.f, w);
      load_params<T, C, WIDE>(a.bias, a.wide_params, c, a.width, 0.f, b);
#pragma unroll
      for (int j = 0; j < C; ++j) s[i][j] = fmaf(s[i][j] * rstd, w[j], b[j]);
      store_values<T, C, WIDE>(static_cast<T*>(a.y) + r * a.width, c, a.width, s[i]);
    }
  }
}

// Rows beyond what registers hold: the row is read three times, from L2 as a rule.
template <class T, int C, bool WIDE>
__global__ void __launch_bounds__(1024) layer_norm_long_kernel(NormArgs a) {
  __shared__ float buf[2][1][32];
  int turn = 0;
  pdl_wait();
  const Random random(a.seed, a.seed != nullptr);
  const float inverse = 1.f / (float)a.width;
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const auto sum_at = [&](int c, float (&s)[C]) {
      load_values<T, C, WIDE>(static_cast<const T*>(a.x) + r * a.x_stride, c, a.width, s);
      if (a.seed) random.drop(s, c, (uint32_t)r, a.below, a.scale);
      if (a.residual) {
        float t[C];
        load_values<T, C, WIDE>(static_cast<const T*>(a.residual) + r * a.residual_stride, c, a.width, t);
#pragma unroll
        for (int j = 0; j < C; ++j) s[j] += t[j];
      }
    };
    float total[1] = {0.f}, s[C];
    for (int c = threadIdx.x * C; c < a.width; c += 1024 * C) {
      sum_at(c, s);
#pragma unroll
      for (int j = 0; j < C; ++j) total[0] += s[j];
    }
    row_sums<1024>(total, buf, turn);
    const float mean = total[0] * inverse;
    total[0] = 0.f;
    for (int c = threadIdx.x * C; c < a.width; c += 1024 * C) {
      sum_at(c, s);
      if (a.sum) store_values<T, C, WIDE>(static_cast<T*>(a.sum) + r * a.width, c, a.width, s);
#pragma unroll
      for (int j = 0; j < C; ++j)
        if (c + j < a.width) total[0] = fmaf(s[j] - mean, s[j] - mean, total[0]);
    }
    row_sums<1024>(total, buf, turn);
    const float rstd = 1.f / sqrtf(fmaf(total[0], inverse, a.eps));
    if (threadIdx.x == 0) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
    for (int c = threadIdx.x * C; c < a.width; c += 1024 * C) {
      float w[C], b[C];
      sum_at(c, s);
      load_params<T, C, WIDE>(a.weight, a.wide_params, c, a.width, 1.f, w);
      load_params<T, C, WIDE>(a.bias, a.wide_params, c, a.width, 0.f, b);
#pragma unroll
      for (int j = 0; j < C; ++j) s[j] = fmaf((s[j] - mean) * rstd, w[j], b[j]);
      store_values<T, C, WIDE>(static_cast<T*>(a.y) + r * a.width, c, a.width, s);
    }
  }
}

// ---- gradients -----------------------------------------------------------------------------------------------------

struct NormGradArgs {
  const void *dy, *x, *weight, *dsum;
  const float *mean, *rstd;
  const unsigned long long* seed;
  void *dx, *dresidual, *dweight, *dbias;
  float* parts;                        // [CTAs][2][width]: sums of dy n and of dy over a CTA's rows; null: not wanted
  long long rows, dy_stride, x_stride, dsum_stride;
  int width, wide_params;
  float scale;
  uint32_t below;
};

// CTAs an SM, by the registers that the columns' sums leave.
constexpr int norm_grad_ctas_an_sm(int l, int tpr) { return (l == 8 ? 768 : 512) / row_threads(tpr); }

// With n = (x - mean) rstd and g = dy weight:  ds = rstd (g - mean(g) - n mean(g n)) + dsum,  dx = ds through the dropout,  dweight = sum over rows of
// dy n,  dbias = sum of dy.  Bound by memory.  A CTA takes every gridDim-th row (TPR = 32: a warp does) and keeps its columns' sums in registers, so
// that rows are read once; the CTAs' sums meet in a second launch, in the CTAs' order.
template <class T, int C, bool WIDE, int L, int TPR>
__global__ void __launch_bounds__(row_threads(TPR), norm_grad_ctas_an_sm(L, TPR)) layer_norm_backward_kernel(NormGradArgs a) {
  constexpr int V = L / C, kRows = row_threads(TPR) / TPR;
  __shared__ float buf[2][2][32];
  const int at = threadIdx.x % TPR;
  int turn = 0;
  float dw[V][C], db[V][C];
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < C; ++j) dw[i][j] = db[i][j] = 0.f;
  pdl_wait();
  const Random random(a.seed, a.seed != nullptr);
  const float inverse = 1.f / (float)a.width;
  for (long long r = (long long)blockIdx.x * kRows + threadIdx.x / TPR; r < a.rows; r += (long long)gridDim.x * kRows) {
    const float mean = a.mean[r], rstd = a.rstd[r];
    float n[V][C], g[V][C];
    Values<T, C, WIDE> x[V], dy[V], d[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x[i].load(static_cast<const T*>(a.x) + r * a.x_stride, (i * TPR + at) * C, a.width);
      dy[i].load(static_cast<const T*>(a.dy) + r * a.dy_stride, (i * TPR + at) * C, a.width);
    }
    if (a.dsum) {
#pragma unroll
      for (int i = 0; i < V; ++i) d[i].load(static_cast<const T*>(a.dsum) + r * a.dsum_stride, (i * TPR + at) * C, a.width);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) d[i].q.zero();
    }
    float sums[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float w[C];
      load_params<T, C, WIDE>(a.weight, a.wide_params, (i * TPR + at) * C, a.width, 1.f, w);
      x[i].get(n[i]);
      dy[i].get(g[i]);
#pragma unroll
      for (int j = 0; j < C; ++j) {
        n[i][j] = (n[i][j] - mean) * rstd;                 // beyond the width g is 0
        dw[i][j] = fmaf(g[i][j], n[i][j], dw[i][j]);
        db[i][j] += g[i][j];
        g[i][j] *= w[j];
        sums[0] += g[i][j];
        sums[1] = fmaf(g[i][j], n[i][j], sums[1]);
      }
    }
    row_sums<TPR>(sums, buf, turn);
    const float first = -(sums[0] * inverse * rstd), second = -(sums[1] * inverse * rstd);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (i * TPR + at) * C;
      float added[C];
      d[i].get(added);
#pragma unroll
      for (int j = 0; j < C; ++j) g[i][j] = fmaf(n[i][j], second, fmaf(g[i][j], rstd, first)) + added[j];
      store_values<T, C, WIDE>(static_cast<T*>(a.dresidual) + r * a.width, c, a.width, g[i]);
      if (a.seed) {
        random.drop(g[i], c, (uint32_t)r, a.below, a.scale);
        store_values<T, C, WIDE>(static_cast<T*>(a.dx) + r * a.width, c, a.width, g[i]);
      }
    }
  }
  if (!a.parts) return;
  float* const mine = a.parts + (size_t)blockIdx.x * 2 * a.width;
  if constexpr (kRows > 1) {                 // the warps' sums, one after the other
    __shared__ float joined[2][L * 32];
    for (int w = 0; w < kRows; ++w) {
      if ((int)threadIdx.x / TPR == w)
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
          for (int j = 0; j < C; ++j) {
            const int c = (i * TPR + at) * C + j;
            joined[0][c] = w ? joined[0][c] + dw[i][j] : dw[i][j];
            joined[1][c] = w ? joined[1][c] + db[i][j] : db[i][j];
          }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < a.width; c += row_threads(TPR)) {
      mine[c] = joined[0][c];
      mine[a.width + c] = joined[1][c];
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const int c = (i * TPR + at) * C + j;
        if (c < a.width) {
          mine[c] = dw[i][j];
          mine[a.width + c] = db[i][j];
        }
      }
  }
}

// Rows beyond what registers hold: read twice, and the columns' sums by the kernel after this one.
template <class T, int C, bool WIDE>
__global__ void __launch_bounds__(1024) layer_norm_backward_long_kernel(NormGradArgs a) {
  __shared__ float buf[2][2][32];
  int turn = 0;
  pdl_wait();
  const Random random(a.seed, a.seed != nullptr);
  const float inverse = 1.f / (float)a.width;
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const float mean = a.mean[r], rstd = a.rstd[r];
    const auto values_at = [&](int c, float (&n)[C], float (&g)[C]) {
      float w[C];
      load_values<T, C, WIDE>(static_cast<const T*>(a.x) + r * a.x_stride, c, a.width, n);
      load_values<T, C, WIDE>(static_cast<const T*>(a.dy) + r * a.dy_stride, c, a.width, g);
      load_params<T, C, WIDE>(a.weight, a.wide_params, c, a.width, 1.f, w);
#pragma unroll
      for (int j = 0; j < C; ++j) {
        n[j] = c + j < a.width ? (n[j] - mean) * rstd : 0.f;
        g[j] *= w[j];
      }
    };
    float sums[2] = {0.f, 0.f}, n[C], g[C];
    for (int c = threadIdx.x * C; c < a.width; c += 1024 * C) {
      values_at(c, n, g);
#pragma unroll
      for (int j = 0; j < C; ++j) {
        sums[0] += g[j];
        sums[1] = fmaf(g[j], n[j], sums[1]);
      }
    }
    row_sums<1024>(sums, buf, turn);
    const float first = sums[0] * inverse, second = sums[1] * inverse;
    for (int c = threadIdx.x * C; c < a.width; c += 1024 * C) {
      values_at(c, n, g);
#pragma unroll
      for (int j = 0; j < C; ++j) g[j] = rstd * (g[j] - first - n[j] * second);
      if (a.dsum) {
        float d[C];
        load_values<T, C, WIDE>(static_cast<const T*>(a.dsum) + r * a.dsum_stride, c, a.width, d);
#pragma unroll
        for (int j = 0; j < C; ++j) g[j] += d[j];
      }
      store_values<T, C, WIDE>(static_cast<T*>(a.dresidual) + r * a.width, c, a.width, g);
      if (a.seed) {
        random.drop(g, c, (uint32_t)r, a.below, a.scale);
        store_values<T, C, WIDE>(static_cast<T*>(a.dx) + r * a.width, c, a.width, g);
      }
    }
  }
}

// blockIdx.x: 256 C columns, blockIdx.y: every gridDim.y-th row.
template <class T, int C, bool WIDE>
__global__ void __launch_bounds__(256) norm_columns_kernel(NormGradArgs a) {
  const int c = (blockIdx.x * 256 + threadIdx.x) * C;
  float dw[C], db[C];
#pragma unroll
  for (int j = 0; j < C; ++j) dw[j] = db[j] = 0.f;
  pdl_wait();
  if (c >= a.width) return;
  for (long long r = blockIdx.y; r < a.rows; r += gridDim.y) {
    float n[C], g[C];
    const float mean = a.mean[r], rstd = a.rstd[r];
    load_values<T, C, WIDE>(static_cast<const T*>(a.x) + r * a.x_stride, c, a.width, n);
    load_values<T, C, WIDE>(static_cast<const T*>(a.dy) + r * a.dy_stride, c, a.width, g);
#pragma unroll
    for (int j = 0; j < C; ++j) {
      dw[j] = fmaf(g[j], (n[j] - mean) * rstd, dw[j]);
      db[j] += g[j];
    }
  }
  float* const mine = a.parts + (size_t)blockIdx.y * 2 * a.width;
#pragma unroll
  for (int j = 0; j < C; ++j)
    if (c + j < a.width) {
      mine[c + j] = dw[j];
      mine[a.width + c + j] = db[j];
    }
}

// dweight and dbias from the CTAs' sums: a warp's lanes on 32 columns, 32 warps on every 32nd part, joined in the warps' order.
template <class P>
__global__ void __launch_bounds__(1024) norm_finish_kernel(const float* __restrict__ parts, int count, int width, P* __restrict__ dweight, P* __restrict__ dbias) {
  __shared__ float joined[32][33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, columns = 2 * width, c = blockIdx.x * 32 + lane;
  pdl_wait();
  float s = 0.f;
  if (c < columns)
#pragma unroll 4
    for (int p = warp; p < count; p += 32) s += parts[(size_t)p * columns + c];
  joined[warp][lane] = s;
  __syncthreads();
  s = joined[lane][warp];
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int mine = blockIdx.x * 32 + warp;
  if (lane == 0 && mine < columns) {
    if (mine < width) dweight[mine] = from_float<P>(s);
    else dbias[mine - width] = from_float<P>(s);
  }
}

// ---- dropout -------------------------------------------------------------------------------------------------------

struct DropoutArgs {
  const void *x, *residual;
  const unsigned long long* seed;
  void* out;
  long long rows, x_stride, residual_stride;
  int width;
  float scale;
  uint32_t below;
};

// out = residual + x keep / (1 - p).  A thread takes C neighbouring columns at a time of the rows laid end to end, and has the next ones' loads under way.
// Bound by memory, with the multiplier close behind: the generator's 19 products of 64 bits for four values keep it busy for four cycles each.
template <class T, int C, bool WIDE>
__global__ void __launch_bounds__(256, 4) dropout_kernel(DropoutArgs a) {
  pdl_wait();
  const Random random(a.seed, true);
  const int pieces = (a.width + C - 1) / C;
  const long long work = a.rows * pieces, step = (long long)gridDim.x * 256;
  const long long row_step = step / pieces;
  const int piece_step = (int)(step - row_step * pieces);
  long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= work) return;
  long long row = i / pieces;
  int piece = (int)(i - row * pieces);
  Values<T, C, WIDE> x, t;
  const auto load = [&] {
    x.load(static_cast<const T*>(a.x) + row * a.x_stride, piece * C, a.width);
    if (a.residual) t.load(static_cast<const T*>(a.residual) + row * a.residual_stride, piece * C, a.width);
  };
  t.q.zero();
  load();
  for (;;) {
    float v[C], added[C];
    x.get(v);
    t.get(added);
    const long long this_row = row;
    const int c = piece * C;
    i += step;
    row += row_step;
    piece += piece_step;
    if (piece >= pieces) {
      piece -= pieces;
      ++row;
    }
    const bool more = i < work;
    if (more) load();
    random.drop(v, added, c, (uint32_t)this_row, a.below, a.scale);
    store_values<T, C, WIDE>(static_cast<T*>(a.out) + this_row * a.width, c, a.width, v);
    if (!more) break;
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------

constexpr int kNormMost = 16384, kNormGradMost = 8192;          // widths that registers hold

static int row_grid(long long rows, int rows_a_cta, long long most) {
  const long long want = (rows + rows_a_cta - 1) / rows_a_cta;
  return (int)(want < 1 ? 1 : want > most ? most : want);
}

template <class T, int C, bool WIDE>
static int norm_typed(const NormArgs& a, cudaStream_t st) {
  const auto go = [&](auto kernel, int tpr) {
    const int threads = row_threads(tpr);
    return launch_pdl(kernel, row_grid(a.rows, threads / tpr, device_sm_count() * (long long)norm_ctas(0, tpr)), threads, 0, st, a);
  };
  if (a.width <= 512) return go(layer_norm_kernel<T, C, WIDE, 16, 32>, 32);
  if (a.width <= 1024) return go(layer_norm_kernel<T, C, WIDE, 8, 128>, 128);
  if (a.width <= 2048) return go(layer_norm_kernel<T, C, WIDE, 16, 128>, 128);
  if (a.width <= 4096) return go(layer_norm_kernel<T, C, WIDE, 16, 256>, 256);
  if (a.width <= 8192) return go(layer_norm_kernel<T, C, WIDE, 16, 512>, 512);
  if (a.width <= kNormMost) return go(layer_norm_kernel<T, C, WIDE, 16, 1024>, 1024);
  return go(layer_norm_long_kernel<T, C, WIDE>, 1024);
}

// CTAs of the gradients: what an SM holds of them, times the SMs.
static int norm_grad_ctas(long long rows, int width) {
  const int sms = device_sm_count();
  if (width <= 512) return row_grid(rows, 8, sms * norm_grad_ctas_an_sm(16, 32));
  if (width <= 1024) return row_grid(rows, 1, sms * norm_grad_ctas_an_sm(8, 128));
  if (width <= 2048) return row_grid(rows, 1, sms * norm_grad_ctas_an_sm(16, 128));
  if (width <= 4096) return row_grid(rows, 1, sms * norm_grad_ctas_an_sm(16, 256));
  if (width <= kNormGradMost) return row_grid(rows, 1, sms);
  return row_grid(rows, 16, sms);
}

template <class T, int C, bool WIDE>
static int norm_grad_typed(const NormGradArgs& a, cudaStream_t st) {
  const int ctas = norm_grad_ctas(a.rows, a.width);
  const auto go = [&](auto kernel, int threads) { return launch_pdl(kernel, (unsigned)ctas, threads, 0, st, a); };
  int e;
  if (a.width <= 512) e = go(layer_norm_backward_kernel<T, C, WIDE, 16, 32>, 256);
  else if (a.width <= 1024) e = go(layer_norm_backward_kernel<T, C, WIDE, 8, 128>, 128);
  else if (a.width <= 2048) e = go(layer_norm_backward_kernel<T, C, WIDE, 16, 128>, 128);
  else if (a.width <= 4096) e = go(layer_norm_backward_kernel<T, C, WIDE, 16, 256>, 256);
  else if (a.width <= kNormGradMost) e = go(layer_norm_backward_kernel<T, C, WIDE, 16, 512>, 512);
  else {
    e = launch_pdl(layer_norm_backward_long_kernel<T, C, WIDE>, row_grid(a.rows, 1, 1 << 20), 1024, 0, st, a);
    if (e || !a.parts) return e;
    norm_columns_kernel<T, C, WIDE><<<dim3((a.width + 256 * C - 1) / (256 * C), ctas), 256, 0, st>>>(a);
    e = (int)cudaGetLastError();
  }
  if (e || !a.parts) return e;
  const int blocks = (2 * a.width + 31) / 32;
  if (a.wide_params) return launch_pdl(norm_finish_kernel<float>, blocks, 1024, 0, st, (const float*)a.parts, ctas, a.width, static_cast<float*>(a.dweight), static_cast<float*>(a.dbias));
  return launch_pdl(norm_finish_kernel<T>, blocks, 1024, 0, st, (const float*)a.parts, ctas, a.width, static_cast<T*>(a.dweight), static_cast<T*>(a.dbias));
}

template <class T, int C, bool WIDE>
static int dropout_typed(const DropoutArgs& a, cudaStream_t st) {
  return launch_pdl(dropout_kernel<T, C, WIDE>, row_grid(a.rows * ((a.width + C - 1) / C), 256, device_sm_count() * 4ll), 256, 0, st, a);
}

// Accesses of 16 bytes where every row allows them.
static bool wide_rows(int type, long long width, long long stride, const void* p) {
  const int each = 16 / type_bytes(type);
  return !p || (width % each == 0 && stride % each == 0 && aligned16(p));
}

template <class F>
static int by_type(int type, const F& f) {
  switch (type) {
    case FLEXSPMV_TYPE_F32: return f(0.f);
    case FLEXSPMV_TYPE_BF16: return f(__nv_bfloat16());
    default: return f(__half());
  }
}

static uint32_t drop_below(double p) { return (uint32_t)(p * 4294967296.0); }
static float drop_scale(double p) { return (float)(1.0 / (1.0 - p)); }

static int check_rows(const flexspmv_rows_desc* d) {
  if (!d || d->rows < 0 || d->width < 1 || !known_type(d->type) || !(d->p >= 0.0 && d->p < 1.0)) return FLEXSPMV_ERR_BAD_ARG;
  for (int i = 0; i < 3; ++i)
    if (d->stride[i] && d->stride[i] < d->width) return FLEXSPMV_ERR_BAD_ARG;
  if (d->rows > 0x7fffffffLL || d->width > FLEXSPMV_MAX_WIDTH) return FLEXSPMV_ERR_TOO_LARGE;
  return 0;
}
static int check_norm(const flexspmv_rows_desc* d) {
  if (int e = check_rows(d)) return e;
  if ((d->param_type != FLEXSPMV_TYPE_F32 && d->param_type != d->type) || !(d->eps >= 0.f)) return FLEXSPMV_ERR_BAD_ARG;
  return 0;
}
// 0: contiguous
static long long stride_of(const flexspmv_rows_desc* d, int i) { return d->stride[i] ? d->stride[i] : d->width; }

}  // namespace flex

extern "C" {

int flexspmv_layer_norm(const flexspmv_rows_desc* d, const void* const* in, void* const* out, void* stream) {
  using namespace flex;
  if (int e = check_norm(d)) return e;
  if (!in || !out) return FLEXSPMV_ERR_BAD_ARG;
  if (d->rows == 0) return 0;
  if (!in[0] || (d->p > 0.0 && !in[4]) || !out[0] || !out[2] || !out[3]) return FLEXSPMV_ERR_BAD_ARG;
  const int bytes = type_bytes(d->type), param = type_bytes(d->param_type);
  if (!aligned_to(bytes, in[0], in[1], out[0], out[1]) || !aligned_to(param, in[2], in[3]) || !aligned_to(8, in[4]) || !aligned_to(4, out[2], out[3]))
    return FLEXSPMV_ERR_ALIGN;
  const long long xs = stride_of(d, 0), rs = stride_of(d, 1), all = d->rows * d->width * bytes, stats = 4 * d->rows, params = (long long)d->width * param;
  if (!apart({{out[0], all}, {out[1], all}, {out[2], stats}, {out[3], stats}},
             {rows_at(in[0], d->rows, d->width, xs, d->type), rows_at(in[1], d->rows, d->width, rs, d->type), {in[2], params}, {in[3], params},
              {d->p > 0.0 ? in[4] : nullptr, 16}}))
    return FLEXSPMV_ERR_BAD_ARG;
  const NormArgs a = {in[0], in[1], in[2], in[3], d->p > 0.0 ? static_cast<const unsigned long long*>(in[4]) : nullptr, out[0], out[1],
                      static_cast<float*>(out[2]), static_cast<float*>(out[3]), d->rows, xs, rs, (int)d->width, d->param_type == FLEXSPMV_TYPE_F32, d->eps,
                      drop_scale(d->p), drop_below(d->p)};
  const bool wide = wide_rows(d->type, d->width, xs, in[0]) && wide_rows(d->type, d->width, rs, in[1]) && wide_rows(d->type, d->width, d->width, out[0]) &&
                    wide_rows(d->type, d->width, d->width, out[1]) && aligned16(in[2]) && aligned16(in[3]);
  return by_type(d->type, [&](auto zero) {
    using T = decltype(zero);
    return wide ? norm_typed<T, 16 / (int)sizeof(T), true>(a, static_cast<cudaStream_t>(stream)) : norm_typed<T, 4, false>(a, static_cast<cudaStream_t>(stream));
  });
}

int flexspmv_layer_norm_backward_bytes(const flexspmv_rows_desc* d, size_t* bytes) {
  if (!bytes) return FLEXSPMV_ERR_BAD_ARG;
  if (int e = flex::check_norm(d)) return e;
  *bytes = (size_t)flex::norm_grad_ctas(d->rows, (int)d->width) * 2 * d->width * 4;
  return 0;
}

int flexspmv_layer_norm_backward(const flexspmv_rows_desc* d, const void* const* in, void* const* out, void* ws, size_t ws_bytes, void* stream) {
  using namespace flex;
  if (int e = check_norm(d)) return e;
  if (!in || !out || !out[2] != !out[3]) return FLEXSPMV_ERR_BAD_ARG;
  if (d->rows && (!in[0] || !in[1] || !in[3] || !in[4] || (d->p > 0.0 && (!in[6] || !out[0])) || !out[1])) return FLEXSPMV_ERR_BAD_ARG;
  if (d->rows == 0 && !out[2]) return 0;
  const int bytes = type_bytes(d->type), param = type_bytes(d->param_type);
  if (!aligned_to(bytes, in[0], in[1], in[5], out[0], out[1]) || !aligned_to(param, in[2], out[2], out[3]) || !aligned_to(4, in[3], in[4]) || !aligned_to(8, in[6]))
    return FLEXSPMV_ERR_ALIGN;
  const size_t need = (size_t)norm_grad_ctas(d->rows, (int)d->width) * 2 * d->width * 4;
  if (out[2] && (!ws || ws_bytes < need)) return FLEXSPMV_ERR_WORKSPACE;
  if (out[2] && !aligned16(ws)) return FLEXSPMV_ERR_ALIGN;
  const long long ys = stride_of(d, 0), xs = stride_of(d, 1), ds = stride_of(d, 2), all = d->rows * d->width * bytes, stats = 4 * d->rows,
                  params = (long long)d->width * param;
  if (!apart({{d->p > 0.0 ? out[0] : nullptr, all}, {out[1], all}, {out[2], params}, {out[3], params}, {out[2] ? ws : nullptr, (long long)need}},
             {rows_at(in[0], d->rows, d->width, ys, d->type), rows_at(in[1], d->rows, d->width, xs, d->type), {in[2], params}, {in[3], stats}, {in[4], stats},
              rows_at(in[5], d->rows, d->width, ds, d->type), {d->p > 0.0 ? in[6] : nullptr, 16}}))
    return FLEXSPMV_ERR_BAD_ARG;
  const NormGradArgs a = {in[0], in[1], in[2], in[5], static_cast<const float*>(in[3]), static_cast<const float*>(in[4]),
                          d->p > 0.0 ? static_cast<const unsigned long long*>(in[6]) : nullptr, out[0], out[1], out[2], out[3],
                          out[2] ? static_cast<float*>(ws) : nullptr, d->rows, ys, xs, ds, (int)d->width, d->param_type == FLEXSPMV_TYPE_F32, drop_scale(d->p),
                          drop_below(d->p)};
  const bool wide = wide_rows(d->type, d->width, ys, in[0]) && wide_rows(d->type, d->width, xs, in[1]) && wide_rows(d->type, d->width, ds, in[5]) &&
                    wide_rows(d->type, d->width, d->width, d->p > 0.0 ? out[0] : nullptr) && wide_rows(d->type, d->width, d->width, out[1]) && aligned16(in[2]);
  return by_type(d->type, [&](auto zero) {
    using T = decltype(zero);
    return wide ? norm_grad_typed<T, 16 / (int)sizeof(T), true>(a, static_cast<cudaStream_t>(stream))
                : norm_grad_typed<T, 4, false>(a, static_cast<cudaStream_t>(stream));
  });
}

int flexspmv_dropout(const flexspmv_rows_desc* d, const void* const* in, void* const* out, void* stream) {
  using namespace flex;
  if (int e = check_rows(d)) return e;
  if (!in || !out) return FLEXSPMV_ERR_BAD_ARG;
  if (d->rows == 0) return 0;
  if (!in[0] || !in[2] || !out[0]) return FLEXSPMV_ERR_BAD_ARG;
  const int bytes = type_bytes(d->type);
  if (!aligned_to(bytes, in[0], in[1], out[0]) || !aligned_to(8, in[2])) return FLEXSPMV_ERR_ALIGN;
  const long long xs = stride_of(d, 0), rs = stride_of(d, 1);
  if (!apart({{out[0], d->rows * d->width * bytes}},
             {rows_at(in[0], d->rows, d->width, xs, d->type), rows_at(in[1], d->rows, d->width, rs, d->type), {in[2], 16}}))
    return FLEXSPMV_ERR_BAD_ARG;
  const DropoutArgs a = {in[0], in[1], static_cast<const unsigned long long*>(in[2]), out[0], d->rows, xs, rs, (int)d->width, drop_scale(d->p), drop_below(d->p)};
  const bool wide = wide_rows(d->type, d->width, xs, in[0]) && wide_rows(d->type, d->width, rs, in[1]) && wide_rows(d->type, d->width, d->width, out[0]);
  return by_type(d->type, [&](auto zero) {
    using T = decltype(zero);
    return wide ? dropout_typed<T, 16 / (int)sizeof(T), true>(a, static_cast<cudaStream_t>(stream)) : dropout_typed<T, 4, false>(a, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
