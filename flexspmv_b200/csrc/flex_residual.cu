// What stands around a layer on the residual stream: layer norm with the sum (and the dropout) in front of it, its gradients, and dropout.
#include <cuda_runtime.h>

#include <type_traits>

#include "flex_common.cuh"
#include "flex_expert_types.cuh"
#include "flex_umma.cuh"

namespace flex {

int device_sm_count();

// ---- random numbers ------------------------------------------------------------------------------------------------

// The product's two halves.  BY_HAND: not as the language's product, for which the compiler chooses registers differently: us, the gradients of 16384 rows of 4096
// 128 / 157, dropout 65 / 72, the norm 95 / 91.5.
template <bool BY_HAND>
__device__ __forceinline__ void product(uint32_t a, uint32_t b, uint32_t& high, uint32_t& low) {
  if constexpr (BY_HAND) {
    asm("{\n\t.reg .b64 p;\n\tmul.wide.u32 p, %2, %3;\n\tmov.b64 {%1, %0}, p;\n\t}" : "=r"(high), "=r"(low) : "r"(a), "r"(b));
  } else {
    const unsigned long long p = (unsigned long long)a * b;
    high = (uint32_t)(p >> 32);
    low = (uint32_t)p;
  }
}

// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers, as easy as 1, 2, 3; 2011).  Four words for four neighbouring columns of
// a row: counter (column / 4, row, offset), key = seed, so that a value's word goes by its place alone, whatever the launch, the strides or the type,
// and the backward pass makes it again.  19 products of 64 bits for four values, of which the multiplier takes some 50 us for 2^26 values: as long as
// DRAM takes for one array and a half of them in 16 bits.
template <bool BY_HAND = true>
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
      uint32_t a, b, low_a, low_b;
      product<BY_HAND>(c0, 0xD2511F53u, a, low_a);
      product<BY_HAND>(c2, 0xCD9E8D57u, b, low_b);
      c0 = b ^ c1 ^ key0[i];
      c1 = low_b;
      c2 = a ^ c3 ^ key1[i];
      c3 = low_a;
    }
    w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
  }
  // C values from column c (a multiple of four) on: t becomes t plus what is kept of them, scaled.  Not by a choice between the value and 0: a product under
  // a predicate is an instruction less.
  template <int C>
  __device__ __forceinline__ void drop(const float (&v)[C], float (&t)[C], int c, uint32_t row, uint32_t below, float scale) const {
    static_assert(C % 4 == 0, "whole groups");
#pragma unroll
    for (int g = 0; g < C / 4; ++g) {
      uint32_t w[4];
      words((uint32_t)(c / 4 + g), row, w);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (w[j] >= below) t[g * 4 + j] = fmaf(v[g * 4 + j], scale, t[g * 4 + j]);
    }
  }
  template <int C>
  __device__ __forceinline__ void drop(float (&v)[C], int c, uint32_t row, uint32_t below, float scale) const {
    float kept[C];
#pragma unroll
    for (int j = 0; j < C; ++j) kept[j] = 0.f;
    drop(v, kept, c, row, below, scale);
#pragma unroll
    for (int j = 0; j < C; ++j) v[j] = kept[j];
  }
};

// ---- two values an instruction -------------------------------------------------------------------------------------

struct Two {
  float a, b;
  __device__ __forceinline__ Two(float x, float y) : a(x), b(y) {}
  __device__ __forceinline__ explicit Two(float x) : a(x), b(x) {}
  __device__ __forceinline__ explicit Two(const float* p) : a(p[0]), b(p[1]) {}
  __device__ __forceinline__ void put(float* p) const { p[0] = a; p[1] = b; }
};
__device__ __forceinline__ Two operator+(const Two& x, const Two& y) {
  float a, b;
  asm("{\n\t.reg .b64 x, y, r;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 r, x, y;\n\tmov.b64 {%0, %1}, r;\n\t}"
      : "=f"(a), "=f"(b)
      : "f"(x.a), "f"(x.b), "f"(y.a), "f"(y.b));
  return Two(a, b);
}
__device__ __forceinline__ Two operator*(const Two& x, const Two& y) {
  float a, b;
  asm("{\n\t.reg .b64 x, y, r;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 r, x, y;\n\tmov.b64 {%0, %1}, r;\n\t}"
      : "=f"(a), "=f"(b)
      : "f"(x.a), "f"(x.b), "f"(y.a), "f"(y.b));
  return Two(a, b);
}
__device__ __forceinline__ Two fma(const Two& x, const Two& y, const Two& z) {
  float a, b;
  asm("{\n\t.reg .b64 x, y, z, r;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 r, x, y, z;\n\tmov.b64 {%0, %1}, r;\n\t}"
      : "=f"(a), "=f"(b)
      : "f"(x.a), "f"(x.b), "f"(y.a), "f"(y.b), "f"(z.a), "f"(z.b));
  return Two(a, b);
}

// ---- rows ----------------------------------------------------------------------------------------------------------

// C values of a row as they are: neighbouring ones in one access (WIDE: all of them exist or none), or one by one, S columns apart.
template <class T, int C, bool WIDE, int S = 1>
struct Values {
  Pack<T, C> q;
  __device__ __forceinline__ void load(const T* row, int c, int width) {
    if constexpr (WIDE) {
      if (c < width) q.load(row + c);
      else q.zero();
    } else {
#pragma unroll
      for (int j = 0; j < C; ++j) q.v[j] = c + j * S < width ? row[c + j * S] : from_float<T>(0.f);
    }
  }
  __device__ __forceinline__ void get(float (&v)[C]) const {
#pragma unroll
    for (int j = 0; j < C; ++j) v[j] = q.get(j);
  }
};
template <class T, int C, bool WIDE, int S = 1>
__device__ __forceinline__ void load_values(const T* row, int c, int width, float (&v)[C]) {
  Values<T, C, WIDE, S> q;
  q.load(row, c, width);
  q.get(v);
}
template <class T, int C, bool WIDE, int S = 1>
__device__ __forceinline__ void store_values(T* row, int c, int width, const float (&v)[C]) {
  if constexpr (WIDE && sizeof(T) == 2) {          // rounded by two: an instruction, and none to put them together
    static_assert(C % 8 == 0, "16 bytes");
#pragma unroll
    for (int j = 0; j < C; j += 8)
      if (c < width)
        *reinterpret_cast<uint4*>(row + c + j) =
            make_uint4(two_of<T>(v[j], v[j + 1]), two_of<T>(v[j + 2], v[j + 3]), two_of<T>(v[j + 4], v[j + 5]), two_of<T>(v[j + 6], v[j + 7]));
  } else if constexpr (WIDE) {
    Pack<T, C> q;
#pragma unroll
    for (int j = 0; j < C; ++j) q.set(j, v[j]);
    if (c < width) q.store(row + c);
  } else {
#pragma unroll
    for (int j = 0; j < C; ++j)
      if (c + j * S < width) row[c + j * S] = from_float<T>(v[j]);
  }
}
// Weights are 32-bit or of the rows' type; none: `value`.
template <class T, int C, bool WIDE, int S = 1>
__device__ __forceinline__ void load_params(const void* p, bool wide_type, int c, int width, float value, float (&v)[C]) {
  if (!p) {
#pragma unroll
    for (int j = 0; j < C; ++j) v[j] = value;
  } else if (std::is_same<T, float>::value || wide_type) {
    load_values<float, C, WIDE, S>(static_cast<const float*>(p), c, width, v);
  } else {
    load_values<T, C, WIDE, S>(static_cast<const T*>(p), c, width, v);
  }
}

// The columns of a thread that shares a row with TPR - 1 others: V times C of them.  Rows that are not WIDE are accessed value by value, neighbouring threads on
// neighbouring values, but for those that are dropped by four.
constexpr int apart_by(bool wide, bool drop, int tpr) { return wide || drop ? 1 : tpr; }
template <int C, int S, int TPR>
__device__ __forceinline__ int first_column(int i, int at) { return S > 1 ? i * C * TPR + at : (i * TPR + at) * C; }

// Sums over the TPR threads of a row, the same bits in all of them; `barrier`: of the row's threads.  `buf` (of the group) alternates between two halves,
// so that a barrier lies between a half's reading and its next writing.
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*buf)[N][32], int& turn, int barrier) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int o = 16; o; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
  if constexpr (TPR > 32) {
    constexpr int kWarps = TPR / 32;
    const int warp = (threadIdx.x % TPR) >> 5, lane = threadIdx.x & 31;
    if (lane == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) buf[turn][n][warp] = v[n];
    named_bar_sync(barrier, TPR);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if constexpr (kWarps == 2) {
        v[n] = buf[turn][n][0] + buf[turn][n][1];
      } else if constexpr (kWarps <= 8) {      // every thread adds them up, in the same order
        float part[kWarps];
#pragma unroll
        for (int w = 0; w < kWarps; w += 4) {
          const float4 q = *reinterpret_cast<const float4*>(&buf[turn][n][w]);
          part[w] = q.x; part[w + 1] = q.y; part[w + 2] = q.z; part[w + 3] = q.w;
        }
#pragma unroll
        for (int o = kWarps / 2; o; o >>= 1)
#pragma unroll
          for (int w = 0; w < o; ++w) part[w] += part[w + o];
        v[n] = part[0];
      } else {
        v[n] = lane < kWarps ? buf[turn][n][lane] : 0.f;
#pragma unroll
        for (int o = 16; o; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
      }
    }
    turn ^= 1;
  }
}

// 1 / sqrt(x): the approximate one and a step of Newton's method.
__device__ __forceinline__ float inverse_root(float x) {
  const float y = rsqrtf(x), z = fmaf(0.5f * y, fmaf(-x * y, y, 1.f), y);
  return x > 0.f && x < INFINITY ? z : y;
}

// ---- rows ahead ----------------------------------------------------------------------------------------------------

// Many rows: one CTA an SM, its THREADS in groups of TPR, a row each.  A thread's pieces of the rows to come are copied to shared memory, to
// places of its own, so that no register holds them and no barrier is needed for them; PARAMS of weight and bias lie there in 32 bits, which all groups
// share.  What it is for is bytes on their way: us, 16384 rows of 4096 in 16 bits with dropout and sum, loads of each row by itself 131.
constexpr int kSmemAnSm = 226 * 1024;
// `bytes`: 4, or 0 for zeros.
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(__cvta_generic_to_global(src)), "r"(bytes));
}
template <class T, int C, bool WIDE, int S, int L, int TPR, int THREADS, int ARRAYS, int PARAMS>
struct Ahead {
  static constexpr int kGroups = THREADS / TPR, kPieces = L * (int)sizeof(T) / 16, kEach = 16 / (int)sizeof(T);
  static constexpr int kStageBytes = ARRAYS * kPieces * THREADS * 16, kParamBytes = PARAMS * L * TPR * 4;
  static constexpr int kRoom = (kSmemAnSm - kParamBytes - 2048) / kStageBytes, kStages = kRoom > 4 ? 4 : kRoom;
  static constexpr bool kFits = kStages >= 2 && (WIDE || sizeof(T) == 4);          // a copy takes 4 bytes at the least
  static constexpr int kBytes = kParamBytes + kStages * kStageBytes;
  uint32_t params, rows;
  int stage = 0;
  __device__ __forceinline__ explicit Ahead(const void* smem) : params(smem_u32(smem)), rows(smem_u32(smem) + kParamBytes) {}
  __device__ __forceinline__ uint32_t place(int stage, int array, int piece) const {
    return rows + (uint32_t)(stage * kStageBytes + ((array * kPieces + piece) * THREADS + (int)threadIdx.x) * 16);
  }
  __device__ __forceinline__ void copy(int stage, int array, const T* row, int at, int width) const {
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      const int c = first_column<C, S, TPR>(p, at);
      if constexpr (WIDE) {
        copy16(place(stage, array, p), c < width ? row + c : row, c < width ? 16 : 0);
      } else {
#pragma unroll
        for (int j = 0; j < C; ++j) copy4(place(stage, array, p) + j * 4, c + j * S < width ? row + c + j * S : row, c + j * S < width ? 4 : 0);
      }
    }
  }
  // Where the row kStages - 1 ahead goes: it has been read.
  __device__ __forceinline__ int last() const { return stage ? stage - 1 : kStages - 1; }
  static __device__ __forceinline__ void done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory"); }
  template <int V>
  __device__ __forceinline__ void take(int array, Values<T, C, WIDE, S> (&v)[V]) const {
    static_assert(C == kEach, "a piece each");
#pragma unroll
    for (int p = 0; p < V; ++p) {
      uint4& q = v[p].q.raw[0];
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "r"(place(stage, array, p)));
    }
  }
  __device__ __forceinline__ void next() { stage = stage + 1 == kStages ? 0 : stage + 1; }
  // four of a thread's columns behind one another: neighbouring threads in neighbouring banks
  __device__ __forceinline__ uint32_t param_place(int which, int four, int at) const { return params + (uint32_t)(((which * (L / 4) + four) * TPR + at) * 16); }
  __device__ __forceinline__ void put_params(int which, int chunk, int at, const float (&v)[C]) const {
#pragma unroll
    for (int j = 0; j < C; j += 4)
      asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(param_place(which, (chunk * C + j) / 4, at)), "f"(v[j]), "f"(v[j + 1]), "f"(v[j + 2]),
                   "f"(v[j + 3])
                   : "memory");
  }
  __device__ __forceinline__ void get_params(int which, int chunk, int at, float (&v)[C]) const {
#pragma unroll
    for (int j = 0; j < C; j += 4)
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(v[j]), "=f"(v[j + 1]), "=f"(v[j + 2]), "=f"(v[j + 3])
                   : "r"(param_place(which, (chunk * C + j) / 4, at)));
  }
};

constexpr int row_threads(int tpr) { return tpr == 32 ? 256 : tpr; }

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

// Rows whose sum, or whose differences' squares, leave 32 bits: their rstd is 0 or no number.  After all rows, from memory once more, with sums of values that are so much
// smaller that none leaves (less than 2^-149 of them does not show there).  us, 16384 rows of 4096 with dropout and sum, without it 91.3, as a function 91.7, as part of the
// kernel 94.1, where such a row is met 111; elsewhere a function's registers cost more than it saves (4000 rows of 20 000: without 360, part of the kernel 363, function 414).
constexpr float kMostSum = 3.402823466e38f;
template <class T, int TPR>
__device__ __forceinline__ void large_rows(const NormArgs& a, long long from, long long step, int at, float (*buf)[1][32], int& turn, int barrier) {
  constexpr float kSmall = 0x1p-60f, kLarge = 0x1p60f, kSmaller = 0x1p-80f;
  if constexpr (TPR > 32) named_bar_sync(barrier, TPR);
  else __syncwarp();
  const Random<> random(a.seed, a.seed != nullptr);
  const float inverse = 1.f / (float)a.width;
#pragma unroll 1
  for (long long r = from; r < a.rows; r += step) {
    if (a.rstd[r] > 0.f) continue;
    const T* const x = static_cast<const T*>(a.x) + r * a.x_stride;
    const T* const t = a.residual ? static_cast<const T*>(a.residual) + r * a.residual_stride : nullptr;
    const auto sum_at = [&](int c) {
      const float v = to_float(x[c]), s = t ? to_float(t[c]) : 0.f;
      if (!a.seed) return s + v;
      uint32_t w[4];
      random.words((uint32_t)(c / 4), (uint32_t)r, w);
      return (c % 4 == 0 ? w[0] : c % 4 == 1 ? w[1] : c % 4 == 2 ? w[2] : w[3]) >= a.below ? fmaf(v, a.scale, s) : s;
    };
    float total[1] = {0.f};
#pragma unroll 1
    for (int c = at; c < a.width; c += TPR) total[0] = fmaf(sum_at(c), kSmall, total[0]);
    row_sums<TPR>(total, buf, turn, barrier);
    const float mean = total[0] * inverse * kLarge;
    total[0] = 0.f;
#pragma unroll 1
    for (int c = at; c < a.width; c += TPR) {
      const float d = (sum_at(c) - mean) * kSmaller;
      total[0] = fmaf(d, d, total[0]);
    }
    row_sums<TPR>(total, buf, turn, barrier);
    const float rstd = inverse_root(fmaf(total[0], inverse, a.eps * kSmaller * kSmaller)) * kSmaller;
    if (at == 0) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
    const auto param = [&](const void* p, int c, float none) {
      return !p ? none : a.wide_params ? static_cast<const float*>(p)[c] : to_float(static_cast<const T*>(p)[c]);
    };
#pragma unroll 1
    for (int c = at; c < a.width; c += TPR)
      static_cast<T*>(a.y)[r * a.width + c] = from_float<T>(fmaf((sum_at(c) - mean) * rstd, param(a.weight, c, 1.f), param(a.bias, c, 0.f)));
  }
}

template <class T, int TPR>
__device__ __noinline__ void large_rows_apart(const NormArgs& a, long long from, long long step, int at, float (*buf)[1][32], int& turn, int barrier) {
  large_rows<T, TPR>(a, from, step, at, buf, turn, barrier);
}

// y = (s - mean) rstd weight + bias, s = residual + dropout(x).  Bound by memory: TPR threads hold a row in registers, L values each, so that every
// array is read or written once; the variance is the mean square of the differences, from the registers too.  Statistics and sums in 32 bits; s is
// normalised as it is there and rounded only where it is stored.  AHEAD: 0 (a CTA a row, or a warp), or the arrays that are read, whose rows are copied ahead.
constexpr int kAheadThreads = 1024;
template <class T, int C, bool WIDE, int L, int TPR, bool DROP, int AHEAD>
__global__ void __launch_bounds__(AHEAD ? kAheadThreads : row_threads(TPR), AHEAD ? 1 : 1024 / row_threads(TPR)) layer_norm_kernel(const __grid_constant__ NormArgs a) {
  constexpr int S = apart_by(WIDE, DROP, TPR), V = L / C, kThreads = AHEAD ? kAheadThreads : row_threads(TPR), kRows = kThreads / TPR;
  extern __shared__ __align__(16) unsigned char rows_sm[];
  __shared__ __align__(16) float buf[kRows][2][1][32];
  // a barrier for each row; 16 of them take the CTA's own, which is done with before the first row
  const int at = threadIdx.x % TPR, group = threadIdx.x / TPR, barrier = kRows > 15 ? group : 1 + group;
  int turn = 0;
  pdl_wait();
  const Random<!(WIDE && AHEAD > 0)> random(a.seed, DROP);
  const float inverse = 1.f / (float)a.width;
  const long long step = (long long)gridDim.x * kRows, from = (long long)blockIdx.x * kRows + group;
  Ahead<T, C, WIDE, S, L, TPR, kThreads, AHEAD ? AHEAD : 1, 2> next(rows_sm);
  const T *next_x = static_cast<const T*>(a.x) + from * a.x_stride, *next_t = static_cast<const T*>(a.residual) + from * a.residual_stride;
  long long ahead = from;
  const auto copy_next = [&](int to) {
    if (ahead < a.rows) {
      next.copy(to, 0, next_x, at, a.width);
      if (AHEAD == 2) next.copy(to, 1, next_t, at, a.width);
    }
    next.done();
    ahead += step;
    next_x += step * a.x_stride;
    next_t += step * a.residual_stride;
  };
  if constexpr (AHEAD > 0) {
    for (int i = 0; i + 1 < next.kStages; ++i) copy_next(i);
    if (group == 0)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float p[C];
        load_params<T, C, WIDE, S>(a.weight, a.wide_params, first_column<C, S, TPR>(i, at), a.width, 1.f, p);
        next.put_params(0, i, at, p);
        load_params<T, C, WIDE, S>(a.bias, a.wide_params, first_column<C, S, TPR>(i, at), a.width, 0.f, p);
        next.put_params(1, i, at, p);
      }
    __syncthreads();
  }
  bool large = false;
  for (long long r = from; r < a.rows; r += step) {
    float s[V][C];
    Values<T, C, WIDE, S> x[V], t[V];
    const bool sum = AHEAD ? AHEAD == 2 : a.residual != nullptr;
    if constexpr (AHEAD > 0) {
      copy_next(next.last());
      next.wait();
      next.take(0, x);
      if (AHEAD == 2) next.take(1, t);
      next.next();
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) x[i].load(static_cast<const T*>(a.x) + r * a.x_stride, first_column<C, S, TPR>(i, at), a.width);
      if (sum)
#pragma unroll
        for (int i = 0; i < V; ++i) t[i].load(static_cast<const T*>(a.residual) + r * a.residual_stride, first_column<C, S, TPR>(i, at), a.width);
    }
    if (!sum)
#pragma unroll
      for (int i = 0; i < V; ++i) t[i].q.zero();
    Two two(0.f);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = first_column<C, S, TPR>(i, at);
      float v[C];
      x[i].get(v);
      t[i].get(s[i]);
      if (DROP) {
        random.drop(v, s[i], c, (uint32_t)r, a.below, a.scale);
      } else {
#pragma unroll
        for (int j = 0; j < C; j += 2) (Two(s[i] + j) + Two(v + j)).put(s[i] + j);
      }
      if (DROP || sum) store_values<T, C, WIDE, S>(static_cast<T*>(a.sum) + r * a.width, c, a.sum ? a.width : 0, s[i]);
#pragma unroll
      for (int j = 0; j < C; j += 2) two = two + Two(s[i] + j);          // beyond the width: zeros
    }
    float total[1] = {two.a + two.b};
    row_sums<TPR>(total, buf[group], turn, barrier);
    const float mean = total[0] * inverse;
    two = Two(0.f);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (first_column<C, S, TPR>(i, at) < a.width)
#pragma unroll
        for (int j = 0; j < C; j += 2) {
          Two d = Two(s[i] + j) + Two(-mean);
          d.put(s[i] + j);
          if (!WIDE && first_column<C, S, TPR>(i, at) + j * S >= a.width) d.a = 0.f;
          if (!WIDE && first_column<C, S, TPR>(i, at) + (j + 1) * S >= a.width) d.b = 0.f;
          two = fma(d, d, two);
        }
    total[0] = two.a + two.b;
    row_sums<TPR>(total, buf[group], turn, barrier);
    large |= !(total[0] <= kMostSum);
    const float rstd = inverse_root(fmaf(total[0], inverse, a.eps));
    if (at == 0) {
      a.mean[r] = mean;
      a.rstd[r] = rstd;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float w[C], b[C];
      const int c = first_column<C, S, TPR>(i, at);
      if constexpr (AHEAD > 0) {
        next.get_params(0, i, at, w);
        next.get_params(1, i, at, b);
      } else {
        load_params<T, C, WIDE, S>(a.weight, a.wide_params, c, a.width, 1.f, w);
        load_params<T, C, WIDE, S>(a.bias, a.wide_params, c, a.width, 0.f, b);
      }
#pragma unroll
      for (int j = 0; j < C; j += 2) fma(Two(s[i] + j) * Two(rstd), Two(w + j), Two(b + j)).put(s[i] + j);
      store_values<T, C, WIDE, S>(static_cast<T*>(a.y) + r * a.width, c, a.width, s[i]);
    }
  }
  if (large) {
    if constexpr (WIDE && DROP && AHEAD > 0) large_rows_apart<T, TPR>(a, from, step, at, buf[group], turn, barrier);
    else large_rows<T, TPR>(a, from, step, at, buf[group], turn, barrier);
  }
}

// Rows beyond what registers hold: the row is read three times, from L2 as a rule.
template <class T, int C, bool WIDE>
__global__ void __launch_bounds__(1024) layer_norm_long_kernel(NormArgs a) {
  __shared__ __align__(16) float buf[2][1][32];
  int turn = 0;
  pdl_wait();
  const Random<> random(a.seed, a.seed != nullptr);
  const float inverse = 1.f / (float)a.width;
  bool large = false;
  for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const auto sum_at = [&](int c, float (&s)[C]) {
      load_values<T, C, WIDE>(static_cast<const T*>(a.x) + r * a.x_stride, c, a.width, s);
      float t[C];
      if (a.residual) {
        load_values<T, C, WIDE>(static_cast<const T*>(a.residual) + r * a.residual_stride, c, a.width, t);
      } else {
#pragma unroll
        for (int j = 0; j < C; ++j) t[j] = 0.f;
      }
      if (a.seed) {
        random.drop(s, t, c, (uint32_t)r, a.below, a.scale);
#pragma unroll
        for (int j = 0; j < C; ++j) s[j] = t[j];
      } else {
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
    row_sums<1024>(total, buf, turn, 1);
    const float mean = total[0] * inverse;
    total[0] = 0.f;
    for (int c = threadIdx.x * C; c < a.width; c += 1024 * C) {
      sum_at(c, s);
      if (a.sum) store_values<T, C, WIDE>(static_cast<T*>(a.sum) + r * a.width, c, a.width, s);
#pragma unroll
      for (int j = 0; j < C; ++j)
        if (c + j < a.width) total[0] = fmaf(s[j] - mean, s[j] - mean, total[0]);
    }
    row_sums<1024>(total, buf, turn, 1);
    large |= !(total[0] <= kMostSum);
    const float rstd = inverse_root(fmaf(total[0], inverse, a.eps));
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
  if (large) large_rows<T, 1024>(a, blockIdx.x, gridDim.x, threadIdx.x, buf, turn, 1);
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

// With n = (x - mean) rstd and g = dy weight:  ds = rstd (g - mean(g) - n mean(g n)) + dsum,  dx = ds through the dropout,  dweight = sum over rows of
// dy n,  dbias = sum of dy.  Bound by memory.  TPR threads take every so-many-th row and keep its columns' sums in registers (which leave room for 512 threads
// an SM), so that rows are read once; the groups' sums meet in shared memory, the CTAs' in a second launch, each in a fixed order.
constexpr int kAheadGradThreads = 512;
constexpr int norm_grad_threads(int l) { return l == 8 ? 768 : 512; }          // an SM
template <class T, int C, bool WIDE, int L, int TPR, bool DROP, bool AHEAD>
__global__ void __launch_bounds__(AHEAD ? kAheadGradThreads : row_threads(TPR), AHEAD ? 1 : norm_grad_threads(L) / row_threads(TPR))
    layer_norm_backward_kernel(NormGradArgs a) {
  constexpr int S = apart_by(WIDE, DROP, TPR), V = L / C, kThreads = AHEAD ? kAheadGradThreads : row_threads(TPR), kRows = kThreads / TPR;
  extern __shared__ __align__(16) unsigned char rows_sm[];
  __shared__ __align__(16) float buf[kRows][2][2][32];
  static_assert(TPR == 32 || kRows <= 15, "a barrier for each row, beside the CTA's");
  const int at = threadIdx.x % TPR, group = threadIdx.x / TPR, barrier = 1 + group;
  int turn = 0;
  float dw[V][C], db[V][C];
#pragma unroll
  for (int i = 0; i < V; ++i)
#pragma unroll
    for (int j = 0; j < C; ++j) dw[i][j] = db[i][j] = 0.f;
  pdl_wait();
  const Random<> random(a.seed, DROP);
  const float inverse = 1.f / (float)a.width;
  const long long step = (long long)gridDim.x * kRows, from = (long long)blockIdx.x * kRows + group;
  Ahead<T, C, WIDE, S, L, TPR, kThreads, 3, 1> next(rows_sm);
  const T *next_x = static_cast<const T*>(a.x) + from * a.x_stride, *next_y = static_cast<const T*>(a.dy) + from * a.dy_stride,
          *next_d = static_cast<const T*>(a.dsum) + from * a.dsum_stride;
  long long ahead = from;
  const auto copy_next = [&](int to) {
    if (ahead < a.rows) {
      next.copy(to, 0, next_x, at, a.width);
      next.copy(to, 1, next_y, at, a.width);
      if (a.dsum) next.copy(to, 2, next_d, at, a.width);
    }
    next.done();
    ahead += step;
    next_x += step * a.x_stride;
    next_y += step * a.dy_stride;
    next_d += step * a.dsum_stride;
  };
  float next_mean = 0.f, next_rstd = 0.f;
  if (from < a.rows) {
    next_mean = a.mean[from];
    next_rstd = a.rstd[from];
  }
  if constexpr (AHEAD) {
    for (int i = 0; i + 1 < next.kStages; ++i) copy_next(i);
    if (group == 0)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float p[C];
        load_params<T, C, WIDE, S>(a.weight, a.wide_params, first_column<C, S, TPR>(i, at), a.width, 1.f, p);
        next.put_params(0, i, at, p);
      }
    __syncthreads();
  }
  for (long long r = from; r < a.rows; r += step) {
    const float mean = next_mean, rstd = next_rstd;
    if (r + step < a.rows) {
      next_mean = a.mean[r + step];
      next_rstd = a.rstd[r + step];
    }
    float n[V][C], g[V][C];
    Values<T, C, WIDE, S> x[V], dy[V], d[V];
    if constexpr (AHEAD) {
      copy_next(next.last());
      next.wait();
      next.take(0, x);
      next.take(1, dy);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        x[i].load(static_cast<const T*>(a.x) + r * a.x_stride, first_column<C, S, TPR>(i, at), a.width);
        dy[i].load(static_cast<const T*>(a.dy) + r * a.dy_stride, first_column<C, S, TPR>(i, at), a.width);
      }
      if (a.dsum)
#pragma unroll
        for (int i = 0; i < V; ++i) d[i].load(static_cast<const T*>(a.dsum) + r * a.dsum_stride, first_column<C, S, TPR>(i, at), a.width);
    }
    Two one(0.f), two(0.f);
    const bool beyond = !(fabsf(mean * rstd) <= 3.402823466e38f);          // what lies beyond the width would be infinite then, and 0 times that
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float w[C];
      if constexpr (AHEAD) next.get_params(0, i, at, w);
      else load_params<T, C, WIDE, S>(a.weight, a.wide_params, first_column<C, S, TPR>(i, at), a.width, 1.f, w);
      x[i].get(n[i]);
      dy[i].get(g[i]);
      if (beyond)
#pragma unroll
        for (int j = 0; j < C; ++j)
          if (first_column<C, S, TPR>(i, at) + j * S >= a.width) n[i][j] = mean;
#pragma unroll
      for (int j = 0; j < C; j += 2) {
        const Two normed = (Two(n[i] + j) + Two(-mean)) * Two(rstd), y(g[i] + j), scaled = y * Two(w + j);          // beyond the width y is 0
        normed.put(n[i] + j);
        scaled.put(g[i] + j);
        fma(y, normed, Two(dw[i] + j)).put(dw[i] + j);
        (Two(db[i] + j) + y).put(db[i] + j);
        one = one + scaled;
        two = fma(scaled, normed, two);
      }
    }
    float sums[2] = {one.a + one.b, two.a + two.b};
    row_sums<TPR>(sums, buf[group], turn, barrier);
    const float first = -(sums[0] * inverse * rstd), second = -(sums[1] * inverse * rstd);
    if constexpr (AHEAD) {
      if (a.dsum) next.take(2, d);
      next.next();
    }
    if (!a.dsum)
#pragma unroll
      for (int i = 0; i < V; ++i) d[i].q.zero();
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = first_column<C, S, TPR>(i, at);
      float added[C];
      d[i].get(added);
#pragma unroll
      for (int j = 0; j < C; j += 2) (fma(Two(n[i] + j), Two(second), fma(Two(g[i] + j), Two(rstd), Two(first))) + Two(added + j)).put(g[i] + j);
      store_values<T, C, WIDE, S>(static_cast<T*>(a.dresidual) + r * a.width, c, a.width, g[i]);
      if (DROP) {
        random.drop(g[i], c, (uint32_t)r, a.below, a.scale);
        store_values<T, C, WIDE, S>(static_cast<T*>(a.dx) + r * a.width, c, a.width, g[i]);
      }
    }
  }
  if (!a.parts) return;
  float* const mine = a.parts + (size_t)blockIdx.x * 2 * a.width;
  if constexpr (kRows > 1) {                 // the groups' sums, one after the other, over the stages
    float* const joined = reinterpret_cast<float*>(rows_sm);
    copy16_wait_all();
    __syncthreads();
    for (int w = 0; w < kRows; ++w) {
      if (group == w)
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
          for (int j = 0; j < C; ++j) {
            const int c = first_column<C, S, TPR>(i, at) + j * S;
            joined[c] = w ? joined[c] + dw[i][j] : dw[i][j];
            joined[L * TPR + c] = w ? joined[L * TPR + c] + db[i][j] : db[i][j];
          }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < a.width; c += kThreads) {
      mine[c] = joined[c];
      mine[a.width + c] = joined[L * TPR + c];
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const int c = first_column<C, S, TPR>(i, at) + j * S;
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
  __shared__ __align__(16) float buf[2][2][32];
  int turn = 0;
  pdl_wait();
  const Random<> random(a.seed, a.seed != nullptr);
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
    row_sums<1024>(sums, buf, turn, 1);
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
// Bound by memory (2^26 values in 16 bits and as many added: 6.26 TB/s), with the generator close behind, which is why C is 32 bytes where the width allows: what a
// thread does for a place and not for a value is shared by twice as many (64.4 us, with 16 bytes 80.6).
template <class T, int C, bool WIDE>
__global__ void __launch_bounds__(256, 4) dropout_kernel(DropoutArgs a) {
  pdl_wait();
  const Random<> random(a.seed, true);
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
    store_values<T, C, WIDE>(static_cast<T*>(a.out) + this_row * a.width, c, a.width, added);
    if (!more) break;
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------

constexpr int kNormMost = 16384, kNormGradMost = 8192;          // widths that registers hold

static int row_grid(long long rows, int rows_a_cta, long long most) {
  const long long want = (rows + rows_a_cta - 1) / rows_a_cta;
  return (int)(want < 1 ? 1 : want > most ? most : want);
}

// Rows are copied ahead where each group of an SM has some to copy.  us, norm, by itself / ahead: 300 rows of 4096 3.8 / 4.8, 1200 10.5 / 10.7, 2000 14.8 / 13.1;
// gradients, whose CTAs leave fewer sums that way: 64 rows of 1000 5.3 / 8.8, 300 of 4096 18.1 / 10.8, 2000 of 1024 17.0 / 10.6, but a warp a row 500 of 256 8.0 / 12.6.
static bool many_rows(long long rows, int groups) { return rows >= 2ll * groups * device_sm_count(); }
static bool many_grad_rows(long long rows, int groups, int tpr) { return tpr > 32 ? 2 * rows >= (long long)groups * device_sm_count() : many_rows(rows, groups); }

template <class T, int C, bool WIDE, int L, int TPR, bool DROP>
static int norm_launch(const NormArgs& a, cudaStream_t st) {
  constexpr int S = apart_by(WIDE, DROP, TPR);
  const auto ahead = [&](auto arrays) {
    using Next = Ahead<T, C, WIDE, S, L, TPR, kAheadThreads, decltype(arrays)::value, 2>;
    constexpr auto kernel = layer_norm_kernel<T, C, WIDE, L, TPR, DROP, decltype(arrays)::value>;
    if (int e = allow_smem<kernel>(Next::kBytes)) return e;
    return launch_pdl(kernel, row_grid(a.rows, Next::kGroups, device_sm_count()), kAheadThreads, Next::kBytes, st, a);
  };
  if constexpr (Ahead<T, C, WIDE, S, L, TPR, kAheadThreads, 2, 2>::kFits)
    if (many_rows(a.rows, kAheadThreads / TPR)) return a.residual ? ahead(std::integral_constant<int, 2>()) : ahead(std::integral_constant<int, 1>());
  constexpr int kThreads = row_threads(TPR);
  return launch_pdl(layer_norm_kernel<T, C, WIDE, L, TPR, DROP, 0>, row_grid(a.rows, kThreads / TPR, device_sm_count() * (1024ll / kThreads)), kThreads, 0, st, a);
}

template <class T, int C, bool WIDE, bool DROP>
static int norm_typed(const NormArgs& a, cudaStream_t st) {
  if (a.width <= 256) return norm_launch<T, C, WIDE, 8, 32, DROP>(a, st);
  if constexpr (sizeof(T) == 2)
    if (a.width <= 512) return norm_launch<T, C, WIDE, 16, 32, DROP>(a, st);
  // Two warps a row where the generator is what costs: us, 40 000 rows of 768, 128 threads / 64: with dropout 65.7 / 55.6, without 40.1 / 46.8.
  if constexpr (sizeof(T) == 2 && WIDE && DROP)
    if (a.width <= 1024) return norm_launch<T, C, WIDE, 16, 64, DROP>(a, st);
  if (a.width <= 1024) return norm_launch<T, C, WIDE, 8, 128, DROP>(a, st);
  // 16 values a thread where they are of 16 bits, else 8: as many bytes
  constexpr int L = (int)sizeof(T) == 2 ? 16 : 8;
  if (a.width <= 128 * L) return norm_launch<T, C, WIDE, L, 128, DROP>(a, st);
  if (a.width <= 256 * L) return norm_launch<T, C, WIDE, L, 256, DROP>(a, st);
  if (a.width <= 512 * L) return norm_launch<T, C, WIDE, L, 512, DROP>(a, st);
  if (a.width <= 1024 * L) return norm_launch<T, C, WIDE, L, 1024, DROP>(a, st);
  if (a.width <= kNormMost) return norm_launch<T, C, WIDE, 16, 1024, DROP>(a, st);
  return launch_pdl(layer_norm_long_kernel<T, C, WIDE>, row_grid(a.rows, 1, 1 << 20), 1024, 0, st, a);
}

// CTAs that may leave sums of their rows, of any variant.
static int norm_grad_ctas(long long rows, int width) {
  const int sms = device_sm_count();
  if (width <= 512) return row_grid(rows, 8, sms * 2);
  if (width <= 1024) return row_grid(rows, 1, sms * 6);
  if (width <= 2048) return row_grid(rows, 1, sms * 4);
  if (width <= 4096) return row_grid(rows, 1, sms * 2);
  if (width <= kNormGradMost) return row_grid(rows, 1, sms);
  return row_grid(rows, 16, sms);
}

template <class T, int C, bool WIDE, int L, int TPR, bool DROP>
static int norm_grad_launch(const NormGradArgs& a, int& ctas, cudaStream_t st) {
  using Next = Ahead<T, C, WIDE, apart_by(WIDE, DROP, TPR), L, TPR, kAheadGradThreads, 3, 1>;
  if constexpr (Next::kFits) {
    static_assert(Next::kBytes >= 8 * L * TPR, "the groups' sums lie over the stages");
    if (many_grad_rows(a.rows, Next::kGroups, TPR)) {
      constexpr auto kernel = layer_norm_backward_kernel<T, C, WIDE, L, TPR, DROP, true>;
      if (int e = allow_smem<kernel>(Next::kBytes)) return e;
      ctas = row_grid(a.rows, Next::kGroups, device_sm_count());
      return launch_pdl(kernel, (unsigned)ctas, kAheadGradThreads, Next::kBytes, st, a);
    }
  }
  constexpr int kThreads = row_threads(TPR);
  return launch_pdl(layer_norm_backward_kernel<T, C, WIDE, L, TPR, DROP, false>, (unsigned)ctas, kThreads, kThreads > TPR ? 8 * L * TPR : 0, st, a);
}

template <class T, int C, bool WIDE, bool DROP>
static int norm_grad_typed(const NormGradArgs& a, cudaStream_t st) {
  int ctas = norm_grad_ctas(a.rows, a.width), e;
  if (a.width <= 512) e = norm_grad_launch<T, C, WIDE, 16, 32, DROP>(a, ctas, st);
  // us, 40 000 rows of 768, 128 threads a row / 64: with dropout 83.5 / 75.5, without 58.1 / 49.6
  else if (sizeof(T) == 2 && WIDE && a.width <= 1024) e = norm_grad_launch<T, C, WIDE, 16, 64, DROP>(a, ctas, st);
  else if (a.width <= 1024) e = norm_grad_launch<T, C, WIDE, 8, 128, DROP>(a, ctas, st);
  else if (a.width <= 2048) e = norm_grad_launch<T, C, WIDE, 16, 128, DROP>(a, ctas, st);
  else if (a.width <= 4096) e = norm_grad_launch<T, C, WIDE, 16, 256, DROP>(a, ctas, st);
  else if (a.width <= kNormGradMost) e = norm_grad_launch<T, C, WIDE, 16, 512, DROP>(a, ctas, st);
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
    const auto go = [&](auto drop) {
      constexpr bool kDrop = decltype(drop)::value;
      return wide ? norm_typed<T, 16 / (int)sizeof(T), true, kDrop>(a, static_cast<cudaStream_t>(stream)) : norm_typed<T, 4, false, kDrop>(a, static_cast<cudaStream_t>(stream));
    };
    return a.seed ? go(std::true_type()) : go(std::false_type());
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
    const auto go = [&](auto drop) {
      constexpr bool kDrop = decltype(drop)::value;
      return wide ? norm_grad_typed<T, 16 / (int)sizeof(T), true, kDrop>(a, static_cast<cudaStream_t>(stream))
                  : norm_grad_typed<T, 4, false, kDrop>(a, static_cast<cudaStream_t>(stream));
    };
    return a.seed ? go(std::true_type()) : go(std::false_type());
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
    if (wide && d->width % (32 / (int)sizeof(T)) == 0) return dropout_typed<T, 32 / (int)sizeof(T), true>(a, static_cast<cudaStream_t>(stream));
    return wide ? dropout_typed<T, 16 / (int)sizeof(T), true>(a, static_cast<cudaStream_t>(stream)) : dropout_typed<T, 4, false>(a, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
