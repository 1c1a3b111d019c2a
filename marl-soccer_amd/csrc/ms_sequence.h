// ms_sequence.h — what the sequence kernels (ms_conv.hip, ms_scan.hip) share: element types, vector
// loads with guarded ends, the activations, and the error text of their entry points.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/marl_soccer.h"

extern thread_local char g_sequence_error[256];  // ms_conv.hip

namespace seq {

// Element types of the [io] arrays: the value is float32 in registers, rounded to nearest even
// (v_cvt_pk_bf16_f32, v_cvt_f16_f32) when it is stored.
typedef __bf16 bf16;
typedef _Float16 f16;

template <typename T, int E>
struct Vec {
  // 16 B at most are assumed aligned: wider vectors are moved as several 16-B accesses
  typedef T type __attribute__((ext_vector_type(E), aligned(sizeof(T) * E < 16 ? sizeof(T) * E : 16)));
};

// E channels from p, of which the first n (<= E) exist; `vec`: p is aligned for Vec<T, E>
template <typename T, int E>
__device__ __forceinline__ typename Vec<T, E>::type load(const T* p, int n, bool vec) {
  typename Vec<T, E>::type v;
  if (vec && n >= E) {
    v = *(const typename Vec<T, E>::type*)p;
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = i < n ? p[i] : (T)0.0f;
  }
  return v;
}
template <typename T, int E>
__device__ __forceinline__ typename Vec<T, E>::type load(const T* p) {  // all of them, aligned
  return *(const typename Vec<T, E>::type*)p;
}
template <typename T, int E>
__device__ __forceinline__ void store(T* p, const float (&x)[E]) {
  typename Vec<T, E>::type v;
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] = (T)x[i];
  *(typename Vec<T, E>::type*)p = v;
}
template <typename T, int E>
__device__ __forceinline__ void store(T* p, const float (&x)[E], int n, bool vec) {
  if (vec && n >= E) {
    typename Vec<T, E>::type v;
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = (T)x[i];
    *(typename Vec<T, E>::type*)p = v;
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (i < n) p[i] = (T)x[i];
  }
}

// 1 / (1 + exp(-x)) and its product with x. v_exp_f32's argument is rounded, which costs |x| 2^-24 of
// exp: less than a unit in the last place of the result where it is not small. Below x = -87.3 the
// result would be subnormal and is 0, and so are the product, off by at most 89 x 2^-126 there, and the
// slope: exp may pass to infinity, whose reciprocal is 0 (holding the argument at 126 left 2^-126, which a
// large x makes large again: silu(-3e38) was -3.5).
__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504f));
}
__device__ __forceinline__ float silu(float x) { return x * sigmoid(x); }
__device__ __forceinline__ float silu_slope(float x) {
  const float s = sigmoid(x);
  return s * (1.0f + x * (1.0f - s));
}
// log(1 + exp(x)) = max(x, 0) + log1p(e), e = exp(-|x|), and its slope, the logistic function of x.
// exp carries the rounding of its argument along (a state's decay feels it at every step). log1p(e) =
// 2 atanh(s), s = e / (2 + e) <= 1/3, by a polynomial in s^2 fitted on Chebyshev nodes, exact to
// 2^-25 of the value for small e too, where log(1 + e) would lose e's digits. A NaN stays one.
__device__ __forceinline__ float softplus(float x, float& slope) {
  const float y = fminf(__builtin_fabsf(x), 87.0f), hi = y * -1.44269504f;
  const float lo = __builtin_fmaf(y, -1.92596299e-8f, __builtin_fmaf(y, -1.44269504f, -hi));
  float e = __builtin_amdgcn_exp2f(hi);
  e = __builtin_fmaf(e * 0.69314718f, lo, e);
  const float s = e * __builtin_amdgcn_rcpf(2.0f + e), q = s * s;
  float p = 0.134337768f;
  p = __builtin_fmaf(p, q, 0.141169772f);
  p = __builtin_fmaf(p, q, 0.200038359f);
  p = __builtin_fmaf(p, q, 0.333333194f);
  p = __builtin_fmaf(p * q, s, s);
  const float r = __builtin_amdgcn_rcpf(1.0f + e);
  slope = x < 0.0f ? e * r : r;
  return __builtin_fmaf(2.0f, p, x < 0.0f ? 0.0f : x);
}

inline bool aligned(const void* p, int64_t a, int64_t b, int64_t elem, int64_t vec) {
  // every row of an array with element strides a and b starts on a multiple of `vec` elements, 16 B at most
  const int64_t bytes = vec * elem < 16 ? vec * elem : 16;
  const int64_t unit = bytes / elem;
  return ((uintptr_t)p % (uint64_t)bytes) == 0 && a % unit == 0 && b % unit == 0;
}

// A launch's threads are counted in 32 bits: past them the runtime cuts the grid without an error
inline bool too_many(int64_t blocks, int64_t threads) { return blocks > 0xffffffffll / threads; }

inline int fail(int code, const char* who, const char* why) {
  snprintf(g_sequence_error, sizeof(g_sequence_error), "%s: %s", who, why);
  return code;
}
inline int launched(const char* who) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MS_OK : fail(MS_ERR_HIP, who, hipGetErrorString(e));
}

// Row sums of partial results: out[y][c] = sum of in[i][c] over the y-th share of the parts, in a fixed
// order. A block owns 64 columns and its waves share the parts of its share; the sum is held in
// float64, so the number of parts does not cost precision.
template <int WAVES>
__device__ __forceinline__ double sum_share(const float* __restrict__ in, int64_t first, int64_t last, int64_t columns,
                                            int64_t c, double (&s)[WAVES][64]) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  constexpr int AHEAD = 8;  // loads in flight
  double x[AHEAD] = {};
  if (c < columns) {
    int64_t i = first + w;
    for (; i + (AHEAD - 1) * WAVES < last; i += AHEAD * WAVES)
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) x[k] += in[(i + k * WAVES) * columns + c];
    for (; i < last; i += WAVES) x[0] += in[i * columns + c];
  }
  s[w][lane] = ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
  __syncthreads();
  double a = 0.0;
  if (w == 0)
#pragma unroll
    for (int k = 0; k < WAVES; ++k) a += s[k][lane];
  return a;  // the first wave's lanes hold the sums
}
template <int WAVES>
__global__ __launch_bounds__(64 * WAVES) void sum_parts(const float* __restrict__ in, int64_t parts, int64_t share,
                                                        int64_t columns, float* __restrict__ out) {
  __shared__ double s[WAVES][64];
  const int64_t c = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63), first = blockIdx.y * share;
  const double a = sum_share<WAVES>(in, first, first + share < parts ? first + share : parts, columns, c, s);
  if (threadIdx.x < 64 && c < columns) out[blockIdx.y * columns + c] = (float)a;
}

}  // namespace seq
