// ms_optim.hip — AdamW over a list of tensors, and the gradients' norm that clips them (gfx950).
//
// Bound by HBM: p, m and v read and written, g read (28 B a value in float32, 16 B with moments in
// 8 bits), some 30 operations between. The list travels in the kernel's arguments (48 tensors of 72 B),
// so a step is one launch whatever the tensors' sizes, needs no table in memory, and a captured graph
// holds its own copy. A block finds its tensor from the running block counts, 4 values a thread and
// round. A short list of small tensors (a policy's) is cut finer than a long one, to fill the chip.
// 201 M values in 8 bits, clipped: 0.78 ms a call, 5.2 TB/s with the norm's read of g (rounded to nearest
// or stochastically alike), in 32 bits 1.25 ms, 5.2 TB/s; the Agent's 423 k
// values: 10 us for the norm and 10 for the step, which is a launch and a chain of two dependent reads.
//
// Step counts stay on the device, one a tensor: every block reads its tensor's count before it takes
// a ticket, and the block with the last ticket raises the counts, so no second launch is needed.
// The clip factor comes from a launch before: each block leaves its part of the norm in float64, and
// the last one adds them in order.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/marl_soccer.h"

static thread_local char g_optim_error[256] = "";

namespace opt {

constexpr int THREADS = 256, E = 4, ROUND = THREADS * E;  // values a block handles at a time
constexpr int LIST = MS_OPTIM_TENSORS;
constexpr int64_t NORM_BLOCKS = 1024;
static_assert(ROUND % MS_ADAMW_BLOCK == 0 && MS_ADAMW_BLOCK == 64 * E, "a wave's round is one scale block");

typedef __bf16 bf16;
typedef _Float16 f16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x4 __attribute__((ext_vector_type(4)));

// the workspace: [0] clip factor, [1] ticket, [2] ticket of the norm, [4..5] the norm's running sum
// (float64), [64..] the blocks' parts (float64)
struct Ws {
  float* f;
  __device__ unsigned* ticket() const { return (unsigned*)f + 1; }
  __device__ unsigned* norm_ticket() const { return (unsigned*)f + 2; }
  __device__ double* total() const { return (double*)(f + 4); }
  __device__ double* parts() const { return (double*)(f + 64); }
};
static_assert(64 + 2 * NORM_BLOCKS <= MS_OPTIM_WORKSPACE, "parts fit the workspace");

struct List {
  ms_optim_tensor t[LIST];
  uint32_t end[LIST];  // blocks up to and including tensor i's
  int32_t count, rounds;  // rounds of ROUND values a block
};
struct NormList {
  const void* grad[LIST];
  int64_t numel[LIST];
  uint32_t end[LIST];
  int32_t dtype[LIST];
  int32_t count, rounds, first, last;
  uint32_t blocks;
};
struct Hyper {
  double lr, beta1, beta2;
  float b1, b2, c1, c2, eps;  // c: 1 - beta
  double weight_decay;
  const float* lr_device;
  int use_clip;
};

template <typename T4, typename T>
__device__ __forceinline__ f32x4 get4(const T* p, int64_t i, int64_t n, bool vec) {
  if (vec && i + 4 <= n) return __builtin_convertvector(*(const T4*)(p + i), f32x4);
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (i + k < n) v[k] = (float)p[i + k];
  return v;
}
template <typename T4, typename T>
__device__ __forceinline__ void put4(T* p, int64_t i, int64_t n, bool vec, f32x4 v) {
  if (vec && i + 4 <= n) {
    *(T4*)(p + i) = __builtin_convertvector(v, T4);
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (i + k < n) p[i + k] = (T)v[k];
}
__device__ __forceinline__ f32x4 get_any(const void* p, int dtype, int64_t i, int64_t n, bool vec) {
  if (dtype == 0) return get4<f32x4>((const float*)p, i, n, vec);
  if (dtype == 1) return get4<bf16x4>((const bf16*)p, i, n, vec);
  return get4<f16x4>((const f16*)p, i, n, vec);
}
__device__ __forceinline__ void put_any(void* p, int dtype, int64_t i, int64_t n, bool vec, f32x4 v) {
  if (dtype == 0) put4<f32x4>((float*)p, i, n, vec, v);
  else if (dtype == 1) put4<bf16x4>((bf16*)p, i, n, vec, v);
  else put4<f16x4>((f16*)p, i, n, vec, v);
}

// OCP e4m3 codes, four in a dword: rounded to nearest even by the hardware's conversions, or to one of the
// two neighbours with the odds that keep the expected value. For these v_cvt_sr_fp8_f32 adds the upper 20
// bits of `odds` to what e4m3 has no bits for and cuts (checked against that on the card, subnormals too);
// 16 random bits will do: the last four stay 0, so that 448 and a unit in the last place is not carried to
// the code after it, which is no number.
__device__ __forceinline__ uint32_t encode(f32x4 v) {
  int c = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], c, true);
}
struct Odds {
  uint32_t h[2];  // 16 bits for each of four values
};
__device__ __forceinline__ uint32_t encode(f32x4 v, Odds o) {
  int c = __builtin_amdgcn_cvt_sr_fp8_f32(v[0], (int)(o.h[0] & 0xffff0000u), 0, 0);
  c = __builtin_amdgcn_cvt_sr_fp8_f32(v[1], (int)(o.h[0] << 16), c, 1);
  c = __builtin_amdgcn_cvt_sr_fp8_f32(v[2], (int)(o.h[1] & 0xffff0000u), c, 2);
  return (uint32_t)__builtin_amdgcn_cvt_sr_fp8_f32(v[3], (int)(o.h[1] << 16), c, 3);
}
// A hash of a tensor's step count (one key a block) and of where in it four values lie, so that a step
// repeats bit for bit: multiplications by odd constants and shifted xors (the constants: the golden ratio,
// the roots of 2, 3, 5 and 7 in 32 bits).
__device__ __forceinline__ uint32_t key_of(int64_t t) {
  uint32_t x = (uint32_t)t * 0x9E3779B9u + (uint32_t)(t >> 32) * 0x6A09E667u;
  x = (x ^ x >> 15) * 0xBB67AE85u;
  return x ^ x >> 13;
}
__device__ __forceinline__ Odds odds_of(int64_t i, uint32_t key) {
  uint32_t x = (uint32_t)(i / E) * 0x9E3779B9u + (uint32_t)((i / E) >> 32) * 0x6A09E667u + key;
  x = (x ^ x >> 16) * 0xBB67AE85u;
  x = (x ^ x >> 15) * 0x3C6EF373u;
  x ^= x >> 16;
  const uint32_t y = x * 0xA54FF53Bu;
  return {{x, y ^ y >> 15}};
}
__device__ __forceinline__ f32x4 decode(uint32_t c) {
  f32x4 v;
  v[0] = __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
  v[1] = __builtin_amdgcn_cvt_f32_fp8((int)c, 1);
  v[2] = __builtin_amdgcn_cvt_f32_fp8((int)c, 2);
  v[3] = __builtin_amdgcn_cvt_f32_fp8((int)c, 3);
  return v;
}
__device__ __forceinline__ uint32_t get_codes(const uint8_t* p, int64_t i, int64_t n, bool vec) {
  if (vec && i + 4 <= n) return *(const uint32_t*)(p + i);
  uint32_t c = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (i + k < n) c |= (uint32_t)p[i + k] << (8 * k);
  return c;
}
__device__ __forceinline__ void put_codes(uint8_t* p, int64_t i, int64_t n, bool vec, uint32_t c) {
  if (vec && i + 4 <= n) {
    *(uint32_t*)(p + i) = c;
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (i + k < n) p[i + k] = (uint8_t)(c >> (8 * k));
}

// the largest of the wave's values, in every lane: within rows of 16 by DPP, across them by swaps
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
template <int CTRL>
__device__ __forceinline__ float max_dpp(float x) {
  return fmaxf(x, __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xf, 0xf, false)));
}
__device__ __forceinline__ float wave_max(float x) {
  x = max_dpp<0x128>(x);  // row_ror:8, 4, 2, 1
  x = max_dpp<0x124>(x);
  x = max_dpp<0x122>(x);
  x = max_dpp<0x121>(x);
  const u32x2 a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const unsigned a0 = a.x, a1 = a.y;
  x = fmaxf(__uint_as_float(a0), __uint_as_float(a1));
  const u32x2 b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const unsigned b0 = b.x, b1 = b.y;
  return fmaxf(__uint_as_float(b0), __uint_as_float(b1));
}

// Eight bits for a moment: a wave's 256 values share the scale max|.| / 448, so the largest is held
// to a unit in the last place of float32 and the others to steps of e4m3, 2^-4 to 2^-3 of the value, down
// to 2^-14.8 of the largest (2^-6 of the scale), and to 2^-9 of the scale below that. The second moment
// is held as its root, which halves the range it spans. Blocks under 2^-100 are held as zeros, where the
// scale's inverse would overflow.
// Rounded to nearest, a step's change of less than half a unit of the codes is lost for good, and with
// beta2 = 0.999 a root moves by some 0.05 % a step: then only the largest moves, by the scale, and the others
// follow it (roots 0.3 to 9 times the 32-bit ones after thousands of steps whose gradients change in
// size). SR keeps such changes in the mean: each rounding is right in expectation, and the held root
// wanders about the 32-bit one, by some 17 % of it at beta2 = 0.999. ROOT: the second moment's, which is
// not rounded down to nothing: the next step without a gradient would divide the first moment by it (values
// of 1e-5 of their block's largest took steps of 400 lr, in either rounding).
template <bool SR, bool ROOT>
__device__ __forceinline__ uint32_t quantise(f32x4 v, float* scale, bool first_lane, Odds odds) {
  float top = 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k) top = fmaxf(top, __builtin_fabsf(v[k]));
  top = wave_max(top);
  if (top > 3.4028234663852886e38f) {  // an infinite one is held as no number, by itself: the scale is the others'
    top = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) top = __builtin_isinf(v[k]) ? top : fmaxf(top, __builtin_fabsf(v[k]));
    top = wave_max(top);
  }
  const bool some = top >= 7.8886090522101181e-31f;
  const float inv = some ? 448.0f / top : 0.0f;
  if (first_lane) *scale = some ? top / 448.0f : 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float x = v[k];
    v[k] = x * inv;
    if constexpr (ROOT) v[k] = v[k] < 0x1p-9f && x > 0.0f ? 0x1p-9f : v[k];
  }
  if constexpr (SR) return encode(v, odds);
  else return encode(v);
}

__device__ __forceinline__ bool aligned(const void* p, int bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }

// b^t by squaring, in float64: off by about t 2^-53 of itself, far below the float32 it ends in
__device__ __forceinline__ double power(double b, int64_t t) {
  double p = 1.0;
  for (; t > 0; t >>= 1) {
    if (t & 1) p *= b;
    b *= b;
  }
  return p;
}

// What all of a tensor's blocks share: the step size and the root's factor of step t
struct Factors {
  float fix1, fix2, keep, clip;
  uint32_t key;
};

struct Moments {
  f32x4 m, v;
};

template <int BITS, bool SR>
__global__ __launch_bounds__(THREADS) void adamw(const List list, const Hyper hp, const Ws ws) {
  __shared__ Factors shared;
  // this block's tensor: as many as end at or before it come before it (the last end is the grid's size)
  const int lane = threadIdx.x & 63;
  const int k = __popcll(__ballot(lane < list.count && blockIdx.x >= list.end[lane]));
  const ms_optim_tensor& a = list.t[k];
  const int64_t block = blockIdx.x - (k ? list.end[k - 1] : 0), n = a.numel;
  const int dtype = a.dtype, size = dtype == 0 ? 16 : 8;
  const bool vp = aligned(a.param, size), vg = aligned(a.grad, size);
  const bool vs = BITS == 32 ? aligned(a.exp_avg, 16) && aligned(a.exp_avg_sq, 16)
                             : aligned(a.exp_avg, 4) && aligned(a.exp_avg_sq, 4);
  const int64_t begin = block * list.rounds * ROUND + threadIdx.x * E;
  f32x4 p, g;
  Moments s;
  float ms = 0.0f, vs8 = 0.0f;
  uint32_t mc = 0, vc = 0;
  auto fetch = [&](int64_t i) __attribute__((always_inline)) {
    p = get_any(a.param, dtype, i, n, vp);
    g = get_any(a.grad, dtype, i, n, vg);
    if constexpr (BITS == 32) {
      s.m = get4<f32x4>((const float*)a.exp_avg, i, n, vs);
      s.v = get4<f32x4>((const float*)a.exp_avg_sq, i, n, vs);
    } else {
      mc = get_codes((const uint8_t*)a.exp_avg, i, n, vs);
      vc = get_codes((const uint8_t*)a.exp_avg_sq, i, n, vs);
      const int64_t q = i / MS_ADAMW_BLOCK;
      ms = a.exp_avg_scale[q];
      vs8 = a.exp_avg_sq_scale[q];
    }
  };
  // whole waves work or leave: the 64 lanes of a wave take one scale block
  const bool some = begin - lane * E < n;
  if (some) fetch(begin);
  if (threadIdx.x < 64) {  // one wave's float64 arithmetic, under the first loads
    const int64_t t = *(volatile int64_t*)a.step + 1;
    const double lr = hp.lr_device ? (double)*hp.lr_device : hp.lr;
    Factors f;
    f.fix1 = (float)(lr / (1.0 - power(hp.beta1, t)));
    f.fix2 = (float)(1.0 / sqrt(1.0 - power(hp.beta2, t)));
    f.keep = (float)(1.0 - lr * hp.weight_decay);
    f.clip = hp.use_clip ? ws.f[0] : 1.0f;
    f.key = SR ? key_of(t) : 0;
    if (threadIdx.x == 0) shared = f;
  }
  __syncthreads();
  const Factors f = shared;
  for (int j = 0; some && j < list.rounds; ++j) {
    const int64_t i = begin + (int64_t)j * ROUND;
    if (i - lane * E >= n) break;
    const f32x4 p0 = p;
    f32x4 g0 = g, m, v, r;
    if constexpr (BITS == 32) {
      m = s.m;
      v = s.v;
    } else {
      m = decode(mc) * ms;
      r = decode(vc) * vs8;
      v = r * r;
    }
    if (j + 1 < list.rounds && i + ROUND - lane * E < n) fetch(i + ROUND);  // the next round's loads under this one's arithmetic
    if (hp.use_clip) g0 = g0 * f.clip;
    m = m * hp.b1 + g0 * hp.c1;
    v = v * hp.b2 + g0 * g0 * hp.c2;
    f32x4 to;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      r[e] = sqrtf(v[e]);
      to[e] = p0[e] * f.keep - f.fix1 * m[e] / (r[e] * f.fix2 + hp.eps);
    }
    put_any(a.param, dtype, i, n, vp, to);
    if constexpr (BITS == 32) {
      put4<f32x4>((float*)a.exp_avg, i, n, vs, m);
      put4<f32x4>((float*)a.exp_avg_sq, i, n, vs, v);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i + e >= n) m[e] = r[e] = 0.0f;  // values past the end count for no scale
      const int64_t q = i / MS_ADAMW_BLOCK;
      Odds o = {};
      if constexpr (SR) o = odds_of(i, f.key);
      put_codes((uint8_t*)a.exp_avg, i, n, vs, quantise<SR, false>(m, a.exp_avg_scale + q, lane == 0, o));
      put_codes((uint8_t*)a.exp_avg_sq, i, n, vs, quantise<SR, true>(r, a.exp_avg_sq_scale + q, lane == 0, {{o.h[1], o.h[0]}}));
    }
  }
  // every block has read its count (and used it) by its ticket; the last one raises them all. The ticket
  // orders nothing else, so it is relaxed: with release and acquire each block would write back and
  // invalidate its XCD's L2, 60 ns a block one after the other.
  __syncthreads();
  if (threadIdx.x < 64) {
    unsigned got = 0;
    if (lane == 0) got = __hip_atomic_fetch_add(ws.ticket(), 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (__builtin_amdgcn_readfirstlane((int)got) == (int)gridDim.x - 1) {
      if (lane < list.count) *list.t[lane].step += 1;
      if (lane == 0) __hip_atomic_store(ws.ticket(), 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  }
}

// four rounds' loads in flight at a time
template <typename T4, typename T>
__device__ __forceinline__ double squares(const T* p, int64_t i, int64_t n, int rounds, bool vec) {
  double sum = 0.0;
  for (int j = 0; j < rounds; j += 4) {
    f32x4 g[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) g[k] = get4<T4>(p, i + (int64_t)(j + k) * ROUND, j + k < rounds ? n : 0, vec);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) sum += (double)g[k][e] * (double)g[k][e];
  }
  return sum;
}

__global__ __launch_bounds__(THREADS) void norm(const NormList list, double max_norm, float* grad_norm, const Ws ws) {
  __shared__ double s[THREADS];
  __shared__ bool last;
  double sum = 0.0;
  const int lane = threadIdx.x & 63;
  for (uint32_t b = blockIdx.x; b < list.blocks; b += gridDim.x) {
    const int k = __popcll(__ballot(lane < list.count && b >= list.end[lane]));
    const int64_t n = list.numel[k];
    const int dtype = list.dtype[k];
    const void* g = list.grad[k];
    const bool vec = aligned(g, dtype == 0 ? 16 : 8);
    const int64_t i = (int64_t)(b - (k ? list.end[k - 1] : 0)) * list.rounds * ROUND + threadIdx.x * E;
    if (dtype == 0) sum += squares<f32x4>((const float*)g, i, n, list.rounds, vec);
    else if (dtype == 1) sum += squares<bf16x4>((const bf16*)g, i, n, list.rounds, vec);
    else sum += squares<f16x4>((const f16*)g, i, n, list.rounds, vec);
  }
  s[threadIdx.x] = sum;
  __syncthreads();
  for (int m = THREADS / 2; m >= 1; m >>= 1) {
    if ((int)threadIdx.x < m) s[threadIdx.x] += s[threadIdx.x + m];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    // the part goes through to where every XCD sees it (an agent-scope store) and has arrived (the wait)
    // before the ticket is taken; the last block reads the parts the same way. Release and acquire on
    // the ticket would write back and invalidate the L2 for every block, for nothing else's sake.
    __hip_atomic_store(ws.parts() + blockIdx.x, s[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    last = __hip_atomic_fetch_add(ws.norm_ticket(), 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  double all = 0.0;
  for (uint32_t b = threadIdx.x; b < gridDim.x; b += THREADS)
    all += __hip_atomic_load(ws.parts() + b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  s[threadIdx.x] = all;
  __syncthreads();
  for (int m = THREADS / 2; m >= 1; m >>= 1) {
    if ((int)threadIdx.x < m) s[threadIdx.x] += s[threadIdx.x + m];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const double total = s[0] + (list.first ? 0.0 : *ws.total());
    *ws.total() = total;
    if (list.last) {
      const double nrm = sqrt(total), f = max_norm / (nrm + 1e-6);
      ws.f[0] = (float)(f > 1.0 ? 1.0 : f);  // a NaN stays one
      if (grad_norm) *grad_norm = (float)nrm;
    }
    __hip_atomic_store(ws.norm_ticket(), 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}

int fail(int code, const char* who, const char* why) {
  snprintf(g_optim_error, sizeof(g_optim_error), "%s: %s", who, why);
  return code;
}
int launched(const char* who) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MS_OK : fail(MS_ERR_HIP, who, hipGetErrorString(e));
}

const char* check(const ms_optim_tensor* t, int64_t count, const float* workspace) {
  if (count < 0 || (count > 0 && !t)) return "no tensors";
  if (!workspace || ((uintptr_t)workspace & 15u)) return "the workspace is missing or misaligned";
  for (int64_t i = 0; i < count; ++i) {
    if (t[i].numel < 0 || t[i].numel > (int64_t)1 << 40) return "a tensor's numel is out of range";
    if (t[i].dtype < 0 || t[i].dtype > 2) return "dtype must be 0 (float32), 1 (bfloat16) or 2 (float16)";
    if (t[i].numel > 0 && !t[i].grad) return "a gradient is NULL";
  }
  return nullptr;
}

// Rounds a block: one for lists that would otherwise leave CUs idle (the Agent's 423 k values, step 10 us
// and norm 10), more for long ones, so that each block's loads run ahead under its arithmetic and fewer
// tickets are taken (201 M values in 8 bits: 0.59-0.68 ms).
int rounds(const ms_optim_tensor* t, int64_t count) {
  int64_t all = 0;
  for (int64_t i = 0; i < count; ++i) all += t[i].numel;
  return all > (int64_t)ROUND * 16384 ? 8 : all > (int64_t)ROUND * 4096 ? 4 : 1;
}

}  // namespace opt

extern "C" {

const char* ms_optim_last_error(void) { return g_optim_error; }

int ms_grad_clip(const ms_optim_tensor* tensors, int64_t count, double max_norm, float* grad_norm, float* workspace,
                 void* stream) {
  const char* who = "ms_grad_clip";
  if (const char* why = opt::check(tensors, count, workspace)) return opt::fail(MS_ERR_INVALID_ARGUMENT, who, why);
  if (!(max_norm > 0.0)) return opt::fail(MS_ERR_INVALID_ARGUMENT, who, "max_norm must be positive");
  const int per = opt::rounds(tensors, count);
  for (int64_t first = 0; first == 0 || first < count; first += opt::LIST) {
    opt::NormList list = {};
    const int64_t n = count - first < opt::LIST ? count - first : opt::LIST;
    uint64_t blocks = 0;
    for (int64_t i = 0; i < n; ++i) {
      const ms_optim_tensor& t = tensors[first + i];
      const int64_t one = (int64_t)per * opt::ROUND;
      blocks += (uint64_t)((t.numel + one - 1) / one);
      if (blocks > 0x7fffffff) return opt::fail(MS_ERR_INVALID_ARGUMENT, who, "too large");
      list.grad[i] = t.grad;
      list.numel[i] = t.numel;
      list.dtype[i] = t.dtype;
      list.end[i] = (uint32_t)blocks;
    }
    list.count = (int32_t)n;
    list.rounds = per;
    list.first = first == 0;
    list.last = first + opt::LIST >= count;
    list.blocks = (uint32_t)blocks;
    const uint64_t grid = blocks < 1 ? 1 : blocks < (uint64_t)opt::NORM_BLOCKS ? blocks : (uint64_t)opt::NORM_BLOCKS;
    hipLaunchKernelGGL(opt::norm, dim3((unsigned)grid), dim3(opt::THREADS), 0, (hipStream_t)stream, list, max_norm,
                       grad_norm, opt::Ws{workspace});
    if (int rc = opt::launched(who)) return rc;
  }
  return MS_OK;
}

int ms_adamw_step(const ms_optim_tensor* tensors, int64_t count, int state_bits, double lr, const float* lr_device,
                  double beta1, double beta2, double eps, double weight_decay, int use_clip, float* workspace,
                  void* stream) {
  const char* who = "ms_adamw_step";
  if (const char* why = opt::check(tensors, count, workspace)) return opt::fail(MS_ERR_INVALID_ARGUMENT, who, why);
  const bool stochastic = state_bits == (8 | MS_ADAMW_STOCHASTIC);
  if (stochastic) state_bits = 8;
  if (state_bits != 32 && state_bits != 8)
    return opt::fail(MS_ERR_INVALID_ARGUMENT, who, "state_bits must be 32, 8 or 8 | MS_ADAMW_STOCHASTIC");
  if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0 && weight_decay >= 0.0) ||
      (!lr_device && !(lr >= 0.0)))
    return opt::fail(MS_ERR_INVALID_ARGUMENT, who, "lr, eps and weight_decay must be >= 0, the betas in [0, 1)");
  for (int64_t i = 0; i < count; ++i) {
    const ms_optim_tensor& t = tensors[i];
    if (!t.step || ((uintptr_t)t.step & 7u)) return opt::fail(MS_ERR_INVALID_ARGUMENT, who, "a step count is missing or misaligned");
    if (t.numel > 0 && (!t.param || !t.exp_avg || !t.exp_avg_sq || (state_bits == 8 && (!t.exp_avg_scale || !t.exp_avg_sq_scale))))
      return opt::fail(MS_ERR_INVALID_ARGUMENT, who, "a tensor's param or state is NULL");
  }
  opt::Hyper hp = {};
  hp.lr = lr; hp.lr_device = lr_device;
  hp.beta1 = beta1; hp.beta2 = beta2;
  hp.b1 = (float)beta1; hp.b2 = (float)beta2;
  hp.c1 = (float)(1.0 - beta1); hp.c2 = (float)(1.0 - beta2);
  hp.eps = (float)eps;
  hp.weight_decay = weight_decay;
  hp.use_clip = use_clip != 0;
  const int per = opt::rounds(tensors, count);
  for (int64_t first = 0; first < count; first += opt::LIST) {
    opt::List list = {};
    const int64_t n = count - first < opt::LIST ? count - first : opt::LIST;
    uint64_t blocks = 0;
    for (int64_t i = 0; i < n; ++i) {
      list.t[i] = tensors[first + i];
      const int64_t one = (int64_t)per * opt::ROUND;
      blocks += (uint64_t)((list.t[i].numel + one - 1) / one);
      if (blocks > 0xffffffffu / opt::THREADS) return opt::fail(MS_ERR_INVALID_ARGUMENT, who, "too large");  // a launch's threads are counted in 32 bits
      list.end[i] = (uint32_t)blocks;
    }
    if (blocks == 0) {  // only empty tensors: a block still raises their counts
      blocks = 1;
      list.end[n - 1] = 1;
    }
    list.count = (int32_t)n;
    list.rounds = per;
    const dim3 grid((unsigned)blocks), block(opt::THREADS);
    if (state_bits == 32)
      hipLaunchKernelGGL((opt::adamw<32, false>), grid, block, 0, (hipStream_t)stream, list, hp, opt::Ws{workspace});
    else if (stochastic)
      hipLaunchKernelGGL((opt::adamw<8, true>), grid, block, 0, (hipStream_t)stream, list, hp, opt::Ws{workspace});
    else
      hipLaunchKernelGGL((opt::adamw<8, false>), grid, block, 0, (hipStream_t)stream, list, hp, opt::Ws{workspace});
    if (int rc = opt::launched(who)) return rc;
  }
  return MS_OK;
}

}  // extern "C"
