// ms_scan.hip — selective state-space scan over time, its gradients, and its single step (gfx950).
//
// Per row r, channel d, state n:  h[t] = a[t] h[t-1] + rate u B[t],  a = exp(rate A),  rate =
// softplus(delta + bias);  y = sum_n C h + D u;  out = y silu(z).  starts[t] sets h[t-1] to zero.
//
// What bounds it: each (t, r, d) moves 6-8 B in half precision but needs N exponentials (v_exp_f32,
// a quarter of the rate of an FMA) and 4 N other VALU operations, so at N = 16 the vector units and
// not HBM set the time. The layout serves them:
//   * a lane is a channel and holds its states, so nothing is exchanged between lanes in the
//     recurrence, and B and C, the same for all channels of a row's step, are scalars: they are read
//     through the constant address space into SGPRs and cost no vector instruction;
//   * a block is 64 channels of one row; its NW waves share the states (NS each) and add their parts
//     of y through LDS. u, delta and z are read 16 B a thread, turned into (rate, rate u) once and
//     laid into LDS as float pairs;
//   * where rows and channels do not fill the chip, the time axis is split into chunks: one pass
//     leaves each chunk's end state from zero and its summed rate (the decay over a chunk is
//     exp(A sum rate)), a small kernel joins the chunks, and the scan proper starts each chunk from
//     its state. The first pass costs another N exponentials, so only few rows are split.
// Backward runs the same tiles from the end: g[t] = C dy + a[t+1] g[t+1]. The states it needs are
// rebuilt from checkpoints of every KC = 8 steps, B and C read as the forward left them; dB and dC are
// sums over channels, folded over the wave's lanes with v_permlane swaps and DPP, and over the channel
// blocks by a last kernel.
// Measured at 16 states (time; share of the vector units' cycles that issue): forward 8 rows of 2,048
// steps x 2,048 channels bf16 233 us, 65 %; one row of 16,411 x 1,536 bf16 in 31 chunks 106 + 133 us,
// 77 and 72 %; with gradients 2,048 rows of 128 x 128 f32 244 us forward, 59 %, and 600 us backward,
// 67 % (108 vector instructions a wave, step and four states).
#include <type_traits>

#include "ms_sequence.h"

namespace scan {
using namespace seq;

constexpr int KC = 8;  // steps between checkpoints
constexpr int SEGMENT = MS_SUM_CHAIN;  // steps that the backward adds up in float32 for dA, dD and ddelta_bias
static_assert(SEGMENT % KC == 0, "whole tiles");
constexpr float LOG2E = 1.44269504f, LN2 = 0.69314718f;

#define CONSTANT(T) const __attribute__((address_space(4))) T

// How a call is cut. NW waves hold NS states each; `tiles` blocks of 64 channels a group.
struct Plan {
  int ns, nw;               // states per wave, waves per block
  int unit;                 // states of a scalar unit: 16 / unit steps of `unit` states
  int64_t units;            // scalar units along time (of all steps, and one more that is only fetched)
  int64_t tiles, blocks_d;  // tiles per group, tiles * groups
  int64_t chunks, chunk;    // over time; steps per chunk (a multiple of 32)
  int64_t kc;               // checkpoints, tiles of the backward pass
  int64_t segments, sums;   // of a chunk and of all: the backward's sums over time are handed on after each
};

struct Work {  // the workspace, in floats
  float *bc, *local, *rates, *parts_bc, *parts, *sums;
  int* cut;
  int64_t floats;
};

// One launch's view: the caller's arrays and what the kernels share
struct Args {
  ms_scan_io io;
  Plan p;
  float *bc, *local, *rates, *parts_bc, *parts;
  int* cut;
  int vec;
};

// B and C (T, R, G, N) of any strides and type -> float32 in the order that the scans' scalar loads
// want: [row][group][states / unit][16 / unit steps][B, C][16], zeros past the last step and state. A
// block takes a unit's steps of some neighbouring rows, so that it reads runs of rows and writes whole
// units: wave c writes the c-th 16 B of each, its lanes the shares of the states, then the rows. vec: units
// of four states and more, whose four neighbours are read in one access.
template <typename T>
__global__ __launch_bounds__(256) void widen(const ms_scan_io io, int unit, int shares, int64_t units, bool vec, float* __restrict__ to) {
  const int lane = threadIdx.x & 63, c = threadIdx.x >> 6;
  const unsigned per_wave = 64 / shares, rgs = (unsigned)(io.rows * io.groups);
  const int64_t first = (int64_t)blockIdx.x * per_wave, v0 = first / rgs;
  const unsigned i = (unsigned)(first - v0 * rgs) + lane / shares;
  const int share = lane % shares;
  const int64_t v = v0 + i / rgs;
  const unsigned rg = i % rgs, r = rg / (unsigned)io.groups, g = rg - r * (unsigned)io.groups;
  if (v >= units) return;
  const int log = 31 - __builtin_clz(unit);
  float* q = to + (((int64_t)rg * shares + share) * units + v) * 32 + c * 4;
#pragma unroll
  for (int kind = 0; kind < 2; ++kind) {
    const T* p = kind ? (const T*)io.C + r * io.C_r + g * io.C_g : (const T*)io.B + r * io.B_r + g * io.B_g;
    const int64_t step = kind ? io.C_t : io.B_t;
    float x[4];
    const int n0 = share * unit + (c * 4 & (unit - 1));
    const int64_t t0 = v * (16 / unit) + (c * 4 >> log);
    if (vec && n0 + 4 <= io.states && t0 < io.steps) {  // four states of one step
      typedef T T4 __attribute__((ext_vector_type(4)));
      const T4 four = *(const T4*)(p + t0 * step + n0);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = (float)four[k];
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int e = c * 4 + k, n = share * unit + (e & (unit - 1));
        const int64_t t = v * (16 / unit) + (e >> log);
        x[k] = n < io.states && t < io.steps ? (float)p[t * step + n] : 0.0f;
      }
    }
    *(float4*)(q + kind * 16) = make_float4(x[0], x[1], x[2], x[3]);
  }
}

typedef float f32x16 __attribute__((ext_vector_type(16)));
struct Scalars {  // a unit's B and C, in SGPRs
  f32x16 b, c;
};
__device__ __forceinline__ Scalars scalars(CONSTANT(f32x16)* p) {
  Scalars s;
  s.b = p[0];
  s.c = p[1];
  return s;
}
__device__ __forceinline__ CONSTANT(f32x16)* scalars_at(const Args& a, int64_t r, int64_t g, int share) {
  const int shares = a.p.ns * a.p.nw / a.p.unit;
  return (CONSTANT(f32x16)*)(a.bc + ((r * a.io.groups + g) * shares + share) * a.p.units * 32);
}
// Every LDS and scalar load issued so far has returned. Scalar loads return in no order, so a wait for
// any of them is a wait for all: the one for a unit's operands has to stand before the next unit's
// loads are issued, or it would wait for those too.
__device__ __forceinline__ void loads_done() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0), the others unbounded
  __builtin_amdgcn_sched_barrier(0);
}
// the checkpoint of step KC k: [k][row][tile][states / 4][64 channels][4]
__device__ __forceinline__ int64_t checkpoint_at(const Args& a, int64_t k, int64_t r, int64_t td, int state, int lane) {
  return (((k * a.io.rows + r) * a.p.blocks_d + td) * (a.p.ns * a.p.nw / 4) + state / 4) * 256 + lane * 4 + state % 4;
}

// Which steps of a tile begin an episode, as a mask the whole wave shares: lane l looks at step l, a tile
// ahead as every other load
struct Starts {
  const uint8_t* p;
  int64_t by;
  int now;
  // `steps`: how many steps of the first tile there are; a tile further is `tile` steps
  __device__ __forceinline__ Starts(const ms_scan_io& io, int64_t r, int64_t t0, int64_t tile, int steps)
      : p(io.starts ? io.starts + r * io.starts_r + (t0 + (threadIdx.x & 63)) * io.starts_t : nullptr), by(tile * io.starts_t) {
    read(steps);
  }
  __device__ __forceinline__ void read(int steps) { now = p && (int)(threadIdx.x & 63) < steps ? *p : 0; }
  __device__ __forceinline__ uint64_t mask() const { return p ? __ballot(now != 0) : 0; }
  __device__ __forceinline__ void move(int steps) {  // to the next tile, of which `steps` steps are there
    if (p) p += by;
    read(steps);
  }
};

struct Place {  // a block's channels
  int64_t r, chunk, g, c0;  // row, chunk, group, first channel
  int64_t td;               // tile over all groups
  int nc;                   // channels of the tile (<= 64)
};
__device__ __forceinline__ Place place(const Args& a) {
  Place p;
  int64_t b = blockIdx.x;
  p.td = b % a.p.blocks_d;
  b /= a.p.blocks_d;
  p.r = b % a.io.rows;
  p.chunk = b / a.io.rows;
  const int64_t per = a.io.channels / a.io.groups;
  p.g = p.td / a.p.tiles;
  const int64_t in = (p.td % a.p.tiles) * 64;
  p.c0 = p.g * per + in;
  p.nc = (int)(per - in < 64 ? per - in : 64);
  return p;
}

// Where channel c of step t lies in its row of LDS. Threads that move 8 neighbouring values reach every
// other 16 B of a row; odd rows are shifted by 16 B, so that the two rows a 16-lane access covers use
// all banks and not half of them twice.
template <int E>
__device__ __forceinline__ int column(int c, int t) {
  return E == 8 ? c ^ (t & 1) << 2 : c;
}

// ---------------------------------------------------------------- forward
// LOCAL: the first pass of a split time axis (states from zero, no outputs).
// The loop over a tile goes by units of 16 / NS steps: 32 scalars (one s_load_dwordx16 for B and one
// for C) and the unit's rates from LDS are fetched a unit ahead, both before the work of the present
// one, since scalar loads return in no order and one wait covers them all.
template <typename T, int NS, int NW, bool LOCAL>
__global__ __launch_bounds__(64 * NW) void forward(const Args a) {
  constexpr int TT = NW < 4 ? 8 * NW : 32, E = TT / NW, TPR = 64 / E;  // a tile: TT steps x 64 channels, E channels of one step a thread
  constexpr int G = 16 / NS;                                          // steps of a unit
  // With one block a CU nothing runs beside the steps between two tiles: the next tile's rates are then
  // computed under the loads of this one's parts (8 rows of 2,048 x 2,048: 262 -> 233 us). Where three
  // blocks share a CU that takes 2 % longer.
  constexpr bool TOGETHER = NW == 8;
  static_assert(TT % G == 0 && TT % 8 == 0, "tiles are whole units");
  __shared__ float s_rate[TT + G][64], s_ru[TT + G][64];  // the last unit is only fetched
  __shared__ float s_y[LOCAL ? 1 : NW][LOCAL ? 1 : TT][64];
  const ms_scan_io& io = a.io;
  const Place at = place(a);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lt = threadIdx.x / TPR, lc = threadIdx.x % TPR * E;  // this thread's step and channels in loads
  const int n = at.nc - lc < 0 ? 0 : at.nc - lc;
  const int64_t t_begin = at.chunk * a.p.chunk;
  const int64_t t_end = t_begin + a.p.chunk < io.steps ? t_begin + a.p.chunk : io.steps;
  const int64_t cl = at.c0 + lc;
  const T* u = (const T*)io.u + at.r * io.u_r + cl + (t_begin + lt) * io.u_t;
  const T* dl = (const T*)io.delta + at.r * io.delta_r + cl + (t_begin + lt) * io.delta_t;
  const T* z = io.z && !LOCAL ? (const T*)io.z + at.r * io.z_r + cl + (t_begin + lt) * io.z_t : nullptr;
  T* out = (T*)io.out + at.r * io.out_r + cl + (t_begin + lt) * io.out_t;
  const int64_t u_step = io.u_t * TT, d_step = io.delta_t * TT, z_step = io.z_t * TT, o_step = io.out_t * TT;
  float bias[E], skip[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    bias[e] = io.delta_bias && e < n ? io.delta_bias[cl + e] : 0.0f;
    skip[e] = io.D && e < n ? io.D[cl + e] : 0.0f;
  }
  // this lane's channel in the recurrence
  const int64_t ch = at.c0 + lane;
  const bool live = lane < at.nc;
  const int N = io.states;
  float A2[NS], h[NS], total = 0.0f;
  bool was_cut = false;
  const int64_t slot = (at.r * io.channels + ch) * N;  // (R, D, N)
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int s = w * NS + i;
    A2[i] = live && s < N ? io.A[ch * N + s] * LOG2E : 0.0f;
    h[i] = 0.0f;
    if (!LOCAL && live && s < N) {
      if (a.p.chunks > 1) h[i] = a.local[at.chunk * io.rows * io.channels * N + slot + s];
      else if (io.state) h[i] = io.state[slot + s];
    }
  }
  CONSTANT(f32x16)* next = scalars_at(a, at.r, at.g, w) + t_begin / G * 2;
  const bool keep = !LOCAL && io.checkpoints;
  float* ckpt = io.checkpoints + (keep ? checkpoint_at(a, t_begin / KC, at.r, at.td, w * NS, lane) : 0);
  const int64_t ckpt_step = io.rows * a.p.blocks_d * (a.p.ns * a.p.nw / 4) * 256;
  const int soft = io.softplus;
  const bool vec = a.vec;
  typedef typename Vec<T, E>::type V;
  V vu, vd, vz;
  auto fetch = [&](bool in) __attribute__((always_inline)) {
    vu = load<T, E>(u, in ? n : 0, vec);
    vd = load<T, E>(dl, in ? n : 0, vec);
    if (z) vz = load<T, E>(z, in ? n : 0, vec);
    u += u_step;
    dl += d_step;
    if (z) z += z_step;
  };
  // a tile's rates into LDS (a step past the end has rate 0: it changes nothing)
  auto stage = [&](bool mine) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float slope, rate = (float)vd[e] + bias[e];
      if (soft) rate = softplus(rate, slope);
      rate = mine ? rate : 0.0f;
      s_rate[lt][column<E>(lc + e, lt)] = rate;
      s_ru[lt][column<E>(lc + e, lt)] = rate * (float)vu[e];
    }
  };
  int left = (int)(t_end - t_begin);  // steps of the chunk not done yet
  fetch(lt < left);
  Scalars s = scalars(next);
  Starts flags(io, at.r, t_begin, TT, left < TT ? left : TT);
  if constexpr (TOGETHER) stage(lt < left);
  for (; left > 0; left -= TT) {
    const V cu = vu, cz = vz;
    const bool mine = lt < left;
    if constexpr (!TOGETHER) stage(mine);
    const uint64_t starts = flags.mask();
    __syncthreads();
    fetch(lt + TT < left);
    flags.move(left - TT < TT ? left - TT : TT);
    float rate[G], ru[G];
#pragma unroll
    for (int j = 0; j < G; ++j) {
      rate[j] = s_rate[j][column<E>(lane, j)];
      ru[j] = s_ru[j][column<E>(lane, j)];
    }
    const int steps = left < TT ? (left + G - 1) / G * G : TT;
    for (int t = 0; t < steps; t += G) {
      if (keep && (G >= KC || (t & (KC - 1)) == 0)) {  // the states before this step: tiles are multiples of KC
        if constexpr (NS == 2) {
          *(float2*)ckpt = make_float2(h[0], h[1]);
        } else {
#pragma unroll
          for (int i = 0; i < NS; i += 4) *(float4*)(ckpt + i * 64) = make_float4(h[i], h[i + 1], h[i + 2], h[i + 3]);
        }
        ckpt += ckpt_step;
      }
      loads_done();
      next += 2;
      const Scalars ns = scalars(next);
      float nrate[G], nru[G];
#pragma unroll
      for (int j = 0; j < G; ++j) {
        const int c = column<E>(lane, G > 1 ? j : t + 1);
        nrate[j] = s_rate[t + G + j][c];
        nru[j] = s_ru[t + G + j][c];
      }
      __builtin_amdgcn_sched_barrier(0);
      const unsigned cut = (unsigned)(starts >> t) & ((1u << G) - 1);
      auto work = [&](auto any) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < G; ++j) {
          if (decltype(any)::value && (cut >> j & 1)) {
#pragma unroll
            for (int i = 0; i < NS; ++i) h[i] = 0.0f;
            if (LOCAL) was_cut = true;
          }
          float y = 0.0f;
#pragma unroll
          for (int i = 0; i < NS; ++i) {
            h[i] = __builtin_fmaf(__builtin_amdgcn_exp2f(rate[j] * A2[i]), h[i], ru[j] * s.b[j * NS + i]);
            if (!LOCAL) y = i ? __builtin_fmaf(s.c[j * NS + i], h[i], y) : s.c[j * NS] * h[0];
          }
          if (LOCAL) total += rate[j];
          else s_y[w][t + j][column<E>(lane, G > 1 ? j : t)] = y;
        }
      };
      if (cut) work(std::true_type{});
      else work(std::false_type{});
      __builtin_amdgcn_sched_barrier(0);
      s = ns;
#pragma unroll
      for (int j = 0; j < G; ++j) {
        rate[j] = nrate[j];
        ru[j] = nru[j];
      }
    }
    __syncthreads();
    float part[TOGETHER ? NW : 1][E];
    if constexpr (TOGETHER) {
#pragma unroll
      for (int k = 0; k < NW; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) part[k][e] = s_y[k][lt][column<E>(lc + e, lt)];
      __builtin_amdgcn_sched_barrier(0);
      if (left > TT) stage(lt + TT < left);
    }
    if constexpr (!LOCAL) {
      if (mine && n > 0) {
        float y[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          float v = 0.0f;
#pragma unroll
          for (int k = 0; k < NW; ++k) {
            const float x = TOGETHER ? part[TOGETHER ? k : 0][e] : s_y[k][lt][column<E>(lc + e, lt)];
            v = k ? v + x : x;
          }
          y[e] = __builtin_fmaf(skip[e], (float)cu[e], v);
          if (z) y[e] *= silu((float)cz[e]);
        }
        store<T, E>(out, y, n, vec);
      }
      out += o_step;
    }
  }
  if (LOCAL) {
    const int64_t of = at.chunk * io.rows * io.channels;
    if (live) {
#pragma unroll
      for (int i = 0; i < NS; ++i)
        if (w * NS + i < N) a.local[of * N + slot + w * NS + i] = h[i];
      if (w == 0) a.rates[of + at.r * io.channels + ch] = total;
    }
    if (threadIdx.x == 0 && at.td == 0) a.cut[at.chunk * io.rows + at.r] = was_cut;
  } else if (io.new_state && live && t_end == io.steps) {
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (w * NS + i < N) io.new_state[slot + w * NS + i] = h[i];
  }
}

// The chunks of a split time axis in turn: what each left from zero becomes the state it starts from.
// BACK: from the last chunk, with the gradients handed back in place of the states.
template <bool BACK>
__global__ __launch_bounds__(256) void join(const Args a) {
  const ms_scan_io& io = a.io;
  const int64_t N = io.states, all = io.rows * io.channels * N;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= all) return;
  const int64_t rc = i / N, r = rc / io.channels, c = rc - r * io.channels;
  const float A2 = io.A[c * N + (i - rc * N)] * LOG2E;
  const float* first = BACK ? io.dnew_state : io.state;
  float h = first ? first[i] : 0.0f;
  const int64_t chunks = a.p.chunks, rd = io.rows * io.channels;
  for (int64_t k0 = 0; k0 < chunks; k0 += 8) {  // eight chunks' loads in flight
    float mine[8], rate[8];
    int cut[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t k = k0 + j < chunks ? k0 + j : chunks - 1, q = BACK ? chunks - 1 - k : k;
      mine[j] = a.local[q * all + i];
      rate[j] = a.rates[q * rd + rc];
      cut[j] = a.cut[q * io.rows + r];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (k0 + j >= chunks) break;
      const int64_t q = BACK ? chunks - 1 - (k0 + j) : k0 + j;
      a.local[q * all + i] = h;
      h = cut[j] ? mine[j] : __builtin_fmaf(__builtin_amdgcn_exp2f(A2 * rate[j]), h, mine[j]);
    }
  }
}

// ---------------------------------------------------------------- one step
// The states are read and written once: HBM-bound (16,384 x 128 x 16 states: 304 MB in
// 63 us a call, 4.8 TB/s; 250 x 4,096, bf16: 140 MB in 28 us, 5.0 TB/s). Q lanes of
// four states each share a channel. Every load is issued before the first is used, the state's too: an
// episode's start is selected after it, where waiting for the flag first took 86 us. Two or four of
// these a thread took longer (73, 94 us).
template <typename T, int Q>
__global__ __launch_bounds__(256) void step4(const ms_scan_io io) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t D = io.channels, rc = i / Q;
  if (rc >= io.rows * D) return;  // a channel's Q lanes leave together: Q divides the wave
  const int q = (int)(threadIdx.x % Q) * 4;
  const int64_t r = rc / D, ch = rc - r * D, g = ch / (D / io.groups);
  float4 h = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (io.state) h = *(const float4*)(io.state + rc * (Q * 4) + q);
  const bool cut = io.starts && io.starts[r * io.starts_r];
  const float u = (float)((const T*)io.u)[r * io.u_r + ch];
  const float d = (float)((const T*)io.delta)[r * io.delta_r + ch] + (io.delta_bias ? io.delta_bias[ch] : 0.0f);
  const float z = io.z ? (float)((const T*)io.z)[r * io.z_r + ch] : 0.0f;
  const float skip = io.D ? io.D[ch] : 0.0f;
  const float4 A = *(const float4*)(io.A + ch * (Q * 4) + q);
  const T* B = (const T*)io.B + r * io.B_r + g * io.B_g + q;
  const T* C = (const T*)io.C + r * io.C_r + g * io.C_g + q;
  float b[4], c[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    b[j] = (float)B[j];
    c[j] = (float)C[j];
  }
  float slope;
  const float rate = io.softplus ? softplus(d, slope) : d, ru = rate * u, r2 = rate * LOG2E;
  if (cut) h = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  h.x = __builtin_fmaf(__builtin_amdgcn_exp2f(r2 * A.x), h.x, ru * b[0]);
  h.y = __builtin_fmaf(__builtin_amdgcn_exp2f(r2 * A.y), h.y, ru * b[1]);
  h.z = __builtin_fmaf(__builtin_amdgcn_exp2f(r2 * A.z), h.z, ru * b[2]);
  h.w = __builtin_fmaf(__builtin_amdgcn_exp2f(r2 * A.w), h.w, ru * b[3]);
  *(float4*)(io.new_state + rc * (Q * 4) + q) = h;
  float y = c[0] * h.x;
  y = __builtin_fmaf(c[1], h.y, y);
  y = __builtin_fmaf(c[2], h.z, y);
  y = __builtin_fmaf(c[3], h.w, y);
#pragma unroll
  for (int m = 1; m < Q; m <<= 1) y += __shfl_xor(y, m);
  if (q == 0) {
    y = __builtin_fmaf(skip, u, y);
    if (io.z) y *= silu(z);
    ((T*)io.out)[r * io.out_r + ch] = (T)y;
  }
}
// any number of states: a thread per channel
template <typename T>
__global__ __launch_bounds__(256) void step1(const ms_scan_io io) {
  const int64_t rc = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t D = io.channels, N = io.states;
  if (rc >= io.rows * D) return;
  const int64_t r = rc / D, c = rc - r * D, g = c / (D / io.groups);
  const float u = (float)((const T*)io.u)[r * io.u_r + c];
  const float d = (float)((const T*)io.delta)[r * io.delta_r + c] + (io.delta_bias ? io.delta_bias[c] : 0.0f);
  float slope;
  const float rate = io.softplus ? softplus(d, slope) : d, ru = rate * u, r2 = rate * LOG2E;
  const bool fresh = !io.state || (io.starts && io.starts[r * io.starts_r]);
  const T* B = (const T*)io.B + r * io.B_r + g * io.B_g;
  const T* C = (const T*)io.C + r * io.C_r + g * io.C_g;
  float y = 0.0f;
  for (int64_t n = 0; n < N; ++n) {
    float h = fresh ? 0.0f : io.state[rc * N + n];
    h = __builtin_fmaf(__builtin_amdgcn_exp2f(r2 * io.A[c * N + n]), h, ru * (float)B[n]);
    io.new_state[rc * N + n] = h;
    y = __builtin_fmaf((float)C[n], h, y);
  }
  if (io.D) y = __builtin_fmaf(io.D[c], u, y);
  if (io.z) y *= silu((float)((const T*)io.z)[r * io.z_r + c]);
  ((T*)io.out)[r * io.out_r + c] = (T)y;
}

// ---------------------------------------------------------------- backward
// Eight values a lane (8 steps' worth of one folded register each) and eight items a step are summed
// over the 64 lanes with the total left in one lane each: at every level two registers become one
// that holds one half of the lanes for each, so 64 sums cost about two operations apiece.
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float fold32(float x0, float x1) {  // lanes 0-31: sum of x0, 32-63: of x1
  const u32x2 s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x0), __float_as_uint(x1), false, false);
  const unsigned lo = s.x, hi = s.y;
  return __uint_as_float(lo) + __uint_as_float(hi);
}
__device__ __forceinline__ float fold16(float x0, float x1) {  // even rows of 16 lanes: x0, odd rows: x1
  const u32x2 s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x0), __float_as_uint(x1), false, false);
  const unsigned lo = s.x, hi = s.y;
  return __uint_as_float(lo) + __uint_as_float(hi);
}
template <int CTRL>
__device__ __forceinline__ float moved(float x) {
  return __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xf, 0xf, false));
}
template <int CTRL>
__device__ __forceinline__ float fold_dpp(float x0, float x1, bool second) {
  const float s0 = x0 + moved<CTRL>(x0), s1 = x1 + moved<CTRL>(x1);
  return second ? s1 : s0;
}
constexpr int ROR8 = 0x128, HALF_MIRROR = 0x141, XOR2 = 0x4e, XOR1 = 0xb1;

// items of one step -> a register whose lanes 8 i .. 8 i + 7 hold parts of item i
__device__ __forceinline__ float fold_items(const float (&x)[8], bool bit3) {
  float a[4], b[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = fold32(x[i], x[i + 4]);
#pragma unroll
  for (int i = 0; i < 2; ++i) b[i] = fold16(a[i], a[i + 2]);
  return fold_dpp<ROR8>(b[0], b[1], bit3);
}
// eight steps' registers, folded two by two as they come: lane 8 i + l then holds item i of the step
// whose three bits are l's in reverse order
__device__ __forceinline__ int lane_of_step(int t) { return (t & 1) << 2 | (t & 2) | (t & 4) >> 2; }

// The first pass of a split time axis: what each chunk hands back from zero.
template <typename T, int NS, int NW>
__global__ __launch_bounds__(64 * NW) void backward_local(const Args a) {
  constexpr int TT = 8 * NW, E = 8, G = 4;  // units as the main pass has them: 4 steps of 4 states
  __shared__ float s_rate[TT][64], s_dy[TT][64];
  const ms_scan_io& io = a.io;
  const Place at = place(a);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lt = threadIdx.x >> 3, lc = (threadIdx.x & 7) * 8;
  const int n = at.nc - lc < 0 ? 0 : at.nc - lc;
  const int64_t t_begin = at.chunk * a.p.chunk;
  const int64_t t_end = t_begin + a.p.chunk < io.steps ? t_begin + a.p.chunk : io.steps;
  const int64_t cl = at.c0 + lc;
  const T* dl = (const T*)io.delta + at.r * io.delta_r + cl;
  const T* dy = (const T*)io.dout + at.r * io.dout_r + cl;
  const T* z = io.z ? (const T*)io.z + at.r * io.z_r + cl : nullptr;
  float bias[E];
#pragma unroll
  for (int e = 0; e < E; ++e) bias[e] = io.delta_bias && e < n ? io.delta_bias[cl + e] : 0.0f;
  const int64_t ch = at.c0 + lane;
  const int N = io.states;
  const bool live = lane < at.nc;
  float A2[NS], carry[NS], total = 0.0f;
  bool was_cut = false;
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    A2[i] = live && w * NS + i < N ? io.A[ch * N + w * NS + i] * LOG2E : 0.0f;
    carry[i] = 0.0f;
  }
  CONSTANT(f32x16)* base[NS / 4];
#pragma unroll
  for (int q = 0; q < NS / 4; ++q) base[q] = scalars_at(a, at.r, at.g, w * (NS / 4) + q);
  const int64_t tiles = (t_end - t_begin + TT - 1) / TT;
  const bool vec = a.vec;
  typedef typename Vec<T, E>::type V;
  V vd, vy, vz;
  auto fetch = [&](int64_t t) __attribute__((always_inline)) {
    const bool in = t >= t_begin && t + lt < t_end;
    vd = load<T, E>(dl + (t + lt) * io.delta_t, in ? n : 0, vec);
    vy = load<T, E>(dy + (t + lt) * io.dout_t, in ? n : 0, vec);
    if (z) vz = load<T, E>(z + (t + lt) * io.z_t, in ? n : 0, vec);
  };
  fetch(t_begin + (tiles - 1) * TT);
  Starts flags(io, at.r, t_begin + (tiles - 1) * TT, -TT, (int)(t_end - t_begin - (tiles - 1) * TT));
  for (int64_t k = tiles - 1; k >= 0; --k) {
    const int64_t t0 = t_begin + k * TT, t1 = t0 + TT < t_end ? t0 + TT : t_end;
    const bool mine = t0 + lt < t1;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float slope, rate = (float)vd[e] + bias[e];
      if (io.softplus) rate = softplus(rate, slope);
      s_rate[lt][column<E>(lc + e, lt)] = mine ? rate : 0.0f;
      s_dy[lt][column<E>(lc + e, lt)] = z ? (float)vy[e] * silu((float)vz[e]) : (float)vy[e];
    }
    const uint64_t starts = flags.mask();
    __syncthreads();
    fetch(t0 - TT);
    flags.move(k > 0 ? TT : 0);
    for (int t = TT - G; t >= 0; t -= G) {
      f32x16 c[NS / 4];
#pragma unroll
      for (int q = 0; q < NS / 4; ++q) c[q] = base[q][(t0 + t) / G * 2 + 1];
      const unsigned cut = (unsigned)(starts >> t) & 15u;
#pragma unroll
      for (int j = G - 1; j >= 0; --j) {
        const float rate = s_rate[t + j][column<E>(lane, j)], d = s_dy[t + j][column<E>(lane, j)];
        total += rate;
#pragma unroll
        for (int i = 0; i < NS; ++i)
          carry[i] = __builtin_amdgcn_exp2f(rate * A2[i]) * __builtin_fmaf(c[i / 4][j * 4 + i % 4], d, carry[i]);
        if (cut >> j & 1) {
          was_cut = true;
#pragma unroll
          for (int i = 0; i < NS; ++i) carry[i] = 0.0f;
        }
      }
    }
    __syncthreads();
  }
  const int64_t of = at.chunk * io.rows * io.channels;
  if (live) {
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (w * NS + i < N) a.local[(of + at.r * io.channels + ch) * N + w * NS + i] = carry[i];
    if (w == 0) a.rates[of + at.r * io.channels + ch] = total;
  }
  if (threadIdx.x == 0 && at.td == 0) a.cut[at.chunk * io.rows + at.r] = was_cut;
}

// The KC steps from a checkpoint at a time, and of them four states at a time: first forwards, keeping
// a[t] and a[t] h[t - 1] in registers (64 of them), then backwards through them. With 16 steps between
// checkpoints they would be 128, and two waves a SIMD would spill.
template <typename T, int NS, int NW>
__global__ __launch_bounds__(64 * NW, NW == 4 && NS == 4 ? 3 : NW == 1 ? 1 : 2) void backward(const Args a) {
  constexpr int TT = KC, E = TT / NW, TPR = 64 / E;  // a tile's values over the threads: E channels each
  __shared__ float s_in[2][3][TT][64];  // rate, rate u and dy of this tile and, while it is finished, the next
  // what a thread needs of its own values again after the recurrence: kept here, 168 registers are few
  enum { U, Z, DOUT, SLOPE, GATE, DSKIP, DBIAS, KEPT };
  __shared__ float s_kept[KEPT][TT][64], s_bias[64], s_skip[64];
  __shared__ float s_gb[NW][TT][64], s_ga[NW][TT][64], s_y[NW][TT][64];
  const ms_scan_io& io = a.io;
  const Place at = place(a);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lt = threadIdx.x / TPR, lc = (threadIdx.x % TPR) * E;
  const int n = at.nc - lc < 0 ? 0 : at.nc - lc;
  const int64_t t_begin = at.chunk * a.p.chunk;
  const int64_t t_end = t_begin + a.p.chunk < io.steps ? t_begin + a.p.chunk : io.steps;
  const int len = (int)(t_end - t_begin), tiles = (len + TT - 1) / TT;
  const int64_t cl = at.c0 + lc, last = t_begin + (tiles - 1) * TT + lt;
  const T* pu = (const T*)io.u + at.r * io.u_r + cl + last * io.u_t;
  const T* pd = (const T*)io.delta + at.r * io.delta_r + cl + last * io.delta_t;
  const T* pz = io.z ? (const T*)io.z + at.r * io.z_r + cl + last * io.z_t : nullptr;
  const T* po = (const T*)io.dout + at.r * io.dout_r + cl + last * io.dout_t;
  T* qu = (T*)io.du + at.r * io.du_r + cl + last * io.du_t;
  T* qd = (T*)io.ddelta + at.r * io.ddelta_r + cl + last * io.ddelta_t;
  T* qz = io.z ? (T*)io.dz + at.r * io.dz_r + cl + last * io.dz_t : nullptr;
  if (threadIdx.x < 64) {
    const bool in = lane < at.nc;
    s_bias[lane] = in && io.delta_bias ? io.delta_bias[at.c0 + lane] : 0.0f;
    s_skip[lane] = in && io.D ? io.D[at.c0 + lane] : 0.0f;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s_kept[DSKIP][lt][lc + e] = s_kept[DBIAS][lt][lc + e] = 0.0f;
  __syncthreads();
  const int64_t ch = at.c0 + lane;
  const int N = io.states;
  const bool live = lane < at.nc;
  const int64_t slot = (at.r * io.channels + ch) * N;
  float A2[NS], carry[NS], dA[NS];
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const int s = w * NS + i;
    A2[i] = live && s < N ? io.A[ch * N + s] * LOG2E : 0.0f;
    carry[i] = dA[i] = 0.0f;
    if (live && s < N) {
      if (a.p.chunks > 1) carry[i] = a.local[at.chunk * io.rows * io.channels * N + slot + s];
      else if (io.dnew_state) carry[i] = io.dnew_state[slot + s];
    }
  }
  CONSTANT(f32x16)* base = scalars_at(a, at.r, at.g, w * (NS / 4)) + (t_begin + (tiles - 1) * TT) / 4 * 2;
  const int64_t share = a.p.units * 2;
  const int soft = io.softplus;
  const bool vec = a.vec;
  typedef typename Vec<T, E>::type V;
  V vu, vd, vz, vo;
  float4 start[NS / 4];  // the checkpoint, a tile ahead as the rest
  const int64_t ckpt_step = io.rows * a.p.blocks_d * (NS * NW / 4) * 256;
  const float* from = io.checkpoints + checkpoint_at(a, t_begin / KC + tiles - 1, at.r, at.td, w * NS, 0);
  const int64_t to_step = io.rows * a.p.blocks_d * (NS * NW / 4) * 64;
  float* to = a.parts_bc + (((t_begin / KC + tiles - 1) * io.rows + at.r) * a.p.blocks_d + at.td) * (NS * NW / 4) * 64 + w * (NS / 4) * 64;
  Starts flags(io, at.r, t_begin + (tiles - 1) * TT, -TT, len - (tiles - 1) * TT);
  auto fetch = [&](bool in) __attribute__((always_inline)) {
    vu = load<T, E>(pu, in ? n : 0, vec);
    vd = load<T, E>(pd, in ? n : 0, vec);
    vo = load<T, E>(po, in ? n : 0, vec);
    if (pz) vz = load<T, E>(pz, in ? n : 0, vec);
  };
  // a segment's parts of dA (D, N), dD (D) and ddelta_bias (D), in one row; the sums begin anew
  auto hand_on = [&](int64_t g) __attribute__((always_inline)) {
    const int64_t D = io.channels;
    float* part = a.parts + ((at.chunk * a.p.segments + g) * io.rows + at.r) * D * (N + 2);
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      if (live && w * NS + i < N) part[ch * N + w * NS + i] = dA[i];
      dA[i] = 0.0f;
    }
    __syncthreads();
    if (threadIdx.x < 64 && live) {  // the threads of the same channels add up
      double dskip = 0.0, dbias = 0.0;
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        dskip += s_kept[DSKIP][i][lane];
        dbias += s_kept[DBIAS][i][lane];
      }
      part[D * N + ch] = (float)dskip;
      part[D * (N + 1) + ch] = (float)dbias;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) s_kept[DSKIP][lt][lc + e] = s_kept[DBIAS][lt][lc + e] = 0.0f;
  };
  fetch((tiles - 1) * TT + lt < len);
#pragma unroll
  for (int q = 0; q < NS / 4; ++q) start[q] = *(const float4*)(from + q * 256 + lane * 4);
  for (int k = tiles - 1; k >= 0; --k) {
    float(&s_rate)[TT][64] = s_in[k & 1][0], (&s_ru)[TT][64] = s_in[k & 1][1], (&s_dy)[TT][64] = s_in[k & 1][2];
    const bool mine = k * TT + lt < len;
#pragma unroll
    for (int e = 0; e < E; ++e) {  // a step past the end has rate 0 and dy 0: it changes nothing
      const int c = lc + e;
      const float u = (float)vu[e], z = pz ? (float)vz[e] : 0.0f, d = (float)vo[e];
      float rate = (float)vd[e] + s_bias[c], slope = 1.0f;
      if (soft) rate = softplus(rate, slope);
      rate = mine ? rate : 0.0f;
      const float gate = pz ? sigmoid(z) : 1.0f;
      s_rate[lt][c] = rate;
      s_ru[lt][c] = rate * u;
      s_dy[lt][c] = pz ? d * (z * gate) : d;
      s_kept[U][lt][c] = u;
      s_kept[Z][lt][c] = z;
      s_kept[DOUT][lt][c] = d;
      s_kept[SLOPE][lt][c] = slope;
      s_kept[GATE][lt][c] = gate;
    }
    const uint64_t starts = flags.mask();
    __syncthreads();
    pu -= TT * io.u_t;
    pd -= TT * io.delta_t;
    po -= TT * io.dout_t;
    if (pz) pz -= TT * io.z_t;
    fetch(k > 0);
    flags.move(k > 0 ? TT : 0);
    if (k > 0) from -= ckpt_step;
    auto tile = [&](auto any) __attribute__((always_inline)) {
      constexpr bool CUTS = decltype(any)::value;
#pragma unroll
      for (int nb = 0; nb < NS; nb += 4) {
        {
          const float4 h0 = start[nb >> 2];
          CONSTANT(f32x16)* p = base + (nb >> 2) * share;
          float h[4] = {h0.x, h0.y, h0.z, h0.w};
          float dec[KC][4], ah[KC][4];  // a[t] and a[t] h[t - 1]
          f32x16 b = p[0], c_last;
#pragma unroll
          for (int t4 = 0; t4 < KC; t4 += 4) {
            float rate[4], ru[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              rate[j] = s_rate[t4 + j][lane];
              ru[j] = s_ru[t4 + j][lane];
            }
            loads_done();
            f32x16 b_next = b;
            if (t4 + 4 < KC) b_next = p[(t4 + 4) / 4 * 2];
            else c_last = p[KC / 4 * 2 - 1];
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int t = t4 + j;
              if (CUTS && (starts >> t & 1)) h[0] = h[1] = h[2] = h[3] = 0.0f;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                dec[t][i] = __builtin_amdgcn_exp2f(rate[j] * A2[nb + i]);
                ah[t][i] = dec[t][i] * h[i];
                h[i] = __builtin_fmaf(ru[j], b[j * 4 + i], ah[t][i]);
              }
            }
            __builtin_amdgcn_sched_barrier(0);
            b = b_next;
          }
          start[nb >> 2] = *(const float4*)(from + nb * 64 + lane * 4);  // the next tile's
          Scalars s;
          s.b = b;
          s.c = c_last;
          float pair = 0.0f, four = 0.0f, eight = 0.0f;  // folded registers of 1, 2 and 4 steps that wait for their other half
#pragma unroll
          for (int t4 = KC - 4; t4 >= 0; t4 -= 4) {
            float rate[4], ru[4], dy[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              dy[j] = s_dy[t4 + j][lane];
              rate[j] = s_rate[t4 + j][lane];
              ru[j] = s_ru[t4 + j][lane];
            }
            loads_done();
            Scalars prev = s;
            if (t4) prev = scalars(p + (t4 - 4) / 4 * 2);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 3; j >= 0; --j) {
              const int t = t4 + j;
              float gb = 0.0f, ga = 0.0f, y = 0.0f, items[8];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float B = s.b[j * 4 + i], C = s.c[j * 4 + i];
                const float g = __builtin_fmaf(C, dy[j], carry[nb + i]);
                const float hh = __builtin_fmaf(ru[j], B, ah[t][i]);
                const float q = g * ah[t][i];
                y = i ? __builtin_fmaf(C, hh, y) : C * hh;
                gb = i ? __builtin_fmaf(B, g, gb) : B * g;
                ga = i ? __builtin_fmaf(q, A2[nb + i], ga) : q * A2[nb];
                dA[nb + i] = __builtin_fmaf(q, rate[j], dA[nb + i]);
                carry[nb + i] = dec[t][i] * g;
                items[i] = ru[j] * g;
                items[4 + i] = dy[j] * hh;
              }
              if (CUTS && (starts >> t & 1)) carry[nb] = carry[nb + 1] = carry[nb + 2] = carry[nb + 3] = 0.0f;
              if (nb) {
                gb += s_gb[w][t][lane];
                ga += s_ga[w][t][lane];
                y += s_y[w][t][lane];
              }
              s_gb[w][t][lane] = gb;
              s_ga[w][t][lane] = ga;
              s_y[w][t][lane] = y;
              float x = fold_items(items, lane & 8);
              if (t & 1) {
                pair = x;
              } else {
                x = fold_dpp<HALF_MIRROR>(x, pair, lane & 4);
                if (t & 2) {
                  four = x;
                } else {
                  x = fold_dpp<XOR2>(x, four, lane & 2);
                  if (t & 4) eight = x;
                  else to[(nb >> 2) * 64 + lane] = fold_dpp<XOR1>(x, eight, lane & 1);
                }
              }
            }
            __builtin_amdgcn_sched_barrier(0);
            s = prev;
          }
        }
      }
    };
    if (starts) tile(std::true_type{});
    else tile(std::false_type{});
    base -= TT / 4 * 2;
    to -= to_step;
    __syncthreads();
    if (mine && n > 0) {
      float du[E], dd[E], dz[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float gb = 0.0f, ga = 0.0f, y = 0.0f;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
          gb += s_gb[i][lt][lc + e];
          ga += s_ga[i][lt][lc + e];
          y += s_y[i][lt][lc + e];
        }
        const int c = lc + e;
        const float u = s_kept[U][lt][c], rt = s_rate[lt][c], dy = s_dy[lt][c], skip = s_skip[c];
        if (pz) {
          const float z = s_kept[Z][lt][c], gate = s_kept[GATE][lt][c];
          dz[e] = s_kept[DOUT][lt][c] * __builtin_fmaf(skip, u, y) * (gate * (1.0f + z * (1.0f - gate)));
        }
        du[e] = __builtin_fmaf(skip, dy, rt * gb);
        dd[e] = __builtin_fmaf(gb, u, ga * LN2) * s_kept[SLOPE][lt][c];
        s_kept[DSKIP][lt][c] += dy * u;
        s_kept[DBIAS][lt][c] += dd[e];
      }
      store<T, E>(qu, du, n, vec);
      store<T, E>(qd, dd, n, vec);
      if (pz) store<T, E>(qz, dz, n, vec);
    }
    qu -= TT * io.du_t;
    qd -= TT * io.ddelta_t;
    if (pz) qz -= TT * io.dz_t;
    if (k % (SEGMENT / TT) == 0) hand_on(k / (SEGMENT / TT));
  }
  if (live && io.dstate && t_begin == 0) {
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (w * NS + i < N) io.dstate[slot + w * NS + i] = carry[i];
  }
}

// The second stage of the sums over rows, chunks and segments, put in place: dA, dD, ddelta_bias
template <int WAVES>
__global__ __launch_bounds__(64 * WAVES) void finish_weights(const float* __restrict__ in, int64_t parts, ms_scan_io io) {
  __shared__ double s[WAVES][64];
  const int64_t c = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63), D = io.channels, dn = D * io.states;
  const float sum = (float)sum_share<WAVES>(in, 0, parts, dn + 2 * D, c, s);
  if (threadIdx.x >= 64) return;
  if (c < dn) io.dA[c] = sum;
  else if (c < dn + D) { if (io.dD) io.dD[c - dn] = sum; }
  else if (c < dn + 2 * D) { if (io.ddelta_bias) io.ddelta_bias[c - dn - D] = sum; }
}

// dB, dC: the tiles of a group added and put in place. A wave takes 8 steps of a row's group, 64 sums
// (4 states of both, one a lane as the folds left them) at a time; `split` waves share a row's states
// where rows and steps alone are too few waves. 128 steps x 2,048 rows x 128, f32: 26 us, 3.9 TB/s (37 with
// one quad of states at a time).
template <typename T>
__global__ __launch_bounds__(256) void finish_bc(const Args a, int split) {
  const ms_scan_io& io = a.io;
  const int lane = threadIdx.x & 63, n4 = a.p.ns * a.p.nw / 4;
  const unsigned wave = blockIdx.x * 4 + (unsigned)__builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const unsigned k = wave / (unsigned)split, first = wave - k * (unsigned)split;
  const unsigned rgs = (unsigned)(io.rows * io.groups), t8 = k / rgs, rg = k - t8 * rgs;
  if (t8 >= (io.steps + 7) / 8) return;
  const unsigned r = rg / (unsigned)io.groups, g = rg - r * (unsigned)io.groups;
  const int64_t one = n4 * 64, tiles = a.p.tiles;  // a tile's floats
  const float* p = a.parts_bc + ((t8 * io.rows + r) * a.p.blocks_d + g * tiles) * one + lane;
  const int item = lane >> 3;
  const int64_t t = (int64_t)t8 * 8 + lane_of_step(lane & 7);  // its own inverse
  T* out = (T*)(item & 4 ? io.dC : io.dB) + ((t * io.rows + r) * io.groups + g) * io.states;
  auto sums = [&](int q, auto many) __attribute__((always_inline)) {  // quads q, q + split, ...: their loads together
    constexpr int K = decltype(many)::value, U = K == 1 ? 4 : 2;
    float sum[K] = {};
    int64_t j = 0;
    for (; j + U <= tiles; j += U) {
      float x[K][U];
#pragma unroll
      for (int i = 0; i < K; ++i)
#pragma unroll
        for (int m = 0; m < U; ++m) x[i][m] = p[(j + m) * one + (q + i * split) * 64];
#pragma unroll
      for (int i = 0; i < K; ++i)
#pragma unroll
        for (int m = 0; m < U; m += 2) sum[i] += x[i][m] + x[i][m + 1];
    }
    for (; j < tiles; ++j)
#pragma unroll
      for (int i = 0; i < K; ++i) sum[i] += p[j * one + (q + i * split) * 64];
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const int s = (q + i * split) * 4 + (item & 3);
      if (s < io.states && t < io.steps) out[s] = (T)sum[i];
    }
  };
  int q = (int)first;
  for (; q + 3 * split < n4; q += 4 * split) sums(q, std::integral_constant<int, 4>{});
  for (; q < n4; q += split) sums(q, std::integral_constant<int, 1>{});
}

// ---------------------------------------------------------------- the host's side

// How many states a wave holds, and whether the time axis is split. Measured at 16 states, bf16, T x D =
// 2,048 x 2,048 a row unless stated (forward alone; forward with backward for the backward's rule):
//   * four states a wave, four waves a block. One wave with all 16 has less to add up but leaves the
//     SIMDs idle: 64 rows of 256 steps 259 us against 181, 8 rows 996 against 310.
//   * forward of 9 to 16 states with at most one block a CU: two states a wave and eight waves, 8 rows
//     221 us against 310; with more blocks the four have it (12 rows of 1,024 steps: 204 against 253).
//   * fewer blocks: chunks of time, 768 blocks in all, where the steps saved pay for three more launches
//     and twice the exponentials: a call takes 25 us + blocks x steps x 0.56 ns split, 5 us + steps x 0.106
//     us unsplit. 3 rows (96 blocks) 136 us against 221, 4 rows 173 against 222, but 500 steps of them 66
//     against 62; 5 rows 243 against 221; 1 row of 200 steps 39 against 30, of 16,411 x 1,536 241 against
//     1,800. Other numbers of states: up to 192 blocks of four waves, or as many waves in smaller ones (4
//     states, 16 rows of 2,048 x 512: 94 us against 526 unsplit and 170 with 768 blocks; 8 states, 40 rows
//     of 377 x 448: 68 against 94).
//   * backward: chunks up to 511 blocks, 1,536 blocks in all. 6 rows of 1,024 steps 406 us against 581,
//     12 rows 714 against 805; 16 rows (512 blocks) 872 against 825, so not there.
//   * chunks of 64 steps at least: 512 steps x 256 channels 39 us, 128 steps at least 50, 32 steps 41.
Plan plan(const ms_scan_io& io, bool back) {
  Plan p = {};
  p.tiles = (io.channels / io.groups + 63) / 64;
  p.blocks_d = p.tiles * io.groups;
  const int64_t blocks = p.blocks_d * io.rows;
  const int np = io.states <= 4 ? 4 : io.states <= 8 ? 8 : io.states <= 16 ? 16 : io.states <= 32 ? 32 : 64;
  p.ns = np <= 16 ? 4 : np / 4;
  const int64_t small = 4 * p.ns / np > 1 ? 4 * p.ns / np : 1;  // blocks of one or two waves: as many times the blocks
  const bool split = blocks > 0 && (back ? blocks <= 511 * small : np == 16 ? (160 - blocks) * io.steps > 30000 : blocks <= 192 * small);
  if (!back && np == 16 && !split && blocks <= 256) p.ns = 2;
  p.nw = np / p.ns;
  const int64_t pieces = (io.steps + 31) / 32;
  int64_t chunks = split ? ((back ? 1536 : 768) * small + blocks - 1) / blocks : 1;
  if (chunks > pieces / 2) chunks = pieces / 2;
  if (chunks < 1) chunks = 1;
  p.chunk = (pieces + chunks - 1) / chunks * 32;
  p.chunk = p.chunk < 32 ? 32 : p.chunk;
  p.chunks = io.steps > 0 ? (io.steps + p.chunk - 1) / p.chunk : 1;
  p.kc = (io.steps + KC - 1) / KC;
  p.segments = (p.chunk + SEGMENT - 1) / SEGMENT;
  p.sums = (p.chunks - 1) * p.segments + (io.steps - (p.chunks - 1) * p.chunk + SEGMENT - 1) / SEGMENT;  // the last chunk may be shorter
  p.unit = back ? 4 : p.ns;
  // whole tiles of 32 steps, and a unit past the end
  p.units = (io.steps + 31) / 32 * 32 * p.unit / 16 + 1;
  return p;
}

int64_t round4(int64_t n) { return (n + 3) / 4 * 4; }

// how many parts the sums over rows, chunks and segments add in the first of their two stages
int64_t share_of(int64_t parts) { return parts <= 64 ? parts : parts <= 4096 ? 64 : (parts + 63) / 64; }

int64_t scalar_floats(const ms_scan_io& io, const Plan& p) { return io.rows * io.groups * (p.ns * p.nw / p.unit) * p.units * 32; }
int64_t checkpoint_floats(const ms_scan_io& io, const Plan& p) { return p.kc * io.rows * p.blocks_d * p.nw * p.ns * 64; }
bool kept_scalars(const ms_scan_io& io, const Plan& p) { return io.checkpoints && p.unit == 4 && plan(io, false).unit == 4; }

Work work(const ms_scan_io& io, const Plan& p, bool back) {
  Work w = {};
  float* at = (float*)io.workspace;
  int64_t used = 0;
  auto take = [&](int64_t n) {
    float* q = at + used;
    used += round4(n);
    return q;
  };
  const int64_t rd = io.rows * io.channels, parts = p.chunks * io.rows, row = io.channels * (io.states + 2);
  // B and C as scalars: kept behind the checkpoints by a forward whose units are the backward's
  if (kept_scalars(io, p)) w.bc = io.checkpoints + checkpoint_floats(io, p);
  else w.bc = take(scalar_floats(io, p));
  if (p.chunks > 1) {
    w.local = take(p.chunks * rd * io.states);
    w.rates = take(p.chunks * rd);
    w.cut = (int*)take(parts);
  }
  if (back) {
    w.parts_bc = take(p.kc * io.rows * p.blocks_d * (p.ns * p.nw / 4) * 64);
    const int64_t sums = p.sums * io.rows, share = share_of(sums);
    w.parts = take(sums * row);
    w.sums = share ? take((sums + share - 1) / share * row) : nullptr;
  }
  w.floats = used;
  return w;
}

const char* check(const ms_scan_io* io, bool back, bool step) {
  if (!io) return "no arguments";
  if (io->dtype < 0 || io->dtype > 2) return "dtype must be 0 (float32), 1 (bfloat16) or 2 (float16)";
  if (io->steps < 0 || io->rows < 0 || io->channels <= 0) return "steps and rows must be >= 0, channels > 0";
  if (io->steps > 0x7fffff00) return "too many steps";
  if (io->states < 1 || io->states > 64) return "1 to 64 states are supported";
  if (io->groups < 1 || io->channels % io->groups) return "groups must divide the channels";
  if (step && io->steps != 1) return "a step has steps = 1";
  if (!io->A) return "A is NULL";
  const bool some = io->steps > 0 && io->rows > 0;
  if (some && (!io->u || !io->delta || !io->B || !io->C)) return "u, delta, B or C is NULL";
  if (some && !back && !io->out) return "out is NULL";
  if (step && io->rows > 0 && !io->new_state) return "a step needs new_state";
  if (back) {
    if (!io->dA) return "dA is NULL";
    if (some && (!io->dout || !io->du || !io->ddelta || !io->dB || !io->dC || !io->checkpoints || (io->z && !io->dz)))
      return "dout, du, ddelta, dz, dB, dC or checkpoints is NULL";
  }
  return nullptr;
}

int64_t widen_blocks(const ms_scan_io& io, const Plan& p) {
  const int64_t each = 64 / (p.ns * p.nw / p.unit);
  return (p.units * io.rows * io.groups + each - 1) / each;
}
int64_t join_blocks(const ms_scan_io& io) { return (io.rows * io.channels * io.states + 255) / 256; }
int64_t finish_waves(const ms_scan_io& io) { return (io.steps + 7) / 8 * io.rows * io.groups; }

// Whether every launch's threads fit 32 bits, looked at before the first of them
bool fits(const ms_scan_io& io, const Plan& p, bool back) {
  if (io.rows > ((int64_t)1 << 40) / io.channels || io.rows > ((int64_t)1 << 40) / (io.steps + 64)) return false;
  if (too_many(p.blocks_d * io.rows * p.chunks, 64 * p.nw) || too_many(widen_blocks(io, p), 256) || io.rows * io.groups > 0x7fffffff) return false;
  if (p.chunks > 1 && too_many(join_blocks(io), 256)) return false;
  return !back || !(too_many((finish_waves(io) * (p.ns * p.nw / 4) + 3) / 4, 256) || too_many((io.channels * (io.states + 2) + 63) / 64, 256));
}

int prepare(const ms_scan_io& io, const Plan& p, const Work& w, bool back, hipStream_t stream, const char* who, Args& a) {
  a.io = io;
  a.p = p;
  a.bc = w.bc;
  a.local = w.local;
  a.rates = w.rates;
  a.cut = w.cut;
  a.parts_bc = w.parts_bc;
  a.parts = w.parts;
  if (back && kept_scalars(io, p)) return MS_OK;
  const int shares = p.ns * p.nw / p.unit;
  const int64_t elem = io.dtype == 0 ? 4 : 2;
  const bool vec = p.unit >= 4 && aligned(io.B, io.B_t, io.B_r, elem, 4) && aligned(io.C, io.C_t, io.C_r, elem, 4) &&
                   (io.groups == 1 || (io.B_g % 4 == 0 && io.C_g % 4 == 0));
  const dim3 grid((unsigned)widen_blocks(io, p)), block(256);
  if (io.dtype == 0) hipLaunchKernelGGL(widen<float>, grid, block, 0, stream, io, p.unit, shares, p.units, vec, w.bc);
  else if (io.dtype == 1) hipLaunchKernelGGL(widen<bf16>, grid, block, 0, stream, io, p.unit, shares, p.units, vec, w.bc);
  else hipLaunchKernelGGL(widen<f16>, grid, block, 0, stream, io, p.unit, shares, p.units, vec, w.bc);
  return launched(who);
}

enum Pass { LOCAL, MAIN, BACK_LOCAL, BACK };

// Whether a pass may move the E channels of a thread at once (2,048 steps of 8 rows x 2,044 bf16, where
// rows are aligned to 8 B: 261 us with four channels at once, 315 guarded one by one)
bool vec_ok(const ms_scan_io& io, Pass pass, int nw) {
  const int64_t elem = io.dtype == 0 ? 4 : 2, E = pass == BACK ? KC / nw : nw == 8 ? 4 : 8;
  if (io.groups > 1 && (io.channels / io.groups) % E) return false;
  auto ok = [&](const void* p, int64_t t, int64_t r) { return !p || aligned(p, t, r, elem, E); };
  bool all = ok(io.delta, io.delta_t, io.delta_r) && ok(io.z, io.z_t, io.z_r);
  if (pass != BACK_LOCAL) all = all && ok(io.u, io.u_t, io.u_r);
  if (pass == MAIN) all = all && ok(io.out, io.out_t, io.out_r);
  if (pass >= BACK_LOCAL) all = all && ok(io.dout, io.dout_t, io.dout_r);
  if (pass == BACK) all = all && ok(io.du, io.du_t, io.du_r) && ok(io.ddelta, io.ddelta_t, io.ddelta_r) && (!io.z || ok(io.dz, io.dz_t, io.dz_r));
  return all;
}

template <typename T, int NS, int NW>
void launch_as(Pass pass, const Args& a, dim3 grid, hipStream_t stream) {
  const dim3 block(64 * NW);
  if (pass == LOCAL) hipLaunchKernelGGL((forward<T, NS, NW, true>), grid, block, 0, stream, a);
  else if (pass == MAIN) hipLaunchKernelGGL((forward<T, NS, NW, false>), grid, block, 0, stream, a);
  else if (pass == BACK_LOCAL) hipLaunchKernelGGL((backward_local<T, NS, NW>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((backward<T, NS, NW>), grid, block, 0, stream, a);
}
template <typename T>
void launch_type(Pass pass, const Args& a, dim3 grid, hipStream_t stream) {
  if (a.p.nw == 8) hipLaunchKernelGGL((forward<T, 2, 8, false>), grid, dim3(512), 0, stream, a);  // never split
  else if (a.p.nw == 1) launch_as<T, 4, 1>(pass, a, grid, stream);
  else if (a.p.nw == 2) launch_as<T, 4, 2>(pass, a, grid, stream);
  else if (a.p.ns == 4) launch_as<T, 4, 4>(pass, a, grid, stream);
  else if (a.p.ns == 8) launch_as<T, 8, 4>(pass, a, grid, stream);
  else launch_as<T, 16, 4>(pass, a, grid, stream);
}
int launch(Pass pass, Args& a, hipStream_t stream, const char* who) {
  a.vec = vec_ok(a.io, pass, a.p.nw);
  const dim3 grid((unsigned)(a.p.blocks_d * a.io.rows * a.p.chunks));
  if (a.io.dtype == 0) launch_type<float>(pass, a, grid, stream);
  else if (a.io.dtype == 1) launch_type<bf16>(pass, a, grid, stream);
  else launch_type<f16>(pass, a, grid, stream);
  return launched(who);
}
template <bool BACK>
int launch_join(const Args& a, hipStream_t stream, const char* who) {
  hipLaunchKernelGGL(join<BACK>, dim3((unsigned)join_blocks(a.io)), dim3(256), 0, stream, a);
  return launched(who);
}

__global__ __launch_bounds__(256) void copy_state(const float* __restrict__ from, int64_t n, float* __restrict__ to) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) to[i] = from ? from[i] : 0.0f;
}
int copied(const float* from, int64_t n, float* to, hipStream_t stream, const char* who) {
  if (!to || n == 0 || to == from) return MS_OK;
  constexpr int64_t MOST = (int64_t)1 << 31;  // values a launch
  for (int64_t i = 0; i < n; i += MOST) {
    const int64_t m = n - i < MOST ? n - i : MOST;
    hipLaunchKernelGGL(copy_state, dim3((unsigned)((m + 255) / 256)), dim3(256), 0, stream, from ? from + i : nullptr, m, to + i);
    if (int rc = launched(who)) return rc;
  }
  return MS_OK;
}

// A step of as many rows at a time as a launch has threads for
template <typename T>
int launch_step(ms_scan_io io, hipStream_t stream) {
  const int q = io.states / 4;
  const bool four = io.states % 4 == 0 && (q & (q - 1)) == 0 && ((uintptr_t)io.A & 15u) == 0 &&
                    ((uintptr_t)io.new_state & 15u) == 0 && (!io.state || ((uintptr_t)io.state & 15u) == 0);
  const int64_t one = io.channels * (four ? q : 1), most = 0xffffff00ll / one;  // a row's threads
  if (most < 1) return fail(MS_ERR_INVALID_ARGUMENT, "ms_scan_step", "too large");
  auto move = [](auto*& p, int64_t by) {
    typedef std::remove_reference_t<decltype(p)> P;
    if (p) p = (P)((const T*)p + by);
  };
  for (int64_t left = io.rows; left > 0; left -= most) {
    io.rows = left < most ? left : most;
    const dim3 grid((unsigned)((io.rows * one + 255) / 256)), block(256);
    if (!four) hipLaunchKernelGGL(step1<T>, grid, block, 0, stream, io);
    else if (q == 1) hipLaunchKernelGGL((step4<T, 1>), grid, block, 0, stream, io);
    else if (q == 2) hipLaunchKernelGGL((step4<T, 2>), grid, block, 0, stream, io);
    else if (q == 4) hipLaunchKernelGGL((step4<T, 4>), grid, block, 0, stream, io);
    else if (q == 8) hipLaunchKernelGGL((step4<T, 8>), grid, block, 0, stream, io);
    else hipLaunchKernelGGL((step4<T, 16>), grid, block, 0, stream, io);
    if (int rc = launched("ms_scan_step")) return rc;
    move(io.u, most * io.u_r);
    move(io.delta, most * io.delta_r);
    move(io.z, most * io.z_r);
    move(io.B, most * io.B_r);
    move(io.C, most * io.C_r);
    move(io.out, most * io.out_r);
    if (io.starts) io.starts += most * io.starts_r;
    if (io.state) io.state += most * io.channels * io.states;
    io.new_state += most * io.channels * io.states;
  }
  return MS_OK;
}

bool space(const ms_scan_io& io, int64_t bytes) {
  return bytes == 0 || (io.workspace && ((uintptr_t)io.workspace & 15u) == 0 && io.workspace_bytes >= bytes);
}

}  // namespace scan

extern "C" {

int64_t ms_scan_checkpoints(const ms_scan_io* io) {
  if (!io || io->states < 1 || io->states > 64 || io->groups < 1 || io->channels <= 0 || io->steps < 0 || io->rows < 0) return 0;
  const scan::Plan p = scan::plan(*io, false);
  return (scan::checkpoint_floats(*io, p) + (p.unit == 4 ? scan::scalar_floats(*io, p) : 0)) * (int64_t)sizeof(float);
}

int64_t ms_scan_workspace(const ms_scan_io* io, int backward) {
  if (!io || io->states < 1 || io->states > 64 || io->groups < 1 || io->channels <= 0 || io->steps < 0 || io->rows < 0) return 0;
  ms_scan_io none = *io;
  none.workspace = nullptr;
  return scan::work(none, scan::plan(*io, backward != 0), backward != 0).floats * (int64_t)sizeof(float);
}

int ms_scan_forward(const ms_scan_io* io, void* stream) {
  const char* who = "ms_scan_forward";
  if (const char* why = scan::check(io, false, false)) return seq::fail(MS_ERR_INVALID_ARGUMENT, who, why);
  const hipStream_t st = (hipStream_t)stream;
  if (io->rows == 0) return MS_OK;
  if (io->steps == 0) return scan::copied(io->state, io->rows * io->channels * io->states, io->new_state, st, who);
  const scan::Plan p = scan::plan(*io, false);
  if (!scan::fits(*io, p, false)) return seq::fail(MS_ERR_INVALID_ARGUMENT, who, "too large");
  const scan::Work w = scan::work(*io, p, false);
  if (!scan::space(*io, w.floats * 4))
    return seq::fail(MS_ERR_INVALID_ARGUMENT, who, "the workspace is missing, misaligned or too small");
  if (io->checkpoints && ((uintptr_t)io->checkpoints & 15u))
    return seq::fail(MS_ERR_INVALID_ARGUMENT, who, "checkpoints must be 16-B aligned");
  scan::Args a = {};
  if (int rc = scan::prepare(*io, p, w, false, st, who, a)) return rc;
  if (p.chunks > 1) {
    if (int rc = scan::launch(scan::LOCAL, a, st, who)) return rc;
    if (int rc = scan::launch_join<false>(a, st, who)) return rc;
  }
  return scan::launch(scan::MAIN, a, st, who);
}

int ms_scan_step(const ms_scan_io* io, void* stream) {
  if (const char* why = scan::check(io, false, true)) return seq::fail(MS_ERR_INVALID_ARGUMENT, "ms_scan_step", why);
  if (io->rows == 0) return MS_OK;
  const hipStream_t st = (hipStream_t)stream;
  return io->dtype == 0 ? scan::launch_step<float>(*io, st) : io->dtype == 1 ? scan::launch_step<seq::bf16>(*io, st) : scan::launch_step<seq::f16>(*io, st);
}

int ms_scan_backward(const ms_scan_io* io, void* stream) {
  const char* who = "ms_scan_backward";
  if (const char* why = scan::check(io, true, false)) return seq::fail(MS_ERR_INVALID_ARGUMENT, who, why);
  const hipStream_t st = (hipStream_t)stream;
  const int64_t dn = io->channels * io->states;
  if (io->rows == 0 || io->steps == 0) {
    if (int rc = scan::copied(nullptr, dn, io->dA, st, who)) return rc;
    if (int rc = scan::copied(nullptr, io->channels, io->dD, st, who)) return rc;
    if (int rc = scan::copied(nullptr, io->channels, io->ddelta_bias, st, who)) return rc;
    return scan::copied(io->dnew_state, io->rows * dn, io->dstate, st, who);
  }
  const scan::Plan p = scan::plan(*io, true);
  if (!scan::fits(*io, p, true)) return seq::fail(MS_ERR_INVALID_ARGUMENT, who, "too large");
  const scan::Work w = scan::work(*io, p, true);
  if (!scan::space(*io, w.floats * 4) || ((uintptr_t)io->checkpoints & 15u))
    return seq::fail(MS_ERR_INVALID_ARGUMENT, who, "the workspace or the checkpoints are missing, misaligned or too small");
  scan::Args a = {};
  if (int rc = scan::prepare(*io, p, w, true, st, who, a)) return rc;
  if (p.chunks > 1) {
    if (int rc = scan::launch(scan::BACK_LOCAL, a, st, who)) return rc;
    if (int rc = scan::launch_join<true>(a, st, who)) return rc;
  }
  if (int rc = scan::launch(scan::BACK, a, st, who)) return rc;
  int64_t waves = scan::finish_waves(*io);
  const int split = waves < 32768 ? p.ns * p.nw / 4 : 1;
  waves *= split;
  const dim3 grid((unsigned)((waves + 3) / 4)), block(256);
  if (io->dtype == 0) hipLaunchKernelGGL(scan::finish_bc<float>, grid, block, 0, st, a, split);
  else if (io->dtype == 1) hipLaunchKernelGGL(scan::finish_bc<seq::bf16>, grid, block, 0, st, a, split);
  else hipLaunchKernelGGL(scan::finish_bc<seq::f16>, grid, block, 0, st, a, split);
  const int64_t parts = p.sums * io->rows, share = scan::share_of(parts), row = io->channels * (io->states + 2);
  const unsigned columns = (unsigned)((row + 63) / 64), shares = (unsigned)((parts + share - 1) / share);
  if (shares > 1)
    hipLaunchKernelGGL(seq::sum_parts<4>, dim3(columns, shares), dim3(256), 0, st, w.parts, parts, share, row, w.sums);
  hipLaunchKernelGGL(scan::finish_weights<4>, dim3(columns), dim3(256), 0, st, shares > 1 ? w.sums : w.parts, shares > 1 ? shares : parts, *io);
  return seq::launched(who);
}

}  // extern "C"
